// capi_varlen.cuh -- extern "C" entry points of the ragged paged-cache operators (included by capi.cu).
#pragma once

namespace mxfa {
namespace {

int paged_varlen_checks(const void* k_cache, const void* v_cache, const void* k_scales, const void* v_scales,
                               const int32_t* cu_seqlens, const int32_t* seqlens, const int32_t* block_table,
                               int total, int B, int HKV, int D, int PS, int BTW, int num_pages) {
  if (D != 64 && D != 128) return fail(MXFA_ERR_UNSUPPORTED, "head dim %d not in {64, 128}", D);
  if (total < 0 || B < 0 || HKV <= 0) return fail(MXFA_ERR_INVALID, "bad ragged batch geometry");
  if (PS <= 0 || num_pages <= 0 || BTW <= 0) return fail(MXFA_ERR_INVALID, "bad cache geometry");
  if (total == 0 || B == 0) return MXFA_OK;
  if (!k_cache || !v_cache || !cu_seqlens || !seqlens || !block_table)
    return fail(MXFA_ERR_INVALID, "null tensor pointer");
  if ((k_scales == nullptr) != (v_scales == nullptr))
    return fail(MXFA_ERR_INVALID, "k_scales and v_scales must both be given");
  if (!aligned16(k_cache) || !aligned16(v_cache)) return fail(MXFA_ERR_INVALID, "caches must be 16-byte aligned");
  int cap = 0;
  return cache_capacity(block_table, BTW, PS, &cap);
}

// Tokens a CTA takes: one while that still fills the GPU's CTA slots (8 of
// 256 threads per SM), so a decode step's few tokens spread over every SM,
// and up to 32 for long prompts, where a CTA's token lookups overlap.
int tokens_per_cta(int total) {
  const int n = (total + 8 * sm_count() - 1) / (8 * sm_count());
  return n > kPvMaxTok ? kPvMaxTok : n;
}

template <typename T, int HD>
int launch_append_varlen(const PagedVarlenParams& p, bool quant, bool vec, cudaStream_t st) {
  const dim3 grid((p.T + p.tok_per_cta - 1) / p.tok_per_cta);
  if (quant)
    vec ? append_varlen_kernel<T, HD, true, true><<<grid, kPvThreads, 0, st>>>(p)
        : append_varlen_kernel<T, HD, true, false><<<grid, kPvThreads, 0, st>>>(p);
  else
    vec ? append_varlen_kernel<T, HD, false, true><<<grid, kPvThreads, 0, st>>>(p)
        : append_varlen_kernel<T, HD, false, false><<<grid, kPvThreads, 0, st>>>(p);
  return check_launch("append_varlen_kernel");
}

template <typename T, int HD>
int launch_gather_varlen(const PagedVarlenParams& p, bool quant, cudaStream_t st) {
  const dim3 grid((p.T + p.tok_per_cta - 1) / p.tok_per_cta);
  quant ? gather_varlen_kernel<T, HD, true><<<grid, kPvThreads, 0, st>>>(p)
        : gather_varlen_kernel<T, HD, false><<<grid, kPvThreads, 0, st>>>(p);
  return check_launch("gather_varlen_kernel");
}

template <typename T, int HD>
int launch_varlen_rows(const VarlenAttnParams& p, bool quant, cudaStream_t st) {
  const long long rows = static_cast<long long>(p.T) * p.HQ;
  const dim3 grid(static_cast<unsigned>((rows + 3) / 4));
  quant ? varlen_rows_kernel<T, HD, true><<<grid, 128, 0, st>>>(p)
        : varlen_rows_kernel<T, HD, false><<<grid, 128, 0, st>>>(p);
  return check_launch("varlen_rows_kernel");
}

}  // namespace
}  // namespace mxfa

extern "C" {

int mxfa_kvcache_append_varlen_launch(const void* k, const void* v, void* k_cache, void* v_cache, void* k_scales,
                                      void* v_scales, const int32_t* cu_seqlens, const int32_t* seqlens,
                                      const int32_t* block_table, int total, int B, int HKV, int D, int PS, int BTW,
                                      int num_pages, size_t k_token_stride, size_t k_head_stride,
                                      size_t v_token_stride, size_t v_head_stride, int bf16, void* stream) {
  if (int rc = paged_varlen_checks(k_cache, v_cache, k_scales, v_scales, cu_seqlens, seqlens, block_table, total, B,
                                   HKV, D, PS, BTW, num_pages))
    return rc;
  if (total == 0 || B == 0) return MXFA_OK;
  if (!k || !v) return fail(MXFA_ERR_INVALID, "null tensor pointer");
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 1)
    return fail(MXFA_ERR_INVALID, "k and v must be 2-byte aligned");
  PagedVarlenParams p{};
  p.k = k;
  p.v = v;
  p.k_tok = k_token_stride;
  p.k_head = k_head_stride;
  p.v_tok = v_token_stride;
  p.v_head = v_head_stride;
  p.k_cache = static_cast<uint8_t*>(k_cache);
  p.v_cache = static_cast<uint8_t*>(v_cache);
  p.k_scales = static_cast<uint8_t*>(k_scales);
  p.v_scales = static_cast<uint8_t*>(v_scales);
  p.cu = cu_seqlens;
  p.seqlens = seqlens;
  p.bt = block_table;
  p.T = total;
  p.B = B;
  p.HKV = HKV;
  p.PS = PS;
  p.BTW = BTW;
  p.P = num_pages;
  p.tok_per_cta = tokens_per_cta(total);
  const bool vec = aligned16(k) && aligned16(v) &&
                   (k_token_stride | k_head_stride | v_token_stride | v_head_stride) % 8 == 0;
  const bool quant = k_scales != nullptr;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (bf16)
    return D == 128 ? launch_append_varlen<__nv_bfloat16, 128>(p, quant, vec, st)
                    : launch_append_varlen<__nv_bfloat16, 64>(p, quant, vec, st);
  return D == 128 ? launch_append_varlen<__half, 128>(p, quant, vec, st)
                  : launch_append_varlen<__half, 64>(p, quant, vec, st);
}

int mxfa_kvcache_gather_varlen_launch(const void* k_cache, const void* v_cache, const void* k_scales,
                                      const void* v_scales, const int32_t* cu_seqlens, const int32_t* seqlens,
                                      const int32_t* block_table, void* k_out, void* v_out, int total, int B, int HKV,
                                      int D, int PS, int BTW, int num_pages, int bf16, void* stream) {
  if (int rc = paged_varlen_checks(k_cache, v_cache, k_scales, v_scales, cu_seqlens, seqlens, block_table, total, B,
                                   HKV, D, PS, BTW, num_pages))
    return rc;
  if (total == 0 || B == 0) return MXFA_OK;
  if (!k_out || !v_out) return fail(MXFA_ERR_INVALID, "null tensor pointer");
  if (!aligned16(k_out) || !aligned16(v_out)) return fail(MXFA_ERR_INVALID, "outputs must be 16-byte aligned");
  PagedVarlenParams p{};
  p.k = k_out;
  p.v = v_out;
  p.k_cache = static_cast<uint8_t*>(const_cast<void*>(k_cache));
  p.v_cache = static_cast<uint8_t*>(const_cast<void*>(v_cache));
  p.k_scales = static_cast<uint8_t*>(const_cast<void*>(k_scales));
  p.v_scales = static_cast<uint8_t*>(const_cast<void*>(v_scales));
  p.cu = cu_seqlens;
  p.seqlens = seqlens;
  p.bt = block_table;
  p.T = total;
  p.B = B;
  p.HKV = HKV;
  p.PS = PS;
  p.BTW = BTW;
  p.P = num_pages;
  p.tok_per_cta = tokens_per_cta(total);
  const bool quant = k_scales != nullptr;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (bf16)
    return D == 128 ? launch_gather_varlen<__nv_bfloat16, 128>(p, quant, st)
                    : launch_gather_varlen<__nv_bfloat16, 64>(p, quant, st);
  return D == 128 ? launch_gather_varlen<__half, 128>(p, quant, st) : launch_gather_varlen<__half, 64>(p, quant, st);
}

int mxfa_kvcache_varlen_attention_launch(const void* q, const void* k_cache, const void* v_cache,
                                         const void* k_scales, const void* v_scales, const int32_t* cu_seqlens_q,
                                         const int32_t* seqlens, const int32_t* block_table, void* out, float* lse,
                                         int total_q, int B, int HQ, int HKV, int D, int PS, int BTW, int num_pages,
                                         size_t q_token_stride, size_t q_head_stride, int causal, int bf16,
                                         float scale, void* stream) {
  if (HKV <= 0 || HQ <= 0 || HQ % HKV != 0)
    return fail(MXFA_ERR_INVALID, "bad head geometry (HQ=%d HKV=%d)", HQ, HKV);
  if (int rc = paged_varlen_checks(k_cache, v_cache, k_scales, v_scales, cu_seqlens_q, seqlens, block_table, total_q,
                                   B, HKV, D, PS, BTW, num_pages))
    return rc;
  if (total_q == 0 || B == 0) return MXFA_OK;
  if (!q || !out) return fail(MXFA_ERR_INVALID, "null tensor pointer");
  if (!aligned16(q) || !aligned16(out) || (q_token_stride | q_head_stride) % 8 != 0)
    return fail(MXFA_ERR_INVALID, "q rows and out must be 16-byte aligned");
  const long long rows = static_cast<long long>(total_q) * HQ;
  if (rows > INT_MAX) return fail(MXFA_ERR_UNSUPPORTED, "%lld query rows above 2^31-1", rows);
  VarlenAttnParams p{};
  p.q = q;
  p.q_tok = q_token_stride;
  p.q_head = q_head_stride;
  p.k = static_cast<const uint8_t*>(k_cache);
  p.v = static_cast<const uint8_t*>(v_cache);
  p.k_scales = static_cast<const uint8_t*>(k_scales);
  p.v_scales = static_cast<const uint8_t*>(v_scales);
  p.cu = cu_seqlens_q;
  p.seqlens = seqlens;
  p.bt = block_table;
  p.out = out;
  p.lse = lse;
  p.T = total_q;
  p.B = B;
  p.HQ = HQ;
  p.HKV = HKV;
  p.GQ = HQ / HKV;
  p.PS = PS;
  p.BTW = BTW;
  p.P = num_pages;
  p.causal = causal ? 1 : 0;
  p.scale_log2 = scale * kLog2e;
  const bool quant = k_scales != nullptr;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (bf16)
    return D == 128 ? launch_varlen_rows<__nv_bfloat16, 128>(p, quant, st)
                    : launch_varlen_rows<__nv_bfloat16, 64>(p, quant, st);
  return D == 128 ? launch_varlen_rows<__half, 128>(p, quant, st) : launch_varlen_rows<__half, 64>(p, quant, st);
}

}  // extern "C"
