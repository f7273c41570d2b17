// capi_varlen.cuh -- extern "C" entry points of the ragged paged-cache operators (included by capi.cu).
#pragma once

namespace mxfa {
namespace {

int paged_varlen_checks(const void* k_cache, const void* v_cache, const void* k_scales, const void* v_scales,
                               const int32_t* cu_seqlens, const int32_t* seqlens, const int32_t* block_table,
                               int total, int B, int HKV, int D, int PS, int BTW, int num_pages) {
  if (D != 64 && D != 128) return fail(MXFA_ERR_UNSUPPORTED, "head dim %d not in {64, 128}", D);
  if (total < 0 || B < 0 || HKV <= 0) return fail(MXFA_ERR_INVALID, "bad ragged batch geometry");
  if (PS <= 0 || num_pages <= 0 || BTW < 0) return fail(MXFA_ERR_INVALID, "bad cache geometry");
  if (total == 0 || B == 0) return MXFA_OK;
  if (BTW == 0) return fail(MXFA_ERR_INVALID, "bad cache geometry");
  if (!k_cache || !v_cache || !cu_seqlens || !seqlens || !block_table)
    return fail(MXFA_ERR_INVALID, "null tensor pointer");
  if ((k_scales == nullptr) != (v_scales == nullptr))
    return fail(MXFA_ERR_INVALID, "k_scales and v_scales must both be given");
  if (!aligned16(k_cache) || !aligned16(v_cache)) return fail(MXFA_ERR_INVALID, "caches must be 16-byte aligned");
  if (!aligned4(k_scales) || !aligned4(v_scales)) return fail(MXFA_ERR_INVALID, "scales must be 4-byte aligned");
  int cap = 0;
  return cache_capacity(block_table, BTW, PS, &cap);
}

// Tokens a CTA takes: one while that still fills the GPU's CTA slots (8 of
// 256 threads per SM), so a decode step's few tokens spread over every SM,
// and up to 16 for long prompts, where a CTA's token lookups overlap (read-back of
// 8 x 16,384 tokens: 91 us at 16, 97 at 32, 93 at 8; the append, 69 now, was at 78, 78, 81 then).
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

// ---------------------------------------------------- tiled attention, plan

// What the tiled kernel takes: whole 8-row groups per page, and at least one
// token's heads per tile.
bool chunk_tiled(int HQ, int HKV, int PS) { return PS % 8 == 0 && HQ / HKV <= kTcRows; }

// CTA slots per KV head a step's work is divided by (one CTA per SM).
int chunk_share(int HKV) {
  const int n = sm_count() / HKV;
  return n < 1 ? 1 : n;
}
int chunk_parts_cap(int HKV) { return 2 * chunk_share(HKV) + 2; }
int chunk_items_cap(int total_q, int B, int HQ, int HKV) {
  const int tok = kTcRows / (HQ / HKV);
  return total_q / tok + (B < total_q ? B : total_q) + chunk_share(HKV) + 1;
}

struct ChunkMaps {
  CUtensorMap k{}, v{};
};
MapCache<ChunkMaps> g_chunk_maps(8192);
MapCache<CUtensorMap> g_chunk_q_maps(4096);

// 5-D view of a 16-bit cache: (64 columns, head, row of an 8-row group,
// 64-column block, group).  A box of g groups lands as [group][block][8 rows]
// [128 B], 128-byte swizzle: boxes of any row count stack into one tile with
// a constant group stride.
bool encode_chunk_kv(CUtensorMap* map, const void* base, int D, int HKV, long long slots, int box) {
  auto enc = tensor_map_encoder();
  if (enc == nullptr) return false;
  const cuuint64_t row = static_cast<cuuint64_t>(HKV) * D * 2;
  cuuint64_t dims[5] = {64, static_cast<cuuint64_t>(HKV), 8, static_cast<cuuint64_t>(D / 64),
                        static_cast<cuuint64_t>(slots / 8)};
  cuuint64_t strides[4] = {static_cast<cuuint64_t>(D) * 2, row, 128, 8 * row};
  cuuint32_t dim[5] = {64, 1, 8, static_cast<cuuint32_t>(D / 64), static_cast<cuuint32_t>(box / 8)};
  cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 5, const_cast<void*>(base), dims, strides, dim, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// 3-D view of an e4m3 cache: (D bytes, head, row), rows unswizzled.
bool encode_chunk_kv8(CUtensorMap* map, const void* base, int D, int HKV, long long slots, int box) {
  auto enc = tensor_map_encoder();
  if (enc == nullptr) return false;
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(HKV), static_cast<cuuint64_t>(slots)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(HKV) * D};
  cuuint32_t dim[3] = {static_cast<cuuint32_t>(D), 1, static_cast<cuuint32_t>(box)};
  cuuint32_t estr[3] = {1, 1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, dim, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Queries [T][HQ][D] with strides: boxes of (64 columns, GQ heads, 128 / GQ
// tokens), so a tile's row is token * GQ + head.
bool encode_chunk_q(CUtensorMap* map, const void* q, int D, int HQ, int T, int GQ, size_t tok, size_t head) {
  auto enc = tensor_map_encoder();
  if (enc == nullptr) return false;
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(HQ), static_cast<cuuint64_t>(T)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(head) * 2, static_cast<cuuint64_t>(tok) * 2};
  cuuint32_t dim[3] = {64, static_cast<cuuint32_t>(GQ), static_cast<cuuint32_t>(kTcRows / GQ)};
  cuuint32_t estr[3] = {1, 1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void*>(q), dims, strides, dim, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int HD, bool kQuant>
int launch_chunk_inst(const ChunkParams& p, dim3 grid, const CUtensorMap& mq, const ChunkMaps& m, cudaStream_t st) {
  static std::atomic<unsigned long long> done{0};
  auto kern = chunk_attn_kernel<T, HD, kQuant>;
  if (int rc = ensure_smem(kern, ChunkCfg<HD, kQuant>::kSmemBytes, done)) return rc;
  kern<<<grid, ChunkCfg<HD, kQuant>::kThreads, ChunkCfg<HD, kQuant>::kSmemBytes, st>>>(p, mq, m.k, m.v);
  return check_launch("chunk_attn_kernel");
}

template <typename T>
int launch_chunk(const ChunkParams& p, int D, bool quant, dim3 grid, const CUtensorMap& mq, const ChunkMaps& m,
                 cudaStream_t st) {
  if (D == 128)
    return quant ? launch_chunk_inst<T, 128, true>(p, grid, mq, m, st)
                 : launch_chunk_inst<T, 128, false>(p, grid, mq, m, st);
  return quant ? launch_chunk_inst<T, 64, true>(p, grid, mq, m, st)
               : launch_chunk_inst<T, 64, false>(p, grid, mq, m, st);
}

int run_chunk(const VarlenAttnParams& a, int D, const void* plan, size_t plan_bytes, void* workspace,
              size_t workspace_bytes, unsigned* counters, bool bf16, cudaStream_t st, const int* inexact = nullptr,
              int unpacked = 0) {
  const bool quant = a.k_scales != nullptr;
  if (plan == nullptr || plan_bytes < mxfa_chunk_plan_bytes(a.T, a.B, a.HQ, a.HKV) || !aligned16(plan))
    return fail(MXFA_ERR_INVALID, "plan missing, too small or unaligned (%zu < %zu bytes)", plan_bytes,
                mxfa_chunk_plan_bytes(a.T, a.B, a.HQ, a.HKV));
  const size_t need = mxfa_chunk_workspace_bytes(a.HKV, D);
  if (workspace == nullptr || workspace_bytes < need || !aligned16(workspace))
    return fail(MXFA_ERR_INVALID, "chunk workspace too small or unaligned (%zu < %zu bytes)", workspace_bytes, need);
  if (counters == nullptr || !aligned4(counters)) return fail(MXFA_ERR_INVALID, "counters missing or unaligned");
  const long long slots = static_cast<long long>(a.P) * a.PS;
  if (slots > INT_MAX) return fail(MXFA_ERR_UNSUPPORTED, "%lld cache slots above 2^31-1", slots);
  ChunkParams p{};
  p.plan = static_cast<const int*>(plan);
  p.bt = a.bt;
  p.out = a.out;
  p.lse = a.lse;
  p.k_scales = a.k_scales;
  p.v_scales = a.v_scales;
  p.inexact = inexact;
  p.unpacked = unpacked;
  p.parts_cap = chunk_parts_cap(a.HKV);
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = p.part_o + static_cast<size_t>(a.HKV) * p.parts_cap * kTcRows * D;
  p.counters = counters;
  p.T = a.T;
  p.B = a.B;
  p.HQ = a.HQ;
  p.HKV = a.HKV;
  p.GQ = a.GQ;
  p.PS = a.PS;
  p.BTW = a.BTW;
  p.P = a.P;
  p.box = quant ? ChunkCfg<128, true>::kRawKeys : kTcKeys;
  while (a.PS % p.box != 0) p.box >>= 1;  // the largest power of two, up to a (half) tile, that divides the page
  p.causal = a.causal;
  p.scale_log2 = a.scale_log2;
  int dev = 0;
  cudaGetDevice(&dev);
  ChunkMaps maps;
  const MapKey key{dev, a.k, a.v, nullptr, D, a.HKV, slots, p.box * 2 + (quant ? 1 : 0)};
  if (!g_chunk_maps.get(key, &maps)) {
    const bool ok = quant ? encode_chunk_kv8(&maps.k, a.k, D, a.HKV, slots, p.box) &&
                                encode_chunk_kv8(&maps.v, a.v, D, a.HKV, slots, p.box)
                          : encode_chunk_kv(&maps.k, a.k, D, a.HKV, slots, p.box) &&
                                encode_chunk_kv(&maps.v, a.v, D, a.HKV, slots, p.box);
    if (!ok) return fail(MXFA_ERR_UNSUPPORTED, "TMA descriptor encoding failed for the cache");
    g_chunk_maps.put(key, maps);
  }
  CUtensorMap mq;
  const MapKey qkey{dev, a.q, nullptr, nullptr, (static_cast<long long>(D) << 32) | a.GQ,
                    (static_cast<long long>(a.HQ) << 32) | static_cast<unsigned>(a.T),
                    static_cast<long long>(a.q_tok), static_cast<long long>(a.q_head)};
  if (!g_chunk_q_maps.get(qkey, &mq)) {
    if (!encode_chunk_q(&mq, a.q, D, a.HQ, a.T, a.GQ, a.q_tok, a.q_head))
      return fail(MXFA_ERR_UNSUPPORTED, "TMA descriptor encoding failed for the queries");
    g_chunk_q_maps.put(qkey, mq);
  }
  const long long blocks = static_cast<long long>(a.HKV) * chunk_items_cap(a.T, a.B, a.HQ, a.HKV);
  if (blocks > INT_MAX) return fail(MXFA_ERR_UNSUPPORTED, "%lld items exceed the grid", blocks);
  const dim3 grid(static_cast<unsigned>(blocks));
  return bf16 ? launch_chunk<__nv_bfloat16>(p, D, quant, grid, mq, maps, st)
              : launch_chunk<__half>(p, D, quant, grid, mq, maps, st);
}

// Checks of a ragged attention call, and its parameters (T = 0 where there is nothing to do).
int varlen_params(VarlenAttnParams* params, const void* q, const void* k_cache, const void* v_cache,
                  const void* k_scales, const void* v_scales, const int32_t* cu_seqlens_q, const int32_t* seqlens,
                  const int32_t* block_table, void* out, float* lse, int total_q, int B, int HQ, int HKV, int D, int PS,
                  int BTW, int num_pages, size_t q_token_stride, size_t q_head_stride, int causal, float scale) {
  VarlenAttnParams& p = *params;
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
  return MXFA_OK;
}

// Unpacks a quantised cache's sequences (mxfa_kvcache_unpack_launch); inexact: see PagedVarlenParams.
int unpack_impl(const void* k_cache, const void* v_cache, const void* k_scales, const void* v_scales,
                const int32_t* seqlens, const int32_t* block_table, void* k_out, void* v_out,
                int32_t* table_out, int B, int rows, int HKV, int D, int PS, int BTW, int num_pages,
                int bf16, int32_t* inexact, cudaStream_t st) {
  // (the lengths stand in for the offsets, which this call has none of)
  if (int rc = paged_varlen_checks(k_cache, v_cache, k_scales, v_scales, seqlens, seqlens, block_table, rows, B, HKV,
                                   D, PS, BTW, num_pages))
    return rc;
  if (rows == 0 || B == 0) return MXFA_OK;
  if (k_scales == nullptr) return fail(MXFA_ERR_INVALID, "unpacking is for quantised caches");
  if (!k_out || !v_out || !table_out) return fail(MXFA_ERR_INVALID, "null tensor pointer");
  if (!aligned16(k_out) || !aligned16(v_out)) return fail(MXFA_ERR_INVALID, "outputs must be 16-byte aligned");
  if (B > 65535) return fail(MXFA_ERR_UNSUPPORTED, "%d sequences exceed the grid", B);
  PagedVarlenParams p{};
  p.k = k_out;
  p.v = v_out;
  p.k_cache = static_cast<uint8_t*>(const_cast<void*>(k_cache));
  p.v_cache = static_cast<uint8_t*>(const_cast<void*>(v_cache));
  p.k_scales = static_cast<uint8_t*>(const_cast<void*>(k_scales));
  p.v_scales = static_cast<uint8_t*>(const_cast<void*>(v_scales));
  p.seqlens = seqlens;
  p.bt = block_table;
  p.T = rows;
  p.B = B;
  p.HKV = HKV;
  p.PS = PS;
  p.BTW = BTW;
  p.P = num_pages;
  p.tok_per_cta = kPvMaxTok;
  p.table = table_out;
  p.inexact = inexact;
  const dim3 grid(unpacked_blocks(rows), B);
  if (bf16)
    D == 128 ? gather_varlen_kernel<__nv_bfloat16, 128, true, true><<<grid, kPvThreads, 0, st>>>(p)
             : gather_varlen_kernel<__nv_bfloat16, 64, true, true><<<grid, kPvThreads, 0, st>>>(p);
  else
    D == 128 ? gather_varlen_kernel<__half, 128, true, true><<<grid, kPvThreads, 0, st>>>(p)
             : gather_varlen_kernel<__half, 64, true, true><<<grid, kPvThreads, 0, st>>>(p);
  return check_launch("gather_varlen_kernel(dense)");
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
  if (total == 0) return MXFA_OK;  // (without sequences every row is one that nobody owns, and becomes zero)
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

size_t mxfa_chunk_plan_bytes(int total_q, int B, int HQ, int HKV) {
  if (total_q <= 0 || B <= 0 || HKV <= 0 || HQ <= 0 || HQ % HKV != 0 || HQ / HKV > kTcRows) return 0;
  return (static_cast<size_t>(kPlanHeader) + B + 1) * 4 +
         static_cast<size_t>(chunk_items_cap(total_q, B, HQ, HKV)) * sizeof(ChunkItem);
}

size_t mxfa_chunk_workspace_bytes(int HKV, int D) {
  if (HKV <= 0 || (D != 64 && D != 128)) return 0;
  return static_cast<size_t>(HKV) * chunk_parts_cap(HKV) * kTcRows * (static_cast<size_t>(D) + 2) * sizeof(float);
}

size_t mxfa_chunk_counter_bytes(int HKV) {
  if (HKV <= 0) return 0;
  return static_cast<size_t>(HKV) * (chunk_parts_cap(HKV) / 2 + 1) * sizeof(unsigned);
}

int mxfa_kvcache_chunk_plan_launch(const int32_t* cu_seqlens_q, const int32_t* seqlens, void* plan, size_t plan_bytes,
                                   int total_q, int B, int HQ, int HKV, int causal, void* stream) {
  if (total_q < 0 || B < 0 || HKV <= 0 || HQ <= 0 || HQ % HKV != 0)
    return fail(MXFA_ERR_INVALID, "bad ragged batch geometry");
  if (HQ / HKV > kTcRows) return fail(MXFA_ERR_UNSUPPORTED, "%d query heads per KV head exceed a tile", HQ / HKV);
  if (total_q == 0 || B == 0) return MXFA_OK;
  if (!cu_seqlens_q || !seqlens || !plan) return fail(MXFA_ERR_INVALID, "null tensor pointer");
  if (plan_bytes < mxfa_chunk_plan_bytes(total_q, B, HQ, HKV) || !aligned16(plan))
    return fail(MXFA_ERR_INVALID, "plan too small or unaligned (%zu bytes)", plan_bytes);
  ChunkPlanParams p{};
  p.cu = cu_seqlens_q;
  p.seqlens = seqlens;
  p.plan = static_cast<int*>(plan);
  p.T = total_q;
  p.B = B;
  p.tok = kTcRows / (HQ / HKV);
  p.items_cap = chunk_items_cap(total_q, B, HQ, HKV);
  p.parts_cap = chunk_parts_cap(HKV);
  p.slots = sm_count();
  p.HKV = HKV;
  p.share = chunk_share(HKV);
  p.min_part = 4;
  p.causal = causal ? 1 : 0;
  chunk_plan_kernel<<<1, kPlanThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
  return check_launch("chunk_plan_kernel");
}

int mxfa_kvcache_varlen_attention_launch(const void* q, const void* k_cache, const void* v_cache,
                                         const void* k_scales, const void* v_scales, const int32_t* cu_seqlens_q,
                                         const int32_t* seqlens, const int32_t* block_table, const void* plan,
                                         size_t plan_bytes, void* out, float* lse, void* workspace,
                                         size_t workspace_bytes, unsigned* counters, int total_q, int B, int HQ, int HKV, int D, int PS, int BTW, int num_pages,
                                         size_t q_token_stride, size_t q_head_stride, int causal, int bf16,
                                         float scale, void* stream) {
  VarlenAttnParams p{};
  if (int rc = varlen_params(&p, q, k_cache, v_cache, k_scales, v_scales, cu_seqlens_q, seqlens, block_table, out, lse,
                             total_q, B, HQ, HKV, D, PS, BTW, num_pages, q_token_stride, q_head_stride, causal, scale))
    return rc;
  if (p.T == 0) return MXFA_OK;
  const bool quant = k_scales != nullptr;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (chunk_tiled(HQ, HKV, PS))
    return run_chunk(p, D, plan, plan_bytes, workspace, workspace_bytes, counters, bf16 != 0, st);
  if (bf16)
    return D == 128 ? launch_varlen_rows<__nv_bfloat16, 128>(p, quant, st)
                    : launch_varlen_rows<__nv_bfloat16, 64>(p, quant, st);
  return D == 128 ? launch_varlen_rows<__half, 128>(p, quant, st) : launch_varlen_rows<__half, 64>(p, quant, st);
}

int mxfa_kvcache_step_attention_launch(const void* q, const void* k_cache, const void* v_cache, const void* k_scales,
                                       const void* v_scales, const int32_t* cu_seqlens_q, const int32_t* seqlens,
                                       const int32_t* block_table, const int32_t* length_order, void* out, float* lse,
                                       void* workspace, size_t workspace_bytes, unsigned* counters, int total_q, int B,
                                       int max_q, int HQ, int HKV, int D, int PS, int BTW, int num_pages,
                                       int num_splits, int chunk_len, int causal, int bf16, float scale,
                                       void* stream) {
  if (HKV <= 0 || HQ <= 0 || HQ % HKV != 0)
    return fail(MXFA_ERR_INVALID, "bad head geometry (HQ=%d HKV=%d)", HQ, HKV);
  if (int rc = paged_varlen_checks(k_cache, v_cache, k_scales, v_scales, cu_seqlens_q, seqlens, block_table, total_q,
                                   B, HKV, D, PS, BTW, num_pages))
    return rc;
  if (total_q == 0 || B == 0 || max_q == 0) return MXFA_OK;
  if (max_q < 0) return fail(MXFA_ERR_INVALID, "max_q must not be negative");
  if (counters == nullptr) return fail(MXFA_ERR_INVALID, "counters is NULL");
  const bool quant = k_scales != nullptr;
  if (quant && (D != 128 || PS % kTileTok != 0))
    return fail(MXFA_ERR_UNSUPPORTED, "a quantised step needs head dim 128 and pages of a multiple of %d", kTileTok);
  if (!aligned16(k_scales) || !aligned16(v_scales)) return fail(MXFA_ERR_INVALID, "scales must be 16-byte aligned");
  return kvcache_attention_impl(q, k_cache, v_cache, block_table, seqlens, out, lse, workspace, workspace_bytes, B,
                                max_q, HQ, HKV, D, PS, BTW, num_pages, 0, num_splits, chunk_len, causal, bf16, scale,
                                nullptr, nullptr, counters, stream, quant, 1.f, 1.f, length_order,
                                static_cast<const uint8_t*>(k_scales), static_cast<const uint8_t*>(v_scales),
                                cu_seqlens_q, total_q);
}

int mxfa_kvcache_unpack_launch(const void* k_cache, const void* v_cache, const void* k_scales, const void* v_scales,
                               const int32_t* seqlens, const int32_t* block_table, void* k_out, void* v_out,
                               int32_t* table_out, int B, int rows, int HKV, int D, int PS, int BTW, int num_pages,
                               int bf16, void* stream) {
  return unpack_impl(k_cache, v_cache, k_scales, v_scales, seqlens, block_table, k_out, v_out, table_out, B, rows, HKV,
                     D, PS, BTW, num_pages, bf16, nullptr, static_cast<cudaStream_t>(stream));
}

size_t mxfa_unpack_flag_bytes(int B, int rows) {
  return B <= 0 || rows <= 0 ? 0 : static_cast<size_t>(B) * unpacked_blocks(rows) * sizeof(int32_t);
}

int mxfa_kvcache_varlen_attention_half_launch(const void* q, const void* k_cache, const void* v_cache,
                                              const void* k_scales, const void* v_scales,
                                              const int32_t* cu_seqlens_q, const int32_t* seqlens,
                                              const int32_t* block_table, const void* plan, size_t plan_bytes,
                                              void* out, float* lse, void* workspace, size_t workspace_bytes,
                                              unsigned* counters, void* k_rows, void* v_rows, int32_t* table_out,
                                              int32_t* inexact, int total_q, int B, int HQ, int HKV, int D, int PS,
                                              int BTW, int num_pages, int rows, size_t q_token_stride,
                                              size_t q_head_stride, int causal, float scale, void* stream) {
  VarlenAttnParams p{};
  if (int rc = varlen_params(&p, q, k_cache, v_cache, k_scales, v_scales, cu_seqlens_q, seqlens, block_table, out, lse,
                             total_q, B, HQ, HKV, D, PS, BTW, num_pages, q_token_stride, q_head_stride, causal, scale))
    return rc;
  if (p.T == 0) return MXFA_OK;
  if (!chunk_tiled(HQ, HKV, PS)) return fail(MXFA_ERR_UNSUPPORTED, "not a call of the tiled kernel (page size %d)", PS);
  if (rows <= 0 || inexact == nullptr) return fail(MXFA_ERR_INVALID, "unpacked rows or their flags missing");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (int rc = unpack_impl(k_cache, v_cache, k_scales, v_scales, seqlens, block_table, k_rows, v_rows, table_out, B, rows,
                           HKV, D, PS, BTW, num_pages, 0, inexact, st))
    return rc;
  VarlenAttnParams unpacked = p;
  unpacked.k = static_cast<const uint8_t*>(k_rows);
  unpacked.v = static_cast<const uint8_t*>(v_rows);
  unpacked.k_scales = unpacked.v_scales = nullptr;
  unpacked.bt = table_out;
  unpacked.PS = rows;
  unpacked.BTW = 1;
  unpacked.P = B;
  if (int rc = run_chunk(unpacked, D, plan, plan_bytes, workspace, workspace_bytes, counters, false, st, inexact, rows))
    return rc;
  return run_chunk(p, D, plan, plan_bytes, workspace, workspace_bytes, counters, false, st, inexact, rows);
}

}  // extern "C"
