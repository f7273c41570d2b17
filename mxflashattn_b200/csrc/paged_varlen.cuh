// paged_varlen.cuh -- a ragged batch over a paged cache: append, read-back, row attention.
//
// Every kernel here takes packed tokens [T, heads, D] whose sequence b owns
// rows cu[b] .. cu[b+1], and seqlens[b], the tokens the cache holds for b
// with those included: packed row t of sequence b is position
// seqlens[b] - cu[b+1] + t of its block-table row.  No reference counterpart
// (the reference appends a uniform block, mxflashattn/reference.py:108-122).
//
// Quantised caches hold e4m3 codes [P, PS, HKV, D] and one e8m0 byte per
// (token, KV head), [P, HKV, PS]: value = code * 2^(byte - 127).  The scale
// is the smallest power of two s >= 2^-126 with max |x| <= 448 s.  e4m3 is a
// floating format, so a power of two costs no precision against max/448
// (only the last binade of the subnormal range differs), and in return x / s
// is exact before its one rounding, the scale is one byte, and code * s is
// exact in bf16: reading back or multiplying through never rounds again.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace mxfa {

// Sequence of packed token t (one warp): the number of entries cu[1..B] that
// are <= t, every lane comparing its own; B when every sequence ends before t.
// (A token before cu[0] comes out as one of the first sequence: callers ask.)
__device__ __forceinline__ int token_sequence(const int* __restrict__ cu, int B, int t, int lane) {
  int n = 0;
  for (int i = 0; i < B; i += 32) {
    const bool before = i + lane < B && cu[1 + i + lane] <= t;
    const int c = __popc(__ballot_sync(0xffffffffu, before));
    n += c;
    if (c < 32) break;  // the rest lie behind t
  }
  return n;
}

// Physical page and slot of position pos of sequence b; page -1, and the flag
// raised, when the table or the cache does not have it.
__device__ __forceinline__ int2 paged_slot(const int* __restrict__ bt, int b, int pos, int PS, int BTW, int P) {
  const int page = pos / PS;
  if (pos < 0 || page >= BTW) {
    raise_flag(MXFA_FLAG_TABLE_TOO_NARROW);
    return make_int2(-1, 0);
  }
  const int phys = bt[static_cast<size_t>(b) * BTW + page];
  if (phys < 0 || phys >= P) {
    raise_flag(MXFA_FLAG_PAGE_OUT_OF_RANGE);
    return make_int2(-1, 0);
  }
  return make_int2(phys, pos - page * PS);
}
// Element offset of a head's row in the cache, and of its scale.
__device__ __forceinline__ size_t row_offset(int2 slot, int h, int PS, int HKV, int D) {
  return ((static_cast<size_t>(slot.x) * PS + slot.y) * HKV + h) * D;
}
__device__ __forceinline__ size_t scale_offset(int2 slot, int h, int PS, int HKV) {
  return (static_cast<size_t>(slot.x) * HKV + h) * PS + slot.y;
}

struct PagedVarlenParams {
  const void* k;  // append: packed input; gather: packed output (written)
  const void* v;
  size_t k_tok, k_head, v_tok, v_head;  // strides of the packed tensors, elements
  uint8_t* k_cache;  // [P, PS, HKV, D]
  uint8_t* v_cache;
  uint8_t* k_scales;  // [P, HKV, PS], quantised caches
  uint8_t* v_scales;
  const int* cu;       // [B+1]
  const int* seqlens;  // [B]
  const int* bt;       // [B, BTW]
  int T, B, HKV, PS, BTW, P;
  int tok_per_cta;
  int* table;  // dense read-back: [B], written
  int* inexact;  // dense read-back to fp16, optional: [B][unpacked_blocks(T)], written for the tokens that exist
};

constexpr int kPvThreads = 256;
constexpr int kPvMaxTok = 16;  // tokens of one CTA (8 to 32 differ by 7%)
// CTAs of a sequence of `rows` unpacked tokens.
__host__ __device__ __forceinline__ int unpacked_blocks(int rows) { return (rows + kPvMaxTok - 1) / kPvMaxTok; }

// The cache slots of this CTA's tokens (page -1: not mapped), a token per lane of
// the first warp: one search for the first token, then each lane walks on to
// its own (consecutive tokens share sequences), so a CTA waits for three
// dependent loads however many tokens it has.
__device__ __forceinline__ void cta_token_rows(const PagedVarlenParams& p, int t0, int n, int2* slots) {
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x, t = t0 + lane;
    int b = token_sequence(p.cu, p.B, t0, lane);
    if (lane < n) {
      while (b < p.B && p.cu[b + 1] <= t) ++b;
      const bool owned = b < p.B && t >= p.cu[0];
      slots[lane] = owned ? paged_slot(p.bt, b, p.seqlens[b] - p.cu[b + 1] + t, p.PS, p.BTW, p.P) : make_int2(-1, 0);
    }
  }
  __syncthreads();
}

// A CTA's share of its rows (token, K heads then V heads): groups of D/8
// lanes take a row each; with fewer rows per token than groups, several
// tokens go side by side.  A thread keeps its head and walks tokens, kPvBatch
// rows at a time with their loads in flight together.
constexpr int kPvBatch = 4;
struct RowWalk {
  int pair, tok, step;  // first (K|V, head) pair, first token, tokens apart
  bool live;
};
template <int kGroup>
__device__ __forceinline__ RowWalk row_walk(int per_tok) {
  constexpr int kGroups = kPvThreads / kGroup;
  const int g = threadIdx.x / kGroup;
  if (per_tok >= kGroups) return {g, 0, 1, true};
  const int side = kGroups / per_tok;
  return {g % per_tok, g / per_tok, side, g / per_tok < side};
}

// Exponent k of the row scale 2^k for the largest finite magnitude amax:
// amax = 1.m * 2^E, 448 = 1.75 * 2^8.
__device__ __forceinline__ int scale_exponent(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  const int E = static_cast<int>(bits >> 23) - 127;
  const int k = E - ((bits & 0x7fffffu) > 0x600000u ? 7 : 8);
  return max(k, -126);
}

// The value of a 16-bit pattern without sign.
template <typename T>
__device__ __forceinline__ float magnitude_to_float(uint32_t bits) {
  if constexpr (std::is_same_v<T, __half>)
    return __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
  else
    return __uint_as_float(bits << 16);
}

// Append: a group of D/8 lanes moves one (token, KV head) row of K or V,
// eight values a lane.  HBM-bound: each value is read once and its code (or
// itself) written once; a group reduces its row's maximum by shuffles, so
// nothing is staged.  kVec: the rows allow 16-byte loads.  Quantising four ragged
// prompts of up to 15,000 tokens (8 heads of 128) takes 69 us on the device (0.69 of the copy bandwidth; 62
// without the scale bytes' stores, 74 with them gathered in shared memory first;
// 8 rows in flight instead of 4: 116 against 78).
template <typename T, int HD, bool kQuant, bool kVec>
__global__ void __launch_bounds__(kPvThreads) append_varlen_kernel(const PagedVarlenParams p) {
  constexpr int kGroup = HD / 8;
  __shared__ int2 s_slots[kPvMaxTok];
  const int t0 = blockIdx.x * p.tok_per_cta;
  const int n = min(p.tok_per_cta, p.T - t0);
  cta_token_rows(p, t0, n, s_slots);
  const int sub = threadIdx.x % kGroup;
  const RowWalk walk = row_walk<kGroup>(2 * p.HKV);
  // loop bounds are the same for every lane: the shuffles need all of them
  for (int pair0 = 0; pair0 < 2 * p.HKV; pair0 += kPvThreads / kGroup) {
    const int pair = pair0 + walk.pair;
    const bool live = walk.live && pair < 2 * p.HKV;
    const int kv = pair >= p.HKV, h = live ? pair - kv * p.HKV : 0;
    const T* src = kv ? static_cast<const T*>(p.v) + h * p.v_head : static_cast<const T*>(p.k) + h * p.k_head;
    const size_t stride = kv ? p.v_tok : p.k_tok;
    uint8_t* cache = kv ? p.v_cache : p.k_cache;
    for (int i0 = 0; i0 < n; i0 += walk.step * kPvBatch) {
      int2 slot[kPvBatch];
      uint4 raw[kPvBatch];
#pragma unroll
      for (int u = 0; u < kPvBatch; ++u) {
        const int i = i0 + walk.tok + u * walk.step;
        slot[u] = live && i < n ? s_slots[i] : make_int2(-1, 0);
        raw[u] = make_uint4(0, 0, 0, 0);
        if (slot[u].x >= 0) {
          const T* at = src + static_cast<size_t>(t0 + i) * stride + sub * 8;
          if constexpr (kVec) {
            raw[u] = *reinterpret_cast<const uint4*>(at);
          } else {
            const uint16_t* s16 = reinterpret_cast<const uint16_t*>(at);
            raw[u].x = s16[0] | (static_cast<uint32_t>(s16[1]) << 16);
            raw[u].y = s16[2] | (static_cast<uint32_t>(s16[3]) << 16);
            raw[u].z = s16[4] | (static_cast<uint32_t>(s16[5]) << 16);
            raw[u].w = s16[6] | (static_cast<uint32_t>(s16[7]) << 16);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < kPvBatch; ++u) {
        if constexpr (!kQuant) {
          if (slot[u].x >= 0)
            *reinterpret_cast<uint4*>(cache + (row_offset(slot[u], h, p.PS, p.HKV, HD) + sub * 8) * 2) = raw[u];
        } else {
          // magnitudes compare as integers, two at a time
          uint32_t top = __vmaxu2(__vmaxu2(raw[u].x & 0x7fff7fffu, raw[u].y & 0x7fff7fffu),
                                  __vmaxu2(raw[u].z & 0x7fff7fffu, raw[u].w & 0x7fff7fffu));
#pragma unroll
          for (int sh = kGroup / 2; sh > 0; sh >>= 1) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, sh));
          top = max(top & 0xffffu, top >> 16);
          constexpr uint32_t kInf = std::is_same_v<T, __half> ? 0x7c00u : 0x7f80u;
          float amax = magnitude_to_float<T>(top);
          const float2 a = Elem<T>::unpack(raw[u].x), b = Elem<T>::unpack(raw[u].y);
          const float2 c = Elem<T>::unpack(raw[u].z), d = Elem<T>::unpack(raw[u].w);
          const float x[8] = {a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
          if (__any_sync(0xffffffffu, top >= kInf)) {
            // the maximum is over finite values: an infinity saturates to 448 s
            // and a NaN stays a NaN, and neither costs the rest of its row
            amax = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float m = fabsf(x[j]);
              amax = m < INFINITY ? fmaxf(amax, m) : amax;
            }
#pragma unroll
            for (int sh = kGroup / 2; sh > 0; sh >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, sh));
          }
          const int k = scale_exponent(amax);
          const float inv = __uint_as_float(static_cast<uint32_t>(127 - k) << 23);
          uint32_t q[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * j] * inv, x[4 * j + 1] * inv),
                                                         __NV_SATFINITE, __NV_E4M3);
            const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * j + 2] * inv, x[4 * j + 3] * inv),
                                                         __NV_SATFINITE, __NV_E4M3);
            q[j] = lo | (hi << 16);
          }
          if (slot[u].x >= 0) {
            *reinterpret_cast<uint2*>(cache + row_offset(slot[u], h, p.PS, p.HKV, HD) + sub * 8) = make_uint2(q[0], q[1]);
            if (sub == 0)
              (kv ? p.v_scales : p.k_scales)[scale_offset(slot[u], h, p.PS, p.HKV)] = static_cast<uint8_t>(k + 127);
          }
        }
      }
    }
  }
}

// 2^(byte - 127) as a float (byte 0 is 2^-127, a subnormal; 255 is NaN).
__device__ __forceinline__ float e8m0_to_float(uint32_t byte) {
  return __uint_as_float(byte == 0 ? 0x00400000u : byte == 255 ? 0x7fffffffu : byte << 23);
}

// Eight e4m3 codes times one scale, as eight floats.
__device__ __forceinline__ void dequant8(uint2 codes, float s, float (&x)[8]) {
  uint32_t h[4];
  e4m3x4_to_f16x2x2(codes.x, h[0], h[1]);
  e4m3x4_to_f16x2x2(codes.y, h[2], h[3]);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = Elem<__half>::unpack(h[j]);
    x[2 * j] = f.x * s;
    x[2 * j + 1] = f.y * s;
  }
}

// Two floats to T, fp16 saturating at its largest value (NaN stays NaN).
template <typename T>
__device__ __forceinline__ uint32_t pack_sat(float lo, float hi) {
  if constexpr (std::is_same_v<T, __half>) {
    uint32_t r;
    asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
  } else {
    return Elem<T>::pack(lo, hi);
  }
}

// Read-back: the append's mirror; packed rows of tokens that are not mapped
// (or that no sequence holds) are zero.  HBM-bound, each code read once and
// each value written once: 91 us for 8 sequences of up to 16,384 tokens, 0.93 of the
// copy bandwidth.
// kDense: every sequence's tokens from position 0 on, sequence b (blockIdx.y)
// to rows b * T .. of the output, T rows a sequence, with the table
// (sequence b: page b) that reads the output as a cache of pages of T tokens.
// Rows past a sequence's length are left alone.  To fp16, p.inexact says of
// each CTA's tokens whether some value is not one of fp16's: past 65,504 (it
// saturates) or with bits under 2^-24.
template <typename T, int HD, bool kQuant, bool kDense = false>
__global__ void __launch_bounds__(kPvThreads) gather_varlen_kernel(const PagedVarlenParams p) {
  constexpr int kGroup = HD / 8;
  __shared__ int2 s_slots[kPvMaxTok];
  const int t0 = blockIdx.x * p.tok_per_cta;
  int n = min(p.tok_per_cta, p.T - t0);
  size_t row0 = t0;
  if constexpr (kDense) {
    const int b = blockIdx.y;
    n = min(n, p.seqlens[b] - t0);
    row0 += static_cast<size_t>(b) * p.T;
    if (blockIdx.x == 0 && threadIdx.x == 0) p.table[b] = b;
    if (n <= 0) return;
    if (threadIdx.x < n) s_slots[threadIdx.x] = paged_slot(p.bt, b, t0 + threadIdx.x, p.PS, p.BTW, p.P);
    __syncthreads();
  } else {
    cta_token_rows(p, t0, n, s_slots);
  }
  const int sub = threadIdx.x % kGroup;
  const RowWalk walk = row_walk<kGroup>(2 * p.HKV);
  constexpr bool kCheck = kDense && std::is_same_v<T, __half>;
  int lost = 0;
  if (!kCheck && !walk.live) return;
  for (int pair = walk.pair; (!kCheck || walk.live) && pair < 2 * p.HKV; pair += kPvThreads / kGroup) {
    const int kv = pair >= p.HKV, h = pair - kv * p.HKV;
    const uint8_t* cache = kv ? p.v_cache : p.k_cache;
    const uint8_t* scales = kv ? p.v_scales : p.k_scales;
    T* dst = static_cast<T*>(const_cast<void*>(kv ? p.v : p.k)) + row0 * p.HKV * HD + h * HD + sub * 8;
    for (int i0 = walk.tok; i0 < n; i0 += walk.step * kPvBatch) {
      uint4 out[kPvBatch];
      uint2 codes[kPvBatch];
      uint32_t byte[kPvBatch];
#pragma unroll
      for (int u = 0; u < kPvBatch; ++u) {
        const int i = i0 + u * walk.step;
        const int2 slot = i < n ? s_slots[i] : make_int2(-1, 0);
        out[u] = make_uint4(0, 0, 0, 0);
        codes[u] = make_uint2(0, 0);
        byte[u] = 127;
        if (slot.x >= 0) {
          const size_t at = row_offset(slot, h, p.PS, p.HKV, HD) + sub * 8;
          if constexpr (!kQuant) {
            out[u] = *reinterpret_cast<const uint4*>(cache + at * 2);
          } else {
            codes[u] = *reinterpret_cast<const uint2*>(cache + at);
            byte[u] = scales[scale_offset(slot, h, p.PS, p.HKV)];
          }
        }
      }
#pragma unroll
      for (int u = 0; u < kPvBatch; ++u) {
        const int i = i0 + u * walk.step;
        if constexpr (kQuant) {
          float x[8];
          dequant8(codes[u], e8m0_to_float(byte[u]), x);
          // read back, a value past fp16's largest is its infinity; as an operand it saturates
          auto pack = [](float lo, float hi) { return kDense ? pack_sat<T>(lo, hi) : Elem<T>::pack(lo, hi); };
          out[u] = make_uint4(pack(x[0], x[1]), pack(x[2], x[3]), pack(x[4], x[5]), pack(x[6], x[7]));
          if (kCheck && byte[u] - 112u > 22u) {  // (448 * 2^7 fits, and so does 2^-9, the codes' last place, times 2^-15)
            const uint32_t w[4] = {out[u].x, out[u].y, out[u].z, out[u].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 f = Elem<T>::unpack(w[j]);
              lost |= f.x != x[2 * j] && x[2 * j] == x[2 * j];
              lost |= f.y != x[2 * j + 1] && x[2 * j + 1] == x[2 * j + 1];
            }
          }
        }
        if (i < n) *reinterpret_cast<uint4*>(dst + static_cast<size_t>(i) * p.HKV * HD) = out[u];
      }
    }
  }
  if constexpr (kCheck) {
    lost = __syncthreads_or(lost);
    if (threadIdx.x == 0 && p.inexact != nullptr)
      p.inexact[static_cast<size_t>(blockIdx.y) * unpacked_blocks(p.T) + blockIdx.x] = lost;
  }
}

// ------------------------------------------------------------- row attention

struct VarlenAttnParams {
  const void* q;  // [T, HQ, D], strides q_tok / q_head
  size_t q_tok, q_head;
  const uint8_t* k;  // [P, PS, HKV, D]
  const uint8_t* v;
  const uint8_t* k_scales;  // [P, HKV, PS], quantised caches
  const uint8_t* v_scales;
  const int* cu;
  const int* seqlens;
  const int* bt;
  void* out;   // [T, HQ, D]
  float* lse;  // optional [T, HQ]
  int T, B, HQ, HKV, GQ, PS, BTW, P;
  int causal;
  float scale_log2;
};

// One warp per (token, query head): 32 keys a round, a key per lane for the
// scores, D/32 columns per lane for P.V.  Every K and V row is read by each
// of its query rows, so this form is for what the tiled kernel does not
// take.  All arithmetic is fp32; P is never rounded.
template <typename T, int HD, bool kQuant>
__global__ void __launch_bounds__(128) varlen_rows_kernel(const VarlenAttnParams p) {
  constexpr int kPer = HD / 32;
  __shared__ float s_q[4][HD];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long r = static_cast<long long>(blockIdx.x) * 4 + warp;
  if (r >= static_cast<long long>(p.T) * p.HQ) return;
  const int t = static_cast<int>(r / p.HQ);
  const int h = static_cast<int>(r - static_cast<long long>(t) * p.HQ);
  const int hk = h / p.GQ;
  const int b = token_sequence(p.cu, p.B, t, lane);
  if (b >= p.B || t < p.cu[0]) return;  // a padding row: nothing is written
  const T* qr = static_cast<const T*>(p.q) + static_cast<size_t>(t) * p.q_tok + h * p.q_head;
#pragma unroll
  for (int j = 0; j < kPer; ++j) s_q[warp][j * 32 + lane] = static_cast<float>(qr[j * 32 + lane]);
  __syncwarp();
  const int total = p.seqlens[b];
  const int pos = total - p.cu[b + 1] + t;
  const int end = p.causal ? min(total, pos + 1) : total;
  float m = -INFINITY, l = 0.f, acc[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) acc[j] = 0.f;
  for (int k0 = 0; k0 < end; k0 += 32) {
    int2 slot = make_int2(-1, 0);
    float vs = 1.f, s = -INFINITY;
    if (k0 + lane < end) slot = paged_slot(p.bt, b, k0 + lane, p.PS, p.BTW, p.P);
    const long long row = slot.x < 0 ? -1 : static_cast<long long>(slot.x) * p.PS + slot.y;
    if (row >= 0) {
      s = 0.f;
      if constexpr (kQuant) {
        const size_t at = scale_offset(slot, hk, p.PS, p.HKV);
        vs = e8m0_to_float(p.v_scales[at]);
        const float ks = e8m0_to_float(p.k_scales[at]);
        const uint8_t* kr = p.k + (row * p.HKV + hk) * HD;
        for (int c = 0; c < HD; c += 8) {
          float x[8];
          dequant8(*reinterpret_cast<const uint2*>(kr + c), ks, x);
#pragma unroll
          for (int j = 0; j < 8; ++j) s = fmaf(s_q[warp][c + j], x[j], s);
        }
      } else {
        const uint8_t* kr = p.k + (row * p.HKV + hk) * HD * 2;
        for (int c = 0; c < HD; c += 8) {
          const uint4 raw = *reinterpret_cast<const uint4*>(kr + c * 2);
          const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 f = Elem<T>::unpack(w[j]);
            s = fmaf(s_q[warp][c + 2 * j], f.x, s);
            s = fmaf(s_q[warp][c + 2 * j + 1], f.y, s);
          }
        }
      }
      s *= p.scale_log2;
    }
    float mx = s;
#pragma unroll
    for (int sh = 16; sh > 0; sh >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, sh));
    const float m_new = fmaxf(m, mx);
    // nothing visible yet; a NaN score (which the maximum ignores) goes on
    if (m_new == -INFINITY && !__any_sync(0xffffffffu, s != s)) continue;
    const float alpha = fast_exp2(m - m_new);
    const float pr = row >= 0 ? fast_exp2(s - m_new) : 0.f;
    m = m_new;
    float sum = pr;
#pragma unroll
    for (int sh = 16; sh > 0; sh >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, sh);
    l = l * alpha + sum;
#pragma unroll
    for (int j = 0; j < kPer; ++j) acc[j] *= alpha;
    const int n = min(32, end - k0);
    for (int i = 0; i < n; ++i) {
      const long long vrow = __shfl_sync(0xffffffffu, row, i);
      const float w = __shfl_sync(0xffffffffu, pr * vs, i);
      if (vrow < 0) continue;
      if constexpr (kQuant) {
        const uint8_t* vr = p.v + (vrow * p.HKV + hk) * HD + lane * kPer;
#pragma unroll
        for (int j = 0; j < kPer; ++j)
          acc[j] = fmaf(w, __half2float(__half(__nv_cvt_fp8_to_halfraw(vr[j], __NV_E4M3))), acc[j]);
      } else {
        const T* vr = reinterpret_cast<const T*>(p.v + (vrow * p.HKV + hk) * HD * 2) + lane * kPer;
#pragma unroll
        for (int j = 0; j < kPer; ++j) acc[j] = fmaf(w, static_cast<float>(vr[j]), acc[j]);
      }
    }
  }
  const float inv = l != 0.f ? 1.f / l : 0.f;  // a NaN sum stays one
  T* orow = static_cast<T*>(p.out) + (static_cast<size_t>(t) * p.HQ + h) * HD + lane * kPer;
#pragma unroll
  for (int j = 0; j < kPer; ++j) orow[j] = Elem<T>::from_float(acc[j] * inv);
  if (p.lse != nullptr && lane == 0)
    p.lse[static_cast<size_t>(t) * p.HQ + h] = l != 0.f ? (m + log2f(l)) * kLn2 : -INFINITY;
}

}  // namespace mxfa
