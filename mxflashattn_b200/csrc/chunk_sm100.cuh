// chunk_sm100.cuh -- attention of a ragged batch over a paged cache on the
// 5th-generation tensor cores, and the plan that divides it.
//
// A tile is 128 query rows of one KV head: 128 / GQ tokens of one sequence
// times the GQ query heads that share the head (row r = token r / GQ, head
// r % GQ).  Packing heads with tokens reads each K/V row once per 128 query
// rows whatever GQ is, fills the tile from 128 / GQ tokens on, and keeps the
// causal diagonal of a tile 128 / GQ keys wide.
//
// An item is a tile and a range of 128-key tiles.  chunk_plan_kernel writes
// the items of a step once (every layer uses them): tiles whose keys exceed
// a CTA's fair share are split, and items go out longest first.  A split
// tile's parts leave (O, m, l) in a workspace, and the part that finishes
// last merges them in split order.
//
// The pipeline of one item is prefill_sm100.cuh's: score and P.V products
// from two issuing threads, three score buffers and one O in tensor memory,
// softmax groups (two, or three at D = 64 on 16-bit caches) on alternating key
// tiles that share a running maximum.
// What differs:
//  - K and V come through the block table: one TMA box per page piece (the
//    largest power of two that divides page size and tile, 8 rows at least),
//    each lane of a producer warp resolving and issuing its own box.  A box
//    lands as [8-row group][64-column block][8 rows][128 B], so any mix of
//    boxes makes one tile with a constant 8-row group stride.
//  - Keys that some row of the tile does not see have P = 0, but 0 * NaN is
//    NaN: V rows past the last visible key are zeroed in shared memory, and a
//    non-finite V element that only some rows see is zeroed and put into
//    those rows' output at the end.
//  - Quantised caches: four converter warpgroups turn the e4m3 tiles that TMA
//    lands into f16 tiles, times each row's scale relative to the tile's
//    largest (see kRefShift); the tile's own power of two goes into the softmax
//    in 32 bits.  bf16 queries become f16 the same way, row by row.  f16 needs
//    two instructions per pair of codes; widening to bf16 took five.  The scale
//    bytes come by a warp of their own.
//
// Measured (HQ 32, HKV 8, D 128, bf16): 2,048 tokens on 14,336 cached take 445 us
// in a burst (1,157 TFLOP/s) and 521 back to back under the power cap, 1,920
// cycles per key tile and SM, all included, against 1,024 of tensor work.  On 512
// tokens issue is active 0.44 per scheduler and the tensor pipe 46%: what remains
// is taken to be the latency from one score buffer's product to its next.  The loops stay
// rolled because all warps' code has to fit the instruction cache (541 -> 515 us).
// Converting e4m3 in the kernel takes 468 us for 1,024 tokens on 15,360, against
// 248 with the rows unpacked first, so only short pieces convert; 722 where every
// tile is wide (see kWideTile).
#pragma once

#include "paged_varlen.cuh"
#include "prefill_sm100.cuh"

namespace mxfa {

// ------------------------------------------------------------------- plan

struct ChunkItem {
  int b, row0, ntok, pos0;     // sequence, packed row of the first token, tokens, position of the first token
  int total, kt0, kt1, nsplit; // cached tokens, key tiles [kt0, kt1), parts of this tile
  int split, part0, group, pad;
};
constexpr int kPlanHeader = 16;  // ints before the items: [0] items
constexpr int kPlanThreads = 1024;
constexpr int kPlanBuckets = 256;
constexpr int kChunkMaxParts = 160;  // parts of one tile (their weights share memory with the K and V stages)

struct ChunkPlanParams {
  const int* cu;
  const int* seqlens;
  int* plan;     // header, items, then B + 1 tile offsets
  int T, B, tok; // tok: tokens per tile
  int items_cap, parts_cap;
  int slots, HKV;  // CTAs the GPU holds at once, KV heads
  int share;     // slots / HKV: what the step's work per KV head is divided by
  int min_part;  // key tiles a part holds at least
  int causal;
};

__device__ __forceinline__ int chunk_tiles_of(const ChunkPlanParams& p, int b) {
  const int lo = min(max(p.cu[b], 0), p.T), hi = min(max(p.cu[b + 1], lo), p.T);
  return (hi - lo + p.tok - 1) / p.tok;
}

// Item fields of tile i (its sequence by binary search in the tile offsets),
// and the key tiles it covers (at least one: a tile without keys still
// writes its rows).
__device__ __forceinline__ int chunk_tile(const ChunkPlanParams& p, const int* off, int i, ChunkItem& it) {
  int lo = 0, hi = p.B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (off[mid] <= i)
      lo = mid;
    else
      hi = mid;
  }
  const int b = lo;
  const int q0 = min(max(p.cu[b], 0), p.T);
  const int n = min(max(p.cu[b + 1], q0), p.T) - q0;
  const int t0 = (i - off[b]) * p.tok;
  it.b = b;
  it.row0 = q0 + t0;
  it.ntok = min(p.tok, n - t0);
  it.total = max(p.seqlens[b], 0);
  it.pos0 = it.total - n + t0;
  it.pad = 0;
  const int k_end = p.causal ? min(max(it.pos0 + it.ntok, 0), it.total) : it.total;
  return max(1, (k_end + kTcKeys - 1) / kTcKeys);
}

// Sum over the block (every thread gets it); s: one int of shared memory.
__device__ __forceinline__ int block_sum(int x, int* s) {
  x = __reduce_add_sync(0xffffffffu, x);
  __syncthreads();
  if (threadIdx.x == 0) *s = 0;
  __syncthreads();
  if ((threadIdx.x & 31) == 0) atomicAdd(s, x);
  __syncthreads();
  return *s;
}

// One block; the work is counted in key tiles.  Let fair = work / share, the
// tiles a CTA slot would get of an even division.
//  - Fewer tiles than slots: every tile is split into parts of at most L,
//    L the smallest for which the parts still go out in one wave.
//  - More: tiles longer than fair are split to it, so one long sequence does
//    not outlast the rest; without such, what remains after whole waves (the
//    shortest tiles) is split over the slots of the last one.  512 equal
//    items on 148 SMs: 3 waves and a split one instead of 4.  The step's one launch
// costs 16 to 25 us with its host call, for all layers; whole waves with a split
// remainder brought a long chunk from 482 to 455 us, one-wave splits with
// per-row merge weights a ragged one from 80 to 48.
// Parts of split tiles never exceed 2 * share.  Buckets of equal length
// order the items, longest first; which item of a bucket comes first is left
// to the atomics, since the order only schedules.
__global__ void __launch_bounds__(kPlanThreads) chunk_plan_kernel(const ChunkPlanParams p) {
  __shared__ int s_scan[kPlanThreads / 32];
  __shared__ int s_sum, s_max, s_parts, s_groups, s_tail, s_bad, s_hist[kPlanBuckets];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  ChunkItem* items = reinterpret_cast<ChunkItem*>(p.plan + kPlanHeader);
  int* off = p.plan + kPlanHeader + p.items_cap * static_cast<int>(sizeof(ChunkItem) / 4);
  if (tid == 0) s_max = s_parts = s_groups = s_tail = s_bad = 0;
  for (int i = tid; i < kPlanBuckets; i += kPlanThreads) s_hist[i] = 0;
  __syncthreads();
  // tile offsets: block-wide exclusive scan over the sequences
  int base = 0;
  for (int b0 = 0; b0 < p.B; b0 += kPlanThreads) {
    const int b = b0 + tid;
    const int n = b < p.B ? chunk_tiles_of(p, b) : 0;
    if (b < p.B && (p.cu[b] < 0 || p.cu[b + 1] < p.cu[b] || p.cu[b + 1] > p.T)) s_bad = 1;
    int x = n;
#pragma unroll
    for (int sh = 1; sh < 32; sh <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, sh);
      if (lane >= sh) x += y;
    }
    if (lane == 31) s_scan[warp] = x;
    __syncthreads();
    if (warp == 0) {
      int w = s_scan[lane];
#pragma unroll
      for (int sh = 1; sh < 32; sh <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, w, sh);
        if (lane >= sh) w += y;
      }
      s_scan[lane] = w;
    }
    __syncthreads();
    if (b < p.B) off[b] = base + x - n + (warp > 0 ? s_scan[warp - 1] : 0);
    base += s_scan[kPlanThreads / 32 - 1];
    __syncthreads();
  }
  int tiles = base;
  // (offsets that never decrease have p.T / p.tok + min(p.B, p.T) tiles at most, which the plan has room for)
  if (s_bad) {
    if (tid == 0) raise_flag(MXFA_FLAG_BAD_ORDER);
    tiles = 0;
  }
  if (tid == 0) off[p.B] = tiles;
  __syncthreads();  // off (global, this block's own writes) and the counters are visible

  // f(tile, its key tiles) over this thread's tiles; the first four lengths
  // stay in registers
  constexpr int kKeep = 4;
  int len[kKeep];
#pragma unroll
  for (int k = 0; k < kKeep; ++k) {
    ChunkItem it;
    const int i = tid + k * kPlanThreads;
    len[k] = i < tiles ? chunk_tile(p, off, i, it) : 0;
  }
  auto each = [&](auto f) {
#pragma unroll
    for (int k = 0; k < kKeep; ++k)
      if (tid + k * kPlanThreads < tiles) f(tid + k * kPlanThreads, len[k]);
    for (int i = tid + kKeep * kPlanThreads; i < tiles; i += kPlanThreads) {
      ChunkItem it;
      f(i, chunk_tile(p, off, i, it));
    }
  };
  long long work = 0;  // 64-bit sum in two halves
  int longest = 0;
  each([&](int, int n) {
    work += n;
    longest = max(longest, n);
  });
  atomicMax(&s_max, longest);
  const int lo16 = block_sum(static_cast<int>(work & 0xffff), &s_sum);
  const int hi16 = block_sum(static_cast<int>(work >> 16), &s_sum);
  const long long total = static_cast<long long>(hi16) * 65536 + lo16;
  longest = s_max;
  const int fair = static_cast<int>(min((total + p.share - 1) / p.share, 1ll << 30));
  int limit = max(max(fair, p.min_part), (longest + kChunkMaxParts - 1) / kChunkMaxParts);
  if (tiles > 0 && tiles < p.share) {
    int lo = limit, hi = max(longest, limit);
    while (lo < hi) {  // the smallest limit whose parts fit one wave
      const int mid = (lo + hi) >> 1;
      int n = 0;
      each([&](int, int m) { n += (m + mid - 1) / mid; });
      if (block_sum(n, &s_sum) <= p.share)
        hi = mid;
      else
        lo = mid + 1;
    }
    limit = lo;
  }
  // tiles that whole waves take unsplit, and the parts of each one behind them
  int whole = tiles, tail_parts = 1;
  if (tiles >= p.share && longest <= limit) {
    const int waves = static_cast<int>(static_cast<long long>(tiles) * p.HKV / p.slots);
    const int rest = tiles - static_cast<int>(static_cast<long long>(waves) * p.slots / p.HKV);
    if (rest > 0 && rest < tiles && p.slots / (rest * p.HKV) > 1) {
      whole = tiles - rest;
      tail_parts = p.slots / (rest * p.HKV);
    }
  }
  const int top = min(longest, limit);
  auto bucket_of = [&](int per) {
    return kPlanBuckets - 1 - static_cast<int>(static_cast<long long>(per) * (kPlanBuckets - 1) / max(top, 1));
  };
  each([&](int, int n) {
    const int parts = (n + limit - 1) / limit;
    atomicAdd(&s_hist[bucket_of((n + parts - 1) / parts)], parts);
  });
  __syncthreads();
  if (warp == 0) {  // exclusive scan of the buckets, longest first
    int run = 0;
    for (int b0 = 0; b0 < kPlanBuckets; b0 += 32) {
      const int n = s_hist[b0 + lane];
      int x = n;
#pragma unroll
      for (int sh = 1; sh < 32; sh <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, sh);
        if (lane >= sh) x += y;
      }
      s_hist[b0 + lane] = run + x - n;
      run += __shfl_sync(0xffffffffu, x, 31);
    }
    if (lane == 0) s_sum = run;
  }
  __syncthreads();
  each([&](int i, int n) {
    int parts = (n + limit - 1) / limit;
    int at = atomicAdd(&s_hist[bucket_of((n + parts - 1) / parts)], parts);
    if (tail_parts > 1 && at >= whole) {  // (parts is 1 wherever whole waves precede split tiles)
      parts = max(1, min(tail_parts, n / p.min_part));
      at = whole + atomicAdd(&s_tail, parts);
    }
    const int per = (n + parts - 1) / parts;
    ChunkItem it;
    chunk_tile(p, off, i, it);
    it.nsplit = parts;
    it.part0 = it.group = -1;
    if (parts > 1) {
      it.part0 = atomicAdd(&s_parts, parts);
      it.group = atomicAdd(&s_groups, 1);
    }
    for (int s = 0; s < parts; ++s) {
      it.split = s;
      it.kt0 = min(s * per, n);
      it.kt1 = min((s + 1) * per, n);
      if (at + s < p.items_cap) items[at + s] = it;
    }
  });
  __syncthreads();
  if (tid == 0) p.plan[0] = min(tail_parts > 1 ? whole + s_tail : s_sum, p.items_cap);
}

// --------------------------------------------------------------- attention

struct ChunkParams {
  const int* plan;
  const int* bt;
  void* out;   // [T, HQ, HD]
  float* lse;  // optional [T, HQ]
  const uint8_t* k_scales;  // [P, HKV, PS], quantised caches
  const uint8_t* v_scales;
  float* part_o;    // [HKV][parts_cap][128][HD]
  float* part_ml;   // [HKV][parts_cap][128][2]
  unsigned* counters;  // [HKV][parts_cap / 2 + 1], zero on entry and on exit
  int parts_cap;
  // fp16 queries over unpacked rows (optional): which blocks of kPvMaxTok
  // tokens of the first `unpacked` of a sequence fp16 does not hold exactly.
  // Items with such a token are left to the converting kernel, which is
  // launched behind the 16-bit one and takes no others.
  const int* inexact;
  int unpacked;
  int T, B, HQ, HKV, GQ, PS, BTW, P;
  int box;       // rows of one TMA box: divides PS and 128, a multiple of 8
  int causal;
  float scale_log2;
};

template <int HD, bool kQuant>
struct ChunkCfg {
  // softmax groups of four warps; group g takes tiles j % kGroups == g.  At D = 64 the products
  // of a tile are short and a third group pays (46.2 -> 43.4 us on ragged pieces, the one case it was
  // tried on; later steps brought them to 32-36); at D = 128 it costs (477 -> 494 us on a long one).
  static constexpr int kGroups = !kQuant && HD == 64 ? 3 : 2;
  static constexpr int kThreads = kQuant ? 1024 : 128 + 128 * kGroups;
  static constexpr int kDBlk = HD / 64;
  static constexpr int kStages = kQuant ? 2 : 3;
  static constexpr int kGroupBytes = kDBlk * 1024;        // 8 rows of a K or V tile
  static constexpr int kQBlk = 128 * 128;                 // one 64-column block of the Q tile
  static constexpr int kTile = 128 * HD * 2;
  // quantised: three e4m3 half tiles (64 keys) of K and three of V in flight
  static constexpr int kRawSlots = 3, kRawKeys = 64;
  static constexpr int kRawTile = kRawKeys * HD;
  static constexpr int kRawBytes = kQuant ? 2 * kRawSlots * kRawTile : 0;
  static constexpr int kQ = 0;
  static constexpr int kK = kQ + kTile;
  static constexpr int kV = kK + kStages * kTile;
  static constexpr int kRaw = kV + kStages * kTile;
  static constexpr int kMl = kQ;                          // epilogue exchange over Q once every product is done
  static constexpr int kMPub = kRaw + kRawBytes;  // [2][128] running maxima
  // quantised: [4 tiles][K|V][128] row factors (f16 pairs), [8] (K, V)
  // exponents of a tile (kWideTile: see there), [128] factors of the query rows
  static constexpr int kScale = kMPub + 2 * kTcRows * 4;
  static constexpr int kTileExp = kScale + (kQuant ? 4 * 2 * 128 * 4 : 0);
  static constexpr int kExpBytes = kTileExp + (kQuant ? 8 * 8 : 0);  // [8 tiles][K|V][128] exponent bytes
  static constexpr int kWide = kExpBytes + (kQuant ? 8 * 256 : 0);  // [8 tiles][128] (K factor, V exponent) of wide tiles
  static constexpr int kQScale = kWide + (kQuant ? 8 * 128 * 8 : 0);
  static constexpr int kBad = kQScale + (kQuant ? 128 * 4 : 0);  // [HD] first keys with a non-finite V
  static constexpr int kBar = kBad + HD * 4;
  static constexpr int kNumBars = 52;
  static constexpr int kSmemBytes = kBar + kNumBars * 8 + 32 + 1024;
  static constexpr uint32_t kTmemCols = 512;
  static constexpr uint32_t kTmemO = 3 * kTcKeys;
  static_assert(kSmemBytes <= 232448, "shared memory of one CTA");
};

struct ChunkBars {
  uint64_t q_full, q_ready, k_full[3], v_full[3], raw_full[2][3], raw_empty[2][3];
  uint64_t s_full[3], p_full[3], pv_done[3];
  uint64_t m_ready[2][4];
  uint64_t scale_ready[4], scale_free[4];  // quantised: the factors of tile t, slot t % 4
  uint64_t v_ok[2];  // 16-bit caches: the guarded V tiles (the last two at most) are clean
  uint64_t all_done;
};
static_assert(sizeof(ChunkBars) <= 52 * 8, "barrier block");

// Pairs of 16-bit values with an exponent of all ones.
template <typename T>
__device__ __forceinline__ bool any_nonfinite(uint4 v) {
  constexpr uint32_t e = std::is_same_v<T, __half> ? 0x7c007c00u : 0x7f807f80u;
  constexpr uint32_t one = std::is_same_v<T, __half> ? 0x04000400u : 0x00800080u;
  // adding one unit of exponent carries into the (masked) sign exactly when all its bits are set
  const uint32_t x = (((v.x & e) + one) | ((v.y & e) + one) | ((v.z & e) + one) | ((v.w & e) + one)) & 0x80008000u;
  return x != 0;
}

// First keys (relative to the first guarded tile, under 256) whose V is NaN,
// +inf and -inf in one column: three 10-bit fields, kNoKey where there is none.
constexpr unsigned kNoKey = 0x3ffu;
constexpr unsigned kNoBad = kNoKey | (kNoKey << 10) | (kNoKey << 20);

// A 16-byte chunk of V of key `rel` (columns d0 .. d0+7): zero its
// non-finite elements and note the key in their columns.
template <typename T>
__device__ __noinline__ uint4 strip_nonfinite(uint4 v, unsigned rel, unsigned* bad, volatile int* any_bad) {
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = Elem<T>::unpack(w[i]);
    const float x[2] = {f.x, f.y};
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (!(fabsf(x[j]) < INFINITY)) {
        const int at = 10 * (x[j] != x[j] ? 0 : x[j] > 0.f ? 1 : 2);
        unsigned old = bad[2 * i + j];
        while (((old >> at) & kNoKey) > rel) {
          const unsigned seen = atomicCAS(&bad[2 * i + j], old, (old & ~(kNoKey << at)) | (rel << at));
          if (seen == old) break;
          old = seen;
        }
        *any_bad = 1;
        w[i] &= j ? 0x0000ffffu : 0xffff0000u;
      }
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Exponent bytes (e8m0) of a tile are taken relative to the tile's largest
// one, ref: a 16-bit operand is code * 2^(byte - ref + 7), at most 448 * 2^7
// < 65504, and exact in f16 for rows down to 2^-22 of the tile's largest.
// 2^(ref - 127 - 7) multiplies the products in 32 bits.  ref is kept from
// 2^-60 up, so that 2^-ref and sums of it stay in range; values under 2^-75
// vanish.
//
// The largest row may be one that a query does not see, or weighs with next
// to nothing, and must not cost the others bits.  K has none to lose down to
// 2^-22.  P is relative to max(score) * 2^ref, which overstates the largest
// contribution by up to the spread of V's scales, and f16 has P's full 11
// bits only down to 2^-14: P is scaled up by 2^kPShift (with the lazy maximum
// at most 2^15), which makes up for a spread of as much.  A tile whose K
// scales are further apart than 2^kWideK or whose V scales are than 2^kWideV
// is *wide*: its operands are the codes as they are, the factors of each key
// are applied to its scores in 32 bits, and V's exponent joins the score key by
// key, as in the decode kernel (slower, on such tiles only).  Rows of zeros (byte 0 or 1, the smallest) have
// no part in this.
constexpr int kRefShift = 7, kRefMin = 127 - 60;
constexpr int kPShift = 7, kWideK = 22, kWideV = kPShift;
constexpr int kWideTile = 1 << 20;  // in place of a tile's K exponent
static_assert(kPShift + kRescaleThreshold <= 15.f, "P in f16");

// 2^e as an f16 pair for e <= 15; under 2^-24 it is 0.
__device__ __forceinline__ uint32_t pow2_f16x2(int e) {
  const uint32_t h = e >= -14 ? static_cast<uint32_t>(e + 15) << 10 : e >= -24 ? 1u << (e + 24) : 0u;
  return h | (h << 16);
}
__device__ __forceinline__ float pow2_f32(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// Eight e4m3 codes times a row's factor, as f16.
__device__ __forceinline__ uint4 codes_to_f16(uint2 codes, uint32_t factor) {
  uint4 h;
  e4m3x4_to_f16x2x2(codes.x, h.x, h.y);
  e4m3x4_to_f16x2x2(codes.y, h.z, h.w);
  return make_uint4(mul_f16x2(h.x, factor), mul_f16x2(h.y, factor), mul_f16x2(h.z, factor), mul_f16x2(h.w, factor));
}

// What a key of a wide tile puts on its scores: K's factor, and V's exponent,
// from the scales' bytes.  (A NaN V scale is in the operand, and takes no part in the
// row sum.)
__device__ __forceinline__ float2 wide_key(int kb, int vb) {
  return make_float2(e8m0_to_float(kb), vb == 255 ? 0.f : static_cast<float>(max(vb, kRefMin) - 127));
}
// 2^-e for a whole e: its bits come out of the sum with 1.5 * 2^23.
__device__ __forceinline__ float pow2_inverse(float e) {
  return __uint_as_float(0x3f800000u - (__float_as_uint(e + 12582912.f) << 23));
}

// Register shares of the quantised kernel's eight warpgroups (launched with 64
// each): producers, issuers, converters and the scale warp give theirs to
// the softmax.
template <int N>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
constexpr int kRegsIssue = 56, kRegsSoftmax = 128, kRegsConvert = 40, kRegsScale = 40;
static_assert(kRegsIssue + 2 * kRegsSoftmax + 4 * kRegsConvert + kRegsScale <= 8 * 64, "the launch's registers");

__device__ __forceinline__ void named_barrier_arrive(int id, int threads) {
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

template <typename T, int HD, bool kQuant>
__global__ void __launch_bounds__(ChunkCfg<HD, kQuant>::kThreads, 1)
    chunk_attn_kernel(const ChunkParams p, const __grid_constant__ CUtensorMap tmq,
                      const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv) {
  using Cfg = ChunkCfg<HD, kQuant>;
  constexpr int NS = Cfg::kStages;
  constexpr int NB = 3;
  constexpr int NG = Cfg::kGroups, kSoft = 128 * NG;  // softmax groups and threads
  using MT = std::conditional_t<kQuant, __half, T>;              // tensor-core operand type
  constexpr bool kConvertQ = kQuant && !std::is_same_v<T, __half>;  // bf16 queries become f16 in shared memory
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  ChunkBars* bars = reinterpret_cast<ChunkBars*>(sm + Cfg::kBar);
  float* ml = reinterpret_cast<float*>(sm + Cfg::kMl);
  unsigned* bad = reinterpret_cast<unsigned*>(sm + Cfg::kBad);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + Cfg::kBar + Cfg::kNumBars * 8);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* any_bad = reinterpret_cast<volatile int*>(tmem_slot + 2);
  int* s_last = reinterpret_cast<int*>(tmem_slot + 3);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // block: KV head, then item (one dimension, which alone has room for more than 65,535)
  const int hk = blockIdx.x % p.HKV, item = blockIdx.x / p.HKV;
  if (item >= p.plan[0]) return;
  const ChunkItem it = reinterpret_cast<const ChunkItem*>(p.plan + kPlanHeader)[item];
  // a plan made for another batch reaches nothing outside this one's tensors
  if (it.b < 0 || it.b >= p.B || it.row0 < 0 || it.ntok < 1 || it.ntok * p.GQ > kTcRows || it.row0 > p.T - it.ntok ||
      it.kt0 < 0 || it.nsplit < 1 || it.nsplit > kChunkMaxParts || it.split < 0 || it.split >= it.nsplit ||
      (it.nsplit > 1 && (it.part0 < 0 || it.part0 > p.parts_cap - it.nsplit || it.group < 0 || it.group > p.parts_cap / 2))) {
    if (threadIdx.x == 0) raise_flag(MXFA_FLAG_BAD_ORDER);
    return;
  }
  if (p.inexact != nullptr) {
    constexpr int kPer = kTcKeys / kPvMaxTok;  // blocks of a key tile
    const int tiles = (p.unpacked + kTcKeys - 1) / kTcKeys;
    const int end = min(min(it.kt1, tiles) * kPer, unpacked_blocks(min(it.total, p.unpacked)));
    const int* f = p.inexact + static_cast<size_t>(it.b) * unpacked_blocks(p.unpacked);
    int lost = 0;
    for (int i = min(it.kt0, tiles) * kPer + threadIdx.x; i < end; i += Cfg::kThreads) lost |= f[i];
    if ((__syncthreads_or(lost) != 0) != kQuant) return;
  }
  // keys the block table can hold; a longer sequence is flagged and cut
  const int k_lim = min(it.total, p.BTW * p.PS);
  if (threadIdx.x == 0 && it.total > k_lim) raise_flag(MXFA_FLAG_TABLE_TOO_NARROW);
  const int k_end = p.causal ? min(max(it.pos0 + it.ntok, 0), k_lim) : k_lim;    // keys some row sees
  const int vis_first = p.causal ? min(max(it.pos0 + 1, 0), k_lim) : k_lim;      // keys every row sees
  const int nkt = max(0, min(it.kt1, (k_end + kTcKeys - 1) / kTcKeys) - it.kt0);  // key tiles of this item
  const int key_base = it.kt0 * kTcKeys;
  const int nrows = it.ntok * p.GQ;

  if (threadIdx.x == 0) {
    mbar_init(&bars->q_full, 1);
    mbar_init(&bars->q_ready, 4);
    for (int i = 0; i < 4; ++i) {
      mbar_init(&bars->scale_ready[i], 1);
      mbar_init(&bars->scale_free[i], 16);
    }
    for (int i = 0; i < 3; ++i) {
      mbar_init(&bars->k_full[i], kQuant ? 8 : 1);
      mbar_init(&bars->v_full[i], kQuant ? 8 : 1);
      for (int kv = 0; kv < 2; ++kv) {
        mbar_init(&bars->raw_full[kv][i], 1);
        mbar_init(&bars->raw_empty[kv][i], 4);
      }
      mbar_init(&bars->s_full[i], 1);
      mbar_init(&bars->p_full[i], kTcGroupWarps);
      mbar_init(&bars->pv_done[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      for (int qd = 0; qd < 4; ++qd) mbar_init(&bars->m_ready[i][qd], 32);
      mbar_init(&bars->v_ok[i], 1);
    }
    mbar_init(&bars->all_done, 1);
    *abort = 0;
    *any_bad = 0;
    fence_mbar_init();
  }
  for (int i = threadIdx.x; i < HD; i += Cfg::kThreads) bad[i] = kNoBad;
  if (warp == 1) {
    tmem_alloc(tmem_slot, Cfg::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // Boxes of this item, numbered from key_base on: the table entry of box g
  // (of the last page past the table), and from it the cache row in units of
  // `unit` rows -- the first row past the cache, where TMA fills zeros and
  // reads nothing, for an entry that names no page.  Entries are read 32
  // boxes ahead, a box per lane, and not looked at before.
  auto box_entry = [&](int g) -> int {
    return p.bt[static_cast<size_t>(it.b) * p.BTW + min((key_base + g * p.box) / p.PS, p.BTW - 1)];
  };
  auto box_row = [&](int g, int phys, int unit) -> int {
    const int pos = key_base + g * p.box;
    if (pos >= k_lim) return 0;
    if (phys < 0 || phys >= p.P) {
      raise_flag(MXFA_FLAG_PAGE_OUT_OF_RANGE);
      return static_cast<int>(static_cast<long long>(p.P) * p.PS / unit);
    }
    return (phys * p.PS + pos % p.PS) / unit;  // slots fit 31 bits
  };
  // first tile (of this item) that some row does not see in full
  const int guard0 = max(0, vis_first / kTcKeys - it.kt0);
  const int guard_key = key_base + guard0 * kTcKeys;

  if (warp < 4) {
   if constexpr (kQuant) regs_dec<kRegsIssue>();
   if (nkt > 0 && (warp == 0 || warp == 3)) {
    // ------------------------------------------------------------ producers
    // Warp 0 loads Q and K, warp 3 loads V; lane i issues box i of a tile.
    const int nbox = kTcKeys / p.box;
    const bool for_v = warp == 3;
    const CUtensorMap* map = for_v ? &tmv : &tmk;
    if (lane == 0 && !for_v) {
      mbar_arrive_expect_tx(&bars->q_full, Cfg::kDBlk * (kTcRows / p.GQ) * p.GQ * 128);
#pragma unroll
      for (int db = 0; db < Cfg::kDBlk; ++db)
        tma_load_3d(sm + Cfg::kQ + db * Cfg::kQBlk, &tmq, &bars->q_full, db * 64, hk * p.GQ, it.row0);
    }
    bool ok = true;
    int filled = 0;  // tiles, or half tiles, whose copies were started
    int entry = box_entry(lane), rows = 0;
    for (int t = 0; t < nkt && ok; ++t) {
      const int g0 = t * nbox;
      if ((g0 & 31) == 0) {
        rows = box_row(g0 + lane, entry, kQuant ? 1 : 8);
        entry = box_entry(g0 + 32 + lane);
      }
      const int row = __shfl_sync(0xffffffffu, rows, (g0 + (lane & (nbox - 1))) & 31);
      const bool has = lane < nbox && key_base + (g0 + lane) * p.box < k_lim;
      if constexpr (!kQuant) {
        const int st = t % NS, use = t / NS;
        uint64_t* full = for_v ? &bars->v_full[st] : &bars->k_full[st];
        const int n = __popc(__ballot_sync(0xffffffffu, has));
        if (lane == 0) {
          // K stage: free once S_{t-3} is done; V stage: once P.V_{t-3} is
          if (use > 0) ok = tc_wait(for_v ? &bars->pv_done[st] : &bars->s_full[st], (use - 1) & 1, abort);
          if (ok) mbar_arrive_expect_tx(full, n * p.box * HD * 2);
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (!ok) break;
        filled = t + 1;
        if (has)
          tma_load_5d(sm + (for_v ? Cfg::kV : Cfg::kK) + st * Cfg::kTile + lane * (p.box / 8) * Cfg::kGroupBytes, map,
                      full, 0, hk, 0, 0, row);
      } else {
        const int half = Cfg::kRawKeys / p.box;  // boxes of a half tile
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          const int slot = filled % Cfg::kRawSlots, use = filled / Cfg::kRawSlots;
          const bool mine = has && lane / half == h;
          const int n = __popc(__ballot_sync(0xffffffffu, mine));
          if (lane == 0) {
            if (use > 0) ok = tc_wait(&bars->raw_empty[for_v][slot], (use - 1) & 1, abort);
            if (ok) mbar_arrive_expect_tx(&bars->raw_full[for_v][slot], n * p.box * HD);
          }
          ok = __shfl_sync(0xffffffffu, ok, 0);
          if (!ok) break;
          ++filled;
          if (mine)
            tma_load_3d(sm + Cfg::kRaw + ((for_v ? Cfg::kRawSlots : 0) + slot) * Cfg::kRawTile + lane % half * p.box * HD,
                        map, &bars->raw_full[for_v][slot], 0, hk, row);
        }
      }
    }
    if constexpr (kQuant) {
      if (*abort && lane == 0)  // leave no copy in flight
        for (int w = max(0, filled - Cfg::kRawSlots); w < filled; ++w)
          mbar_wait(&bars->raw_full[for_v][w % Cfg::kRawSlots], (w / Cfg::kRawSlots) & 1);
    } else {
      if (for_v) {
        // V guard: keys [vis_first, end of tile) of the last tiles
        for (int t = guard0; t < nkt && ok; ++t) {
          ok = __all_sync(0xffffffffu, tc_wait(&bars->v_full[t % NS], (t / NS) & 1, abort));
          if (!ok) break;
          uint8_t* vt = sm + Cfg::kV + (t % NS) * Cfg::kTile;
          const int key0 = key_base + t * kTcKeys;
          constexpr int kCh = HD / 8;
          for (int c = max(0, vis_first - key0) * kCh + lane; c < kTcKeys * kCh; c += 32) {
            const int r = c / kCh, ch = c % kCh;
            uint4* at = reinterpret_cast<uint4*>(vt + (r >> 3) * Cfg::kGroupBytes + (ch >> 3) * 1024 +
                                                 swz128(r & 7, ch & 7));
            if (key0 + r >= k_end) {
              *at = make_uint4(0, 0, 0, 0);
            } else if (any_nonfinite<T>(*at)) {
              *at = strip_nonfinite<T>(*at, key0 + r - guard_key, bad + ch * 8, any_bad);
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars->v_ok[t - guard0]);
        }
      }
      if (*abort && lane == 0)
        for (int t = max(0, filled - NS); t < filled; ++t)
          mbar_wait(for_v ? &bars->v_full[t % NS] : &bars->k_full[t % NS], (t / NS) & 1);
    }
    __syncwarp();
   } else if (nkt > 0 && (warp == 1 || warp == 2)) {
    // ------------------------------------------------------------ MMA issue
    if (lane == 0) {
      constexpr uint32_t idesc_s = umma_idesc<MT>(kTcRows, kTcKeys, false);
      constexpr uint32_t idesc_o = umma_idesc<MT>(kTcRows, HD, true);
      constexpr int kS = HD / 16;
      constexpr int kP = kTcKeys / 16;
      if (warp == 2) {
        uint64_t qd[kS];
        {
          const uint64_t base = smem_desc(smem_u32(sm + Cfg::kQ), 16, 1024);
#pragma unroll
          for (int kk = 0; kk < kS; ++kk) qd[kk] = base + (kk >> 2) * (Cfg::kQBlk >> 4) + (kk & 3) * 2;
        }
        bool ok = tc_wait(kConvertQ ? &bars->q_ready : &bars->q_full, 0, abort);
        for (int t = 0; t < nkt && ok; ++t) {
          const int buf = t % NB, ks = t % NS;
          uint64_t kd[kS];
          {
            const uint64_t base = smem_desc(smem_u32(sm + Cfg::kK + ks * Cfg::kTile), 16, Cfg::kGroupBytes);
#pragma unroll
            for (int kk = 0; kk < kS; ++kk) kd[kk] = base + (kk >> 2) * (1024 >> 4) + (kk & 3) * 2;
          }
          pin_regs(kd);
          if (t >= NB && !tc_wait(&bars->pv_done[buf], ((t - NB) / NB) & 1, abort)) break;  // buffer free
          if (!tc_wait(&bars->k_full[ks], (t / NS) & 1, abort)) break;
          tc_fence_after();
          umma_ss_chain(tmem + buf * kTcKeys, qd, kd, idesc_s);
          umma_commit(&bars->s_full[buf]);
        }
      } else {
        for (int j = 0; j < nkt; ++j) {
          const int buf = j % NB, vs = j % NS;
          uint64_t vd[kP];
          uint32_t pa[kP];
          {
            const uint64_t vbase = smem_desc(smem_u32(sm + Cfg::kV + vs * Cfg::kTile), 1024, Cfg::kGroupBytes);
#pragma unroll
            for (int kk = 0; kk < kP; ++kk) {
              vd[kk] = vbase + kk * (2 * Cfg::kGroupBytes >> 4);
              pa[kk] = tmem + buf * kTcKeys + kk * 8;
            }
          }
          pin_regs(vd);
          pin_regs(pa);
          if (!tc_wait(&bars->v_full[vs], (j / NS) & 1, abort)) break;
          if (!kQuant && j >= guard0 && !tc_wait(&bars->v_ok[j - guard0], 0, abort)) break;
          if (!tc_wait(&bars->p_full[buf], (j / NB) & 1, abort)) break;
          tc_fence_after();
          umma_ts_chain(tmem + Cfg::kTmemO, pa, vd, idesc_o, j > 0 ? 1u : 0u);
          umma_commit(&bars->pv_done[buf]);
          if (j == nkt - 1) umma_commit(&bars->all_done);
        }
      }
    }
    __syncwarp();
   }
   if (warp == 1) {  // tensor memory goes back once the softmax warps have read it
     named_barrier_sync(3, kSoft + 32);
     tc_fence_after();
     tmem_dealloc(tmem, Cfg::kTmemCols);
   }
  } else if (kQuant && warp >= 28) {
   if constexpr (kQuant) regs_dec<kRegsScale>();
   if (nkt > 0 && warp == 28) {
    // --------------------------------------------------------------- scales
    // The exponent bytes of a tile become f16 factors relative to the tile's
    // largest byte.  Lane i has keys 4i .. 4i+3 (one page: pages hold a
    // multiple of 8), copied to its own words of a ring four tiles ahead.
    uint32_t* factors = reinterpret_cast<uint32_t*>(sm + Cfg::kScale);
    int2* tile_exp = reinterpret_cast<int2*>(sm + Cfg::kTileExp);
    uint32_t* ring = reinterpret_cast<uint32_t*>(sm + Cfg::kExpBytes);  // [8][K|V][32]
    float4* wide_keys = reinterpret_cast<float4*>(sm + Cfg::kWide);  // [8][128 / 2]
    const int nbox = kTcKeys / p.box;
    // box g's first byte in units of 8, ~0u without a page
    auto box_bytes = [&](int g, int phys) -> unsigned {
      const int pos = key_base + g * p.box;
      if (pos >= k_lim || phys < 0 || phys >= p.P) return ~0u;
      return static_cast<unsigned>(((static_cast<size_t>(phys) * p.HKV + hk) * p.PS + pos % p.PS) >> 3);
    };
    int entry = box_entry(lane);
    unsigned base = 0;
    auto fetch = [&](int t) {
      const int g0 = t * nbox;
      if ((g0 & 31) == 0) {
        base = box_bytes(g0 + lane, entry);
        entry = box_entry(g0 + 32 + lane);
      }
      const unsigned at8 = __shfl_sync(0xffffffffu, base, (g0 + 4 * lane / p.box) & 31);
      const bool has = at8 != ~0u;
      const size_t at = (has ? static_cast<size_t>(at8) << 3 : 0) + (4 * lane) % p.box;
      uint32_t* dst = ring + (t & 7) * 64 + lane;
      cp_async_4_zfill(dst, p.k_scales + at, has);
      cp_async_4_zfill(dst + 32, p.v_scales + at, has);
    };
    // the word's bytes of keys past the sequence become 0, which takes no part in the maximum
    auto cut = [&](uint32_t w, int t) -> uint32_t {
      const int left = k_lim - (key_base + t * kTcKeys + 4 * lane);  // keys of this word that exist
      return left >= 4 ? w : w & ((1u << (8 * max(left, 0))) - 1u);
    };
    auto largest = [&](uint32_t w) -> int {  // over the tile's 128 bytes; NaN scales (255) do not count
      uint32_t m = w & ~__vcmpeq4(w, 0xffffffffu);
      m = __vmaxu4(m, m >> 16);
      m = __vmaxu4(m, m >> 8) & 255u;
      return max(static_cast<int>(__reduce_max_sync(0xffffffffu, m)), kRefMin);
    };
    // whether some row of the tile lies more than `most` under the largest; rows under `floor` count as that,
    // bytes 0, 1 and 255 do not
    auto spread_over = [&](uint32_t w, int ref, int floor, int most) -> bool {
      uint32_t m = w | __vcmpltu4(w, 0x02020202u);
      m = __vminu4(m, m >> 16);
      m = __vminu4(m, m >> 8) & 255u;
      return ref - max(static_cast<int>(__reduce_min_sync(0xffffffffu, m)), floor) > most;
    };
    // f16 factors of the rows relative to 2^ref, or of a wide tile: 1 for K, and for V what a byte lacks to kRefMin
    auto factor4 = [&](uint32_t w, int ref, bool wide, bool v) -> uint4 {
      uint32_t f[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int byte = (w >> (8 * i)) & 255;
        const int e = !wide ? byte - ref + kRefShift : v ? min(byte - kRefMin, 0) : 0;
        f[i] = byte == 255 ? 0x7fff7fffu : pow2_f16x2(e);
      }
      return make_uint4(f[0], f[1], f[2], f[3]);
    };
#pragma unroll 1
    for (int t = -4; t < nkt; ++t) {
      if (t + 4 < nkt) fetch(t + 4);
      cp_async_commit();
      if (t < 0) continue;
      cp_async_wait<4>();  // tile t's group
      const uint32_t kw = cut(ring[(t & 7) * 64 + lane], t), vw = cut(ring[(t & 7) * 64 + 32 + lane], t);
      const int rk = largest(kw), rv = largest(vw);
      const bool wide = spread_over(kw, rk, kRefMin - kWideK, kWideK) || spread_over(vw, rv, kRefMin, kWideV);
      // slot t % 4 is free once tile t-4's K and V are converted
      const bool ok = t < 4 || tc_wait(&bars->scale_free[t & 3], (t / 4 - 1) & 1, abort);
      if (!__all_sync(0xffffffffu, ok)) break;
      uint4* f = reinterpret_cast<uint4*>(factors + (t & 3) * 256);
      f[lane] = factor4(kw, rk, wide, false);
      f[32 + lane] = factor4(vw, rv, wide, true);
      if (wide) {
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          const float2 a = wide_key((kw >> (8 * i)) & 255, (vw >> (8 * i)) & 255);
          const float2 b = wide_key((kw >> (8 * i + 8)) & 255, (vw >> (8 * i + 8)) & 255);
          wide_keys[(t & 7) * 64 + lane * 2 + i / 2] = make_float4(a.x, a.y, b.x, b.y);
        }
      }
      if (lane == 0) tile_exp[t & 7] = make_int2(wide ? kWideTile : rk - 127 - kRefShift, rv - 127 - kRefShift);
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->scale_ready[t & 3]);
    }
    cp_async_wait_all();
   }
  } else if (kQuant && warp >= 12) {
   if constexpr (kQuant) regs_dec<kRegsConvert>();
   if (nkt > 0) {
    // ----------------------------------------------------------- converters
    // Warps 12-19 turn the e4m3 K tiles into f16 tiles, warps 20-27 the V
    // tiles; each warpgroup takes one half (64 keys) of every tile.  A thread
    // has the eight codes c of rows kRowStep apart, one 16-byte store each:
    // eight lanes fill a row of one 64-column block, all banks once.
    const bool is_v = warp >= 20;
    const int h = (warp >> 2) & 1 ? 0 : 1;  // warps 12-15 and 20-23: the first half
    const int tid = (threadIdx.x - 384) & 127;
    if (kConvertQ && is_v && h == 0) {
      // Query row tid to f16, times the power of two that brings its largest
      // finite element to [2^14, 2^15): exact for elements down to 2^-28 of it.
      if (__all_sync(0xffffffffu, tc_wait(&bars->q_full, 0, abort))) {
        float top = 0.f;
#pragma unroll 1
        for (int ch = 0; ch < HD / 8; ++ch) {
          const uint4 v = *reinterpret_cast<const uint4*>(sm + Cfg::kQ + (ch >> 3) * Cfg::kQBlk + swz128(tid, ch & 7));
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = Elem<T>::unpack(w[i]);
            top = fabsf(f.x) < INFINITY ? fmaxf(top, fabsf(f.x)) : top;
            top = fabsf(f.y) < INFINITY ? fmaxf(top, fabsf(f.y)) : top;
          }
        }
        const int e = top > 0.f ? max(static_cast<int>(__float_as_uint(top) >> 23) - 127 - 14, -100) : 0;
        const float down = pow2_f32(-e);
#pragma unroll 1
        for (int ch = 0; ch < HD / 8; ++ch) {
          uint4* at = reinterpret_cast<uint4*>(sm + Cfg::kQ + (ch >> 3) * Cfg::kQBlk + swz128(tid, ch & 7));
          const uint4 v = *at;
          const float2 a = Elem<T>::unpack(v.x), b = Elem<T>::unpack(v.y), cc = Elem<T>::unpack(v.z),
                       d = Elem<T>::unpack(v.w);
          *at = make_uint4(Elem<__half>::pack(a.x * down, a.y * down), Elem<__half>::pack(b.x * down, b.y * down),
                           Elem<__half>::pack(cc.x * down, cc.y * down), Elem<__half>::pack(d.x * down, d.y * down));
        }
        reinterpret_cast<float*>(sm + Cfg::kQScale)[tid] = pow2_f32(e);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->q_ready);
      }
    }
    constexpr int kCh = HD / 8;            // eight-code chunks of a row
    constexpr int kRowStep = 128 / kCh;    // 8 or 16: a thread's rows share their place in an 8-row group
    constexpr int kSteps = Cfg::kRawKeys / kRowStep;
    const int c = tid % kCh, r0 = tid / kCh;
    // shared-space addresses of this thread's first chunk in a raw slot, in a
    // 16-bit stage and of its first row's factor; the others follow at
    // constant distances (generic addresses took twice the instructions)
    const uint32_t raw_0 = smem_u32(sm + Cfg::kRaw) + (is_v ? Cfg::kRawSlots : 0) * Cfg::kRawTile + r0 * HD + c * 8;
    const uint32_t dst_off = ((h * Cfg::kRawKeys + r0) >> 3) * Cfg::kGroupBytes + (c >> 3) * 1024 + swz128(r0 & 7, c & 7);
    const uint32_t dst_0 = smem_u32(sm + (is_v ? Cfg::kV : Cfg::kK)) + dst_off;
    const uint32_t factor_0 = smem_u32(sm + Cfg::kScale) + ((is_v ? 128 : 0) + h * Cfg::kRawKeys + r0) * 4;
    for (int t = 0; t < nkt; ++t) {
      const int st = t % NS, key0 = key_base + t * kTcKeys;
      // the codes go to registers as soon as they are there, and their slot
      // back to the producer: a slot held through the waits below bounded the
      // kernel by its round trip
      const int w = 2 * t + h, slot = w % Cfg::kRawSlots;
      bool ready = tc_wait(&bars->raw_full[is_v][slot], (w / Cfg::kRawSlots) & 1, abort);
      uint2 x[kSteps];
      const uint32_t src = raw_0 + slot * Cfg::kRawTile;
#pragma unroll
      for (int i = 0; i < kSteps; ++i) x[i] = lds_v2(src + i * kRowStep * HD);
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->raw_empty[is_v][slot]);
      ready = tc_wait(&bars->scale_ready[t & 3], (t >> 2) & 1, abort) && ready;
      // the 16-bit stage is free once the product that read it is done
      if (t >= NS)
        ready = tc_wait(is_v ? &bars->pv_done[(t - NS) % NB] : &bars->s_full[(t - NS) % NB], ((t - NS) / NB) & 1, abort) &&
                ready;
      if (!__all_sync(0xffffffffu, ready)) break;
      const uint32_t dst = dst_0 + st * Cfg::kTile, fac = factor_0 + (t & 3) * 1024;
#pragma unroll
      for (int i = 0; i < kSteps; ++i)
        sts_v4(dst + i * (kRowStep / 8) * Cfg::kGroupBytes, codes_to_f16(x[i], lds_u32(fac + i * kRowStep * 4)));
      if (is_v && t >= guard0) {  // V guard, each thread over its own chunks
#pragma unroll 1
        for (int r = h * Cfg::kRawKeys + r0; r < (h + 1) * Cfg::kRawKeys; r += kRowStep) {
          const int key = key0 + r;
          if (key < vis_first) continue;
          uint4* at = reinterpret_cast<uint4*>(sm + Cfg::kV + st * Cfg::kTile + (r >> 3) * Cfg::kGroupBytes +
                                               (c >> 3) * 1024 + swz128(r & 7, c & 7));
          if (key >= k_end)
            *at = make_uint4(0, 0, 0, 0);
          else if (any_nonfinite<MT>(*at))
            *at = strip_nonfinite<MT>(*at, key - guard_key, bad + c * 8, any_bad);
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(is_v ? &bars->v_full[st] : &bars->k_full[st]);
        mbar_arrive(&bars->scale_free[t & 3]);
      }
    }
   }
  } else {
    if constexpr (kQuant) regs_inc<kRegsSoftmax>();
    // ------------------------------------------------------------ softmax
    const int g = (warp - 4) >> 2;
    const int quad = warp & 3;
    const int r = quad * 32 + lane;
    const uint32_t lane_base = tmem + ((static_cast<uint32_t>(quad) * 32u) << 16);
    const uint32_t o_base = lane_base + Cfg::kTmemO;
    const bool warp_live = quad * 32 < nrows;  // some row of this warp exists
    const bool row_live = r < nrows;
    const int pos = it.pos0 + r / p.GQ;
    // keys [0, vis_end) are visible; rows that do not exist see everything
    const int vis_end = !row_live ? 0x7fffffff : p.causal ? min(k_lim, max(pos + 1, 0)) : k_lim;
    // Quantised: scores count in units of the query row's and the tile's K
    // factor, so each tile has its own scale.  V counts in units of 2^v_exp:
    // the exponent joins the score before the maximum, so P is relative to
    // the largest contribution to O, and leaves the row sum again.  In a wide
    // tile both belong to the key.
    float sc = p.scale_log2;
    float v_exp = 0.f, v_inv = 1.f;
    const bool pos_scale = sc >= 0.f;
    float row_scale = sc;
    float m_own = -INFINITY, l_own = 0.f;
    const uint32_t mpub_r = smem_u32(sm + Cfg::kMPub) + r * 4;  // [tile parity][row] running maxima
    bool ok = true;
    if (kConvertQ && nkt > 0) {
      ok = __all_sync(0xffffffffu, tc_wait(&bars->q_ready, 0, abort));
      row_scale = sc * reinterpret_cast<const float*>(sm + Cfg::kQScale)[r];
    }
    for (int j = g; j < nkt && ok; j += NG) {
      const int buf = j % NB;
      if (!__all_sync(0xffffffffu, tc_wait(&bars->s_full[buf], (j / NB) & 1, abort))) {
        ok = false;
        break;
      }
      if (!warp_live) {  // P of rows that do not exist is never read back
        if (lane == 0) mbar_arrive(&bars->p_full[buf]);
        continue;
      }
      tc_fence_after();
      const uint32_t sbuf = lane_base + buf * kTcKeys;
      const int key0 = key_base + j * kTcKeys;
      bool wide = false;
      if constexpr (kQuant) {
        const uint2 e = lds_v2(smem_u32(sm + Cfg::kTileExp) + (j & 7) * 8);
        wide = e.x == kWideTile;
        sc = row_scale * pow2_f32(static_cast<int>(e.x));
        v_exp = static_cast<float>(static_cast<int>(e.y));
        v_inv = wide ? 1.f : pow2_f32(-static_cast<int>(e.y));
      }
      const uint32_t wide_keys = smem_u32(sm + Cfg::kWide) + (j & 7) * 1024;
      // (a negative scale, which looks for the least score, takes the masked loops)
      const bool all_full = __all_sync(0xffffffffu, key0 + kTcKeys <= vis_end) && pos_scale && !wide;
      const float ext0 = pos_scale ? -INFINITY : INFINITY;
      float ext = ext0;
      uint32_t ra[32], rb[32];
      // Two chunks of 32 columns a turn, the second's load in flight while the
      // first is worked on.  Loops, not straight code: all warps' loops
      // together have to stay in the instruction cache (unrolled over the
      // tile the kernel took 5% longer, the quantised one 20%).  Tiles with
      // masked columns take short loops of their own, for the same reason.
      if (all_full) {
        float e[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
        for (int c = 0; c < kTcKeys; c += 64) {
          tmem_ld32_async(sbuf + c, ra);
          tmem_wait_ld(ra);
          tmem_ld32_async(sbuf + c + 32, rb);
          ext_chunk32(ra, true, e);
          tmem_wait_ld(rb);
          ext_chunk32(rb, true, e);
        }
        ext = fmaxf(fmaxf(e[0], e[1]), fmaxf(e[2], e[3]));
      } else if (kQuant && wide) {
        ext = -INFINITY;
#pragma unroll 1
        for (int c = 0; c < kTcKeys; c += 16) {
          uint32_t raw[16];
          tmem_ld16(sbuf + c, raw);
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            const float4 w = lds_f32x4(wide_keys + (c + i) * 8);
            const float a = fmaf(__uint_as_float(raw[i]) * row_scale, w.x, w.y);
            const float b = fmaf(__uint_as_float(raw[i + 1]) * row_scale, w.z, w.w);
            ext = key0 + c + i < vis_end ? fmaxf(ext, a) : ext;
            ext = key0 + c + i + 1 < vis_end ? fmaxf(ext, b) : ext;
          }
        }
      } else {
#pragma unroll 1
        for (int c = 0; c < kTcKeys; c += 16) {
          uint32_t raw[16];
          tmem_ld16(sbuf + c, raw);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float v = __uint_as_float(raw[i]);
            const bool vis = key0 + c + i < vis_end;
            ext = vis ? (pos_scale ? fmaxf(ext, v) : fminf(ext, v)) : ext;
          }
        }
      }
      float mx = kQuant ? (wide ? ext : fmaf(ext, sc, v_exp)) - kPShift : ext * sc;
      mx = (ext == INFINITY || ext == -INFINITY) ? -INFINITY : mx;
      float m_in = -INFINITY;
      if (j > 0) {
        const int pj = j - 1;
        if (!__all_sync(0xffffffffu, tc_wait(&bars->m_ready[pj & 1][quad], (pj >> 1) & 1, abort))) {
          ok = false;
          break;
        }
        m_in = lds_f32(mpub_r + (pj & 1) * kTcRows * 4);
      }
      const float m_j = mx > m_in + kRescaleThreshold ? mx : m_in;
      sts_f32(mpub_r + (j & 1) * kTcRows * 4, m_j);
      mbar_arrive(&bars->m_ready[j & 1][quad]);
      if (m_j != m_own) {
        l_own *= fast_exp2(m_own - m_j);
        m_own = m_j;
      }
      const bool grow = j > 0 && m_j != m_in;
      if (__any_sync(0xffffffffu, grow)) {
        const int pj = j - 1;
        if (!__all_sync(0xffffffffu, tc_wait(&bars->pv_done[pj % NB], (pj / NB) & 1, abort))) {
          ok = false;
          break;
        }
        tc_fence_after();
        const float alpha = grow ? fast_exp2(m_in - m_j) : 1.f;
#pragma unroll 1
        for (int c = 0; c < HD; c += 32) {
          uint32_t o[32];
          tmem_ld32(o_base + c, o);
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
          tmem_st32(o_base + c, o);
        }
      }
      float rs = 0.f;
      const float neg_m = kQuant ? v_exp - m_j : -m_j;
      if (all_full) {
        const uint64_t sc2 = f2_pack(sc, sc), nm2 = f2_pack(neg_m, neg_m);
        uint64_t acc0 = 0, acc1 = 0;
        uint32_t pka[16], pkb[16];
#pragma unroll 1
        for (int c = 0; c < kTcKeys; c += 64) {
          tmem_ld32_async(sbuf + c, ra);
          tmem_wait_ld(ra);
          tmem_ld32_async(sbuf + c + 32, rb);
          exp2_chunk32<MT>(ra, sc2, nm2, acc0, acc1, pka);
          tmem_st16_async(sbuf + (c >> 1), pka);
          tmem_wait_ld(rb);
          exp2_chunk32<MT>(rb, sc2, nm2, acc0, acc1, pkb);
          tmem_st16_async(sbuf + (c >> 1) + 16, pkb);
          tmem_wait_st();
        }
        float a, bb;
        f2_unpack(f2_add(acc0, acc1), a, bb);
        rs = a + bb;
      } else if (kQuant && wide) {
#pragma unroll 1
        for (int c = 0; c < kTcKeys; c += 16) {
          uint32_t raw[16];
          tmem_ld16(sbuf + c, raw);
          uint32_t packed[8];
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            const float4 w = lds_f32x4(wide_keys + (c + i) * 8);
            const float a = fmaf(__uint_as_float(raw[i]) * row_scale, w.x, w.y - m_j);
            const float b = fmaf(__uint_as_float(raw[i + 1]) * row_scale, w.z, w.w - m_j);
            const float p0 = key0 + c + i < vis_end ? fast_exp2(a) : 0.f;
            const float p1 = key0 + c + i + 1 < vis_end ? fast_exp2(b) : 0.f;
            rs = fmaf(p0, pow2_inverse(w.y), fmaf(p1, pow2_inverse(w.w), rs));
            packed[i >> 1] = Elem<MT>::pack(p0, p1);
          }
          tmem_st8(sbuf + (c >> 1), packed);
        }
      } else {
#pragma unroll 1
        for (int c = 0; c < kTcKeys; c += 16) {
          uint32_t raw[16];
          tmem_ld16(sbuf + c, raw);
          uint32_t packed[8];
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            const bool v0 = key0 + c + i < vis_end;
            const bool v1 = key0 + c + i + 1 < vis_end;
            const float p0 = v0 ? fast_exp2(fmaf(__uint_as_float(raw[i]), sc, neg_m)) : 0.f;
            const float p1 = v1 ? fast_exp2(fmaf(__uint_as_float(raw[i + 1]), sc, neg_m)) : 0.f;
            rs += p0 + p1;
            packed[i >> 1] = Elem<MT>::pack(p0, p1);
          }
          tmem_st8(sbuf + (c >> 1), packed);
        }
      }
      l_own += kQuant ? rs * v_inv : rs;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->p_full[buf]);
    }
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");  // a load left in flight by an aborted tile

    // ---------------------------------------------------------- merge + store
    const bool done_ok =
        nkt == 0 || __all_sync(0xffffffffu, ok && tc_wait(&bars->all_done, 0, abort));
    fence_proxy_async_smem();
    ml[(g * 2) * kTcRows + r] = m_own;
    ml[(g * 2 + 1) * kTcRows + r] = l_own;
    named_barrier_sync(1, kSoft);
    tc_fence_after();
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int gg = 0; gg < NG; ++gg) M = fmaxf(M, ml[(gg * 2) * kTcRows + r]);
#pragma unroll
    for (int gg = 0; gg < NG; ++gg) {
      const float mg = ml[(gg * 2) * kTcRows + r], lg = ml[(gg * 2 + 1) * kTcRows + r];
      L += lg * (mg == -INFINITY ? 1.f : fast_exp2(mg - M));  // at maximum -inf a sum is 0, or NaN when every score was
    }
    const bool split = it.nsplit > 1;
    const float inv = split ? 1.f : (L != 0.f ? 1.f / L : 0.f);
    const int head = hk * p.GQ + r % p.GQ;
    const size_t R = static_cast<size_t>(it.row0 + r / p.GQ) * p.HQ + head;
    const size_t prow = (static_cast<size_t>(hk) * p.parts_cap + it.part0 + it.split) * kTcRows + r;
    T* orow = static_cast<T*>(p.out) + R * HD;
    if (warp_live && done_ok) {
      const bool patch = *any_bad != 0;
      for (int c = g * 32; c < HD; c += 32 * NG) {
        uint32_t o[32];
        if (nkt > 0)
          tmem_ld32(o_base + c, o);
        else
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0u;
        if (patch) {
          // non-finite V elements taken out of the products go into the rows that see their key
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const unsigned b3 = bad[c + i];
            const int seen = vis_end - guard_key;  // relative keys below it are visible
            const int kn = b3 & kNoKey, kp = (b3 >> 10) & kNoKey, km = (b3 >> 20) & kNoKey;
            const bool n = kn != kNoKey && kn < seen, pi = kp != kNoKey && kp < seen, mi = km != kNoKey && km < seen;
            if (n || (pi && mi))
              o[i] = 0x7fffffffu;
            else if (pi || mi)
              o[i] = __float_as_uint(__uint_as_float(o[i]) + (pi ? INFINITY : -INFINITY));
          }
        }
        if (row_live && split) {
          float* dst = p.part_o + prow * HD + c;
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            *reinterpret_cast<uint4*>(dst + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
        } else if (row_live) {
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            uint4 v;
            v.x = Elem<T>::pack(__uint_as_float(o[i + 0]) * inv, __uint_as_float(o[i + 1]) * inv);
            v.y = Elem<T>::pack(__uint_as_float(o[i + 2]) * inv, __uint_as_float(o[i + 3]) * inv);
            v.z = Elem<T>::pack(__uint_as_float(o[i + 4]) * inv, __uint_as_float(o[i + 5]) * inv);
            v.w = Elem<T>::pack(__uint_as_float(o[i + 6]) * inv, __uint_as_float(o[i + 7]) * inv);
            *reinterpret_cast<uint4*>(orow + c + i) = v;
          }
        }
        __syncwarp();
      }
    }
    if (g == 0 && row_live && done_ok) {
      if (split)
        *reinterpret_cast<float2*>(p.part_ml + prow * 2) = make_float2(M, L);
      else if (p.lse != nullptr)
        p.lse[R] = L != 0.f ? (M + log2f(L)) * kLn2 : -INFINITY;
    }
    tc_fence_before();
    named_barrier_arrive(3, kSoft + 32);  // tensor memory is read
    if (split) {
      // publish this part; the last one of the tile merges them all, in split order
      __threadfence();
      named_barrier_sync(1, kSoft);
      unsigned* counter = p.counters + static_cast<size_t>(hk) * (p.parts_cap / 2 + 1) + it.group;
      const int tid = threadIdx.x - 128;
      if (tid == 0) *s_last = atomicAdd(counter, 1u) == static_cast<unsigned>(it.nsplit) - 1u;
      named_barrier_sync(1, kSoft);
      if (*s_last) {
        __threadfence();
        // Weights first, one thread per row, over the K and V stages (every
        // product is done): w = 2^(m_z - M) / L.  Then O = sum w_z O_z, four
        // loads in flight per thread.
        const size_t first = (static_cast<size_t>(hk) * p.parts_cap + it.part0) * kTcRows;
        float* wz = reinterpret_cast<float*>(sm + Cfg::kK);  // [part][row]
        static_assert(2 * Cfg::kStages * Cfg::kTile + Cfg::kRawBytes >= kChunkMaxParts * kTcRows * 4, "room for weights");
        if (tid < nrows) {
          const float2* pm = reinterpret_cast<const float2*>(p.part_ml) + first + tid;
          float Mx = -INFINITY, Ls = 0.f;
#pragma unroll 8
          for (int z = 0; z < it.nsplit; ++z) Mx = fmaxf(Mx, __ldcg(pm + static_cast<size_t>(z) * kTcRows).x);
#pragma unroll 8
          for (int z = 0; z < it.nsplit; ++z) {
            const float2 s = __ldcg(pm + static_cast<size_t>(z) * kTcRows);
            // a part at -inf saw no key (sum 0), or only NaN scores
            const float w = s.x != -INFINITY ? fast_exp2(s.x - Mx) : s.y == 0.f ? 0.f : 1.f;
            Ls = fmaf(s.y, w, Ls);
            wz[z * kTcRows + tid] = w;
          }
          const float iv = Ls != 0.f ? 1.f / Ls : 0.f;
          for (int z = 0; z < it.nsplit; ++z) wz[z * kTcRows + tid] *= iv;
          const size_t RR = static_cast<size_t>(it.row0 + tid / p.GQ) * p.HQ + hk * p.GQ + tid % p.GQ;
          if (p.lse != nullptr) p.lse[RR] = Ls != 0.f ? (Mx + log2f(Ls)) * kLn2 : -INFINITY;
        }
        named_barrier_sync(1, kSoft);
        constexpr int kQuads = HD / 4, kBatch = 4;
        for (int idx0 = tid; idx0 < nrows * kQuads; idx0 += kSoft * kBatch) {
          float4 acc[kBatch];
#pragma unroll
          for (int u = 0; u < kBatch; ++u) acc[u] = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int z = 0; z < it.nsplit; ++z) {
            const float* po = p.part_o + (first + static_cast<size_t>(z) * kTcRows) * HD;
            float4 o4[kBatch];
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
              const int idx = idx0 + u * kSoft;
              o4[u] = idx < nrows * kQuads ? __ldcg(reinterpret_cast<const float4*>(po) + idx) : acc[0];
            }
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
              const int row = min(idx0 + u * kSoft, nrows * kQuads - 1) / kQuads;
              const float w = wz[z * kTcRows + row];
              if (w == 0.f) continue;  // its O may be anything
              acc[u].x = fmaf(o4[u].x, w, acc[u].x);
              acc[u].y = fmaf(o4[u].y, w, acc[u].y);
              acc[u].z = fmaf(o4[u].z, w, acc[u].z);
              acc[u].w = fmaf(o4[u].w, w, acc[u].w);
            }
          }
#pragma unroll
          for (int u = 0; u < kBatch; ++u) {
            const int idx = idx0 + u * kSoft;
            if (idx >= nrows * kQuads) break;
            const int row = idx / kQuads, d4 = (idx % kQuads) * 4;
            const size_t RR = static_cast<size_t>(it.row0 + row / p.GQ) * p.HQ + hk * p.GQ + row % p.GQ;
            uint2 v;
            v.x = Elem<T>::pack(acc[u].x, acc[u].y);
            v.y = Elem<T>::pack(acc[u].z, acc[u].w);
            *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + RR * HD + d4) = v;
          }
        }
        if (tid == 0) *counter = 0u;
      }
    }
  }
}

}  // namespace mxfa
