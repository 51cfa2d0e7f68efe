// Decode attention over the key blocks that a cheap score selects for each query.
//
// Keys are taken in blocks of 64. For each block and KV head the pool keeps the elementwise
// minimum lo and maximum hi of its keys (key_block_bounds_kernel). For a query q,
//   sum_d max(q_d lo_d, q_d hi_d) = sum_d min(q_d, 0) lo_d + max(q_d, 0) hi_d
// is at least q . k for every key of the block. A block's score is the largest of these over
// the query heads that share the KV head; of a row's blocks the first `sink` and the last
// `recent` are always taken, then those with the largest scores (equal scores: the lower block;
// NaN counts as the largest, so a damaged block shows in the output) up to `top` in all. The
// output is softmax attention over the keys of these blocks alone, its weights held in fp32 and
// multiplied with V as two bf16 values each (decode_tile's FINE), so that the output's rounding to
// bf16 is the only one that counts. (One bf16 value per weight, as in dense decode, was not faster.)
//
// The right-hand form is a product over 256 dims, [min(q, 0) | max(q, 0)] . [lo | hi], so the
// scores of all heads of a group come from m16n8k16 MMAs (blocks as M, heads as N) at the cost
// of reading the bounds: 512 bytes per block where the block's K and V are 32 KB. Their fp32
// error is at most eps = 2^-15 sum |terms| (256 exact products, each addition rounded or
// truncated at 2^-23 or better). Blocks further than 2 eps from the threshold, the k-th largest
// computed score, are settled by it; the few within are scored again in 64 bits, where 256
// products of two 8-bit significands sum exactly or very nearly so, and ranked by that. The
// selection is therefore that of exact scores. With infinite bounds the two forms differ: 0 times the
// bound that max() leaves out is NaN in the right-hand one. The sum of |terms| is not finite then, so
// every block is in doubt and the scores compared are those in 64 bits, taken as the left-hand form.
#pragma once

#include "attention_decode.cuh"
#include "linear_w4.cuh"

namespace hb {

constexpr int kBlockKeys = kDecTileKeys;  // keys per block: one tile of the decode ring

// ---------------------------------------------------------------- bounds
struct BlockBoundsParams {
  const __nv_bfloat16* keys;  // [num_pages, page_size, kv_heads, 128]
  __nv_bfloat16* bounds;      // [num_pages, kv_heads, page_size / 64, 2, 128]
  const int32_t* block_table;  // [rows, width]
  const int32_t* cu_seq_q;     // [rows + 1]
  const int32_t* seqused_k;    // [rows]
  const int32_t* token_row;    // [tokens]
  int32_t rows, tokens, width, num_pages, page_size, kv_heads;
};

constexpr int kBoundsThreads = 512;

// The bounds of the n keys from key `at` of a page, by the whole CTA.
__device__ __forceinline__ void block_bounds_of(const BlockBoundsParams& p, int page, int at, int n, uint4 (*other)[2][16]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int pair = warp >> 1, part = warp & 1, half = lane >> 4, col = lane & 15;  // 16 bytes per lane
  const int blocks = p.page_size / kBlockKeys;
  const int64_t step = static_cast<int64_t>(p.kv_heads) * 128;
  for (int h0 = 0; h0 < p.kv_heads; h0 += kBoundsThreads / 64) {  // the same for the whole CTA
    const int h = h0 + pair;
    __nv_bfloat162 lo[4], hi[4];
    if (h < p.kv_heads) {
      const __nv_bfloat16* src =
          p.keys + ((static_cast<int64_t>(page) * p.page_size + at) * p.kv_heads + h) * 128 + 8 * col;
      uint4 v[kBlockKeys / 4];
#pragma unroll
      for (int i = 0; i < kBlockKeys / 4; ++i) {
        const int key = min(32 * part + 2 * i + half, n - 1);
        v[i] = *reinterpret_cast<const uint4*>(src + key * step);
      }
      *reinterpret_cast<uint4*>(lo) = v[0];
      *reinterpret_cast<uint4*>(hi) = v[0];
#pragma unroll
      for (int i = 1; i < kBlockKeys / 4; ++i) {
        const __nv_bfloat162* k = reinterpret_cast<const __nv_bfloat162*>(&v[i]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          lo[e] = __hmin2_nan(lo[e], k[e]);
          hi[e] = __hmax2_nan(hi[e], k[e]);
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {  // the other half-warp's keys
        lo[e] = __hmin2_nan(lo[e], __shfl_xor_sync(0xffffffffu, lo[e], 16));
        hi[e] = __hmax2_nan(hi[e], __shfl_xor_sync(0xffffffffu, hi[e], 16));
      }
      if (part == 1 && half == 0) {
        other[pair][0][col] = *reinterpret_cast<uint4*>(lo);
        other[pair][1][col] = *reinterpret_cast<uint4*>(hi);
      }
    }
    __syncthreads();
    if (h < p.kv_heads && part == 0) {  // half-warp 0 writes the minima, 1 the maxima
      const uint4 o = other[pair][half][col];
      const __nv_bfloat162* k = reinterpret_cast<const __nv_bfloat162*>(&o);
      __nv_bfloat162 r[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) r[e] = half == 0 ? __hmin2_nan(lo[e], k[e]) : __hmax2_nan(hi[e], k[e]);
      __nv_bfloat16* dst = p.bounds + ((static_cast<int64_t>(page) * p.kv_heads + h) * blocks + at / kBlockKeys) * 256;
      *reinterpret_cast<uint4*>(dst + 128 * half + 8 * col) = *reinterpret_cast<uint4*>(r);
    }
    __syncthreads();  // `other` is written again
  }
}

constexpr int kBoundsCtas = 293;  // two per SM, and a number that spreads every 64th token over them

// The first token that a row has in a block (in this tick) stands for the block, and its bounds are
// computed anew from the pool, over the keys the row has there by now. Nothing is carried over from
// earlier bounds, so truncated and rewritten keys leave no trace. CTA b looks at tokens b, b + grid,
// ..., a thread each, and then takes the blocks that it found one after the other: a decode tick has
// a block per CTA, and a chunk's blocks, one in 64 tokens, spread evenly. (A CTA per token took 11
// us for a 2048-token chunk and 80 us for 16,384.) What bounds it is latency: the row's description
// is two reads deep, then the page, then the keys. Two warps share a KV head, a half-warp reads a
// key's 256 bytes, and a warp's 32 keys are all asked for at once. Keys past the row's end repeat its
// last one.
__global__ void __launch_bounds__(kBoundsThreads) key_block_bounds_kernel(BlockBoundsParams p) {
  __shared__ uint4 other[kBoundsThreads / 64][2][16];  // a head's second warp: minima, maxima
  __shared__ int3 found[kBoundsThreads];               // page, first key in it, keys
  __shared__ int n_found;
  pdl_wait();  // the keys, from the kernel ahead
  pdl_trigger();
  for (int64_t t0 = blockIdx.x; t0 < p.tokens; t0 += static_cast<int64_t>(kBoundsThreads) * gridDim.x) {
    if (threadIdx.x == 0) n_found = 0;
    __syncthreads();
    const int64_t token = t0 + static_cast<int64_t>(threadIdx.x) * gridDim.x;
    const int row = token < p.tokens ? p.token_row[token] : 0;
    if (row < 0 || row >= p.rows) raise_status(kStatusBadRow);
    else if (token < p.tokens) {
      const int q0 = p.cu_seq_q[row], count = p.cu_seq_q[row + 1] - q0, end = p.seqused_k[row];
      const int pos = end - count + static_cast<int>(token - q0);
      if (pos >= 0 && pos < end && (token == q0 || pos % kBlockKeys == 0)) {
        const int first = pos - pos % kBlockKeys, pidx = first / p.page_size;
        const int page = pidx < p.width ? p.block_table[static_cast<int64_t>(row) * p.width + pidx] : -1;
        if (page < 0 || page >= p.num_pages) raise_status(kStatusBadPage);
        else found[atomicAdd(&n_found, 1)] = make_int3(page, first % p.page_size, min(kBlockKeys, end - first));
      }
    }
    __syncthreads();
    const int blocks = n_found;
    for (int b = 0; b < blocks; ++b) block_bounds_of(p, found[b].x, found[b].y, found[b].z, other);
  }
}

// ---------------------------------------------------------------- selection and attention
struct SparseAttentionParams {
  const __nv_bfloat16* q;       // [tokens, H, 128]
  __nv_bfloat16* out;           // [tokens, H, 128]
  const __nv_bfloat16* bounds;  // [num_pages, kv_heads, page_size / 64, 2, 128]
  const int32_t* block_table;   // [rows, width]
  const int32_t* seqused_k;     // [rows]
  const int32_t* cu_seq_q;      // [rows + 1]: rows with other than one token are left alone; null: row r has token r
  int32_t* selected;            // [rows, kv_heads, top] or null
  int32_t width, num_pages, page_size, heads, kv_heads;
  int32_t per_page;        // blocks per page
  uint32_t per_page_inv;   // ceil(2^32 / per_page), 0 for one block per page
  int32_t top, sink, recent;
  float scale_log2;
};

constexpr int kSparseThreads = kDecSubThreads;
constexpr int kSparseWarps = kSparseThreads / 32;
// Keys, border indices and border scores of a row's blocks share the ring's memory.
constexpr int kSparseMaxBlocks = kDecRingBytes / 16;
constexpr int kSparseMaxTop = 1024;
static_assert(kDecRingBytes % 16 == 0, "three arrays in the ring");

// Order-preserving integers of scores: NaN above everything, -0 as +0.
__device__ __forceinline__ uint32_t score_key(float s) {
  if (s != s) return 0xFFFFFFFFu;
  const uint32_t b = __float_as_uint(s + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ unsigned long long score_key(double s) {
  if (s != s) return ~0ull;
  const unsigned long long b = static_cast<unsigned long long>(__double_as_longlong(s + 0.0));
  return (b >> 63) ? ~b : (b | (1ull << 63));
}
__device__ __forceinline__ float key_score(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}
__device__ __forceinline__ void cluster_store(uint32_t* local, uint32_t rank, uint32_t v) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(local)), "r"(rank));
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory");
}

// b / per_page, exact for b x per_page < 2^32.
__device__ __forceinline__ int block_page(const SparseAttentionParams& p, int b) {
  return p.per_page_inv ? static_cast<int>(__umulhi(static_cast<uint32_t>(b), p.per_page_inv)) : b;
}

// The bounds of block b for KV head h, or null where the row's pages (shared memory) name none.
__device__ __forceinline__ const __nv_bfloat16* block_bounds(const SparseAttentionParams& p, const int* pages, int h,
                                                             int b) {
  const int pidx = block_page(p, b), page = pages[pidx];
  if (page < 0 || page >= p.num_pages) return nullptr;
  return p.bounds + ((static_cast<int64_t>(page) * p.kv_heads + h) * p.per_page + (b - pidx * p.per_page)) * 256;
}

// Scores of blocks [b0, b1) (b0 a multiple of 8) into the keys[] of every CTA of the cluster (0
// for the first `sink` and, from block `last`, the forced ones), by the CTA's warps; returns the
// lane's largest sum |terms|. `frags` is scratch of 4 KB.
template <int GROUP>
__device__ __forceinline__ float score_blocks(const SparseAttentionParams& p, const int* pages, int token, int h, int b0,
                                              int b1, int last, uint32_t* keys, uint4* frags, int ranks) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g4 = lane >> 2, c4 = lane & 3;
  float worst = 0.f;
  // A warp takes 16 blocks at a time, as the MMAs' rows: lane (g4, c4) has dims 32 j + 8 c4 .. + 7 of
  // blocks g4 and g4 + 8. The next 16 blocks' bounds are asked for as these are used up.
  auto source = [&](int b) {
    const __nv_bfloat16* src = b < b1 ? block_bounds(p, pages, h, b) : nullptr;
    if (b < b1 && src == nullptr) raise_status(kStatusBadPage);
    return src;
  };
  auto load = [&](const __nv_bfloat16* src, int j) {
    return src ? *reinterpret_cast<const uint4*>(src + 32 * j + 8 * c4) : make_uint4(0, 0, 0, 0);
  };
  constexpr int kStep = 16 * kSparseWarps;
  uint4 va[8], vb[8];
  {
    const __nv_bfloat16 *sa = source(b0 + 16 * warp + g4), *sb = source(b0 + 16 * warp + 8 + g4);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      va[j] = load(sa, j);
      vb[j] = load(sb, j);
    }
  }
  // Query fragments, the same for every warp: head g4, dims 32 j + 8 c4 .. + 7; the negative parts (j
  // 0..3), then the positive ones. They stay in shared memory: 32 registers more than the 168 that
  // two CTAs per SM leave would be spilled, and what L1 the rings leave does not hold spills (16 rows
  // of 40,960 keys: 21 us for the scores, 13 without the spills).
  if (warp == 0) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint4 v = make_uint4(0, 0, 0, 0);
      if (g4 < GROUP)
        v = *reinterpret_cast<const uint4*>(p.q + (static_cast<int64_t>(token) * p.heads + h * GROUP + g4) * 128 + 32 * j +
                                            8 * c4);
      uint32_t w[4] = {v.x, v.y, v.z, v.w}, n[4], m[4];
      const __nv_bfloat162 zero = __float2bfloat162_rn(0.f);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 x = *reinterpret_cast<const __nv_bfloat162*>(&w[i]);
        const __nv_bfloat162 lo = __hmin2_nan(x, zero), hi = __hmax2_nan(x, zero);
        n[i] = *reinterpret_cast<const uint32_t*>(&lo);
        m[i] = *reinterpret_cast<const uint32_t*>(&hi);
      }
      frags[32 * j + lane] = make_uint4(n[0], n[1], n[2], n[3]);
      frags[32 * (j + 4) + lane] = make_uint4(m[0], m[1], m[2], m[3]);
    }
  }
  __syncthreads();
  if (ranks > 1) cluster_wait();  // every CTA of the cluster has started
  for (int base = b0 + 16 * warp; base < b1; base += kStep) {
    const __nv_bfloat16 *sa = source(base + kStep + g4), *sb = source(base + kStep + 8 + g4);
    // Two chains each for the scores and for sum |terms|: a warp MMA's result is 20 cycles away.
    float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
    float a0[4] = {0.f, 0.f, 0.f, 0.f}, a1[4] = {0.f, 0.f, 0.f, 0.f};
    constexpr uint32_t kAbs = 0x7FFF7FFFu;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint4 q = frags[32 * j + lane];
      const uint32_t f0[4] = {va[j].x, vb[j].x, va[j].y, vb[j].y}, f1[4] = {va[j].z, vb[j].z, va[j].w, vb[j].w};
      mma_16816(s0, f0, q.x, q.y);
      mma_16816(s1, f1, q.z, q.w);
      const uint32_t e0[4] = {f0[0] & kAbs, f0[1] & kAbs, f0[2] & kAbs, f0[3] & kAbs};
      const uint32_t e1[4] = {f1[0] & kAbs, f1[1] & kAbs, f1[2] & kAbs, f1[3] & kAbs};
      mma_16816(a0, e0, q.x & kAbs, q.y & kAbs);
      mma_16816(a1, e1, q.z & kAbs, q.w & kAbs);
      va[j] = load(sa, j);
      vb[j] = load(sb, j);
    }
    // Blocks base + g4 and + 8, heads 2 c4 and + 1: the largest over the group's heads.
    uint32_t key[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t k = 2 * c4 < GROUP ? score_key(s0[2 * i] + s1[2 * i]) : 0u;
      if (2 * c4 + 1 < GROUP) k = max(k, score_key(s0[2 * i + 1] + s1[2 * i + 1]));
      k = max(k, __shfl_xor_sync(0xffffffffu, k, 1));
      key[i] = max(k, __shfl_xor_sync(0xffffffffu, k, 2));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = a0[i] + a1[i];
      worst = a < INFINITY ? fmaxf(worst, a) : INFINITY;
    }
    // The lanes of a block hand it to CTAs c4 and c4 + 4.
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int b = base + 8 * i + g4;
      if (b < p.sink || b >= last) key[i] = 0u;
      if (c4 < ranks && b < b1) cluster_store(keys + b, c4, key[i]);
      if (c4 + 4 < ranks && b < b1) cluster_store(keys + b, c4 + 4, key[i]);
    }
  }
  return worst;
}

struct SparseShared {
  uint64_t full[kDecStages], empty[kDecStages];
  int abort_flag;
  uint32_t worst;  // largest sum |terms| (float bits; the CTAs' maxima meet here)
  int n_border;
  int taken[kSparseWarps];
  float merge_ml[kDecConsumerWarps][16][2];
  alignas(16) float part[8][128];  // unnormalised output of each head of the group over this CTA's blocks
  float part_ml[8][2];    // its running maximum and sum
};

// Exact score of block b (see the head of this file) by a whole warp, as an ordered integer.
template <int GROUP>
__device__ unsigned long long exact_score(const SparseAttentionParams& p, const int* pages, int token, int h, int b) {
  const int lane = threadIdx.x & 31;
  const __nv_bfloat16* src = block_bounds(p, pages, h, b);
  unsigned long long best = 0ull;
  if (src == nullptr) return best;
  const uint2 lo2 = *reinterpret_cast<const uint2*>(src + 4 * lane);
  const uint2 hi2 = *reinterpret_cast<const uint2*>(src + 128 + 4 * lane);
  const __nv_bfloat16 *lo = reinterpret_cast<const __nv_bfloat16*>(&lo2), *hi = reinterpret_cast<const __nv_bfloat16*>(&hi2);
  uint2 q2[GROUP];
#pragma unroll
  for (int g = 0; g < GROUP; ++g)
    q2[g] = *reinterpret_cast<const uint2*>(p.q + (static_cast<int64_t>(token) * p.heads + h * GROUP + g) * 128 + 4 * lane);
  double s[GROUP];
#pragma unroll
  for (int g = 0; g < GROUP; ++g) {
    const __nv_bfloat16* q = reinterpret_cast<const __nv_bfloat16*>(&q2[g]);
    s[g] = 0.0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // max(x lo, x hi): the bound on x's side. The other one counts where its product is NaN.
      const float x = __bfloat162float(q[i]), l = __bfloat162float(lo[i]), r = __bfloat162float(hi[i]);
      const float near = x > 0.f ? r : l, far = x > 0.f ? l : r;
      const float other = x * far;
      s[g] += static_cast<double>(x) * static_cast<double>(other == other ? near : NAN);  // exact in 64 bits
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)  // the heads' sums side by side
#pragma unroll
    for (int g = 0; g < GROUP; ++g) s[g] += __shfl_xor_sync(0xffffffffu, s[g], o);
#pragma unroll
  for (int g = 0; g < GROUP; ++g) best = max(best, score_key(s[g]));
  return best;
}

// A threshold on keys[] such that the keys above it are those of the `need` (>= 1) best blocks
// with non-zero keys; keys[] is padded with zeros to a multiple of 128. Every warp finds the
// need-th largest key for itself, by bisection: the scores of one row differ in their low 20 bits
// or so. With at most 128 KEEP keys (KEEP > 0) a lane holds its keys in registers. Only where the
// computed scores near the cut do not settle it do the warps work together: the keys there are
// replaced by the largest or the smallest one, by exact score (`index` and `score` are scratch).
template <int GROUP, int KEEP>
__device__ uint32_t cut_blocks(const SparseAttentionParams& p, const int* pages, int token, int h, int nb, int need,
                               float worst, uint32_t* keys, uint32_t* index, unsigned long long* score,
                               int* n_border) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint4* k4 = reinterpret_cast<const uint4*>(keys) + lane;
  const int passes = KEEP > 0 ? KEEP : (nb + 127) / 128;
  uint4 kept[KEEP > 0 ? KEEP : 1];
  if constexpr (KEEP > 0) {
#pragma unroll
    for (int i = 0; i < KEEP; ++i) kept[i] = 128 * i < nb ? k4[32 * i] : make_uint4(0, 0, 0, 0);
  }
  // f for every four keys of the lane, or for each of them.
  auto each4 = [&](auto f) {
    if constexpr (KEEP > 0) {
#pragma unroll
      for (int i = 0; i < KEEP; ++i) f(kept[i].x, kept[i].y, kept[i].z, kept[i].w);
    } else {
      for (int i = 0; i < passes; ++i) {
        const uint4 v = k4[32 * i];
        f(v.x, v.y, v.z, v.w);
      }
    }
  };
  auto each = [&](auto f) {
    each4([&](uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
      f(a);
      f(b);
      f(c);
      f(d);
    });
  };
  uint32_t hi = 0u, lo = 0xFFFFFFFFu;
  each([&](uint32_t k) {
    hi = max(hi, k);
    lo = min(lo, k - 1u);  // 0 wraps to the largest
  });
  hi = __reduce_max_sync(0xffffffffu, hi);
  lo = __reduce_min_sync(0xffffffffu, lo) + 1u;
  bool met = false;  // exactly `need` keys reach lo; always: count(key >= lo) >= need > count(key > hi)
  while (lo < hi && !met) {
    const uint32_t mid = lo + (hi - lo) / 2 + 1;  // lo < mid <= hi
    int n = 0;
    each4([&](uint32_t a, uint32_t b, uint32_t c, uint32_t d) { n += ((a >= mid) + (b >= mid)) + ((c >= mid) + (d >= mid)); });
    n = __reduce_add_sync(0xffffffffu, n);
    if (n >= need) {
      lo = mid;
      met = n == need;
    } else {
      hi = mid - 1;
    }
  }
  uint32_t kth = 0xFFFFFFFFu;  // the need-th largest key
  each([&](uint32_t k) { kth = min(kth, k >= lo ? k : 0xFFFFFFFFu); });
  kth = __reduce_min_sync(0xffffffffu, kth);
  const float eps2 = 2.f * 3.0517578125e-5f * worst;  // 2 eps, eps = 2^-15 sum |terms|
  const float cut = key_score(kth);
  // Every block within 2 eps of the cut (all of them where scores are not finite), one more step
  // outwards for the rounding of these sums.
  uint32_t low = 1u, high = 0xFFFFFFFFu;
  if (eps2 < INFINITY && fabsf(cut) < INFINITY && kth != 0xFFFFFFFFu) {
    low = score_key(__fsub_rd(cut, eps2));
    high = score_key(__fadd_ru(cut, eps2));
  }
  int count = 0;  // keys above the border, and in its low half those in it
  each([&](uint32_t k) { count += k > high ? 0x10000 : k >= low ? 1 : 0; });  // low >= 1: never a forced block
  count = __reduce_add_sync(0xffffffffu, count);
  const int left = need - (count >> 16), border = count & 0xFFFF;
  if (left >= border) return low - 1u;  // all of them: no doubt
  // The same decision in every warp: the CTA goes on together.
  for (int b = threadIdx.x; b < nb; b += kSparseThreads)
    if (keys[b] >= low && keys[b] <= high) index[atomicAdd(n_border, 1)] = static_cast<uint32_t>(b);
  __syncthreads();
  for (int i = warp; i < border; i += kSparseWarps) {
    const unsigned long long s = exact_score<GROUP>(p, pages, token, h, static_cast<int>(index[i]));
    if (lane == 0) score[i] = s;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < border; i += kSparseThreads) {  // the larger score, then the lower block
    const unsigned long long s = score[i];
    const uint32_t b = index[i];
    int rank = 0;
    for (int j = 0; j < border; ++j) rank += score[j] > s || (score[j] == s && index[j] < b);
    keys[b] = rank < left ? 0xFFFFFFFFu : 1u;
  }
  __syncthreads();
  return min(high, 0xFFFFFFFEu);
}

// One cluster per (row, KV head): its CTAs score a share of the row's blocks each and hand the
// scores to one another, select alike, attend to a share of the selected blocks each (the
// decode ring and tile of attention_decode.cuh), and merge through shared memory. One launch,
// no workspace. Clusters are as large as two CTAs per SM allow, so that few rows use every SM.
//
// Measured (8 KV heads of 4 query heads): 64 rows of 8 to 20 thousand keys, 48 blocks each, 143 us: 0.94
// of what the bounds and the selected K and V take at the measured copy rate, and bound by it. 16
// rows of 500 to 41,000 keys, 32 blocks: 36 us (floor 24); the longest row's scores take 11 of them
// (their loads go through what L1 the rings leave, 18 KB per SM), its selection 2.
// 1 row of 40,000: 12.7 us (floor 1.7), steps one after the other: launch 1.5, scores 2.7, selection
// 1.9, list 0.9, the first K and V, tiles and merges 5.7.
template <int GROUP>
__global__ void __launch_bounds__(kSparseThreads, 2) sparse_attention_kernel(SparseAttentionParams p,
                                                                            const __grid_constant__ CUtensorMap kmap,
                                                                            const __grid_constant__ CUtensorMap vmap) {
  extern __shared__ __align__(1024) uint8_t dsm[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dsm) + 1023) & ~uintptr_t(1023));
  __shared__ SparseShared sh;
  uint32_t* keys = reinterpret_cast<uint32_t*>(smem);
  uint32_t* index = keys + kSparseMaxBlocks;
  unsigned long long* score = reinterpret_cast<unsigned long long*>(index + kSparseMaxBlocks);
  int* list = reinterpret_cast<int*>(smem + kDecRingBytes);  // [top] selected blocks, ascending
  int* where = list + p.top;                                 // [top] first pool token, -1: no page
  int* pages = where + p.top;                                // [width] the row's pages
  pdl_wait();  // keys, bounds and queries, from the kernels ahead
  pdl_trigger();

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int ranks = static_cast<int>(cluster_size()), rank = static_cast<int>(cluster_rank());
  const int h = blockIdx.y, row = blockIdx.z;
  int len = p.seqused_k[row], token = row;
  if (p.cu_seq_q != nullptr) {
    token = p.cu_seq_q[row];
    if (p.cu_seq_q[row + 1] - token != 1) return;  // the whole cluster
  }
  for (int i = tid; i < p.width; i += kSparseThreads) pages[i] = p.block_table[static_cast<int64_t>(row) * p.width + i];
  if (len > p.width * p.page_size) {  // more keys than the table has pages for
    if (tid == 0 && rank == 0) raise_status(kStatusBadPage);
    len = p.width * p.page_size;
  }
  const int nb = len > 0 ? (len - 1) / kBlockKeys + 1 : 0;
  if (tid == 0) {
    for (int s = 0; s < kDecStages; ++s) {
      mbar_init(&sh.full[s], 1);
      mbar_init(&sh.empty[s], kDecConsumerWarps);
    }
    sh.abort_flag = 0;
    sh.worst = 0u;
    sh.n_border = 0;
    fence_barrier_init();
  }
  const bool choose = nb > p.top;  // row-uniform: the whole cluster agrees
  const int need = choose ? p.top - p.sink - p.recent : 0;
  uint32_t above = 0u;  // blocks with keys above this are taken, and the forced ones
  __syncthreads();
  if (need > 0) {
    if (ranks > 1) cluster_arrive();  // the words that the others write are set
    const int last = nb - p.recent, groups = (nb + 7) / 8;
    const int b0 = 8 * (groups * rank / ranks), b1 = min(nb, 8 * (groups * (rank + 1) / ranks));
    for (int b = nb + tid; b < (nb + 127) / 128 * 128; b += kSparseThreads) keys[b] = 0u;
    float worst = score_blocks<GROUP>(p, pages, token, h, b0, b1, last, keys, reinterpret_cast<uint4*>(sh.part), ranks);
    worst = warp_max(worst);
    if (lane < ranks) {  // non-negative floats compare as their bits do
      uint32_t a;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(&sh.worst)), "r"(lane));
      asm volatile("red.relaxed.cluster.shared::cluster.max.u32 [%0], %1;" ::"r"(a), "r"(__float_as_uint(worst)) : "memory");
    }
    if (ranks > 1) cluster_sync();
    else __syncthreads();
    const float size = __uint_as_float(sh.worst);
    // Up to 640 blocks a lane holds its keys in 20 registers (8 rows of 40,960 keys: 25.0 us, 26.6 with the
    // keys read from shared memory in every step); with 40, for up to 1,280, shorter rows lose more (26.4)
    // than longer ones gain (8 rows of 80,000: 34.1 -> 32.4).
    above = nb <= 640 ? cut_blocks<GROUP, 5>(p, pages, token, h, nb, need, size, keys, index, score, &sh.n_border)
                      : cut_blocks<GROUP, 0>(p, pages, token, h, nb, need, size, keys, index, score, &sh.n_border);
  }
  // Ascending list: four blocks per thread at a time, places by a scan over the CTA.
  int n_sel = 0;
  if (!choose) {
    n_sel = nb;
    for (int i = tid; i < nb; i += kSparseThreads) list[i] = i;
  } else {
    for (int b0 = 0; b0 < nb; b0 += 4 * kSparseThreads) {
      const int b = b0 + 4 * tid;
      uint32_t take = 0;
      uint4 k = make_uint4(0, 0, 0, 0);
      if (need > 0 && b < nb) k = *reinterpret_cast<const uint4*>(keys + b);
      const uint32_t w[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        take |= (b + e < nb && (w[e] > above || b + e < p.sink || b + e >= nb - p.recent) ? 1u : 0u) << e;
      const int mine = __popc(take);
      int incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      if (lane == 31) sh.taken[warp] = incl;
      __syncthreads();
      int at = n_sel + incl - mine;
#pragma unroll
      for (int x = 0; x < kSparseWarps; ++x) {
        if (x < warp) at += sh.taken[x];
        n_sel += sh.taken[x];
      }
      for (; take; take &= take - 1, ++at)
        if (at < p.top) list[at] = b + __ffs(take) - 1;
      __syncthreads();
    }
    n_sel = min(n_sel, p.top);  // it is p.top
  }
  __syncthreads();
  for (int i = tid; i < n_sel; i += kSparseThreads) {
    const int b = list[i], pidx = block_page(p, b), page = pages[pidx];
    const bool ok = page >= 0 && page < p.num_pages;
    if (!ok) raise_status(kStatusBadPage);
    where[i] = ok ? page * p.page_size + (b - pidx * p.per_page) * kBlockKeys : -1;
  }
  if (p.selected != nullptr && rank == 0) {
    int32_t* dst = p.selected + (static_cast<int64_t>(row) * p.kv_heads + h) * p.top;
    for (int i = tid; i < p.top; i += kSparseThreads) dst[i] = i < n_sel ? list[i] : -1;
  }
  fence_proxy_async_smem();  // the ring's generic reads and writes precede its TMA fills
  __syncthreads();

  const int i0 = n_sel * rank / ranks, i1 = n_sel * (rank + 1) / ranks;  // this CTA's blocks
  if (warp == kDecConsumerWarps) {
    if (lane == 0) {
      int t = 0;
      for (int i = i0; i < i1; ++i) {
        const int tok = where[i];
        if (tok < 0) continue;
        const int s = t % kDecStages;
        if (t >= kDecStages && !mbar_wait(&sh.empty[s], ((t / kDecStages) - 1) & 1, &sh.abort_flag)) break;
        uint8_t* stage = smem + s * kDecStageBytes;
        mbar_expect_tx(&sh.full[s], kDecStageBytes);
        tma_load_3d(stage, &kmap, &sh.full[s], 0, h, tok);
        tma_load_3d(stage + kDecHalfBytes, &kmap, &sh.full[s], 64, h, tok);
        tma_load_3d(stage + kDecTileBytes, &vmap, &sh.full[s], 0, h, tok);
        tma_load_3d(stage + kDecTileBytes + kDecHalfBytes, &vmap, &sh.full[s], 64, h, tok);
        ++t;
      }
      // Never leave with copies in flight.
      if (sh.abort_flag)
        for (int j = max(0, t - kDecStages); j < t; ++j) mbar_drain(&sh.full[j % kDecStages], (j / kDecStages) & 1);
    }
    __syncwarp();
  } else {
    AttentionParams ap{};
    ap.q = p.q;
    ap.heads = p.heads;
    ap.scale_log2 = p.scale_log2;
    DecodeUnit u{};
    u.h = h;
    u.row = row;
    u.q0 = token;
    u.count = 1;
    u.end = u.ke = len;
    u.qrows = GROUP;
    u.key_split = kDecConsumerWarps;
    u.kpw = kBlockKeys / kDecConsumerWarps;
    u.mt = 0;
    u.kpart = warp;
    const int g4 = lane >> 2, c4 = lane & 3;
    uint32_t qa[8][4];
    decode_load_q<GROUP>(ap, u, lane, qa);
    const int qpos_a = decode_qpos<GROUP>(u, g4), qpos_b = -1;
    float acc[16][4];
#pragma unroll
    for (int n = 0; n < 16; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
    float m_a = -INFINITY, m_b = -INFINITY, l_a = 0.f, l_b = 0.f;
    int t = 0;
    for (int i = i0; i < i1; ++i) {
      if (where[i] < 0) continue;
      const int s = t % kDecStages;
      if (!mbar_wait(&sh.full[s], (t / kDecStages) & 1, &sh.abort_flag)) break;
      decode_tile<GROUP, true>(ap, u, smem + s * kDecStageBytes, list[i] * kBlockKeys, lane, qpos_a, qpos_b, qa, acc, m_a, m_b,
                         l_a, l_b);
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.empty[s]);
      ++t;
    }
#pragma unroll
    for (int n = 0; n < 16; ++n) {  // the rounded weights' sums and what their rounding left
      acc[n][0] += acc[n][2];
      acc[n][1] += acc[n][3];
    }
    l_a += __shfl_xor_sync(0xffffffffu, l_a, 1);
    l_a += __shfl_xor_sync(0xffffffffu, l_a, 2);
    l_b += __shfl_xor_sync(0xffffffffu, l_b, 1);
    l_b += __shfl_xor_sync(0xffffffffu, l_b, 2);
    named_barrier_sync(1, kDecConsumerWarps * 32);  // the ring is idle: it becomes the merge scratch
    // After a wait that gave up this merges garbage, but every warp still meets every barrier.
    decode_merge(u, warp, lane, reinterpret_cast<float*>(smem), sh.merge_ml, acc, m_a, m_b, l_a, l_b,
                 [] { named_barrier_sync(1, kDecConsumerWarps * 32); });
    if (warp == 0 && g4 < GROUP) {
#pragma unroll
      for (int n = 0; n < 16; ++n) {
        sh.part[g4][n * 8 + 2 * c4] = acc[n][0];
        sh.part[g4][n * 8 + 2 * c4 + 1] = acc[n][1];
      }
      if (c4 == 0) {
        sh.part_ml[g4][0] = m_a;
        sh.part_ml[g4][1] = l_a;
      }
    }
    __syncwarp();
  }
  if (ranks > 1) cluster_sync();
  else __syncthreads();
  // out = sum_c 2^(m_c - m) acc_c / sum_c 2^(m_c - m) l_c, in rank order; a row without keys gives 0
  // (den is 0 then alone: a NaN or infinite score leaves den NaN, and shows).
  for (int i = rank * kSparseThreads + tid; i < GROUP * 128; i += ranks * kSparseThreads) {
    const int g = i / 128, d = i % 128;
    float m[8], l[8], v[8];  // every CTA's parts are asked for before any is used
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      if (r < ranks) {
        m[r] = cluster_load(&sh.part_ml[g][0], r);
        l[r] = cluster_load(&sh.part_ml[g][1], r);
        v[r] = cluster_load(&sh.part[g][d], r);
      }
    }
    float mx = -INFINITY, num = 0.f, den = 0.f;
#pragma unroll
    for (int r = 0; r < 8; ++r)
      if (r < ranks) mx = fmaxf(mx, m[r]);
    const float base = mx == -INFINITY ? 0.f : mx;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      if (r < ranks) {
        const float w = exp2f(m[r] - base);
        num += w * v[r];
        den += w * l[r];
      }
    }
    p.out[(static_cast<int64_t>(token) * p.heads + h * GROUP + g) * 128 + d] = __float2bfloat16_rn(den == 0.f ? 0.f : num / den);
  }
  if (ranks > 1) cluster_sync();  // the parts stay until every CTA has read them
}

}  // namespace hb
