// Projections with 4-bit weights and group scales, for the few token rows of a small decode tick.
//
//   out[t, n] = bf16( sum_g s[g, n] * sum_{k in group g} (q[n, k] - z[g, n]) * x[t, k] )
//
// q is 0..15; z is 8 where no zero points are given. The weight is read as it is stored:
// packed int32 [N, K / 8], word j of a row holding k = 8j .. 8j + 7 with the even k's in its low
// 16 bits and the odd k's in its high 16 bits, four bits each in ascending k, so
// (word >> 4i) & 0x000F000F is the pair k = 8j + 2i, 8j + 2i + 1, and OR-ing 0x4300 into each half
// makes the bf16 values 128 + q, from which 128 + z is subtracted, exactly: two weights q - z for a
// shift, a LOP3 and a packed subtraction. The products (q - z) x are exact in fp32, so the error is
// that of adding them up: an activation whose code is the zero point adds nothing, however large it is.
// (Multiplying 128 + q and taking (128 + z) sum x off afterwards, from MMAs with a row of ones, leaves
// some 136 |x| 2^-24 of it behind at every addition: in one group of 128 with x = 2^15 at a zero point, errors
// of 0.89 on average beside results of 38 and 0.05 of rounding, which is all there is this way. It was also
// slower, by the ones' MMAs: 19456 x 2560 at 1 token 10.9 us, 10.3 as it is.)
//
// Products run on m16n8k16 warp MMAs with 16 weight rows as M and 8 tokens as N. The sum over k
// does not depend on which k a fragment register holds, as long as A and B agree, so a thread
// takes its k's as consecutive words of the packed row (16 bytes per row for groups of 128) and
// its activations as the matching 16-byte pieces: no reordering on either side. Every group is
// summed in a fresh fp32 accumulator and scaled once, in fp32, so the only rounding to bf16 is the
// output's.
//
// Two kernels share this: up to 8 tokens warps load their own fragments (the second one below); from
// 9 to 16, with twice the activations per weight, a ring filled by TMA brings both. There a CTA has
// 64 weight rows, two warps for every 16, and all tokens; one more warp copies stages of 256 k's, so that
// every SM keeps 130 KB on the way whatever the others do, and a cluster of CTAs shares k where there are
// few weight rows. 16 tokens, weights from DRAM: 19456 x 2560 in 16.1 us (1.6 TB/s), 2560 x 9728 in 9.8,
// 6144 x 2560 in 7.5, 2560 x 4096 in 6.3. Both kernels are bound by latency (launch, first bytes, the sums
// over warps and CTAs) more than by HBM: 0.9 to 2.5 TB/s.
#pragma once

#include "hb_common.cuh"

namespace hb {

struct LinearW4Params {
  const __nv_bfloat16* x;  // [m, x_stride]
  int64_t x_stride;
  const uint32_t* packed;        // [n, k / 8]
  const __nv_bfloat16* scales;   // [k / G, n]
  const uint8_t* zeros;          // [k / G, n] or null
  __nv_bfloat16* out;            // [m, n]
  int32_t m, n, k;
};

constexpr int kW4Tiles = 4;             // MMA tiles of 16 weight rows per CTA
constexpr int kW4Halves = 2;            // warps per tile, taking the two halves of every stage's k's
constexpr int kW4Warps = kW4Tiles * kW4Halves;
constexpr int kW4Threads = 32 * (kW4Warps + 1);  // and the copying one
constexpr int kW4Rows = 16 * kW4Tiles;  // weight rows per CTA
constexpr int kW4StageK = 256;          // k's per stage: 128 bytes of a packed row
constexpr int kW4MaxSplits = 8;
// Most token rows here; the tcgen05 kernel (gemm_w4.cuh) has more. 19456 x 2560: 16.1 us at 16 rows here and
// 22.3 at 17 there, 32.7 at 32 with two tiles more of tokens here; 2560 x 9728: 9.8, 13.2 and 18.4.
constexpr int kW4MaxTokens = 16;

struct W4Stage {
  static constexpr int kWeightBytes = kW4Rows * kW4StageK / 2;  // one box of 128-byte rows
  static constexpr int kBoxBytes = kW4MaxTokens * 128;          // activations: a box per 64 k's
  static constexpr int kBytes = kWeightBytes + kW4StageK / 64 * kBoxBytes;
  static constexpr int kStages = 4;
  static constexpr int kSmem = kStages * kBytes + 1024;  // 65 KB
  static constexpr int kPerSm = 2;                       // CTAs that fit an SM, by registers
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  __syncwarp();  // the barrier wants whole warps
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The two halves of cluster_sync, for work in between (each thread once, in this order).
__device__ __forceinline__ void cluster_arrive() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// A float of another CTA's shared memory, at the place `local` has in this CTA's.
__device__ __forceinline__ float cluster_load(const float* local, uint32_t rank) {
  uint32_t a;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(local)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}

__device__ __forceinline__ float4 cluster_load4(const float* local, uint32_t rank) {
  uint32_t a;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(local)), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(a)
               : "memory");
  return v;
}

// The bf16 pair (128 + z, 128 + z) of a zero point.
__device__ __forceinline__ uint32_t w4_zero_pair(uint32_t z) { return (0x4300u | (z & 15u)) * 0x00010001u; }

// Four bf16 pairs (q - z) of one packed word, exact; zz as w4_zero_pair gives it.
__device__ __forceinline__ void w4_unpack(uint32_t w, uint32_t zz, uint32_t (&p)[4]) {
  const __nv_bfloat162 z2 = *reinterpret_cast<const __nv_bfloat162*>(&zz);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t v = ((w >> (4 * i)) & 0x000F000Fu) | 0x43004300u;
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), z2);
    p[i] = *reinterpret_cast<const uint32_t*>(&d);
  }
}

template <int WORDS>
__device__ __forceinline__ void shared_load(uint32_t src, uint32_t (&v)[WORDS]) {
  if constexpr (WORDS == 4)
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(src));
  else if constexpr (WORDS == 2)
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(src));
  else
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v[0]) : "r"(src));
}
template <int WORDS>
__device__ __forceinline__ void global_load(const uint32_t* src, uint32_t* v) {
  if constexpr (WORDS == 4) {
    const uint4 q = __ldg(reinterpret_cast<const uint4*>(src));
    v[0] = q.x, v[1] = q.y, v[2] = q.z, v[3] = q.w;
  } else if constexpr (WORDS == 2) {
    const uint2 q = __ldg(reinterpret_cast<const uint2*>(src));
    v[0] = q.x, v[1] = q.y;
  } else {
    v[0] = __ldg(src);
  }
}
// Grid (cluster of K splits, row tiles). Rank r of a cluster has the stages r, r +
// splits, ...; the CTAs' sums are added in rank order, from shared memory, so results do not
// depend on timing. Weight rows, tokens and k's past the end arrive as zeros.
template <int G, bool ZEROS>
__global__ void __launch_bounds__(kW4Threads, W4Stage::kPerSm)
    linear_w4_kernel(LinearW4Params p, const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap) {
  using Stage = W4Stage;
  constexpr int NT = kW4MaxTokens / 8;  // MMA tiles of tokens
  constexpr int WPG = G / 32;         // words of one group that a thread holds
  constexpr int GPT = kW4StageK / G / kW4Halves;  // groups per stage and warp
  constexpr int kTokens = 8 * NT, kStages = Stage::kStages;
  extern __shared__ __align__(1024) uint8_t dsm[];
  const uint32_t ring = (smem_u32(dsm) + 1023u) & ~1023u;
  // The sums, once the ring is idle: [token][row].
  constexpr int kPartStride = kW4Rows + 4;
  static_assert(kTokens * kPartStride * 4 <= Stage::kSmem - 1024, "the sums fit the ring");
  float* parts = reinterpret_cast<float*>(dsm + (ring - smem_u32(dsm)));
  __shared__ uint64_t full[kStages], empty[kStages];
  __shared__ int abort_flag;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g4 = lane >> 2, c4 = lane & 3;
  const int splits = static_cast<int>(cluster_size()), rank = static_cast<int>(cluster_rank());
  const int row0 = blockIdx.y * kW4Rows;
  const int all = (p.k + kW4StageK - 1) / kW4StageK;
  const int n = rank < all ? (all - rank + splits - 1) / splits : 0;  // this CTA's stages
  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], kW4Warps);
    }
    abort_flag = 0;
    fence_barrier_init();
  }
  __syncthreads();
  pdl_wait();  // the activations, from the kernel ahead (it may have written weights, too)
  pdl_trigger();

  float acc[NT][4];
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t][0] = acc[t][1] = acc[t][2] = acc[t][3] = 0.f;
  if (warp == kW4Warps) {
    if (lane == 0) {
      int s = 0;
      for (; s < n; ++s) {
        const int st = s % kStages, k0 = (rank + s * splits) * kW4StageK;
        if (s >= kStages && !mbar_wait(&empty[st], ((s / kStages) - 1) & 1, &abort_flag)) break;
        const uint32_t dst = ring + st * Stage::kBytes;
        mbar_expect_tx(&full[st], Stage::kBytes);
        tma_load_2d_at(dst, &wmap, &full[st], k0 / 8, row0);
#pragma unroll
        for (int b = 0; b < kW4StageK / 64; ++b)
          tma_load_2d_at(dst + Stage::kWeightBytes + b * Stage::kBoxBytes, &xmap, &full[st], k0 + 64 * b, 0);
      }
      for (int j = max(0, s - kStages); j < s; ++j) mbar_drain(&full[j % kStages], (j / kStages) & 1);
    }
    __syncwarp();
  } else {
    // Scales and zero points of this thread's rows, two stages ahead in registers (DRAM is further
    // away than one). Past k's end any scale does.
    const int tile = warp % kW4Tiles, half = warp / kW4Tiles;
    const int ra = min(row0 + 16 * tile + g4, p.n - 1), rb = min(row0 + 16 * tile + g4 + 8, p.n - 1);
    const int groups = p.k / G;
    struct Scales {
      __nv_bfloat16 a[GPT], b[GPT];
      uint8_t za[GPT], zb[GPT];
    };
    auto load_scales = [&](int s, Scales& v) {
      const int first = ((rank + s * splits) * kW4Halves + half) * GPT;
#pragma unroll
      for (int g = 0; g < GPT; ++g) {
        const int64_t at = static_cast<int64_t>(min(first + g, groups - 1)) * p.n;
        v.a[g] = p.scales[at + ra];
        v.b[g] = p.scales[at + rb];
        if (ZEROS) {
          v.za[g] = p.zeros[at + ra];
          v.zb[g] = p.zeros[at + rb];
        }
      }
    };
    Scales now, next;
    load_scales(0, now);
    load_scales(1, next);
    const uint32_t wfrag = ring + 128 * (16 * tile + g4);
    // The half's activations start two boxes on.
    const uint32_t xfrag = ring + Stage::kWeightBytes + half * (kW4StageK / 64 / kW4Halves) * Stage::kBoxBytes + 128 * g4;
    for (int s = 0; s < n; ++s) {
      const int st = s % kStages;
      float fa[GPT], fb[GPT];
      uint32_t za[GPT], zb[GPT];
#pragma unroll
      for (int g = 0; g < GPT; ++g) {
        fa[g] = __bfloat162float(now.a[g]);
        fb[g] = __bfloat162float(now.b[g]);
        za[g] = w4_zero_pair(ZEROS ? now.za[g] : 8);
        zb[g] = w4_zero_pair(ZEROS ? now.zb[g] : 8);
      }
      now = next;
      load_scales(s + 2, next);
      if (!mbar_wait_fast(&full[st], (s / kStages) & 1, &abort_flag)) break;
      const uint32_t wst = wfrag + st * Stage::kBytes, xst = xfrag + st * Stage::kBytes;
#pragma unroll
      for (int g = 0; g < GPT; ++g) {
        // Rows 16 tile + g4 and + 8 (the same swizzle): 4 WPG bytes from 64 half + g G / 2 + 4 WPG c4.
        uint32_t qa[WPG], qb[WPG];
        const int piece = 4 * half + g * (G / 32) + (WPG == 4 ? c4 : WPG == 2 ? c4 >> 1 : 0);
        const int within = WPG == 4 ? 0 : WPG == 2 ? (c4 & 1) * 8 : c4 * 4;
        shared_load<WPG>(wst + ((piece ^ g4) << 4) + within, qa);
        shared_load<WPG>(wst + ((piece ^ g4) << 4) + within + 8 * 128, qb);
        float part[NT][4];
#pragma unroll
        for (int t = 0; t < NT; ++t) part[t][0] = part[t][1] = part[t][2] = part[t][3] = 0.f;
#pragma unroll
        for (int w = 0; w < WPG; ++w) {
          uint32_t a[4], b[4];
          w4_unpack(qa[w], za[g], a);
          w4_unpack(qb[w], zb[g], b);
          const uint32_t a0[4] = {a[0], b[0], a[1], b[1]}, a1[4] = {a[2], b[2], a[3], b[3]};
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            uint32_t x[4];
            const int at = g * (G / 8) + WPG * c4 + w;  // 16-byte piece of the half's 16
            shared_load<4>(xst + (at >> 3) * Stage::kBoxBytes + (((at & 7) ^ g4) << 4) + 8 * 128 * t, x);
            mma_16816(part[t], a0, x[0], x[1]);
            mma_16816(part[t], a1, x[2], x[3]);
          }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          acc[t][0] += fa[g] * part[t][0];
          acc[t][1] += fa[g] * part[t][1];
          acc[t][2] += fb[g] * part[t][2];
          acc[t][3] += fb[g] * part[t][3];
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
    }
    named_barrier_sync(1, 32 * kW4Warps);  // every warp has read its last stage
    if (half == 1) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) parts[(8 * t + 2 * c4 + (e & 1)) * kPartStride + 16 * tile + g4 + 8 * (e >> 1)] = acc[t][e];
    }
    named_barrier_sync(1, 32 * kW4Warps);
    if (half == 0) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) parts[(8 * t + 2 * c4 + (e & 1)) * kPartStride + 16 * tile + g4 + 8 * (e >> 1)] += acc[t][e];
    }
    __syncwarp();
  }
  if (splits > 1) cluster_sync();
  else __syncthreads();
  const int tokens = p.m;
  // Every CTA finishes a share of the outputs, four rows at a time.
  const bool wide = p.n % 4 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 7) == 0;
  for (int i = rank * kW4Threads + tid; i < tokens * kW4Rows / 4; i += splits * kW4Threads) {
    const int token = i / (kW4Rows / 4), r = 4 * (i % (kW4Rows / 4)), row = row0 + r;
    if (row >= p.n) continue;
    float4 v[kW4MaxSplits];
#pragma unroll
    for (int q = 0; q < kW4MaxSplits; ++q)
      if (q < splits) v[q] = cluster_load4(parts + token * kPartStride + r, q);
    float4 s = v[0];
#pragma unroll
    for (int q = 1; q < kW4MaxSplits; ++q)
      if (q < splits) {
        s.x += v[q].x;
        s.y += v[q].y;
        s.z += v[q].z;
        s.w += v[q].w;
      }
    const float o[4] = {s.x, s.y, s.z, s.w};
    __nv_bfloat16* dst = p.out + static_cast<int64_t>(token) * p.n + row;
    if (wide) {
      *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3]));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (row + e < p.n) dst[e] = __float2bfloat16_rn(o[e]);
    }
  }
  if (splits > 1) cluster_sync();  // the sums stay until every CTA has read them
}

// Up to 8 tokens: no ring and no cluster. A CTA has 16 weight rows; each of its warps takes every
// `warps`-th unit of 128 k's, loads the next one's weights and scales into registers when it has done
// with one, and the warps' sums are added in shared memory, in warp order. Many warps keep the loads
// on the way here, so registers count: 64 a thread, 32 warps per SM. One token, weights from DRAM: 19456 x
// 2560 in 10.3 us (2.5 TB/s), 6144 x 2560 in 5.1, 2560 x 4096 in 5.1, 2560 x 9728 in 9.3; 8 tokens 12.4, 5.4, 5.7
// and 10.5. Before the exact subtraction, when 19456 x 2560 took 11.0, four units ahead in 124 registers
// took 13.9, prefetches into L2 12.3, 40 registers 15.2, two chains of MMAs per sum 13.3 and the ring kernel
// with one tile of tokens 15.0.
constexpr int kW4DirectTokens = 8;
constexpr int kW4DirectWarps = 16;  // at most
constexpr int kW4DirectFewest = 5;  // where the units allow

template <int G, bool ZEROS>
__global__ void __launch_bounds__(32 * kW4DirectWarps, 2) linear_w4_direct_kernel(LinearW4Params p) {
  constexpr int WPG = G / 32, GPU = 128 / G;  // words of a group that a thread holds, groups per unit
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g4 = lane >> 2, c4 = lane & 3;
  const int warps = blockDim.x >> 5, row0 = blockIdx.x * 16;
  const int ra = min(row0 + g4, p.n - 1), rb = min(row0 + g4 + 8, p.n - 1);
  const int groups = p.k / G, units = (groups + GPU - 1) / GPU;
  const uint32_t* wa = p.packed + static_cast<int64_t>(ra) * (p.k / 8) + WPG * c4;
  const uint32_t* wb = p.packed + static_cast<int64_t>(rb) * (p.k / 8) + WPG * c4;
  const __nv_bfloat16* x = p.x + min(g4, p.m - 1) * p.x_stride + 8 * WPG * c4;
  uint32_t qa[4], qb[4];
  __nv_bfloat16 sa[GPU], sb[GPU];
  uint8_t za[GPU], zb[GPU];
  auto load = [&](int unit) {
#pragma unroll
    for (int g = 0; g < GPU; ++g) {
      const int group = unit * GPU + g;
      if (group >= groups) continue;
      const int64_t at = static_cast<int64_t>(group) * p.n;
      global_load<WPG>(wa + group * (G / 8), &qa[g * WPG]);
      global_load<WPG>(wb + group * (G / 8), &qb[g * WPG]);
      sa[g] = p.scales[at + ra];
      sb[g] = p.scales[at + rb];
      if (ZEROS) {
        za[g] = p.zeros[at + ra];
        zb[g] = p.zeros[at + rb];
      }
    }
  };
  pdl_wait();  // the activations, from the kernel ahead (it may have written weights, too)
  pdl_trigger();
  load(warp);
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int unit = warp; unit < units; unit += warps) {
#pragma unroll
    for (int g = 0; g < GPU; ++g) {
      const int group = unit * GPU + g;
      if (group >= groups) break;
      const float fa = __bfloat162float(sa[g]), fb = __bfloat162float(sb[g]);
      const uint32_t zza = w4_zero_pair(ZEROS ? za[g] : 8), zzb = w4_zero_pair(ZEROS ? zb[g] : 8);
      float part[4] = {0.f, 0.f, 0.f, 0.f};
      uint4 xv[WPG];
#pragma unroll
      for (int w = 0; w < WPG; ++w)
        xv[w] = g4 < p.m ? *reinterpret_cast<const uint4*>(x + group * G + 8 * w) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int w = 0; w < WPG; ++w) {
        uint32_t a[4], b[4];
        w4_unpack(qa[g * WPG + w], zza, a);
        w4_unpack(qb[g * WPG + w], zzb, b);
        const uint32_t a0[4] = {a[0], b[0], a[1], b[1]}, a1[4] = {a[2], b[2], a[3], b[3]};
        mma_16816(part, a0, xv[w].x, xv[w].y);
        mma_16816(part, a1, xv[w].z, xv[w].w);
      }
      acc[0] += fa * part[0];
      acc[1] += fa * part[1];
      acc[2] += fb * part[2];
      acc[3] += fb * part[3];
    }
    load(unit + warps);
  }
  __shared__ float parts[kW4DirectWarps][16 * kW4DirectTokens];  // [token][row]
#pragma unroll
  for (int e = 0; e < 4; ++e) parts[warp][(2 * c4 + (e & 1)) * 16 + g4 + 8 * (e >> 1)] = acc[e];
  __syncthreads();
  for (int i = tid; i < p.m * 16; i += blockDim.x) {
    float sum = parts[0][i];
    for (int w = 1; w < warps; ++w) sum += parts[w][i];
    const int row = row0 + i % 16;
    if (row < p.n) p.out[static_cast<int64_t>(i / 16) * p.n + row] = __float2bfloat16_rn(sum);
  }
}

}  // namespace hb
