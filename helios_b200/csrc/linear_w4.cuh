// Projections with 4-bit weights and group scales, for the few token rows of a decode tick.
//
//   out[t, n] = bf16( sum_g s[g, n] * sum_{k in group g} (q[n, k] - z[g, n]) * x[t, k] )
//
// q is 0..15; z is 8 where no zero points are given. The weight is read as it is stored:
// packed int32 [N, K / 8], word j of a row holding k = 8j .. 8j + 7 with the even k's in its low
// 16 bits and the odd k's in its high 16 bits, four bits each in ascending k, so
// (word >> 4i) & 0x000F000F is the pair k = 8j + 2i, 8j + 2i + 1. OR-ing 0x4300 into each half
// makes the bf16 values 128 + q, and subtracting 128 + z (also a bf16 value) is exact, so two
// weights cost one LOP3 and one packed subtraction.
//
// Products run on m16n8k16 warp MMAs with 16 weight rows as M and 8 tokens as N. The sum over k
// does not depend on which k a fragment register holds, as long as A and B agree, so a thread
// takes its k's as consecutive words of the packed row (one 16-byte load per row for groups of
// 128) and its activations as the matching 16-byte loads: no reordering on either side. A
// group's products are summed in a fresh fp32 accumulator and scaled once, in fp32, so the only
// rounding to bf16 is the output's.
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

constexpr int kW4Warps = 8;
constexpr int kW4Rows = 16;   // weight rows per CTA (the MMA M)
constexpr int kW4Chunk = 128;  // k's a warp takes at a time
constexpr int kW4Batch = 2;   // chunks whose loads are issued before any is used

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

// Four bf16 pairs (q - z) of one packed word; zz = (128 + z, 128 + z).
__device__ __forceinline__ void w4_unpack(uint32_t w, uint32_t zz, uint32_t (&p)[4]) {
  const __nv_bfloat162 z2 = *reinterpret_cast<const __nv_bfloat162*>(&zz);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t v = ((w >> (4 * i)) & 0x000F000Fu) | 0x43004300u;
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), z2);
    p[i] = *reinterpret_cast<const uint32_t*>(&d);
  }
}

// One warp's share of the products of 16 weight rows (row0 ..) with 8 NT tokens (t0 ..): chunks
// first, first + step, ... of 128 k's, into acc (the MMA's C layout: rows lane / 4 and + 8,
// tokens 8 nt + 2 (lane % 4) and + 1).
template <int G, int NT>
__device__ __forceinline__ void w4_rows(const LinearW4Params& p, int row0, int t0, int first, int step,
                                        float (&acc)[NT][4]) {
  constexpr int WPG = G / 32;        // words of one group that a thread holds
  constexpr int GPC = kW4Chunk / G;  // groups per chunk
  const int lane = threadIdx.x & 31, g4 = lane >> 2, c4 = lane & 3;
  const int chunks = (p.k + kW4Chunk - 1) / kW4Chunk, words = p.k / 8;
  const int ra = row0 + g4, rb = ra + 8;
  const bool ok_a = ra < p.n, ok_b = rb < p.n;
  const uint32_t* wa = p.packed + static_cast<int64_t>(ok_a ? ra : 0) * words;
  const uint32_t* wb = p.packed + static_cast<int64_t>(ok_b ? rb : 0) * words;
  for (int c0 = first; c0 < chunks; c0 += step * kW4Batch) {
    uint32_t qa[kW4Batch][4], qb[kW4Batch][4];
    float sa[kW4Batch][GPC], sb[kW4Batch][GPC];
    uint32_t za[kW4Batch][GPC], zb[kW4Batch][GPC];
#pragma unroll
    for (int b = 0; b < kW4Batch; ++b) {
      const int c = c0 + b * step;
#pragma unroll
      for (int gi = 0; gi < GPC; ++gi) {
        const int k0 = c * kW4Chunk + gi * G;
        const bool in = k0 < p.k;  // k is a multiple of G: a group is there whole or not at all
        const int word = k0 / 8 + c4 * WPG;
        sa[b][gi] = sb[b][gi] = 0.f;
        za[b][gi] = zb[b][gi] = 0x43084308u;
#pragma unroll
        for (int i = 0; i < WPG; ++i) qa[b][gi * WPG + i] = qb[b][gi * WPG + i] = 0u;
        if (in && ok_a) {
          if constexpr (WPG == 4) {
            *reinterpret_cast<uint4*>(&qa[b][0]) = __ldg(reinterpret_cast<const uint4*>(wa + word));
          } else if constexpr (WPG == 2) {
            *reinterpret_cast<uint2*>(&qa[b][gi * 2]) = __ldg(reinterpret_cast<const uint2*>(wa + word));
          } else {
            qa[b][gi] = __ldg(wa + word);
          }
        }
        if (in && ok_b) {
          if constexpr (WPG == 4) {
            *reinterpret_cast<uint4*>(&qb[b][0]) = __ldg(reinterpret_cast<const uint4*>(wb + word));
          } else if constexpr (WPG == 2) {
            *reinterpret_cast<uint2*>(&qb[b][gi * 2]) = __ldg(reinterpret_cast<const uint2*>(wb + word));
          } else {
            qb[b][gi] = __ldg(wb + word);
          }
        }
        if (in) {
          const int64_t at = static_cast<int64_t>(k0 / G) * p.n;
          if (ok_a) sa[b][gi] = __bfloat162float(p.scales[at + ra]);
          if (ok_b) sb[b][gi] = __bfloat162float(p.scales[at + rb]);
          if (p.zeros != nullptr) {
            if (ok_a) za[b][gi] = (0x4300u | (p.zeros[at + ra] & 15u)) * 0x00010001u;
            if (ok_b) zb[b][gi] = (0x4300u | (p.zeros[at + rb] & 15u)) * 0x00010001u;
          }
        }
      }
    }
#pragma unroll
    for (int b = 0; b < kW4Batch; ++b) {
      const int c = c0 + b * step;
      if (c >= chunks) break;
#pragma unroll
      for (int gi = 0; gi < GPC; ++gi) {
        const int k0 = c * kW4Chunk + gi * G + c4 * 8 * WPG;
        float part[NT][4];
#pragma unroll
        for (int t = 0; t < NT; ++t) part[t][0] = part[t][1] = part[t][2] = part[t][3] = 0.f;
#pragma unroll
        for (int i = 0; i < WPG; ++i) {
          uint32_t pa[4], pb[4];
          w4_unpack(qa[b][gi * WPG + i], za[b][gi], pa);
          w4_unpack(qb[b][gi * WPG + i], zb[b][gi], pb);
          const uint32_t a0[4] = {pa[0], pb[0], pa[1], pb[1]}, a1[4] = {pa[2], pb[2], pa[3], pb[3]};
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            const int token = t0 + 8 * t + g4, k = k0 + 8 * i;
            uint4 xv = make_uint4(0, 0, 0, 0);
            if (token < p.m && k < p.k) xv = *reinterpret_cast<const uint4*>(p.x + token * p.x_stride + k);
            mma_16816(part[t], a0, xv.x, xv.y);
            mma_16816(part[t], a1, xv.z, xv.w);
          }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          acc[t][0] += sa[b][gi] * part[t][0];
          acc[t][1] += sa[b][gi] * part[t][1];
          acc[t][2] += sb[b][gi] * part[t][2];
          acc[t][3] += sb[b][gi] * part[t][3];
        }
      }
    }
  }
}

// Grid (cluster of K splits, row tiles, token tiles). The chunks of a row go round the cluster's
// warps; a CTA sums its warps' parts in warp order, rank 0 the CTAs' in rank order (from their
// shared memory), so results do not depend on timing.
template <int G, int NT>
__global__ void __launch_bounds__(32 * kW4Warps) linear_w4_kernel(LinearW4Params p) {
  __shared__ float parts[kW4Warps][NT * 8][kW4Rows];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g4 = lane >> 2, c4 = lane & 3;
  const int splits = static_cast<int>(cluster_size()), rank = static_cast<int>(cluster_rank());
  const int row0 = blockIdx.y * kW4Rows, t0 = blockIdx.z * (8 * NT);
  float acc[NT][4];
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t][0] = acc[t][1] = acc[t][2] = acc[t][3] = 0.f;
  w4_rows<G, NT>(p, row0, t0, rank * kW4Warps + warp, splits * kW4Warps, acc);
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    parts[warp][8 * t + 2 * c4][g4] = acc[t][0];
    parts[warp][8 * t + 2 * c4 + 1][g4] = acc[t][1];
    parts[warp][8 * t + 2 * c4][g4 + 8] = acc[t][2];
    parts[warp][8 * t + 2 * c4 + 1][g4 + 8] = acc[t][3];
  }
  __syncthreads();
  constexpr int kOut = NT * 8 * kW4Rows;
  float* mine = &parts[0][0][0];
  for (int i = threadIdx.x; i < kOut; i += 32 * kW4Warps) {
    float s = mine[i];
#pragma unroll
    for (int w = 1; w < kW4Warps; ++w) s += mine[w * kOut + i];
    mine[i] = s;
  }
  if (splits > 1) cluster_sync();
  else __syncthreads();
  if (rank == 0) {
    for (int i = threadIdx.x; i < kOut; i += 32 * kW4Warps) {
      const int token = t0 + i / kW4Rows, row = row0 + i % kW4Rows;
      float s = mine[i];
      for (int r = 1; r < splits; ++r) s += cluster_load(mine + i, r);
      if (token < p.m && row < p.n) p.out[static_cast<int64_t>(token) * p.n + row] = __float2bfloat16_rn(s);
    }
  }
  if (splits > 1) cluster_sync();  // the other CTAs' shared memory stays until rank 0 has read it
}

}  // namespace hb
