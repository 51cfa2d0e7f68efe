// Projections with 4-bit weights for more token rows than a warp MMA serves well: tcgen05.
//
// Formula and storage: linear_w4.cuh. The MMA's M is 128 weight rows, its N the tokens of a
// tile (NT = 64 or 128). The codes become bf16 values q - z, exactly, on the way into tensor
// memory, where the MMA reads them as its A operand; the activations come by TMA as its B
// operand. Group scales are applied to the products, not to the weights: each group of k's has
// an accumulator of its own (two in turn), which other warps multiply by the row's scale and add
// to fp32 registers while the next group's MMAs run. So the output's rounding to bf16 is the only
// one, at the cost of one fp32 FMA per output and group.
//
//   warp 0         TMA of the activations: per step of 128 k's two [NT tokens x 64 k] boxes
//   warps 1, 3     issue the MMAs, eight of K 16 per step, taking steps in turn; tensor memory
//   warp 2         TMA of the packed weights: [128 rows x 256 k] boxes of 16 KB; scales and zero
//                  points into shared memory, eight groups at a time
//   warps 4..11    unpack: thread = weight row (TMEM lane), two warps per lane quadrant taking
//                  steps in turn
//   warps 12..19   scale and add: thread = weight row and half of the tokens; then the output
//
// The issuing warp is the narrow place: it shares its scheduler with four busy warps, and each
// completed wait it made cost it 200 cycles, four MMAs' time. So a step is as long as tensor
// memory allows, it starts on one barrier that the activations' bytes, the unpacked A operand
// and the drained accumulators all arrive on, and its one commit frees the operands and hands
// over the accumulators. The packed boxes and the scales have rings of their own, deep enough to
// cover HBM latency. CTAs walk tiles with the token tiles fastest (a
// weight tile is read from HBM once and then from L2). With few weight rows a cluster splits k;
// its CTAs exchange their fp32 parts through shared memory and sum them in rank order.
//
// Measured, weights from DRAM, groups of 128 (us at 64, 512 and 2048 tokens): 6144 x 2560 11.3, 29, 74;
// 2560 x 4096 9.9, 26, 54; 19456 x 2560 22.8, 62, 220 (928 TFLOP/s, 0.57 of the measured bf16 rate);
// 2560 x 9728 13.9, 43, 118. At 64 tokens some 5 us are start and end (launch, first bytes, the first
// step through all warps, the sum over a cluster) and a step of 128 k's takes 0.55 us: 730 issue slots
// of every scheduler, and waits. Fewer MMAs, no reads of the accumulators or activations twice as far
// ahead changed nothing there; unpacking without its arithmetic would take 0.47. At 64 tokens the
// bf16 weights' cuBLAS products are as fast; what 4 bits save there is memory.
#pragma once

#include "fused_gemm.cuh"
#include "linear_w4.cuh"

namespace hb {

struct GemmW4Params {
  const __nv_bfloat16* scales;  // [k / G, n]
  const uint8_t* zeros;         // [k / G, n] or null
  __nv_bfloat16* out;           // [m, n]
  int32_t m, n, k, tiles_m;  // token tiles
  int32_t tile0, tiles;      // of the tiles in order (token tiles fastest), the first and the number of this launch
};

constexpr int kW4gRows = 128;
constexpr int kW4gUnpackWarps = 8;
constexpr int kW4gAddWarps = 8;
constexpr int kW4gFirstUnpack = 4, kW4gFirstAdd = kW4gFirstUnpack + kW4gUnpackWarps;
constexpr int kW4gThreads = 32 * (kW4gFirstAdd + kW4gAddWarps);
constexpr int kW4gStepK = 128;
constexpr int kW4gBoxK = 64;                             // k's per activation box (128 swizzled bytes)
constexpr int kW4gPackedK = 256;                         // k's per packed box
constexpr int kW4gPackedStages = 4;
constexpr uint32_t kW4gPackedBytes = kW4gRows * kW4gPackedK / 2;  // 16 KB
constexpr int kW4gStages = 4;                            // steps in flight: activations and A operand
constexpr int kW4gACols = kW4gStepK / 2;                 // tensor-memory columns of a step's A operand
constexpr uint32_t kW4gTmemCols = 512;
constexpr int kW4gScaleGroups = 8;                       // groups per batch of scales
constexpr int kW4gScaleStages = 3;

template <int NT>
struct GemmW4Shape {
  static constexpr uint32_t kBoxBytes = NT * 128;
  static constexpr uint32_t kXBytes = 2 * kBoxBytes;
  static constexpr int kAccs = 256 / NT;  // accumulators: half of tensor memory, A has the other
  static constexpr uint32_t kSmem = kW4gPackedStages * kW4gPackedBytes + kW4gStages * kXBytes + 1024;
  static_assert(256 + kW4gACols * kW4gStages <= static_cast<int>(kW4gTmemCols), "accumulators and A in tensor memory");
  static_assert(NT * kW4gRows * 4 <= kW4gPackedStages * kW4gPackedBytes, "the fp32 part fits the packed ring");
};

// a0 += s v0 and a1 += s v1, each rounded once, in one instruction.
__device__ __forceinline__ void fma_pair(float& a0, float& a1, float s, float v0, float v1) {
  asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %2};\n\tmov.b64 c, {%3, %4};\n\t"
      "fma.rn.f32x2 a, b, c, a;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "+f"(a0), "+f"(a1)
      : "f"(s), "f"(v0), "f"(v1));
}

template <int G, int NT>
__global__ void __launch_bounds__(kW4gThreads, 1) gemm_w4_kernel(GemmW4Params p, const __grid_constant__ CUtensorMap xmap,
                                                                 const __grid_constant__ CUtensorMap wmap) {
  using Shape = GemmW4Shape<NT>;
  constexpr int S = kW4gStages, SP = kW4gPackedStages;
  constexpr int kGroupMmas = G / 16;                  // MMAs (16 k's each) per group
  constexpr int kStepMmas = kW4gStepK / 16;
  constexpr int GPS = kW4gStepK / G;                  // groups per step, one accumulator each
  constexpr int kLag = Shape::kAccs / GPS;            // steps until a step's accumulators come round again
  static_assert(kLag >= 1 && S % kLag == 0, "a step's accumulators");
  // An issuing warp looks at the barrier of its next step, two on, while that step's predecessor there
  // (S earlier) may count as its phase only if it is complete: one of the warp's own steps before this.
  static_assert(S % 2 == 0 && S >= 4, "the barrier looked at ahead is at most one phase behind");
  extern __shared__ __align__(1024) uint8_t dsm[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dsm) + 1023) & ~uintptr_t(1023));
  uint8_t* packed = smem;
  uint8_t* xs = smem + SP * kW4gPackedBytes;
  __shared__ uint64_t full_p[SP], empty_p[SP], ready[S], done[S], full_s[kW4gScaleStages], empty_s[kW4gScaleStages], drain_bar[2];
  __shared__ __nv_bfloat16 scale_s[kW4gScaleStages][kW4gScaleGroups][kW4gRows];
  __shared__ uint8_t zero_s[kW4gScaleStages][kW4gScaleGroups][kW4gRows];
  __shared__ uint32_t tmem_base_s;
  __shared__ int abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int splits = static_cast<int>(cluster_size()), rank = static_cast<int>(cluster_rank());
  const int tiles = p.tile0 + p.tiles;  // their end
  const int first_tile = p.tile0 + static_cast<int>(blockIdx.x) / splits, tile_step = static_cast<int>(gridDim.x) / splits;
  // This CTA's k's: whole units of 128, up to k's end.
  const int units = (p.k + 127) / 128;
  const int k0 = 128 * (units * rank / splits), k1 = min(p.k, 128 * (units * (rank + 1) / splits));
  const int steps = (k1 - k0 + kW4gStepK - 1) / kW4gStepK;
  const int groups = (k1 - k0) / G;
  const int batches = (groups + kW4gScaleGroups - 1) / kW4gScaleGroups;

  if (threadIdx.x == 0) {
    for (int s = 0; s < SP; ++s) {
      mbar_init(&full_p[s], 1);
      mbar_init(&empty_p[s], kW4gUnpackWarps);  // both warps of a quadrant: each takes one step of a box
    }
    for (int s = 0; s < S; ++s) {
      // The activations' producer (and their bytes), a warp per quadrant of A, the drained sums.
      mbar_init(&ready[s], 1 + kW4gUnpackWarps / 2 + kW4gAddWarps);
      mbar_init(&done[s], 1);
    }
    for (int s = 0; s < kW4gScaleStages; ++s) {
      mbar_init(&full_s[s], 1);
      mbar_init(&empty_s[s], kW4gAddWarps + (p.zeros != nullptr ? kW4gUnpackWarps : 0));
    }
    mbar_init(&drain_bar[0], 1);
    mbar_init(&drain_bar[1], 1);
    abort_flag = 0;
    fence_barrier_init();
  }
  // Tensor memory is taken after the kernel ahead has ended, which may still have had to take its own,
  // and before the kernel behind may start. (A launch for the remaining tiles starts after the first
  // one's wait here, and its CTAs find room only where that one's have left.)
  if (p.tile0 == 0) pdl_wait();
  if (warp == 1) {
    tmem_alloc(&tmem_base_s, kW4gTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_s;
  const uint32_t tmem_a = tmem + 256;
  pdl_trigger();

  float acc[NT / 2];
  if (warp == 0) {
    // ------------------------------------------------------------ activations
    if (lane == 0) {
      tma_prefetch_desc(&xmap);
      int it = 0;
      bool ok = true;
      for (int t = first_tile; ok && t < tiles; t += tile_step) {
        const int m0 = (t % p.tiles_m) * NT;
        for (int s = 0; s < steps; ++s, ++it) {
          const int st = it % S;
          if (it >= S && !mbar_wait(&done[st], ((it / S) - 1) & 1, &abort_flag)) {
            ok = false;
            break;
          }
          mbar_expect_tx(&ready[st], Shape::kXBytes);
          uint8_t* dst = xs + st * Shape::kXBytes;
          const int k = k0 + s * kW4gStepK;
          tma_load_2d(dst, &xmap, &ready[st], k, m0);
          tma_load_2d(dst + Shape::kBoxBytes, &xmap, &ready[st], k + kW4gBoxK, m0);  // zeros past k's end
        }
      }
      // A step's operands were waited for by its MMAs; after an abort its barrier may stay open, so
      // the boxes in flight are given the time limit to land.
      for (int j = max(0, it - S); j < it; ++j) mbar_drain(&done[j % S], (j / S) & 1);
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------ scales, zero points, packed weights
    // A batch of scales, then the boxes it belongs to: neither waits for the other's consumers
    // longer than the rings are deep.
    constexpr int kBatchK = kW4gScaleGroups * G;
    static_assert(kBatchK % kW4gPackedK == 0, "whole boxes per batch");
    auto box = [&](int i, int k, int n0) {  // the i-th box of this CTA
      mbar_expect_tx(&full_p[i % SP], kW4gPackedBytes);
      tma_load_2d(packed + (i % SP) * kW4gPackedBytes, &wmap, &full_p[i % SP], k / 8, n0);
    };
    int ib = 0, it = 0;
    bool ok = true;
    int early = 0;  // boxes of the first tile that fill the ring before its scales are read
    if (lane == 0 && first_tile < tiles)
      for (; early < SP && k0 + early * kW4gPackedK < k1; ++early)
        box(early, k0 + early * kW4gPackedK, (first_tile / p.tiles_m) * kW4gRows);
    for (int t = first_tile; ok && t < tiles; t += tile_step) {
      const int n0 = (t / p.tiles_m) * kW4gRows;
      for (int b = 0; ok && b < batches; ++b, ++ib) {
        const int st = ib % kW4gScaleStages;
        ok = ib < kW4gScaleStages || mbar_wait(&empty_s[st], ((ib / kW4gScaleStages) - 1) & 1, &abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const int g0 = k0 / G + b * kW4gScaleGroups, n_groups = min(kW4gScaleGroups, groups - b * kW4gScaleGroups);
#pragma unroll
        for (int q = 0; q < kW4gRows / 32; ++q) {
          const int row = min(n0 + 32 * q + lane, p.n - 1);
          __nv_bfloat16 s[kW4gScaleGroups];
          uint8_t z[kW4gScaleGroups];
#pragma unroll
          for (int g = 0; g < kW4gScaleGroups; ++g) {
            const int64_t at = static_cast<int64_t>(g0 + min(g, n_groups - 1)) * p.n + row;
            s[g] = p.scales[at];
            z[g] = p.zeros != nullptr ? p.zeros[at] : 8;
          }
#pragma unroll
          for (int g = 0; g < kW4gScaleGroups; ++g) {
            scale_s[st][g][32 * q + lane] = s[g];
            zero_s[st][g][32 * q + lane] = z[g];
          }
        }
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&full_s[st]);
          const int end = min(k1, k0 + (b + 1) * kBatchK);
          for (int k = k0 + b * kBatchK; k < end; k += kW4gPackedK, ++it) {
            if (it < early) continue;
            if (it >= SP && !mbar_wait(&empty_p[it % SP], ((it / SP) - 1) & 1, &abort_flag)) {
              ok = false;
              break;
            }
            box(it, k, n0);
          }
        }
        ok = __all_sync(0xffffffffu, ok);
      }
    }
    if (lane == 0) {
      it = max(it, early);
      for (int j = max(0, it - SP); j < it; ++j) mbar_drain(&full_p[j % SP], (j / SP) & 1);
    }
    __syncwarp();
  } else if (warp == 1 || warp == 3) {
    // ------------------------------------------------------------ MMA issue (converged warps)
    constexpr uint32_t idesc = idesc_bf16(kW4gRows, NT, false, false);
    const uint64_t desc0 = smem_desc(smem_u32(xs), 16, 1024, kSwizzle128B);
    const int mine = first_tile < tiles ? (tiles - first_tile + tile_step - 1) / tile_step : 0;
    const int total = mine * steps;  // steps of all this CTA's tiles
    const int turn = warp == 1 ? 0 : 1;
    bool seen = false;               // the step's barrier was found complete during the step before
#pragma unroll 1
    for (int it = turn; it < total; it += 2) {
      const int st = it % S;
      if (!seen && !mbar_wait_fast(&ready[st], (it / S) & 1, &abort_flag)) break;
      tc_fence_after();
      seen = mbar_poll(&ready[(it + 2) % S], ((it + 2) / S) & 1);
      const uint64_t b = desc0 + static_cast<uint64_t>((st * Shape::kXBytes) >> 4);
      const uint32_t a = tmem_a + kW4gACols * st;
      const uint32_t d = tmem + (it % kLag) * (GPS * NT);
      // Past k's end the codes and activations are zeros: whole groups of them, never added.
#pragma unroll
      for (int j = 0; j < kStepMmas; ++j)
        mma_ts_warp(d + (j / kGroupMmas) * NT, a + 8 * j,
                    b + (j / 4) * static_cast<uint64_t>(Shape::kBoxBytes >> 4) + 2 * (j % 4), idesc,
                    j % kGroupMmas != 0 ? 1u : 0u);
      mma_commit_warp(&done[st]);
    }
    mma_commit_warp(&drain_bar[turn]);  // nothing may still write tensor memory when it is freed
    mbar_drain(&drain_bar[turn], 0);
  } else if (warp >= kW4gFirstUnpack && warp < kW4gFirstAdd) {
    // ------------------------------------------------------------ codes -> bf16 A operand
    const int quad = warp & 3, r = quad * 32 + lane, turn = (warp - kW4gFirstUnpack) >> 2;
    const uint32_t lane_base = static_cast<uint32_t>(quad * 32) << 16;
    int it = 0, ip = 0, ib = 0;
    bool ok = true;
    for (int t = first_tile; ok && t < tiles; t += tile_step) {
      // This warp's steps: s with s % 2 == turn, the turn-th half of each packed box.
      int batch = -1;  // of the tile's scale batches, the one this warp holds (with zero points)
      auto hold_batch = [&](int b) {
        while (ok && batch < b) {
          __syncwarp();
          if (batch >= 0 && lane == 0) mbar_arrive(&empty_s[(ib + batch) % kW4gScaleStages]);
          ++batch;
          ok = mbar_wait_fast(&full_s[(ib + batch) % kW4gScaleStages], ((ib + batch) / kW4gScaleStages) & 1, &abort_flag);
        }
      };
      for (int s0 = 0; s0 < steps; s0 += 2, ++ip) {
        const int s = s0 + turn, sp = ip % SP, st = (it + s) % S, round = (it + s) / S;
        const bool mine = s < steps;  // the box's second half may lie past the end
        uint32_t zz[GPS];
#pragma unroll
        for (int h = 0; h < GPS; ++h) zz[h] = 0x43084308u;
        if (p.zeros != nullptr && mine) {
          hold_batch(s * GPS / kW4gScaleGroups);
          if (!ok) break;
#pragma unroll
          for (int h = 0; h < GPS; ++h)
            zz[h] = (0x4300u | (zero_s[(ib + batch) % kW4gScaleStages][(s * GPS + h) % kW4gScaleGroups][r] & 15u)) * 0x00010001u;
        }
        ok = mbar_wait_fast(&full_p[sp], (ip / SP) & 1, &abort_flag) &&
             (!mine || round == 0 || mbar_wait_fast(&done[st], (round - 1) & 1, &abort_flag));
        if (!ok) break;
        if (mine) {
          tc_fence_after();
          const uint8_t* src = packed + sp * kW4gPackedBytes;
          uint4 w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = *reinterpret_cast<const uint4*>(src + sw128(r, 4 * turn + i));
#pragma unroll
          for (int i = 0; i < 4; i += 2) {  // 64 k's at a time
            uint32_t a[32];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t c[4] = {w[i + e].x, w[i + e].y, w[i + e].z, w[i + e].w};
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                uint32_t v[4];
                w4_unpack(c[j], zz[(i + e) * GPS / 4], v);
#pragma unroll
                for (int q = 0; q < 4; ++q) a[16 * e + 4 * j + q] = v[q];
              }
            }
            tmem_st32u(tmem_a + kW4gACols * st + 16 * i + lane_base, a);
          }
          tmem_wait_st();
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) {
          if (mine) mbar_arrive(&ready[st]);
          mbar_arrive(&empty_p[sp]);
        }
      }
      it += steps;
      if (p.zeros != nullptr) {  // every batch of the tile is waited for and released once
        hold_batch(batches - 1);
        __syncwarp();
        if (ok && lane == 0) mbar_arrive(&empty_s[(ib + batch) % kW4gScaleStages]);
        ib += batches;
      }
    }
  } else if (warp >= kW4gFirstAdd) {
    // ------------------------------------------------------------ scale and add
    const int half = (warp - kW4gFirstAdd) >> 2, r = (warp & 3) * 32 + lane;
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    int it = 0, ib = 0;
    bool ok = true;
    if (lane == 0)
      for (int s = 0; s < kLag; ++s) mbar_arrive(&ready[s]);  // the first steps' accumulators are free
    for (int t = first_tile; ok && t < tiles; t += tile_step) {
      const int row = (t / p.tiles_m) * kW4gRows + r;
#pragma unroll
      for (int i = 0; i < NT / 2; ++i) acc[i] = 0.f;
      for (int s = 0; s < steps; ++s, ++it) {
        const int sb = ib % kW4gScaleStages, g0 = s * GPS;
        if (g0 % kW4gScaleGroups == 0) {
          ok = mbar_wait_fast(&full_s[sb], (ib / kW4gScaleStages) & 1, &abort_flag);
          if (!ok) break;
        }
        float scale[GPS];
#pragma unroll
        for (int h = 0; h < GPS; ++h) scale[h] = __bfloat162float(scale_s[sb][(g0 + h) % kW4gScaleGroups][r]);
        if ((g0 + GPS) % kW4gScaleGroups == 0 || s == steps - 1) {  // the batch is read
          __syncwarp();
          if (lane == 0) mbar_arrive(&empty_s[sb]);
          ++ib;
        }
        ok = mbar_wait_fast(&done[it % S], (it / S) & 1, &abort_flag);
        if (!ok) break;
        tc_fence_after();
        const uint32_t src = tmem + (it % kLag) * (GPS * NT) + half * (NT / 2) + lane_base;
#pragma unroll
        for (int h = 0; h < GPS; ++h) {
          if (GPS > 1 && g0 + h >= groups) break;
#pragma unroll
          for (int c = 0; c < NT / 32; ++c) {
            float v[16];
            tmem_ld16(src + h * NT + 16 * c, v);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; i += 2) fma_pair(acc[16 * c + i], acc[16 * c + i + 1], scale[h], v[i], v[i + 1]);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ready[(it + kLag) % S]);
      }
      if (splits == 1 && ok) {
        const int t0 = (t % p.tiles_m) * NT + half * (NT / 2);
        __nv_bfloat16* dst = p.out + static_cast<int64_t>(t0) * p.n + row;
        if (p.n % 2 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 3) == 0) {
          // Neighbouring lanes (rows) swap one value of each pair of tokens: the even lane stores
          // both rows of the first, the odd lane of the second. (n is even: a pair is in or out.)
          const bool odd = lane & 1;
          if (odd) dst += p.n - 1;
#pragma unroll
          for (int i = 0; i < NT / 2; i += 2) {
            const float other = __shfl_xor_sync(0xffffffffu, odd ? acc[i] : acc[i + 1], 1);
            const uint32_t v = odd ? pack_bf16(other, acc[i + 1]) : pack_bf16(acc[i], other);
            if (row < p.n && t0 + i + odd < p.m) *reinterpret_cast<uint32_t*>(dst) = v;
            dst += 2 * static_cast<int64_t>(p.n);
          }
        } else if (row < p.n) {
#pragma unroll
          for (int i = 0; i < NT / 2; ++i)
            if (t0 + i < p.m) dst[static_cast<int64_t>(i) * p.n] = __float2bfloat16_rn(acc[i]);
        }
      }
    }
  }
  if (splits > 1) {  // one tile per cluster
    __syncthreads();  // the packed ring is idle: it holds the parts
    float* part = reinterpret_cast<float*>(packed);  // [NT][128]
    if (warp >= kW4gFirstAdd) {
      const int half = (warp - kW4gFirstAdd) >> 2, r = (warp & 3) * 32 + lane;
#pragma unroll
      for (int i = 0; i < NT / 2; ++i) part[(half * (NT / 2) + i) * kW4gRows + r] = acc[i];
    }
    cluster_sync();
    const int n0 = (first_tile / p.tiles_m) * kW4gRows, t0 = (first_tile % p.tiles_m) * NT;
    for (int i = rank * kW4gThreads + static_cast<int>(threadIdx.x); i < NT * kW4gRows / 4; i += splits * kW4gThreads) {
      const int token = t0 + i / (kW4gRows / 4), row = n0 + 4 * (i % (kW4gRows / 4));
      if (token < p.m && row < p.n) {
        float4 v[8];
#pragma unroll
        for (int q = 0; q < 8; ++q)
          if (q < splits) v[q] = cluster_load4(part + 4 * i, q);
        float4 s = v[0];
#pragma unroll
        for (int q = 1; q < 8; ++q)
          if (q < splits) {
            s.x += v[q].x;
            s.y += v[q].y;
            s.z += v[q].z;
            s.w += v[q].w;
          }
        const float o[4] = {s.x, s.y, s.z, s.w};
        __nv_bfloat16* dst = p.out + static_cast<int64_t>(token) * p.n + row;
        if (p.n % 4 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 7) == 0) {
          *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3]));
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (row + e < p.n) dst[e] = __float2bfloat16_rn(o[e]);
        }
      }
    }
    cluster_sync();  // the parts stay until every CTA has read them
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kW4gTmemCols);
  }
  if (p.tile0 > 0) pdl_wait();  // the launch ahead (the other tiles, same inputs) completes before this one
}

}  // namespace hb
