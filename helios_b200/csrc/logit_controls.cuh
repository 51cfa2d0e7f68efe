// Request controls on logits ahead of the sampler: penalties for tokens a request already
// holds, a sparse list of biases, and a grammar mask.
//
// For row r with history h (its request's prompt, then the tokens it has produced):
//   x = logit, in fp32
//   x = x > 0 ? x / repetition : x * repetition      where the token occurs in h
//   x = x - frequency * c                            c = its occurrences past the prompt
//   x = x - presence                                 where c > 0
//   x = x + bias                                     where the row's list has the token
//   x = -inf                                         where the row's mask does not allow it
// each step rounded to fp32 (no contraction), the result once to bf16.
//
// One cluster of CTAs per row, each CTA owning a contiguous segment of the vocabulary with one
// 32-bit word per token in shared memory: bit 31 says that the prompt holds the token, the rest
// counts its produced occurrences. The cluster reads the history once, spread over its threads,
// and each entry becomes one integer atomic on the owning CTA's word (distributed shared
// memory), so counts are exact whatever the order. Every CTA then streams its segment: 16 bytes
// of logits and two 16-byte reads of words at a time. Biased tokens are marked in a bitmap,
// passed over by the stream and done one thread per list entry.
#pragma once

#include "linear_w4.cuh"

namespace hb {

struct LogitControlParams {
  const __nv_bfloat16* in;
  __nv_bfloat16* out;
  int64_t in_stride, out_stride;  // elements per row
  int32_t rows, vocab;
  const float *repetition, *frequency, *presence;  // [rows], each may be null (1, 0, 0)
  const int32_t* history;  // [arena_rows, arena_width] or null
  int64_t arena_width;
  int32_t arena_rows;
  const int32_t* slots;           // [rows]: the row's history, -1 for none
  const int32_t* lengths;         // [arena_rows]
  const int32_t* prompt_lengths;  // [arena_rows]
  const int32_t* bias_offsets;    // [rows + 1] or null
  const int32_t* bias_tokens;     // ascending within a row
  const float* bias_values;
  int32_t bias_entries;
  const uint32_t* mask;  // [masks, mask_words] or null
  int32_t masks, mask_words;
  const int32_t* mask_rows;  // [rows]: the row's mask, -1 for none
  int32_t segment;           // tokens per CTA and pass, a multiple of 32
};

constexpr int kControlThreads = 512;
constexpr int kControlMaxSegment = 19456;  // 76 KB of words: two CTAs per SM

__device__ __forceinline__ void cluster_add(uint32_t* local, uint32_t rank, uint32_t v) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(local)), "r"(rank));
  asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory");
}
__device__ __forceinline__ void cluster_or(uint32_t* local, uint32_t rank, uint32_t v) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(local)), "r"(rank));
  asm volatile("red.relaxed.cluster.shared::cluster.or.b32 [%0], %1;" ::"r"(a), "r"(v) : "memory");
}

struct RowControls {
  float repetition, frequency, presence;
};

// The formula above up to the bias; `word` as the shared-memory words hold it.
__device__ __forceinline__ float penalised(float x, uint32_t word, const RowControls& rc) {
  if (word == 0u) return x;
  x = x > 0.f ? __fdiv_rn(x, rc.repetition) : __fmul_rn(x, rc.repetition);
  const uint32_t count = word & 0x7FFFFFFFu;
  if (count) x = __fsub_rn(__fsub_rn(x, __fmul_rn(rc.frequency, static_cast<float>(count))), rc.presence);
  return x;
}

__global__ void __launch_bounds__(kControlThreads, 2) logit_controls_kernel(LogitControlParams p) {
  extern __shared__ __align__(16) uint32_t control_smem[];
  uint32_t* words = control_smem;                   // [segment]
  uint32_t* biased = control_smem + p.segment;      // [segment / 32]
  const int tid = threadIdx.x, row = blockIdx.y;
  const int ranks = static_cast<int>(cluster_size()), rank = static_cast<int>(cluster_rank());
  const __nv_bfloat16* in = p.in + row * p.in_stride;
  __nv_bfloat16* out = p.out + row * p.out_stride;

  RowControls rc{1.f, 0.f, 0.f};
  if (p.repetition) rc.repetition = p.repetition[row];
  if (p.frequency) rc.frequency = p.frequency[row];
  if (p.presence) rc.presence = p.presence[row];
  // Row-uniform, and so the same in every CTA of the cluster.
  const int32_t* hist = nullptr;
  int hist_len = 0, prompt_len = 0;
  if (p.history != nullptr && (rc.repetition != 1.f || rc.frequency != 0.f || rc.presence != 0.f)) {
    const int slot = p.slots[row];
    if (slot >= 0 && slot < p.arena_rows) {
      hist = p.history + slot * p.arena_width;
      hist_len = static_cast<int>(max(int64_t(0), min(int64_t(p.lengths[slot]), p.arena_width)));
      prompt_len = p.prompt_lengths[slot];
    } else if (slot != -1 && tid == 0 && rank == 0) {
      raise_status(kStatusBadRow);
    }
  }
  const uint32_t* mask = nullptr;
  if (p.mask != nullptr) {
    const int which = p.mask_rows[row];
    if (which >= 0 && which < p.masks) mask = p.mask + static_cast<int64_t>(which) * p.mask_words;
    else if (which != -1 && tid == 0 && rank == 0) raise_status(kStatusBadRow);
  }
  int bias0 = 0, bias1 = 0;
  if (p.bias_offsets != nullptr) {
    bias0 = p.bias_offsets[row];
    bias1 = p.bias_offsets[row + 1];
    if (bias0 < 0 || bias1 < bias0 || bias1 > p.bias_entries) {
      if (tid == 0 && rank == 0) raise_status(kStatusBadRow);
      bias0 = bias1 = 0;
    }
  }
  const bool vec = ((reinterpret_cast<uintptr_t>(in) | reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  const bool in_place = in == out;

  const int64_t per_pass = static_cast<int64_t>(ranks) * p.segment;
  for (int64_t pass0 = 0; pass0 < p.vocab; pass0 += per_pass) {
    const int64_t first = pass0 + static_cast<int64_t>(rank) * p.segment;  // this CTA's tokens
    const int n = static_cast<int>(max(int64_t(0), min(int64_t(p.segment), p.vocab - first)));
    if (hist_len > 0)
      for (int i = tid; i < p.segment / 4; i += kControlThreads) reinterpret_cast<uint4*>(words)[i] = make_uint4(0, 0, 0, 0);
    if (bias1 > bias0)
      for (int i = tid; i < p.segment / 32; i += kControlThreads) biased[i] = 0u;
    if (hist_len > 0) {
      if (ranks > 1) cluster_sync();  // every CTA's words are zero
      else __syncthreads();
      for (int i = rank * kControlThreads + tid; i < hist_len; i += ranks * kControlThreads) {
        const int token = hist[i];
        if (token < 0 || token >= p.vocab) {
          raise_status(kStatusBadToken);
          continue;
        }
        const int64_t at = token - pass0;
        if (at < 0 || at >= per_pass) continue;
        const uint32_t owner = static_cast<uint32_t>(at) / static_cast<uint32_t>(p.segment);
        uint32_t* word = words + (static_cast<uint32_t>(at) - owner * static_cast<uint32_t>(p.segment));
        if (i < prompt_len) cluster_or(word, owner, 0x80000000u);
        else cluster_add(word, owner, 1u);
      }
      if (ranks > 1) cluster_sync();
      else __syncthreads();
    } else if (bias1 > bias0) {
      __syncthreads();
    }
    // A list entry counts when its token is below the next entry's: ascending lists count whole,
    // of equal neighbours the last one does.
    for (int j = bias0 + tid; j < bias1; j += kControlThreads) {
      const int token = p.bias_tokens[j];
      const bool ordered = j + 1 >= bias1 || token <= p.bias_tokens[j + 1];
      if (token < 0 || token >= p.vocab || !ordered) {
        if (rank == 0) raise_status(kStatusBadToken);
        continue;
      }
      const int64_t at = token - first;
      if (at >= 0 && at < n) atomicOr(&biased[at >> 5], 1u << (at & 31));
    }
    if (bias1 > bias0) __syncthreads();

    if (vec) {
      for (int i = 8 * tid; i < n; i += 8 * kControlThreads) {
        uint32_t w[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        uint32_t any = 0;
        if (hist_len > 0) {
          *reinterpret_cast<uint4*>(&w[0]) = *reinterpret_cast<const uint4*>(words + i);
          *reinterpret_cast<uint4*>(&w[4]) = *reinterpret_cast<const uint4*>(words + i + 4);
#pragma unroll
          for (int e = 0; e < 8; ++e) any |= w[e];
        }
        uint32_t banned = 0;
        if (mask) banned = ~(mask[(first + i) >> 5] >> ((first + i) & 31)) & 0xFFu;
        if (in_place && any == 0u && banned == 0u) continue;
        const uint32_t skip = bias1 > bias0 ? (biased[i >> 5] >> (i & 31)) & 0xFFu : 0u;
        if (n - i >= 8 && skip == 0u) {
          const uint4 v = *reinterpret_cast<const uint4*>(in + first + i);
          float f[8];
          unpack8(v, f);
          if (any) {
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = penalised(f[e], w[e], rc);
          }
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if ((banned >> e) & 1u) f[e] = -INFINITY;
          *reinterpret_cast<uint4*>(out + first + i) = pack8(f);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {  // unrolled: w stays in registers
            if (e >= n - i || ((skip >> e) & 1u)) continue;
            float x = penalised(__bfloat162float(in[first + i + e]), w[e], rc);
            if ((banned >> e) & 1u) x = -INFINITY;
            out[first + i + e] = __float2bfloat16_rn(x);
          }
        }
      }
    } else {
      for (int i = tid; i < n; i += kControlThreads) {
        const uint32_t word = hist_len > 0 ? words[i] : 0u;
        const bool banned = mask && !((mask[(first + i) >> 5] >> ((first + i) & 31)) & 1u);
        if (in_place && word == 0u && !banned) continue;
        if (bias1 > bias0 && ((biased[i >> 5] >> (i & 31)) & 1u)) continue;
        const float x = banned ? -INFINITY : penalised(__bfloat162float(in[first + i]), word, rc);
        out[first + i] = __float2bfloat16_rn(x);
      }
    }
    for (int j = bias0 + tid; j < bias1; j += kControlThreads) {
      const int token = p.bias_tokens[j];
      const int64_t at = token - first;
      if (at < 0 || at >= n || (j + 1 < bias1 && token >= p.bias_tokens[j + 1])) continue;
      const bool banned = mask && !((mask[token >> 5] >> (token & 31)) & 1u);
      const float x = penalised(__bfloat162float(in[token]), hist_len > 0 ? words[at] : 0u, rc);
      out[token] = __float2bfloat16_rn(banned ? -INFINITY : __fadd_rn(x, p.bias_values[j]));
    }
    if (pass0 + per_pass < p.vocab) {  // the words are zeroed again
      if (ranks > 1) cluster_sync();
      else __syncthreads();
    }
  }
}

}  // namespace hb
