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
// One CTA per row and segment of the vocabulary, with one 32-bit word per token of the segment in
// shared memory: occurrences in the prompt in its high half, past the prompt in its low half.
// Every CTA reads its row's whole history (from L2 after the first) and counts the tokens of its
// own segment with shared-memory integer atomics, so counts are exact whatever the order.
// (Counting each entry once, in the owning CTA of a cluster through distributed shared memory,
// took 107 us at 128 rows with histories of up to 16,000: frequent tokens have neighbouring ids,
// and their owner took the remote atomics one by one.) The words that are not zero then go on a
// list, and the penalties, with their division, are done one thread per listed token: done
// inside the stream they cost every warp that met one such token the arithmetic for all of its
// tokens. The stream itself is a copy with masked tokens replaced, 16 bytes at a time, asked for
// before the counting. Biased tokens are marked in a bitmap, passed over by the list and done
// one thread per entry.
#pragma once

#include <climits>

#include "hb_common.cuh"

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
  int32_t segment;           // tokens per CTA, a multiple of 32
};

constexpr int kControlThreads = 512;
constexpr int kControlGroups = 4;  // groups of 8 tokens per thread: a whole segment
constexpr int kControlMaxSegment = kControlGroups * 8 * kControlThreads;
constexpr int kControlMinSegment = 2048;
static_assert(kControlMaxSegment == 8 * 4 * kControlThreads && kControlMaxSegment <= 65536, "the touched list");
constexpr int kControlAhead = 4;   // 16-byte pieces of the history a thread loads before it counts any
constexpr int kControlMaxHistory = 65535;  // entries per row: the halves of a word cannot overflow

// Shared memory of a segment: words and touched list (with a history), bias bitmap (with biases).
__host__ __device__ inline int control_smem_bytes(int segment, bool history, bool bias) {
  return (history ? 6 * segment : 0) + (bias ? segment / 8 : 0);
}

struct RowControls {
  float repetition, frequency, presence;
};

// The formula above up to the bias; `word` as the shared-memory words hold it.
__device__ __forceinline__ float penalised(float x, uint32_t word, const RowControls& rc) {
  if (word == 0u) return x;
  x = x > 0.f ? __fdiv_rn(x, rc.repetition) : __fmul_rn(x, rc.repetition);
  const uint32_t count = word & 0xFFFFu;
  if (count) x = __fsub_rn(__fsub_rn(x, __fmul_rn(rc.frequency, static_cast<float>(count))), rc.presence);
  return x;
}

__global__ void __launch_bounds__(kControlThreads, 2) logit_controls_kernel(LogitControlParams p) {
  extern __shared__ __align__(16) uint32_t control_smem[];
  uint32_t* words = control_smem;                                               // [segment]
  uint16_t* touched = reinterpret_cast<uint16_t*>(control_smem + p.segment);    // [segment]
  uint32_t* biased = control_smem + (p.history != nullptr ? p.segment + p.segment / 2 : 0);  // [segment / 32]
  __shared__ int n_touched;
  const int tid = threadIdx.x, row = blockIdx.y;
  const bool first_cta = blockIdx.x == 0;  // reports what concerns the whole row
  const __nv_bfloat16* in = p.in + row * p.in_stride;
  __nv_bfloat16* out = p.out + row * p.out_stride;

  pdl_wait();  // the logits, from the kernel ahead
  pdl_trigger();
  const bool vec = ((reinterpret_cast<uintptr_t>(in) | reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  const bool in_place = in == out;

  const int first = blockIdx.x * p.segment;  // this CTA's tokens
  const int n = min(p.segment, p.vocab - first);
  // The logits are asked for first: they arrive while the row's settings are read, the words
  // zeroed and the history counted. (In place only touched logits are needed, or masked ones.)
  const bool eager = vec && !in_place;
  uint4 raw[kControlGroups];
#pragma unroll
  for (int u = 0; u < kControlGroups; ++u) {
    const int i = 8 * (tid + u * kControlThreads);
    if (eager && n - i >= 8) raw[u] = *reinterpret_cast<const uint4*>(in + first + i);
  }

  // The row's settings; the words and the bitmap are zeroed while they arrive.
  RowControls rc{1.f, 0.f, 0.f};
  if (p.repetition) rc.repetition = p.repetition[row];
  if (p.frequency) rc.frequency = p.frequency[row];
  if (p.presence) rc.presence = p.presence[row];
  const int slot = p.history != nullptr ? p.slots[row] : -1;
  const int which = p.mask != nullptr ? p.mask_rows[row] : -1;
  int bias0 = 0, bias1 = 0;
  if (p.bias_offsets != nullptr) {
    bias0 = p.bias_offsets[row];
    bias1 = p.bias_offsets[row + 1];
  }
  if (p.history != nullptr)
    for (int i = tid; i < p.segment / 4; i += kControlThreads) reinterpret_cast<uint4*>(words)[i] = make_uint4(0, 0, 0, 0);
  if (p.bias_offsets != nullptr)
    for (int i = tid; i < p.segment / 32; i += kControlThreads) biased[i] = 0u;
  if (tid == 0) n_touched = 0;

  if (bias0 < 0 || bias1 < bias0 || bias1 > p.bias_entries) {
    if (tid == 0 && first_cta) raise_status(kStatusBadRow);
    bias0 = bias1 = 0;
  }
  const uint32_t* mask = nullptr;
  if (which >= 0 && which < p.masks) mask = p.mask + static_cast<int64_t>(which) * p.mask_words;
  else if (which != -1 && tid == 0 && first_cta) raise_status(kStatusBadRow);
  uint32_t allowed[kControlGroups];
#pragma unroll
  for (int u = 0; u < kControlGroups; ++u) {
    const int i = 8 * (tid + u * kControlThreads);
    allowed[u] = mask != nullptr && vec && i < n ? reinterpret_cast<const uint8_t*>(mask)[(first + i) >> 3] : 0xFFu;
  }
  // The history in 16-byte pieces, with up to three entries before the first and after the last.
  // Its first pieces are read up to the arena's width, beside the row's length, not after it.
  const int32_t* hist = nullptr;
  int hist_len = 0, prompt_len = 0, lead = 0;
  int4 ahead[kControlAhead];
  if (slot >= 0 && slot < p.arena_rows) {
    if (rc.repetition != 1.f || rc.frequency != 0.f || rc.presence != 0.f) {
      hist = p.history + slot * p.arena_width;
      const int width = static_cast<int>(p.arena_width);
      lead = min(width, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(hist) & 15)) & 15) / 4);
#pragma unroll
      for (int u = 0; u < kControlAhead; ++u)
        if (tid + u * kControlThreads < (width - lead) / 4)
          ahead[u] = reinterpret_cast<const int4*>(hist + lead)[tid + u * kControlThreads];
      hist_len = max(0, min(p.lengths[slot], width));
      prompt_len = p.prompt_lengths[slot];
      lead = min(lead, hist_len);
    }
  } else if (slot != -1 && tid == 0 && first_cta) {
    raise_status(kStatusBadRow);
  }
  const int4* body = reinterpret_cast<const int4*>(hist + lead);
  const int pieces = (hist_len - lead) / 4;
  // A thread's first list entry.
  const int j0 = bias0 + tid;
  int bias_token = 0, bias_next = INT_MAX;
  float bias_value = 0.f;
  if (j0 < bias1) {
    bias_token = p.bias_tokens[j0];
    bias_value = p.bias_values[j0];
    if (j0 + 1 < bias1) bias_next = p.bias_tokens[j0 + 1];
  }
  if (hist_len > 0 || bias1 > bias0) __syncthreads();
  // Every CTA looks at every entry, so an entry's few instructions are what counts here: the
  // atomic is predicated, and one maximum replaces a test of every entry (128 rows: 44.3 -> 43.1 us).
  const uint32_t words0 = smem_u32(words);
  unsigned largest = 0;  // entry, as unsigned: whether one is no token
  auto count = [&](int i, int token) {
    const unsigned at = static_cast<unsigned>(token) - static_cast<unsigned>(first);  // below the segment wraps round
    largest = max(largest, static_cast<unsigned>(token));
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.lt.u32 p, %0, %1;\n\t"
        "@p red.shared.add.u32 [%2], %3;\n\t}" ::"r"(at),
        "r"(n), "r"(words0 + 4u * at), "r"(i < prompt_len ? 0x10000u : 1u)
        : "memory");
  };
  for (int i0 = tid; i0 < pieces; i0 += kControlAhead * kControlThreads) {
#pragma unroll
    for (int u = 0; u < kControlAhead; ++u) {
      const int piece = i0 + u * kControlThreads;
      if (piece >= pieces) break;
      const int i = lead + 4 * piece;
      count(i, ahead[u].x);
      count(i + 1, ahead[u].y);
      count(i + 2, ahead[u].z);
      count(i + 3, ahead[u].w);
    }
#pragma unroll
    for (int u = 0; u < kControlAhead; ++u) {
      const int piece = i0 + (kControlAhead + u) * kControlThreads;
      if (piece < pieces) ahead[u] = body[piece];
    }
  }
  const int tail = hist_len - lead - 4 * pieces;
  if (tid < lead + tail) {
    const int i = tid < lead ? tid : hist_len - tail + tid - lead;
    count(i, hist[i]);
  }
  if (first_cta && largest >= static_cast<unsigned>(p.vocab)) raise_status(kStatusBadToken);
  // A list entry counts when its token is below the next entry's: ascending lists count whole,
  // of equal neighbours the last one does.
  for (int j = j0; j < bias1; j += kControlThreads) {
    const int token = j == j0 ? bias_token : p.bias_tokens[j];
    const int next = j == j0 ? bias_next : j + 1 < bias1 ? p.bias_tokens[j + 1] : INT_MAX;
    if (token < 0 || token >= p.vocab || token > next) {
      if (first_cta) raise_status(kStatusBadToken);
      continue;
    }
    const int at = token - first;
    if (at >= 0 && at < n) atomicOr(&biased[at >> 5], 1u << (at & 31));
  }

  // The stream: a copy with masked tokens replaced.
  constexpr uint32_t kBanned = 0xFF80u;  // -inf
  if (vec) {
#pragma unroll
    for (int u = 0; u < kControlGroups; ++u) {
      const int i = 8 * (tid + u * kControlThreads);
      if (i >= n) break;
      const uint32_t banned = ~allowed[u] & 0xFFu;
      if (in_place && banned == 0u) continue;
      if (n - i >= 8) {
        if (in_place) raw[u] = *reinterpret_cast<const uint4*>(in + first + i);
        uint32_t w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
        if (banned) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if ((banned >> (2 * e)) & 1u) w[e] = (w[e] & 0xFFFF0000u) | kBanned;
            if ((banned >> (2 * e)) & 2u) w[e] = (w[e] & 0x0000FFFFu) | (kBanned << 16);
          }
        }
        *reinterpret_cast<uint4*>(out + first + i) = make_uint4(w[0], w[1], w[2], w[3]);
      } else {
        for (int e = 0; e < n - i; ++e) {
          if ((banned >> e) & 1u) out[first + i + e] = __ushort_as_bfloat16(kBanned);
          else if (!in_place) out[first + i + e] = in[first + i + e];
        }
      }
    }
  } else {
    for (int i0 = tid; i0 < n; i0 += 8 * kControlThreads) {
      __nv_bfloat16 x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (!in_place && i0 + e * kControlThreads < n) x[e] = in[first + i0 + e * kControlThreads];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int i = i0 + e * kControlThreads;
        if (i >= n) break;
        const bool banned = mask && !((mask[(first + i) >> 5] >> ((first + i) & 31)) & 1u);
        if (banned) out[first + i] = __ushort_as_bfloat16(kBanned);
        else if (!in_place) out[first + i] = x[e];
      }
    }
  }
  if (hist_len == 0 && bias1 == bias0) return;
  __syncthreads();  // the words and the bitmap are complete
  if (hist_len > 0) {
    // Which of its tokens 4 (tid + u T) + e a thread finds touched: bit 4 u + e. Every lane takes
    // as many places on the list as it has bits.
    uint32_t bits = 0;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int i = 4 * (tid + u * kControlThreads);
      if (i < p.segment) {
        const uint4 w = *reinterpret_cast<const uint4*>(words + i);
        bits |= ((w.x ? 1u : 0u) | (w.y ? 2u : 0u) | (w.z ? 4u : 0u) | (w.w ? 8u : 0u)) << (4 * u);
      }
    }
    const int mine = __popc(bits), lane = tid & 31;
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    int at0 = 0;
    if (lane == 31 && incl > 0) at0 = atomicAdd(&n_touched, incl);
    int place = __shfl_sync(0xffffffffu, at0, 31) + incl - mine;
    for (; bits; bits &= bits - 1) {
      const int b = __ffs(bits) - 1;
      touched[place++] = static_cast<uint16_t>(4 * (tid + (b >> 2) * kControlThreads) + (b & 3));
    }
    __syncthreads();  // the list is complete, and the stream's writes precede the ones below
  }
  // A touched or biased token that is allowed still holds its logit in `in`, in place too.
  if (hist_len > 0) {
    for (int j = tid; j < n_touched; j += kControlThreads) {
      const int at = touched[j], token = first + at;
      if (bias1 > bias0 && ((biased[at >> 5] >> (at & 31)) & 1u)) continue;
      if (mask && !((mask[token >> 5] >> (token & 31)) & 1u)) continue;
      out[token] = __float2bfloat16_rn(penalised(__bfloat162float(in[token]), words[at], rc));
    }
  }
  for (int j = j0; j < bias1; j += kControlThreads) {
    const int token = j == j0 ? bias_token : p.bias_tokens[j];
    const int next = j == j0 ? bias_next : j + 1 < bias1 ? p.bias_tokens[j + 1] : INT_MAX;
    const int at = token - first;
    if (at < 0 || at >= n || token >= next) continue;
    if (mask && !((mask[token >> 5] >> (token & 31)) & 1u)) continue;
    const float x = penalised(__bfloat162float(in[token]), hist_len > 0 ? words[at] : 0u, rc);
    out[token] = __float2bfloat16_rn(__fadd_rn(x, j == j0 ? bias_value : p.bias_values[j]));
  }
}

}  // namespace hb
