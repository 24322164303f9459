// Rules on the logits of a step, and the record of tokens they go by.
//
// For row w of a request whose record is slot s, token v with logit x:
//   seen in its prompt or answer:   x <- x / r  if x > 0,  else x * r          (repetition)
//   generated c > 0 times:          x <- x - f c - p                           (frequency, presence)
//   biased by b:                    x <- x + b
//   ruled out by the row's mask:    x <- -inf      (whatever it was, NaN included)
//
// The record of a slot is two bit rows over the vocabulary (bit v % 32 of word v / 32: v stands in
// the prompt; v has been generated) and a row of counts, read only where the second bit is set: a
// logit costs a quarter of a byte of record beside the eight of its own way, not four more.
//
// Bound by the bytes of the logits where there are many (256 rows of 131,072 with everything: 46.8 us,
// 43.2 at the copy rate), and by a chain of five dependent trips to memory and two barriers in a
// block where there are few (one row of 50,257: 3.7 us, 64 rows with 100 biases each 9.0; the copy
// alone takes 5.6 there).  us in a graph.
#include "common.cuh"
#include <string.h>

namespace hs {

constexpr int LR_THREADS = 256, LR_BLOCKS = 6;     // of a block; of an SM
constexpr int LR_MOST = 8192;             // the widest tile: a word of bits a thread
constexpr int LR_BIASES = 512;            // biases of a tile that are kept at hand
constexpr int LH_THREADS = 512, LH_TILE = 8192;    // of the record's kernel

struct LogitRules {
  float* out;
  const float* logits;
  int vocab, words, tile;
  const int *prompt, *output, *counts;    // the records
  int n_slots;
  const int* slots;
  const float *repetition, *presence, *frequency;
  const int *bias_start, *bias_ids;
  const float* bias_values;
  int n_bias;
  const int* mask;
  int n_masks;
  const int* mask_row;
  int* status;
};

// Why this split.  A row is cut into as many tiles as run at a time (six blocks an SM), so that few rows
// use every SM and many rows take wide tiles: tiles of a fixed 4,096 places left 64 rows in two waves
// (11.6 us against 9.5) and 256 rows of 131,072 with 74 us against 47.  A table of the tile's biases
// in place of the list cost its initialisation and two blocks an SM; a thread for every seen token
// in place of a test in the copying loop is what took 256 rows from 4,117 us.  Doing the first listed
// token before the copies spilled registers and was slower with biases (9.0 -> 9.6 us).

// Bits i .. i + 3 of a row of words (one word more than the row has is readable).
__device__ __forceinline__ uint32_t lr_four(const uint32_t* words, int i) {
  return __funnelshift_r(words[i >> 5], words[(i >> 5) + 1], i & 31) & 15u;
}

// One block a tile of a row.  Most logits are only copied (or ruled out, and then not read at all);
// the few that stand in the record or are biased are listed first, and computed once the tile has
// been copied, a thread each, in 64 bits.  In place nothing is copied: only what a rule changes is
// written.
template <bool BIAS>
__global__ void __launch_bounds__(LR_THREADS, LR_BLOCKS)
logit_rules_kernel(const LogitRules a) {
  __shared__ uint32_t s_seen[LR_MOST / 32];      // in the record, or biased
  __shared__ uint32_t s_known[LR_MOST / 32], s_said[LR_MOST / 32], s_mask[LR_MOST / 32 + 1];
  __shared__ uint16_t s_list[LR_MOST];
  __shared__ int s_n;
  // (place in the tile, bias entry) in any order; where they are too many, the last entry of each of
  // so many places at a time
  __shared__ int2 s_entry[BIAS ? LR_BIASES : 1];
  __shared__ int s_entries;
  pdl_trigger();
  pdl_wait();
  const int w = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
  const int lo = blockIdx.x * a.tile, n = min(a.vocab - lo, a.tile), n_words = (n + 31) / 32;
  const int slot = a.slots ? a.slots[w] : -1, mrow = a.mask ? a.mask_row[w] : -1;
  const bool known = slot >= 0 && slot < a.n_slots, masked = mrow >= 0 && mrow < a.n_masks;
  int b0 = 0, b1 = 0;
  if (BIAS) {
    b0 = max(0, a.bias_start[w]);
    b1 = min(a.n_bias, a.bias_start[w + 1]);
  }
  if (tid == 0) {
    s_n = s_entries = 0;
    if (blockIdx.x == 0 && (slot >= a.n_slots || mrow >= a.n_masks))      // (without tables: -1 >= 0)
      atomicOr(a.status, HS_STATUS_BAD_ROW);
  }
  const size_t first = (size_t)w * a.vocab + lo;
  const float* from = a.logits + first;
  float* to = a.out + first;
  const bool in_place = from == to;
  const int off = (int)(((uintptr_t)from >> 2) & 3);
  const bool even = (((uintptr_t)from ^ (uintptr_t)to) & 15) == 0;
  // pieces of four that begin on 16 bytes: piece p holds the places 4 p - off + 0..3.  Where every
  // logit is copied, the first of them are under way while the record is read.
  const int pieces = even ? (n + off + 3) / 4 : 0;
  const bool ahead = !in_place && !masked;
  constexpr int INFLIGHT = 4;
  float4 x[INFLIGHT];
  if (ahead) {
#pragma unroll
    for (int k = 0; k < INFLIGHT; ++k) {
      const int i = 4 * (tid + k * LR_THREADS) - off;
      if (i >= 0 && i + 3 < n && even) x[k] = *(const float4*)(from + i);
    }
  }

  uint32_t seen = 0, said = 0;
  if (tid < n_words) {
    const size_t word = (size_t)(lo >> 5) + tid;
    if (known) {
      said = (uint32_t)a.output[(size_t)slot * a.words + word];
      seen = (uint32_t)a.prompt[(size_t)slot * a.words + word] | said;
      const int left = n - 32 * tid;      // (bits behind the vocabulary say nothing)
      if (left < 32) seen &= (1u << left) - 1u;
    }
    s_seen[tid] = seen;
    s_known[tid] = seen;
    s_said[tid] = said;
    s_mask[tid] = masked ? (uint32_t)a.mask[(size_t)mrow * a.words + word] : 0xffffffffu;
  }
  if (tid == 0) s_mask[n_words] = 0;
  int entry_id = -1;                      // the first round of the row's biases
  if (BIAS && b0 + tid < b1) entry_id = a.bias_ids[b0 + tid];
  __syncthreads();
  if (BIAS && b1 > b0) {
    for (int j = b0 + tid; j < b1; j += LR_THREADS) {
      const int v = j == b0 + tid ? entry_id : a.bias_ids[j], i = v - lo;
      if (v < 0 || v >= a.vocab) {
        if (blockIdx.x == 0) atomicOr(a.status, HS_STATUS_BAD_TOKEN);
      } else if (i >= 0 && i < n) {
        const int at = atomicAdd(&s_entries, 1);
        if (at < LR_BIASES) s_entry[at] = make_int2(i, j);
        atomicOr(&s_seen[i >> 5], 1u << (i & 31));
      }
    }
    __syncthreads();
    if (tid < n_words) seen = s_seen[tid];
  }
  // list what has to be computed: ruled-out tokens need not be
  uint32_t todo = tid < n_words ? seen & s_mask[tid] : 0u;
  if (__any_sync(0xffffffffu, todo != 0u)) {
    const int c = __popc(todo);
    int incl = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += u;
    }
    int at = 0;
    if (lane == 31) at = atomicAdd(&s_n, incl);
    at = __shfl_sync(0xffffffffu, at, 31) + incl - c;
    for (uint32_t bits = todo; bits; bits &= bits - 1) s_list[at++] = (uint16_t)(32 * tid + __ffs(bits) - 1);
  }

  if (even && (!in_place || masked)) {
    for (int p0 = tid; p0 < pieces; p0 += INFLIGHT * LR_THREADS) {
      uint32_t keep[INFLIGHT];
#pragma unroll
      for (int k = 0; k < INFLIGHT; ++k) {
        const int i = 4 * (p0 + k * LR_THREADS) - off;
        keep[k] = 15u;
        if (i >= 0 && i + 3 < n) {
          if (masked) keep[k] = lr_four(s_mask, i);
          if (keep[k] != 0u && !(in_place && keep[k] == 15u) && !(ahead && p0 == tid))
            x[k] = *(const float4*)(from + i);
        }
      }
#pragma unroll
      for (int k = 0; k < INFLIGHT; ++k) {
        const int i = 4 * (p0 + k * LR_THREADS) - off;
        if (i >= 0 && i + 3 < n) {
          if (in_place && keep[k] == 15u) continue;
          if (!(keep[k] & 1u)) x[k].x = -INFINITY;
          if (!(keep[k] & 2u)) x[k].y = -INFINITY;
          if (!(keep[k] & 4u)) x[k].z = -INFINITY;
          if (!(keep[k] & 8u)) x[k].w = -INFINITY;
          *(float4*)(to + i) = x[k];
        } else if (p0 + k * LR_THREADS < pieces) {
          for (int j = max(i, 0); j < min(i + 4, n); ++j) {
            const bool kept = (s_mask[j >> 5] >> (j & 31)) & 1u;
            if (!in_place || !kept) to[j] = kept ? from[j] : -INFINITY;
          }
        }
      }
    }
  } else if (!even) {
    for (int j = tid; j < n; j += LR_THREADS) to[j] = (s_mask[j >> 5] >> (j & 31)) & 1u ? from[j] : -INFINITY;
  }
  __syncthreads();
  const int listed = s_n;
  auto compute = [&](int i, int entry) {
    double y = from[i];
    const uint32_t bit = 1u << (i & 31);
    if (known && (s_known[i >> 5] & bit)) {
      const double r = a.repetition[w];
      y = y > 0. ? y / r : y * r;
      if (s_said[i >> 5] & bit) {
        const int c = a.counts[(size_t)slot * a.vocab + lo + i];
        y -= (double)a.frequency[w] * c + (c > 0 ? (double)a.presence[w] : 0.);
      }
    }
    if (BIAS && entry >= 0) y += a.bias_values[entry];
    to[i] = (float)y;
  };
  if (!BIAS || s_entries <= LR_BIASES) {
    const int entries = BIAS ? s_entries : 0;
    for (int l = tid; l < listed; l += LR_THREADS) {
      const int i = s_list[l];
      int last = -1;
      for (int e = 0; e < entries; ++e)
        if (s_entry[e].x == i) last = max(last, s_entry[e].y);
      compute(i, last);
    }
  } else {
    constexpr int PLACES = 2 * LR_BIASES;
    int* s_last = (int*)s_entry;
    for (int from_place = 0; from_place < n; from_place += PLACES) {
      __syncthreads();
      for (int i = tid; i < PLACES; i += LR_THREADS) s_last[i] = -1;
      __syncthreads();
      for (int j = b0 + tid; j < b1; j += LR_THREADS) {
        const unsigned i = (unsigned)a.bias_ids[j] - (unsigned)(lo + from_place);
        if (i < PLACES) atomicMax(&s_last[i], j);
      }
      __syncthreads();
      for (int l = tid; l < listed; l += LR_THREADS) {
        const int i = s_list[l];
        if (i >= from_place && i < from_place + PLACES) compute(i, s_last[i - from_place]);
      }
    }
  }
}

// One block a tile of the vocabulary and slot: the tile's bits and counts are formed in shared memory
// from all of the slot's tokens and written whole, so that nothing has to be cleared first.  Bound by
// the chain slots - offsets - tokens - shared atomics - stores: 64 slots of 3,900 tokens take 7.7 us
// (5.1 without tokens; 2.2 at the copy rate), one of 900 2.5.  Sums of ones: the order of the atomics
// changes nothing.
__global__ void __launch_bounds__(LH_THREADS)
history_begin_kernel(int* prompt, int* output, int* counts, int vocab, int words, int n_slots,
                     const int* slots, int n_rows, const int* tokens, int n_tokens, const int* start,
                     const int* n_prompt, int* status) {
  __shared__ int4 s_count4[LH_TILE / 4 + 1];
  __shared__ uint32_t s_bits[2][LH_TILE / 32];
  int* s_count = (int*)s_count4;
  pdl_trigger();
  pdl_wait();
  const int k = blockIdx.y, tid = threadIdx.x, slot = slots[k];
  if (slot < 0) return;
  if (slot >= n_slots) {
    if (blockIdx.x == 0 && tid == 0) atomicOr(status, HS_STATUS_BAD_ROW);
    return;
  }
  const int t0 = max(0, start[k]), t1 = min(n_tokens, start[k + 1]);
  // (a prompt may be said to be longer than its tokens are, up to any number)
  const int p1 = (int)min(max((long long)start[k] + n_prompt[k], 0ll), (long long)n_tokens);
  // of two rows of one slot the last counts
  bool again = false;
  for (int j = k + 1 + tid; j < n_rows; j += LH_THREADS) again |= slots[j] == slot;
  for (int i = tid; i < LH_TILE / 4 + 1; i += LH_THREADS) s_count4[i] = make_int4(0, 0, 0, 0);
  if (tid < 2 * LH_TILE / 32) (&s_bits[0][0])[tid] = 0u;
  if (__syncthreads_or(again)) return;
  const int lo = blockIdx.x * LH_TILE, n = min(LH_TILE, vocab - lo);
  int* to = counts + (size_t)slot * vocab + lo;
  const int off = (int)(((uintptr_t)to >> 2) & 3);      // counts stand as they do in their row's pieces
  constexpr int INFLIGHT = 8;
  for (int t = t0 + tid; t < t1; t += INFLIGHT * LH_THREADS) {
    int v[INFLIGHT];
#pragma unroll
    for (int j = 0; j < INFLIGHT; ++j) v[j] = t + j * LH_THREADS < t1 ? tokens[t + j * LH_THREADS] : 0;
#pragma unroll
    for (int j = 0; j < INFLIGHT; ++j) {
      const int at = t + j * LH_THREADS, i = v[j] - lo;
      if (at >= t1) break;
      if (v[j] >= lo && i < n) {
        const bool said = at >= p1;
        if (said) atomicAdd(&s_count[off + i], 1);
        atomicOr(&s_bits[said][i >> 5], 1u << (i & 31));
      } else if (blockIdx.x == 0 && (v[j] < 0 || v[j] >= vocab)) {
        atomicOr(status, HS_STATUS_BAD_TOKEN);
      }
    }
  }
  __syncthreads();
  if (tid < (n + 31) / 32) {
    const size_t word = (size_t)slot * words + (lo >> 5) + tid;
    prompt[word] = (int)s_bits[0][tid];
    output[word] = (int)s_bits[1][tid];
  }
  const int pieces = (n + off + 3) / 4;
  for (int p = tid; p < pieces; p += LH_THREADS) {
    const int i = 4 * p - off;
    if (i >= 0 && i + 3 < n) {
      *(int4*)(to + i) = s_count4[p];
    } else {
      for (int j = max(i, 0); j < min(i + 4, n); ++j) to[j] = s_count[off + j];
    }
  }
}

__global__ void history_add_kernel(int* output, int* counts, int vocab, int words, int n_slots,
                                   const int* slots, const int* tokens, int n, int* status) {
  pdl_trigger();
  pdl_wait();
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  const int slot = slots[i], v = tokens[i];
  if (slot < 0) return;
  if (slot >= n_slots || v < 0 || v >= vocab) {
    atomicOr(status, slot >= n_slots ? HS_STATUS_BAD_ROW : HS_STATUS_BAD_TOKEN);
    return;
  }
  atomicOr((unsigned*)&output[(size_t)slot * words + (v >> 5)], 1u << (v & 31));
  atomicAdd(&counts[(size_t)slot * vocab + v], 1);
}

}  // namespace hs

// The arguments of hs_logit_rules, eight bytes each.  The record's three tensors, slots and the
// three penalties are null together, so are the bias's three and the mask's two.  bias_start holds
// rows + 1 offsets into n_bias entries; of an id that a row lists twice the last entry counts.  out
// may be logits itself.
struct HsLogitRules {
  float* out;
  const float* logits;
  long long rows, vocab;
  const int *prompt, *output, *counts;
  long long n_slots;
  const int* slots;
  const float *repetition, *presence, *frequency;
  const int *bias_start, *bias_ids;
  const float* bias_values;
  long long n_bias;
  const int* mask;
  long long n_masks;
  const int* mask_row;
  int* status;
};
static_assert(sizeof(HsLogitRules) == 20 * 8, "");

HS_EXPORT int hs_logit_rules(const HsLogitRules* in, void* stream) {
  if (!in) return HS_ERR_ARGUMENT;
  HsLogitRules a;
  memcpy(&a, in, sizeof a);
  if (!a.out || !a.logits || !a.status || a.vocab <= 0) return HS_ERR_ARGUMENT;
  if (a.slots && (!a.prompt || !a.output || !a.counts || !a.repetition || !a.presence || !a.frequency))
    return HS_ERR_ARGUMENT;
  if (a.bias_start && (!a.bias_ids || !a.bias_values)) return HS_ERR_ARGUMENT;
  if ((a.mask == nullptr) != (a.mask_row == nullptr)) return HS_ERR_ARGUMENT;
  if (a.rows <= 0) return HS_OK;
  if (a.rows > 65535 || a.vocab > 0x7fff0000 || a.n_slots > 0x7fffffff || a.n_bias > 0x7fffffff ||
      a.n_masks > 0x7fffffff)
    return HS_ERR_UNSUPPORTED;
  const int rows = (int)a.rows, vocab = (int)a.vocab;
  // as many tiles as run at a time, none narrower than a round of a block's loads
  const int fit = hs::LR_BLOCKS * hs_sm_count(), tiles = fit / rows > 1 ? fit / rows : 1;
  int tile = ((vocab + tiles - 1) / tiles + 1023) / 1024 * 1024;
  if (tile > hs::LR_MOST) tile = hs::LR_MOST;
  const hs::LogitRules args{a.out, a.logits, vocab, (vocab + 31) / 32, tile, a.prompt, a.output, a.counts,
                            (int)a.n_slots, a.slots, a.repetition, a.presence, a.frequency, a.bias_start,
                            a.bias_ids, a.bias_values, (int)a.n_bias, a.mask, (int)a.n_masks, a.mask_row,
                            a.status};
  const dim3 grid((vocab + tile - 1) / tile, rows);
  const cudaError_t e =
      a.bias_start ? hs_launch(hs::logit_rules_kernel<true>, grid, dim3(hs::LR_THREADS), 0,
                             (cudaStream_t)stream, hs_pdl_enabled(), args)
                 : hs_launch(hs::logit_rules_kernel<false>, grid, dim3(hs::LR_THREADS), 0,
                             (cudaStream_t)stream, hs_pdl_enabled(), args);
  return e == cudaSuccess ? HS_OK : (int)e;
}

// Slot slots[k] gets the record of tokens[start[k] .. start[k + 1]), the first n_prompt[k] of them
// the prompt's.  Whatever the slot held before is gone.
HS_EXPORT int hs_history_begin(int* prompt, int* output, int* counts, int n_slots, int vocab,
                               const int* slots, int n_rows, const int* tokens, int n_tokens,
                               const int* start, const int* n_prompt, int* status, void* stream) {
  if (!prompt || !output || !counts || !slots || !start || !n_prompt || !status || vocab <= 0)
    return HS_ERR_ARGUMENT;
  if (n_tokens > 0 && !tokens) return HS_ERR_ARGUMENT;
  if (n_rows <= 0) return HS_OK;
  if (n_rows > 65535) return HS_ERR_UNSUPPORTED;
  const cudaError_t e = hs_launch(
      hs::history_begin_kernel, dim3((vocab + hs::LH_TILE - 1) / hs::LH_TILE, n_rows),
      dim3(hs::LH_THREADS), 0, (cudaStream_t)stream, hs_pdl_enabled(), prompt, output, counts, vocab,
      (vocab + 31) / 32, n_slots, slots, n_rows, tokens, n_tokens, start, n_prompt, status);
  return e == cudaSuccess ? HS_OK : (int)e;
}

// One more generated token in slot slots[i] for every i < n; a slot below zero is skipped.
HS_EXPORT int hs_history_add(int* output, int* counts, int n_slots, int vocab, const int* slots,
                             const int* tokens, int n, int* status, void* stream) {
  if (!output || !counts || !slots || !tokens || !status || vocab <= 0) return HS_ERR_ARGUMENT;
  if (n <= 0) return HS_OK;
  const cudaError_t e = hs_launch(hs::history_add_kernel, dim3((n + 127) / 128), dim3(128), 0,
                                  (cudaStream_t)stream, hs_pdl_enabled(), output, counts, vocab,
                                  (vocab + 31) / 32, n_slots, slots, tokens, n, status);
  return e == cudaSuccess ? HS_OK : (int)e;
}
