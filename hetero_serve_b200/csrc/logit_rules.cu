// Rules on the logits of a step, and the record of tokens they go by.
//
// For row w of a request whose record is slot s, token v with logit x:
//   seen in its prompt or answer:   x <- x / r  if x > 0,  else x * r          (repetition)
//   generated c > 0 times:          x <- x - f c - p                           (frequency, presence)
//   biased by b:                    x <- x + b
//   ruled out by the row's mask:    x <- -inf      (whatever it was, NaN included)
//
// The record of a slot is two bit rows over the vocabulary (bit v % 32 of word v / 32: v stands in
// the prompt; v has been generated) and a row of counts, read only where the second bit is set.
#include "common.cuh"

namespace hs {

constexpr int LR_THREADS = 256, LR_TILE = 4096;

__global__ void __launch_bounds__(LR_THREADS)
logit_rules_kernel(float* out, const float* logits, int vocab, int words, const int* prompt,
                   const int* output, const int* counts, int n_slots, const int* slots,
                   const float* repetition, const float* presence, const float* frequency,
                   const int* bias_start, const int* bias_ids, const float* bias_values, int n_bias,
                   const int* mask, int n_masks, const int* mask_row, int* status) {
  pdl_trigger();
  pdl_wait();
  const int w = blockIdx.y;
  const int slot = slots ? slots[w] : -1;
  const bool known = slot >= 0 && slot < n_slots;
  const int mrow = mask ? mask_row[w] : -1;
  const bool masked = mrow >= 0 && mrow < n_masks;
  if (blockIdx.x == 0 && threadIdx.x == 0 && (slot >= n_slots || mrow >= n_masks) && (slots || mask))
    if ((slots && slot >= n_slots) || (mask && mrow >= n_masks)) atomicOr(status, HS_STATUS_BAD_ROW);
  int b0 = 0, b1 = 0;
  if (bias_start) {
    b0 = max(0, bias_start[w]);
    b1 = min(n_bias, bias_start[w + 1]);
  }
  const int lo = blockIdx.x * LR_TILE, hi = min(vocab, lo + LR_TILE);
  for (int v = lo + threadIdx.x; v < hi; v += LR_THREADS) {
    const size_t at = (size_t)w * vocab + v;
    const uint32_t bit = 1u << (v & 31);
    float x = logits[at];
    double y = x;
    bool changed = false;
    if (known) {
      const size_t word = (size_t)slot * words + (v >> 5);
      const bool said = (uint32_t)output[word] & bit;
      if (said || ((uint32_t)prompt[word] & bit)) {
        const double r = repetition[w];
        y = y > 0. ? y / r : y * r;
        if (said) {
          const int c = counts[(size_t)slot * vocab + v];
          y -= (double)frequency[w] * c + (c > 0 ? (double)presence[w] : 0.);
        }
        changed = true;
      }
    }
    for (int j = b1 - 1; j >= b0; --j)
      if (bias_ids[j] == v) {
        y += bias_values[j];
        changed = true;
        break;
      }
    if (changed) x = (float)y;
    if (masked && !((uint32_t)mask[(size_t)mrow * words + (v >> 5)] & bit)) x = -INFINITY;
    out[at] = x;
  }
  if (blockIdx.x == 0)
    for (int j = b0 + threadIdx.x; j < b1; j += LR_THREADS)
      if (bias_ids[j] < 0 || bias_ids[j] >= vocab) atomicOr(status, HS_STATUS_BAD_TOKEN);
}

// One block a tile of the vocabulary and slot: the tile's counts are formed in shared memory from
// all of the slot's tokens and written whole, so that nothing has to be cleared first.
__global__ void __launch_bounds__(LR_THREADS)
history_begin_kernel(int* prompt, int* output, int* counts, int vocab, int words, int n_slots,
                     const int* slots, int n_rows, const int* tokens, int n_tokens, const int* start,
                     const int* n_prompt, int* status) {
  __shared__ int s_count[LR_TILE];
  __shared__ uint32_t s_prompt[LR_TILE / 32];
  pdl_trigger();
  pdl_wait();
  const int k = blockIdx.y, slot = slots[k];
  if (slot < 0) return;
  if (slot >= n_slots) {
    if (blockIdx.x == 0 && threadIdx.x == 0) atomicOr(status, HS_STATUS_BAD_ROW);
    return;
  }
  for (int j = k + 1; j < n_rows; ++j)      // of two rows of one slot the last counts
    if (slots[j] == slot) return;
  const int lo = blockIdx.x * LR_TILE;
  for (int i = threadIdx.x; i < LR_TILE; i += LR_THREADS) s_count[i] = 0;
  for (int i = threadIdx.x; i < LR_TILE / 32; i += LR_THREADS) s_prompt[i] = 0;
  __syncthreads();
  const int t0 = max(0, start[k]), t1 = min(n_tokens, start[k + 1]), p1 = start[k] + n_prompt[k];
  for (int t = t0 + threadIdx.x; t < t1; t += LR_THREADS) {
    const int v = tokens[t];
    if (v < 0 || v >= vocab) {
      if (blockIdx.x == 0) atomicOr(status, HS_STATUS_BAD_TOKEN);
      continue;
    }
    const int i = v - lo;
    if (i < 0 || i >= LR_TILE) continue;
    if (t < p1) atomicOr(&s_prompt[i >> 5], 1u << (i & 31));
    else atomicAdd(&s_count[i], 1);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < LR_TILE; i += LR_THREADS) {
    const int v = lo + i;
    const int c = s_count[i];
    const uint32_t said = __ballot_sync(0xffffffffu, c > 0);
    if (v < vocab) counts[(size_t)slot * vocab + v] = c;
    if ((i & 31) == 0 && (v >> 5) < words) {
      output[(size_t)slot * words + (v >> 5)] = (int)said;
      prompt[(size_t)slot * words + (v >> 5)] = (int)s_prompt[i >> 5];
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

// prompt / output / counts / slots (and the three penalties) are null together, so are the bias's
// three and the mask's two.  bias_start holds rows + 1 offsets into n_bias entries; of an id that a
// row lists twice the last entry counts.  out may be logits itself.
HS_EXPORT int hs_logit_rules(float* out, const float* logits, int rows, int vocab, const int* prompt,
                             const int* output, const int* counts, int n_slots, const int* slots,
                             const float* repetition, const float* presence, const float* frequency,
                             const int* bias_start, const int* bias_ids, const float* bias_values,
                             int n_bias, const int* mask, int n_masks, const int* mask_row,
                             int* status, void* stream) {
  if (!out || !logits || !status || vocab <= 0) return HS_ERR_ARGUMENT;
  if (slots && (!prompt || !output || !counts || !repetition || !presence || !frequency))
    return HS_ERR_ARGUMENT;
  if (bias_start && (!bias_ids || !bias_values)) return HS_ERR_ARGUMENT;
  if ((mask == nullptr) != (mask_row == nullptr)) return HS_ERR_ARGUMENT;
  if (rows <= 0) return HS_OK;
  if (rows > 65535) return HS_ERR_UNSUPPORTED;
  const cudaError_t e = hs_launch(
      hs::logit_rules_kernel, dim3((vocab + hs::LR_TILE - 1) / hs::LR_TILE, rows), dim3(hs::LR_THREADS),
      0, (cudaStream_t)stream, hs_pdl_enabled(), out, logits, vocab, (vocab + 31) / 32, prompt, output,
      counts, n_slots, slots, repetition, presence, frequency, bias_start, bias_ids, bias_values, n_bias,
      mask, n_masks, mask_row, status);
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
      hs::history_begin_kernel, dim3((vocab + hs::LR_TILE - 1) / hs::LR_TILE, n_rows),
      dim3(hs::LR_THREADS), 0, (cudaStream_t)stream, hs_pdl_enabled(), prompt, output, counts, vocab,
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
