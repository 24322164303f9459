// Log-probabilities of given tokens, their ranks, and the largest alternatives.
//
// For row w with logits x and token t:  lp = (x_t - m) - log(sum_v exp(x_v - m)),  m = max_v x_v;
// rank = how many tokens stand before t, those of a larger logit and those of an equal one with a
// lower index (0: the greedy choice).  The n largest come in that order with their own lp.
// A row that is -inf throughout has no probabilities: every lp is -inf.  A NaN or +inf in a row makes
// all of its lp NaN; in the order a NaN stands behind everything else.
#include "common.cuh"

namespace hs {

constexpr int TL_THREADS = 256;

// order of (logit, index): larger logits first, among equal ones the lower index; zeros of both
// signs are equal, NaN is the smallest
__device__ __forceinline__ unsigned long long tl_key(float x, int v) {
  uint32_t b = x != x ? 0u : __float_as_uint(x + 0.f);
  if (x == x) b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return ((unsigned long long)b << 32) | (uint32_t)~(uint32_t)v;
}

__global__ void __launch_bounds__(TL_THREADS)
token_logprobs_kernel(float* logprob, int* rank, int* top_ids, float* top_logprobs, int top,
                      const float* logits, const int* tokens, int vocab, int* status) {
  __shared__ float s_f[TL_THREADS / 32];
  __shared__ int s_i[TL_THREADS / 32];
  __shared__ unsigned long long s_k[TL_THREADS / 32];
  pdl_trigger();
  pdl_wait();
  const int w = blockIdx.x, tid = threadIdx.x;
  const float* row = logits + (size_t)w * vocab;
  const int t = tokens[w];
  const bool given = t >= 0 && t < vocab;
  const float xt = given ? row[t] : 0.f;
  const unsigned long long mine = given ? tl_key(xt, t) : ~0ull;
  float m = -INFINITY;
  bool nan = false;
  for (int v = tid; v < vocab; v += TL_THREADS) {
    m = fmaxf(m, row[v]);
    nan |= row[v] != row[v];
  }
  m = warp_max(m);
  if ((tid & 31) == 0) s_f[tid >> 5] = m;
  nan = __syncthreads_or(nan);
  for (int i = 0; i < TL_THREADS / 32; ++i) m = fmaxf(m, s_f[i]);
  __syncthreads();
  float sum = 0.f;
  int before = 0;
  for (int v = tid; v < vocab; v += TL_THREADS) {
    sum += expf(row[v] - m);
    before += tl_key(row[v], v) > mine;
  }
  sum = warp_sum(sum);
  before = __reduce_add_sync(0xffffffffu, before);
  if ((tid & 31) == 0) {
    s_f[tid >> 5] = sum;
    s_i[tid >> 5] = before;
  }
  __syncthreads();
  sum = 0.f;
  before = 0;
  for (int i = 0; i < TL_THREADS / 32; ++i) {
    sum += s_f[i];
    before += s_i[i];
  }
  const float log_sum = logf(sum);
  auto lp = [&](float x) { return m == -INFINITY && !nan ? -INFINITY : (x - m) - log_sum; };
  if (tid == 0) {
    logprob[w] = given ? lp(xt) : __int_as_float(0x7fffffff);
    rank[w] = given ? before : -1;
    if (!given && t != -1) atomicOr(status, HS_STATUS_BAD_TOKEN);
  }
  unsigned long long last = ~0ull;
  for (int n = 0; n < top; ++n) {
    unsigned long long best = 0;
    for (int v = tid; v < vocab; v += TL_THREADS) {
      const unsigned long long key = tl_key(row[v], v);
      if (key < last && key > best) best = key;
    }
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
      if (other > best) best = other;
    }
    __syncthreads();
    if ((tid & 31) == 0) s_k[tid >> 5] = best;
    __syncthreads();
    for (int i = 0; i < TL_THREADS / 32; ++i)
      if (s_k[i] > best) best = s_k[i];
    last = best;
    if (tid == 0) {
      const int v = (int)~(uint32_t)best;
      top_ids[(size_t)w * top + n] = v;
      top_logprobs[(size_t)w * top + n] = lp(row[v]);
    }
  }
}

}  // namespace hs

// tokens[w] == -1: no token (lp NaN, rank -1); any other index outside the vocabulary is reported.
HS_EXPORT int hs_token_logprobs(float* logprob, int* rank, int* top_ids, float* top_logprobs, int top,
                                const float* logits, const int* tokens, int rows, int vocab,
                                int* status, void* stream) {
  if (!logprob || !rank || !logits || !tokens || !status || vocab <= 0) return HS_ERR_ARGUMENT;
  if (top < 0 || top > 32 || top > vocab) return HS_ERR_UNSUPPORTED;
  if (top > 0 && (!top_ids || !top_logprobs)) return HS_ERR_ARGUMENT;
  if (rows <= 0) return HS_OK;
  const cudaError_t e = hs_launch(hs::token_logprobs_kernel, dim3(rows), dim3(hs::TL_THREADS), 0,
                                  (cudaStream_t)stream, hs_pdl_enabled(), logprob, rank, top_ids,
                                  top_logprobs, top, logits, tokens, vocab, status);
  return e == cudaSuccess ? HS_OK : (int)e;
}
