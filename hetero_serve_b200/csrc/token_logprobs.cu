// Log-probabilities of given tokens, their ranks, and the largest alternatives.
//
// For row w with logits x and token t:  lp = (x_t - m) - log(sum_v exp(x_v - m)),  m = max_v x_v;
// rank = how many tokens stand before t, those of a larger logit and those of an equal one with a
// lower index (0: the greedy choice).  The n largest come in that order with their own lp.
// A row that is -inf throughout has no probabilities: every lp is -inf.  A NaN or +inf in a row makes
// all of its lp NaN; in the order a NaN stands behind everything else.
//
// One pass over the row: every thread keeps a running maximum with the sum of exp against it, counts
// the logits before x_t, and remembers which of its pieces held its maximum.  The n largest of the
// row lie in the n threads whose maxima are the largest (each of those threads holds one at least as
// large as the n-th of them), so that only their logits are looked at again: n / threads of the row.
// A row is shared by the blocks of a cluster where there are few rows.
#include "common.cuh"

namespace hs {

constexpr int TL_TOP = 32;                // a warp's lanes hold the alternatives, in order
constexpr int TL_INFLIGHT = 4;            // 16-byte loads a thread has under way
constexpr int TL_CAND = 4096;             // logits looked at again at a time

typedef unsigned long long tl_key_t;

// order of (logit, index): larger logits first, among equal ones the lower index; zeros of both
// signs are equal, NaN is the smallest; 0 stands for no logit at all
__device__ __forceinline__ tl_key_t tl_key(float x, int v) {
  uint32_t b = __float_as_uint(x + 0.f);
  b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  if (x != x) b = 0u;
  return ((tl_key_t)b << 32) | (uint32_t)~(uint32_t)v;
}
__device__ __forceinline__ float tl_value(tl_key_t key) {
  const uint32_t b = (uint32_t)(key >> 32);
  return __uint_as_float((b & 0x80000000u) ? b ^ 0x80000000u : ~b);
}
__device__ __forceinline__ int tl_index(tl_key_t key) { return (int)~(uint32_t)key; }

// Bitonic steps over a warp: lane l ends with the l-th largest.
__device__ __forceinline__ tl_key_t tl_step(tl_key_t k, int lane, int o, bool down) {
  const tl_key_t other = __shfl_xor_sync(0xffffffffu, k, o);
  const bool first = (lane & o) == 0;
  return (first == down) == (k > other) ? k : other;
}
__device__ __forceinline__ tl_key_t tl_sorted(tl_key_t k, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int o = size >> 1; o > 0; o >>= 1) k = tl_step(k, lane, o, (lane & size) == 0 || size == 32);
  return k;
}
// The 32 largest of two sorted lists (b from its end), sorted.
__device__ __forceinline__ tl_key_t tl_merged(tl_key_t a, tl_key_t b_reversed, int lane) {
  tl_key_t k = a > b_reversed ? a : b_reversed;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) k = tl_step(k, lane, o, true);
  return k;
}

// A running maximum and the sum of exp against it.  Nothing is subtracted from an infinite maximum:
// -inf stands for no logit yet (every term is then 0), +inf makes the sum NaN by itself.
struct TlSum {
  float m, s;
};
__device__ __forceinline__ float tl_term(float x, float m) {
  return __expf(x - (m == -INFINITY ? 0.f : m));
}
__device__ __forceinline__ TlSum tl_join(TlSum a, TlSum b) {
  const float m = fmaxf(a.m, b.m);
  return TlSum{m, a.s * tl_term(a.m, m) + b.s * tl_term(b.m, m)};
}

__device__ __forceinline__ uint32_t tl_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void tl_cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
template <typename T>
__device__ __forceinline__ T tl_remote(const T* p, int rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
               : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  if constexpr (sizeof(T) == 8) {
    tl_key_t v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
    return (T)v;
  } else {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    T out;
    memcpy(&out, &v, 4);
    return out;
  }
}

// A row as pieces of four logits that begin on 16 bytes: piece p holds the indices 4 p - off + 0..3;
// places outside the row read as -inf.
struct TlRow {
  const float* row;
  int vocab, off;
  __device__ __forceinline__ float4 load(int p) const {
    const int v = 4 * p - off;
    if (v >= 0 && v + 3 < vocab) return *(const float4*)(row + v);
    float x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = v + j >= 0 && v + j < vocab ? row[v + j] : -INFINITY;
    return make_float4(x[0], x[1], x[2], x[3]);
  }
};

template <int THREADS, int BLOCKS>
__global__ void __launch_bounds__(THREADS)
token_logprobs_kernel(float* __restrict__ logprob, int* __restrict__ rank, int* __restrict__ top_ids,
                      float* __restrict__ top_logprobs, int top, const float* __restrict__ logits,
                      const int* __restrict__ tokens, int vocab, int* status) {
  constexpr int WARPS = THREADS / 32;
  __shared__ TlSum s_sum[WARPS];
  __shared__ int s_before[WARPS];
  __shared__ tl_key_t s_list[WARPS][TL_TOP];
  __shared__ int s_found;
  __shared__ TlSum s_block;             // what the cluster's first block reads of the others
  __shared__ int s_block_before;
  extern __shared__ tl_key_t s_cand[];  // [TL_CAND] where alternatives are wanted
  pdl_trigger();
  pdl_wait();
  const int w = blockIdx.x / BLOCKS, part = BLOCKS > 1 ? (int)tl_rank() : 0;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const float* base = logits + (size_t)w * vocab;
  const TlRow row{base, vocab, (int)(((uintptr_t)base >> 2) & 3)};
  const int pieces = (vocab + row.off + 3) / 4, per = (pieces + BLOCKS - 1) / BLOCKS;
  const int p0 = min(pieces, part * per), p1 = min(pieces, p0 + per);

  const int t = tokens[w];
  const bool given = t >= 0 && t < vocab;
  const float xt = given ? base[t] + 0.f : INFINITY;
  // x stands before x_t where x > x_t, and where x = x_t with a lower index: that is x > the number
  // below x_t there.  (x_t NaN or -inf has no number below it: those rows compare keys.)
  const bool by_key = !(xt > -INFINITY);
  const float below = xt == INFINITY ? 3.402823466e38f : nextafterf(xt, -INFINITY);
  const tl_key_t mine = given ? tl_key(xt, t) : ~0ull;

  TlSum own{-INFINITY, 0.f};
  int before = 0, best_at = p0 + tid;
  for (int p = p0 + tid; p < p1; p += TL_INFLIGHT * THREADS) {
    float x[TL_INFLIGHT][4];
#pragma unroll
    for (int i = 0; i < TL_INFLIGHT; ++i) {
      float4 f = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      if (p + i * THREADS < p1) f = row.load(p + i * THREADS);
      x[i][0] = f.x; x[i][1] = f.y; x[i][2] = f.z; x[i][3] = f.w;
    }
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < TL_INFLIGHT; ++i)
      m = fmaxf(m, fmaxf(fmaxf(x[i][0], x[i][1]), fmaxf(x[i][2], x[i][3])));
    if (m > own.m) {
      own.s *= tl_term(own.m, m);
      own.m = m;
      best_at = p;
    }
    const float ref = own.m == -INFINITY ? 0.f : own.m;
#pragma unroll
    for (int i = 0; i < TL_INFLIGHT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) own.s += __expf(x[i][j] - ref);
#pragma unroll
    for (int i = 0; i < TL_INFLIGHT; ++i) {
      const int v = 4 * (p + i * THREADS) - row.off;
      if (!by_key) {
#pragma unroll
        for (int j = 0; j < 4; ++j) before += x[i][j] > (v + j < t ? below : xt);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          before += p + i * THREADS < p1 && v + j >= 0 && v + j < vocab && tl_key(x[i][j], v + j) > mine;
      }
    }
  }

  // the thread's largest key: the first logit equal to its maximum, in the pieces that brought it
  // (without a maximum: the first -inf, wherever it stands, or its first NaN)
  tl_key_t key = 0;
  if (top > 0 && p0 + tid < p1) {
    const tl_key_t lowest = tl_key(-INFINITY, 0x7fffffff);
    for (int from = best_at; from < p1; from += TL_INFLIGHT * THREADS) {
#pragma unroll
      for (int i = 0; i < TL_INFLIGHT; ++i) {
        const int p = from + i * THREADS;
        if (p < p1) {
          const float4 f = row.load(p);
          const float x[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int v = 4 * p - row.off + j;
            const tl_key_t k = v >= 0 && v < vocab ? tl_key(x[j], v) : 0;
            if (k > key) key = k;
          }
        }
      }
      if (key >= lowest) break;
    }
  }

  TlSum all = own;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    all = tl_join(all, TlSum{__shfl_xor_sync(0xffffffffu, all.m, o), __shfl_xor_sync(0xffffffffu, all.s, o)});
  before = __reduce_add_sync(0xffffffffu, before);
  if (lane == 0) {
    s_sum[warp] = all;
    s_before[warp] = before;
  }
  if (tid == 0) s_found = 0;

  // joins the warps' sorted lists; warp 0 is left with the block's
  auto join_lists = [&](tl_key_t mine_sorted, int lists) {
    tl_key_t k = mine_sorted;
    if (warp < lists) s_list[warp][lane] = k;
    __syncthreads();
    for (int half = lists / 2; half > 0; half >>= 1) {
      if (warp < half) {
        k = tl_merged(k, s_list[warp + half][31 - lane], lane);
        s_list[warp][lane] = k;
      }
      __syncthreads();
    }
    return k;
  };
  tl_key_t best = 0;                        // warp 0: the block's alternatives, in order
  if (top > 0) {
    join_lists(tl_sorted(key, lane), WARPS);
    tl_key_t bound = s_list[0][top - 1];    // the top-th largest of the threads' maxima
    const int rounds = (p1 - p0 + THREADS - 1) / THREADS;
    int owners = 0;                         // threads whose maximum reaches it
    for (int i = 0; i < top; ++i) owners += s_list[0][i] != 0;
    const tl_key_t owner_key = s_list[0][lane];
    __syncthreads();
    // item q: piece q % rounds of owner q / rounds; owners are spread over the block
    for (int from = 0; from < owners * rounds; from += TL_CAND / 4) {
      const int to = min(owners * rounds, from + TL_CAND / 4);
      for (int q0 = from + warp * 32; q0 < to; q0 += THREADS) {
        const int q = q0 + lane;
        const int o = min(q / rounds, TL_TOP - 1);
        const tl_key_t ok = __shfl_sync(0xffffffffu, owner_key, o);
        const int p = (int)(((unsigned)(tl_index(ok) + row.off) / 4 - p0) % THREADS) + p0 +
                      (q % rounds) * THREADS;
        if (q < to && p < p1) {
          const float4 f = row.load(p);
          const float x[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int v = 4 * p - row.off + j;
            if (v < 0 || v >= vocab) continue;
            const tl_key_t k = tl_key(x[j], v);
            if (k >= bound) s_cand[atomicAdd(&s_found, 1)] = k;
          }
        }
      }
      __syncthreads();
      const int found = s_found;
      if (warp == 0) {
        for (int i = 0; i < found; i += 32)
          best = tl_merged(best, __shfl_sync(0xffffffffu, tl_sorted(i + lane < found ? s_cand[i + lane] : 0, lane),
                                             31 - lane), lane);
        s_list[0][lane] = best;
        if (lane == 0) s_found = 0;
      }
      __syncthreads();
      const tl_key_t reached = s_list[0][top - 1];
      if (reached > bound) bound = reached;
    }
  }
  __syncthreads();
  if (warp == 0) {
    all = lane < WARPS ? s_sum[lane] : TlSum{-INFINITY, 0.f};
    before = lane < WARPS ? s_before[lane] : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      all = tl_join(all, TlSum{__shfl_xor_sync(0xffffffffu, all.m, o), __shfl_xor_sync(0xffffffffu, all.s, o)});
    before = __reduce_add_sync(0xffffffffu, before);
  }
  if constexpr (BLOCKS > 1) {
    if (warp == 0) {
      s_list[0][lane] = best;
      if (lane == 0) {
        s_block = all;
        s_block_before = before;
      }
    }
    tl_cluster_sync();
    if (part == 0) {
      if (top > 0) {
        const tl_key_t k = warp < BLOCKS ? tl_remote(&s_list[0][lane], warp) : 0;
        __syncthreads();                    // (this block's own list is read before it is replaced)
        best = join_lists(k, BLOCKS);
      }
      if (warp == 0) {
        all = lane < BLOCKS ? TlSum{tl_remote(&s_block.m, lane), tl_remote(&s_block.s, lane)}
                            : TlSum{-INFINITY, 0.f};
        before = lane < BLOCKS ? tl_remote(&s_block_before, lane) : 0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
          all = tl_join(all, TlSum{__shfl_xor_sync(0xffffffffu, all.m, o), __shfl_xor_sync(0xffffffffu, all.s, o)});
        before = __reduce_add_sync(0xffffffffu, before);
      }
    }
    tl_cluster_sync();                      // the others stay until their memory has been read
  }
  if (part != 0 || warp != 0) return;
  const float log_sum = logf(all.s);
  // (without a maximum the sum is 0, or NaN where a NaN was: -inf then, or NaN)
  auto lp = [&](float x) { return all.m == -INFINITY ? log_sum : (x - all.m) - log_sum; };
  if (lane == 0) {
    logprob[w] = given ? lp(xt) : __int_as_float(0x7fffffff);
    rank[w] = given ? before : -1;
    if (!given && t != -1) atomicOr(status, HS_STATUS_BAD_TOKEN);
  }
  if (lane < top) {
    top_ids[(size_t)w * top + lane] = tl_index(best);
    top_logprobs[(size_t)w * top + lane] = lp(tl_value(best));
  }
}

template <int THREADS, int BLOCKS>
cudaError_t token_logprobs(float* logprob, int* rank, int* top_ids, float* top_logprobs, int top,
                           const float* logits, const int* tokens, int rows, int vocab, int* status,
                           cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(rows * BLOCKS);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = top > 0 ? TL_CAND * sizeof(tl_key_t) : 0;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (BLOCKS > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = BLOCKS;
    attr[n].val.clusterDim.y = 1;
    attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (hs_pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, token_logprobs_kernel<THREADS, BLOCKS>, logprob, rank, top_ids,
                            top_logprobs, top, logits, tokens, vocab, status);
}

}  // namespace hs

// tokens[w] == -1: no token (lp NaN, rank -1); any other index outside the vocabulary is reported.
HS_EXPORT int hs_token_logprobs(float* logprob, int* rank, int* top_ids, float* top_logprobs, int top,
                                const float* logits, const int* tokens, int rows, int vocab,
                                int* status, void* stream) {
  if (!logprob || !rank || !logits || !tokens || !status || vocab <= 0) return HS_ERR_ARGUMENT;
  if (((uintptr_t)logits & 3) != 0) return HS_ERR_ARGUMENT;
  if (top < 0 || top > hs::TL_TOP || top > vocab) return HS_ERR_UNSUPPORTED;
  if (top > 0 && (!top_ids || !top_logprobs)) return HS_ERR_ARGUMENT;
  if (rows <= 0) return HS_OK;
  if (rows > (1 << 27) || vocab > 0x7ffffff0) return HS_ERR_UNSUPPORTED;
  cudaStream_t st = (cudaStream_t)stream;
  const int blocks = vocab <= 4096 ? 1 : rows <= 74 ? 8 : rows <= 148 ? 4 : rows <= 296 ? 2 : 1;
  cudaError_t e;
#define TL_GO(THREADS, BLOCKS)                                                                      \
  e = hs::token_logprobs<THREADS, BLOCKS>(logprob, rank, top_ids, top_logprobs, top, logits, tokens, \
                                          rows, vocab, status, st)
  if (blocks == 8) TL_GO(512, 8);
  else if (blocks == 4) TL_GO(512, 4);
  else if (blocks == 2) TL_GO(512, 2);
  else if (vocab <= 4096) TL_GO(256, 1);
  else TL_GO(512, 1);
#undef TL_GO
  return e == cudaSuccess ? HS_OK : (int)e;
}
