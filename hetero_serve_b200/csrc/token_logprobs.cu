// Log-probabilities of given tokens, their ranks, and the largest alternatives.
//
// For row w with logits x and token t:  lp = (x_t - m) - log(sum_v exp(x_v - m)),  m = max_v x_v;
// rank = how many tokens stand before t, those of a larger logit and those of an equal one with a
// lower index (0: the greedy choice).  The n largest come in that order with their own lp.
// A row that is -inf throughout has no probabilities: every lp is -inf.  A NaN or +inf in a row makes
// all of its lp NaN; in the order a NaN stands behind everything else.
//
// One pass over the row: every thread keeps a running maximum with the sum of exp against it, and
// counts the logits before x_t.  For the alternatives the threads form 32 groups: the n-th largest of
// the groups' maxima is a bound that at least n logits reach, and not many more (about 30 of a row of
// any length for n = 20).  Only the threads whose own maximum reaches the bound look at their logits
// again, the block together; what they find is put in order by counting.  Where too many logits are
// equal for that (a row of zeros, of -inf), or NaNs leave too few, the threads' largest logits are
// ordered with their indices instead, which bounds what is looked at whatever the values are.
// A row is shared by the blocks of a cluster where there are few rows.
//
// Bound by the bytes of the logits where there are many rows (2,048 x 50,257 without alternatives:
// 66 us in a graph, 63 at the copy rate; the exponentials' pipe is half busy), by the chain of barriers
// behind the pass where there are few (one row: 3.8 us, 6.0 with 5 alternatives; 64 rows with 20: 9.6).
// Two numbers an instruction (add and mul on pairs), 2^x without the scaling of results below 2^-126,
// and counting before x_t only where a chunk holds something larger took the pass from 24
// instructions a logit to 11 (82 -> 69 us).
#include "common.cuh"

namespace hs {

constexpr int TL_TOP = 32;                // a warp's lanes hold the alternatives, in order
constexpr int TL_GROUPS = 32;             // of threads, whose maxima give the bound
constexpr int TL_CAND = 1024;             // logits looked at again at a time
constexpr int TL_FEW = 256;               // ... that are put in order by counting

typedef unsigned long long tl_key_t;

// order of (logit, index): larger logits first, among equal ones the lower index; zeros of both
// signs are equal, NaN is the smallest; 0 stands for no logit at all
__device__ __forceinline__ uint32_t tl_order(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return x != x ? 0u : (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ tl_key_t tl_key(float x, int v) {
  return ((tl_key_t)tl_order(x) << 32) | (uint32_t)~(uint32_t)v;
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

// 2^x, to two steps; what lies below the range of normal numbers is 0 (beside a sum of 1 or more)
__device__ __forceinline__ float tl_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float TL_LOG2E = 1.4426950408889634f;

// A running maximum and the sum of exp against it.  Nothing is subtracted from an infinite maximum:
// -inf stands for no logit yet (every term is then 0), +inf makes the sum NaN by itself.
struct TlSum {
  float m, s;
};
__device__ __forceinline__ float tl_term(float x, float m) {
  return tl_exp2((x - (m == -INFINITY ? 0.f : m)) * TL_LOG2E);
}
__device__ __forceinline__ TlSum tl_join(TlSum a, TlSum b) {
  const float m = fmaxf(a.m, b.m);
  return TlSum{m, a.s * tl_term(a.m, m) + b.s * tl_term(b.m, m)};
}

// two numbers at a time
typedef unsigned long long tl_pair;
__device__ __forceinline__ tl_pair tl_two(float a, float b) {
  tl_pair p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(a), "f"(b));
  return p;
}
__device__ __forceinline__ float2 tl_apart(tl_pair p) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p));
  return f;
}
__device__ __forceinline__ tl_pair tl_add(tl_pair a, tl_pair b) {
  tl_pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ tl_pair tl_mul(tl_pair a, tl_pair b) {
  tl_pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
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

// INFLIGHT: 16-byte loads a thread has under way
template <int THREADS, int BLOCKS, int INFLIGHT>
__global__ void __launch_bounds__(THREADS)
token_logprobs_kernel(float* __restrict__ logprob, int* __restrict__ rank, int* __restrict__ top_ids,
                      float* __restrict__ top_logprobs, int top, const float* __restrict__ logits,
                      const int* __restrict__ tokens, int vocab, int* status) {
  constexpr int WARPS = THREADS / 32, STEP = INFLIGHT * THREADS;
  static_assert(THREADS >= 2 * TL_GROUPS && THREADS >= BLOCKS * TL_TOP && BLOCKS * TL_TOP <= TL_CAND, "");
  __shared__ TlSum s_sum[WARPS];
  __shared__ int s_before[WARPS];
  __shared__ __align__(16) uint32_t s_group[TL_GROUPS];
  __shared__ tl_key_t s_list[WARPS][TL_TOP];
  __shared__ tl_key_t s_top[TL_TOP];    // the block's alternatives, in order
  __shared__ uint16_t s_owner[THREADS];
  __shared__ int s_owners, s_found, s_block_before;
  __shared__ TlSum s_block;
  extern __shared__ tl_key_t s_cand[];  // [TL_CAND] where alternatives are wanted
  pdl_trigger();
  pdl_wait();
  const int w = blockIdx.x / BLOCKS, part = BLOCKS > 1 ? (int)tl_rank() : 0;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // a row is up to three logits, pieces of four that begin on 16 bytes, and up to three logits
  const float* base = logits + (size_t)w * vocab;
  const int head = min(vocab, (int)((4 - (((uintptr_t)base >> 2) & 3)) & 3));
  const int pieces = (vocab - head) / 4, tail = (vocab - head) % 4;
  const int per = (pieces + BLOCKS - 1) / BLOCKS;
  const int p0 = min(pieces, part * per), p1 = min(pieces, p0 + per);
  const float4* row = (const float4*)(base + head);
  // the logits outside the pieces: a thread each, of the first block
  const int edge = part != 0 || tid >= head + tail ? -1 : tid < head ? tid : head + 4 * pieces + tid - head;

  const int t = tokens[w];
  const bool given = t >= 0 && t < vocab;
  const float xt = given ? base[t] + 0.f : INFINITY;
  // x stands before x_t where x > x_t, and where x = x_t with a lower index: that is x > the number
  // below x_t there.  (x_t NaN or -inf has no number below it: those rows compare keys.)
  const bool by_key = !(xt > -INFINITY);
  const float below = xt == INFINITY ? 3.402823466e38f : nextafterf(xt, -INFINITY);
  const tl_key_t mine = given ? tl_key(xt, t) : ~0ull;

  TlSum own{-INFINITY, 0.f};
  int before = 0;
  if (edge >= 0) {
    const float x = base[edge];
    own = TlSum{fmaxf(x, -INFINITY), x != x ? x : x == -INFINITY ? 0.f : tl_term(x, x)};
    before = tl_key(x, edge) > mine;
  }
  float m_pieces = -INFINITY;             // the largest in the thread's pieces
  auto chunk = [&](int at, bool whole) {  // pieces at + tid, + THREADS, ...
    float4 f[INFLIGHT];
#pragma unroll
    for (int i = 0; i < INFLIGHT; ++i) {
      f[i] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      if (whole || at + tid + i * THREADS < p1) f[i] = row[at + tid + i * THREADS];
    }
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < INFLIGHT; ++i)
      m = fmaxf(fmaxf(fmaxf(m, f[i].x), f[i].y), fmaxf(f[i].z, f[i].w));
    m_pieces = fmaxf(m_pieces, m);
    if (m > own.m) {
      own.s *= tl_term(own.m, m);
      own.m = m;
    }
    const float ref = own.m == -INFINITY ? 0.f : -own.m;
    const tl_pair ref2 = tl_two(ref, ref), scale2 = tl_two(TL_LOG2E, TL_LOG2E);
    tl_pair sum2 = tl_two(own.s, 0.f);
#pragma unroll
    for (int i = 0; i < INFLIGHT; ++i) {
      const float2 a = tl_apart(tl_mul(tl_add(tl_two(f[i].x, f[i].y), ref2), scale2));
      const float2 b = tl_apart(tl_mul(tl_add(tl_two(f[i].z, f[i].w), ref2), scale2));
      sum2 = tl_add(sum2, tl_two(tl_exp2(a.x), tl_exp2(a.y)));
      sum2 = tl_add(sum2, tl_two(tl_exp2(b.x), tl_exp2(b.y)));
    }
    const float2 sum = tl_apart(sum2);
    own.s = sum.x + sum.y;
    if (by_key) {
#pragma unroll
      for (int i = 0; i < INFLIGHT; ++i) {
        const int p = at + tid + i * THREADS, v = head + 4 * p;
        if (p < p1)
          before += (tl_key(f[i].x, v) > mine) + (tl_key(f[i].y, v + 1) > mine) +
                    (tl_key(f[i].z, v + 2) > mine) + (tl_key(f[i].w, v + 3) > mine);
      }
    } else if (m > below) {               // (most often nothing here stands before the token)
#pragma unroll
      for (int i = 0; i < INFLIGHT; ++i) {
        const int v = head + 4 * (at + tid + i * THREADS);
        before += (f[i].x > (v < t ? below : xt)) + (f[i].y > (v + 1 < t ? below : xt)) +
                  (f[i].z > (v + 2 < t ? below : xt)) + (f[i].w > (v + 3 < t ? below : xt));
      }
    }
  };
  int at = p0;
  for (; at + STEP <= p1; at += STEP) chunk(at, true);
  if (at < p1) chunk(at, false);

  TlSum all = own;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    all = tl_join(all, TlSum{__shfl_xor_sync(0xffffffffu, all.m, o), __shfl_xor_sync(0xffffffffu, all.s, o)});
  before = __reduce_add_sync(0xffffffffu, before);
  if (lane == 0) {
    s_sum[warp] = all;
    s_before[warp] = before;
  }

  if (top > 0) {
    const bool holds = p0 + tid < p1;
    const int rounds = (p1 - p0 + THREADS - 1) / THREADS;
    const int elements = 4 * (p1 - p0) + (part == 0 ? head + tail : 0);
    // piece `round` of thread `who`, or one behind the block's
    auto again = [&](int who, int round, tl_key_t bound) {
      const int p = p0 + who + round * THREADS;
      if (p >= p1) return;
      const float4 f = row[p];
      const float x[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const tl_key_t k = tl_key(x[j], head + 4 * p + j);
        if (k >= bound) {
          const int i = atomicAdd(&s_found, 1);
          if (i < TL_CAND) s_cand[i] = k;
        }
      }
    };
    auto again_edge = [&](tl_key_t bound) {
      if (edge < 0) return;
      const tl_key_t k = tl_key(base[edge], edge);
      if (k >= bound) {
        const int i = atomicAdd(&s_found, 1);
        if (i < TL_CAND) s_cand[i] = k;
      }
    };
    const uint32_t own_order = holds ? tl_order(m_pieces) : 0u;
    uint32_t g = own_order;
#pragma unroll
    for (int o = THREADS / TL_GROUPS / 2; o > 0; o >>= 1) g = max(g, __shfl_xor_sync(0xffffffffu, g, o));
    if (tid % (THREADS / TL_GROUPS) == 0) s_group[tid / (THREADS / TL_GROUPS)] = g;
    if (tid == 0) s_owners = s_found = 0;
    if (tid < TL_TOP) s_top[tid] = 0;
    __syncthreads();
    uint32_t reach = s_group[lane];
    int larger = 0;
#pragma unroll
    for (int i = 0; i < TL_GROUPS; i += 4) {
      const uint4 o = *(const uint4*)&s_group[i];
      larger += (o.x >= reach) + (o.y >= reach) + (o.z >= reach) + (o.w >= reach);
    }
    reach = __reduce_max_sync(0xffffffffu, larger >= top ? reach : 0u);
    if (holds && own_order >= reach) s_owner[atomicAdd(&s_owners, 1)] = (uint16_t)tid;
    __syncthreads();
    const int owners = s_owners;
    bool done = owners <= TL_FEW;         // else more is equal than a list takes, or nearly so
    if (done) {
      for (int q = tid; q < owners * rounds; q += THREADS)
        again(s_owner[q / rounds], q % rounds, (tl_key_t)reach << 32);
      again_edge((tl_key_t)reach << 32);
      __syncthreads();
      const int found = s_found;
      done = found <= TL_FEW && found >= min(top, elements);
      if (done) {
        for (int i = tid; i < found; i += THREADS) {
          const tl_key_t k = s_cand[i];
          int place = 0;
          for (int j = 0; j < found; ++j) place += s_cand[j] > k;
          if (place < TL_TOP) s_top[place] = k;
        }
      }
      __syncthreads();
    }
    if (!done) {
      // the threads' largest keys in order: those of the first `top` hold what is looked for
      tl_key_t key = 0;
      for (int p = p0 + tid; p < p1; p += THREADS) {
        const float4 f = row[p];
        const float x[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const tl_key_t k = tl_key(x[j], head + 4 * p + j);
          if (k > key) key = k;
        }
      }
      tl_key_t k = tl_sorted(key, lane);
      s_list[warp][lane] = k;
      if (tid == 0) s_found = 0;
      __syncthreads();
      for (int half = WARPS / 2; half > 0; half >>= 1) {
        if (warp < half) {
          k = tl_merged(k, s_list[warp + half][31 - lane], lane);
          s_list[warp][lane] = k;
        }
        __syncthreads();
      }
      tl_key_t bound = s_list[0][top - 1];
      const int who = (int)((unsigned)(tl_index(s_list[0][lane]) - head) / 4 - p0) % THREADS;
      const int last = __popc(__ballot_sync(0xffffffffu, lane < top && s_list[0][lane] != 0));
      __syncthreads();
      tl_key_t best = 0;                  // warp 0: what has been found so far, in order
      again_edge(bound);
      constexpr int ITEMS = (TL_CAND - 8) / 4;
      for (int from = 0; from == 0 || from < last * rounds; from += ITEMS) {
        const int to = min(last * rounds, from + ITEMS);
        for (int q0 = from + warp * 32; q0 < to; q0 += THREADS) {
          const int q = q0 + lane, thread = __shfl_sync(0xffffffffu, who, min(q / rounds, 31));
          if (q < to) again(thread, q % rounds, bound);
        }
        __syncthreads();
        const int found = s_found;
        __syncthreads();
        if (warp == 0) {
          for (int i = 0; i < found; i += 32) {
            const tl_key_t next = tl_sorted(i + lane < found ? s_cand[i + lane] : 0, lane);
            best = tl_merged(best, __shfl_sync(0xffffffffu, next, 31 - lane), lane);
          }
          s_top[lane] = best;
          if (lane == 0) s_found = 0;
        }
        __syncthreads();
        if (s_top[top - 1] > bound) bound = s_top[top - 1];
        __syncthreads();
      }
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
    if (lane == 0) {
      s_block = all;
      s_block_before = before;
    }
  }
  if constexpr (BLOCKS > 1) {
    tl_cluster_sync();
    if (part == 0) {
      tl_key_t k = 0;
      if (tid < BLOCKS * top) {
        k = tl_remote(&s_top[tid % top], tid / top);
        s_cand[tid] = k;
      }
      if (warp == WARPS - 1) {            // (a warp that has no list to fetch where there are others)
        all = lane < BLOCKS ? TlSum{tl_remote(&s_block.m, lane), tl_remote(&s_block.s, lane)}
                            : TlSum{-INFINITY, 0.f};
        before = lane < BLOCKS ? tl_remote(&s_block_before, lane) : 0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
          all = tl_join(all, TlSum{__shfl_xor_sync(0xffffffffu, all.m, o), __shfl_xor_sync(0xffffffffu, all.s, o)});
        before = __reduce_add_sync(0xffffffffu, before);
      }
      __syncthreads();                    // (the block's own share has been read as well)
      if (warp == WARPS - 1 && lane == 0) {
        s_block = all;
        s_block_before = before;
      }
      if (k != 0) {
        int place = 0;
        for (int j = 0; j < BLOCKS * top; ++j) place += s_cand[j] > k;
        if (place < top) s_list[0][place] = k;
      }
    }
    tl_cluster_sync();                    // the others stay until their memory has been read
    if (part != 0) return;
  } else {
    __syncthreads();
  }
  const tl_key_t* found = BLOCKS > 1 ? s_list[0] : s_top;
  const TlSum total = s_block;
  const float log_sum = logf(total.s);
  // (without a maximum the sum is 0, or NaN where a NaN was: -inf then, or NaN)
  auto lp = [&](float x) { return total.m == -INFINITY ? log_sum : (x - total.m) - log_sum; };
  if (tid == 0) {
    logprob[w] = given ? lp(xt) : __int_as_float(0x7fffffff);
    rank[w] = given ? s_block_before : -1;
    if (!given && t != -1) atomicOr(status, HS_STATUS_BAD_TOKEN);
  }
  if (tid < top) {
    const tl_key_t k = found[tid];
    top_ids[(size_t)w * top + tid] = tl_index(k);
    top_logprobs[(size_t)w * top + tid] = lp(tl_value(k));
  }
}

template <int THREADS, int BLOCKS, int INFLIGHT>
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
  return cudaLaunchKernelEx(&cfg, token_logprobs_kernel<THREADS, BLOCKS, INFLIGHT>, logprob, rank, top_ids,
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
  // A long row over 8, 4 or 2 blocks of 512 threads, as many as find room at once: two such blocks fit an
  // SM, and a cluster of 8 or 4 needs its SMs in one group of the chip, so that 35 clusters of 8, and 74 of
  // 4, take turns on 148 SMs.  us in a graph over 8, 4, 2 and 1 blocks, rows of 50,257 logits:
  //   rows   without alternatives     with 20
  //     1     3.7  4.1  4.8  5.8       7.4  7.2  7.3  8.8
  //    12     4.2  4.6  5.2  6.1       8.4  7.3  7.7  9.3
  //    24     4.8  5.0  5.4  6.2       9.1  8.1  8.2  9.4
  //    35     6.9  5.3  5.3  6.1      14.2  8.7  8.2  9.2
  //    64     8.6  5.9  6.9  6.3      17.1  9.1  9.8  9.3
  //    74    10.9  8.2  5.5  6.4      22.3 13.9  8.2  9.7
  //   148    18.5 12.6  7.4  6.5      37.1 21.0 10.8  9.5
  // (131,072 logits, 20 alternatives: 12 rows 9.1, 8.6, 10.3, 15.2; 128 rows 34.9, 20.9, 15.0, 21.2).  One rule
  // by rows for both, which costs up to 1.6 us where they differ: 12 rows with 20 alternatives are faster over 4,
  // 24 without over 8, 148 over one.  Rows up to 24,576 long go to one block: longer ones gain from the cluster
  // without alternatives first (1 x 24,577 over 8 3.7, over one 3.9; with 20 alternatives 7.0 and 6.1, 64 rows
  // over 4 8.2, over one 6.6).
  // Short rows take half the threads (128 x 4,096: 4.8, with 512 threads 6.1) or a quarter (512 x 1,000:
  // 5.9, with 256 threads 7.2); long ones that want no alternatives take half of them too once four
  // blocks an SM do not hold them all (600 x 50,257: 26 and 28, 2,048 x 50,257: 66 and 69; but 512 x
  // 50,257: 22 and 17).  Rows that fill the SMs have three loads a thread under way, which leaves an SM
  // the registers for another block (512 x 50,257 with four: 19.8, with three 16.5).
  const int sms = hs_sm_count();
  const int blocks = vocab <= 24576 ? 1 : rows <= 12 ? 8 : rows <= 64 ? 4 : rows <= sms ? 2 : 1;
  cudaError_t e;
#define TL_GO(THREADS, BLOCKS, INFLIGHT)                                                              \
  e = hs::token_logprobs<THREADS, BLOCKS, INFLIGHT>(logprob, rank, top_ids, top_logprobs, top, logits, \
                                                    tokens, rows, vocab, status, st)
  if (blocks == 8) TL_GO(512, 8, 4);
  else if (blocks == 4) TL_GO(512, 4, 4);
  else if (blocks == 2) TL_GO(512, 2, 4);
  else if (vocab <= 2048) TL_GO(128, 1, 4);
  else if (vocab <= 8192) TL_GO(256, 1, 4);
  else if (top == 0 && rows > 4 * sms) TL_GO(256, 1, 3);
  else TL_GO(512, 1, 3);
#undef TL_GO
  return e == cudaSuccess ? HS_OK : (int)e;
}
