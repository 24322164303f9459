// Copies of cache pages, in every cache entry of a group at once.
//
// A pool is [entries, pages, tiles, rows, row bytes] (tiles: planes x heads).  For each listed pair
// i and each entry e:  dst[e, d_i, :, :r_i] = src[e, s_i, :, :r_i];  rows behind the first r_i of a
// page stay as they were.  dst and src may be one pool: the caller sees to it that no page is
// written twice, nor written and read.  The list travels as a kernel argument, so that no copy of
// it has to be made on the device, and kept there, before the launch.
//
// Bound by the bytes, each read and written once: 2,500 pages of 12 entries (1.47 GB one way) take 454 us,
// 6.5 TB/s, the rate of a plain copy.  A few pages are bound by the launch: 7 half pages of 24
// entries 3.0 us.  48 pages of 24 entries in float32, half filled, took 25 us as a block a page and
// entry and 18 in shares with four 16-byte loads a thread under way (mostly from the L2); 20 pages of 13
// entries of 48 KB filled 9.7 us with shares of 64 KB and 5.5 with shares that give an SM eight blocks.
#include "common.cuh"

namespace hs {

constexpr int PC_THREADS = 256, PC_INFLIGHT = 4;
constexpr int PC_FEW = 32, PC_MANY = 1024;     // pairs a launch takes

template <int PAIRS>
struct PageList {
  int dst[PAIRS], src[PAIRS];
  short rows[PAIRS];
};

// One block a pair, an entry and a share of the page's filled rows, counted in pieces of V.
template <typename V, int PAIRS>
__global__ void __launch_bounds__(PC_THREADS)
copy_pages_kernel(V* dst, const V* src, long long dst_pages, long long src_pages, int tiles,
                  int page_rows, int row_vecs, int share, const __grid_constant__ PageList<PAIRS> list) {
  pdl_trigger();
  pdl_wait();
  const int i = blockIdx.x, e = blockIdx.y;
  const int tile_vecs = page_rows * row_vecs, live = list.rows[i] * row_vecs;
  const bool whole = live == tile_vecs;
  const size_t page_vecs = (size_t)tiles * tile_vecs;
  V* to = dst + (e * dst_pages + list.dst[i]) * page_vecs;
  const V* from = src + (e * src_pages + list.src[i]) * page_vecs;
  const int j0 = blockIdx.z * share, j1 = min(tiles * live, j0 + share);
  for (int j = j0 + threadIdx.x; j < j1; j += PC_INFLIGHT * PC_THREADS) {
    V x[PC_INFLIGHT];
    int at[PC_INFLIGHT];
#pragma unroll
    for (int k = 0; k < PC_INFLIGHT; ++k) {
      const int q = j + k * PC_THREADS;
      at[k] = whole ? q : q / live * tile_vecs + q % live;
      if (q < j1) x[k] = from[at[k]];
    }
#pragma unroll
    for (int k = 0; k < PC_INFLIGHT; ++k)
      if (j + k * PC_THREADS < j1) to[at[k]] = x[k];
  }
}

template <typename V, int PAIRS>
cudaError_t copy_pages(void* dst, const void* src, int n, const int* dst_list, const int* src_list,
                       const int* rows, int entries, int dst_pages, int src_pages, int tiles,
                       int page_rows, int row_bytes, cudaStream_t stream) {
  const int sms = hs_sm_count();
  for (int from = 0; from < n; from += PAIRS) {
    const int count = n - from < PAIRS ? n - from : PAIRS;
    PageList<PAIRS> list;
    for (int i = 0; i < count; ++i) {
      list.dst[i] = dst_list[from + i];
      list.src[i] = src_list[from + i];
      list.rows[i] = (short)(rows ? rows[from + i] : page_rows);
    }
    // shares of a page of up to four rounds of a block's loads, eight of them an SM where the page gives them
    const int row_vecs = (int)(row_bytes / sizeof(V)), page_vecs = tiles * page_rows * row_vecs;
    const int round = PC_INFLIGHT * PC_THREADS;
    int share = 4 * round;
    while (share > round && (long long)count * entries * ((page_vecs + share - 1) / share) < 8LL * sms) share /= 2;
    const int shares = (page_vecs + share - 1) / share;
    if (shares > 65535) return cudaErrorInvalidValue;
    const cudaError_t e = hs_launch(copy_pages_kernel<V, PAIRS>, dim3(count, entries, shares),
                                    dim3(PC_THREADS), 0, stream, hs_pdl_enabled(), (V*)dst,
                                    (const V*)src, (long long)dst_pages, (long long)src_pages, tiles,
                                    page_rows, row_vecs, share, list);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace hs

// The lists (n numbers each; rows may be null: whole pages) are in host memory and are read before
// this returns.  Numbers outside the pools are refused here, before anything is launched.
HS_EXPORT int hs_copy_pages(void* dst, const void* src, int n, const int* dst_list,
                            const int* src_list, const int* rows, int entries, int dst_pages,
                            int src_pages, int tiles, int page_rows, int row_bytes, void* stream) {
  if (n <= 0) return HS_OK;
  if (!dst || !src || !dst_list || !src_list) return HS_ERR_ARGUMENT;
  if (entries <= 0 || entries > 65535 || tiles <= 0 || page_rows <= 0 || page_rows > 32767 ||
      row_bytes <= 0 || row_bytes % 2 || (long long)tiles * page_rows * row_bytes > (1LL << 27))
    return HS_ERR_UNSUPPORTED;
  for (int i = 0; i < n; ++i)
    if (dst_list[i] < 0 || dst_list[i] >= dst_pages || src_list[i] < 0 || src_list[i] >= src_pages ||
        (rows && (rows[i] < 0 || rows[i] > page_rows)))
      return HS_ERR_ARGUMENT;
  if (!rows) {                 // whole pages lie in one piece
    row_bytes *= tiles * page_rows;
    tiles = page_rows = 1;
  }
  const uintptr_t bits = (uintptr_t)dst | (uintptr_t)src | (uintptr_t)row_bytes;
  cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e;
#define PC_GO(V)                                                                                     \
  e = n <= hs::PC_FEW                                                                                \
          ? hs::copy_pages<V, hs::PC_FEW>(dst, src, n, dst_list, src_list, rows, entries, dst_pages, \
                                          src_pages, tiles, page_rows, row_bytes, st)                \
          : hs::copy_pages<V, hs::PC_MANY>(dst, src, n, dst_list, src_list, rows, entries, dst_pages, \
                                           src_pages, tiles, page_rows, row_bytes, st)
  if (bits % 16 == 0) PC_GO(uint4);
  else if (bits % 8 == 0) PC_GO(uint2);
  else if (bits % 4 == 0) PC_GO(uint32_t);
  else PC_GO(uint16_t);
#undef PC_GO
  return e == cudaSuccess ? HS_OK : (int)e;
}
