// Plans for the low-rank adapters: rows sorted by the adapter of their request, cut into tiles of rows of one adapter.
//
// A bin is an adapter 0 .. n-1, or n for the rows without one (request without an adapter, an adapter outside [0, n), a row
// behind the last request). The rows of a bin keep their order (a stable counting sort), so a plan depends on its input alone.
//
// Tile list, int32: [0] count, [1..3] unused, then count + 1 pairs (first position, matrix); a tile ends where the next one
// starts, matrix -1: rows without an adapter.
#include <algorithm>

#include "dst_common.cuh"

namespace dst {
namespace {

constexpr int PLAN_THREADS = 1024, PLAN_WARPS = 32, PLAN_ROWS = 16384, PLAN_BINS = 1024;  // of the one-block forms

// The bin of a row: the request that it lies in is the last one that starts at or before it.
__device__ __forceinline__ int bin_of_row(const int32_t* __restrict__ offsets, const int32_t* __restrict__ slots, int64_t requests, int64_t row,
                                          int n) {
  int64_t r = row;
  if (offsets) {
    int64_t lo = 0, hi = requests + 1;  // the first index whose offset is above the row
    while (lo < hi) {
      const int64_t mid = (lo + hi) >> 1;
      if (offsets[mid] <= row) lo = mid + 1;
      else hi = mid;
    }
    r = lo - 1;
  }
  if (r < 0 || r >= requests) return n;
  const int s = slots[r];
  return s >= 0 && s < n ? s : n;
}

// Exclusive sums of val[0 .. count) in place by the whole block, count <= 1024 per pass of its threads; returns the total.
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int incl = v;
  for (int d = 1; d < 32; d <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += up;
  }
  if (lane == 31) warp_sums[warp] = incl;
  __syncthreads();
  int before = 0;
  total = 0;
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) {
    if (w < warp) before += warp_sums[w];
    total += warp_sums[w];
  }
  __syncthreads();
  return before + incl - v;
}

// The whole plan by one block: each warp counts and places a run of consecutive rows of its own.
__global__ void __launch_bounds__(PLAN_THREADS)
plan_kernel(const int32_t* __restrict__ offsets, const int32_t* __restrict__ slots, int64_t requests, int rows, int n, int tile,
            int32_t* __restrict__ order, int32_t* __restrict__ bins, int32_t* __restrict__ bin_offsets, int32_t* __restrict__ tiles) {
  extern __shared__ int32_t sh[];
  const int nb = n + 1, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int32_t* hist = sh;                       // [PLAN_WARPS][nb]
  int32_t* start = hist + PLAN_WARPS * nb;  // [nb + 1]
  int32_t* tstart = start + nb + 1;         // [nb + 1]
  uint16_t* bin_s = reinterpret_cast<uint16_t*>(tstart + nb + 1);  // [rows]
  __shared__ int sums[32];
  for (int i = tid; i < PLAN_WARPS * nb; i += PLAN_THREADS) hist[i] = 0;
  __syncthreads();
  const int per = ((rows + PLAN_WARPS - 1) / PLAN_WARPS + 31) & ~31;
  const int r0 = min(warp * per, rows), r1 = min(r0 + per, rows);
  int32_t* mine = hist + warp * nb;
  for (int r = r0; r < r1; r += 32) {
    const bool in = r + lane < r1;
    const int b = in ? bin_of_row(offsets, slots, requests, r + lane, n) : -1;
    const unsigned peers = __match_any_sync(0xffffffffu, b);
    if (in) {
      bin_s[r + lane] = (uint16_t)b;
      if (lane == __ffs(peers) - 1) mine[b] += __popc(peers);
    }
    __syncwarp();
  }
  __syncthreads();
  int count = 0;
  if (tid < nb)
    for (int w = 0; w < PLAN_WARPS; ++w) {
      const int v = hist[w * nb + tid];
      hist[w * nb + tid] = count;
      count += v;
    }
  int total, n_tiles;
  const int at = block_scan(count, sums, total);
  const int tat = block_scan((count + tile - 1) / tile, sums, n_tiles);
  if (tid < nb) start[tid] = at, tstart[tid] = tat, bin_offsets[tid] = at;
  if (tid == 0) start[nb] = rows, tstart[nb] = n_tiles, bin_offsets[nb] = rows, tiles[0] = n_tiles;
  __syncthreads();
  int2* list = reinterpret_cast<int2*>(tiles + 4);
  for (int i = tid; i <= n_tiles; i += PLAN_THREADS) {
    int lo = 0, hi = nb;  // the last bin whose tiles start at or before i and which has some
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (mid <= nb - 1 && tstart[mid] <= i) lo = mid;
      else hi = mid - 1;
    }
    list[i] = i == n_tiles ? make_int2(rows, -1) : make_int2(start[lo] + (i - tstart[lo]) * tile, lo < n ? lo : -1);
  }
  for (int r = r0; r < r1; r += 32) {
    const bool in = r + lane < r1;
    const int b = in ? (int)bin_s[r + lane] : -1;
    const unsigned peers = __match_any_sync(0xffffffffu, b);
    if (in) {
      const int p = start[b] + mine[b] + __popc(peers & ((1u << lane) - 1u));
      order[p] = r + lane;
      bins[p] = b;
    }
    __syncwarp();
    if (in && lane == __ffs(peers) - 1) mine[b] += __popc(peers);
    __syncwarp();
  }
}

// More rows or adapters: the bins, the routing sort over them, then the lists from its result.
__global__ void bins_kernel(const int32_t* __restrict__ offsets, const int32_t* __restrict__ slots, int64_t requests, int64_t rows, int n,
                            int32_t* __restrict__ bin) {
  const int64_t r = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (r < rows) bin[r] = bin_of_row(offsets, slots, requests, r, n);
}

__global__ void __launch_bounds__(PLAN_THREADS)
lists_kernel(const int64_t* __restrict__ order64, const int64_t* __restrict__ offsets64, const int32_t* __restrict__ bin, int64_t rows, int n,
             int tile, int32_t* __restrict__ order, int32_t* __restrict__ bins, int32_t* __restrict__ bin_offsets, int32_t* __restrict__ tiles) {
  for (int64_t p = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; p < rows; p += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = order64[p];
    order[p] = (int32_t)r;
    bins[p] = bin[r];
  }
  if (blockIdx.x) return;
  __shared__ int sums[32];
  int2* list = reinterpret_cast<int2*>(tiles + 4);
  int done = 0;
  for (int b0 = 0; b0 <= n; b0 += PLAN_THREADS) {
    const int b = b0 + threadIdx.x;
    const int64_t a = b <= n ? offsets64[b] : 0, e = b <= n ? offsets64[b + 1] : 0;
    int total;
    const int at = done + block_scan((int)((e - a + tile - 1) / tile), sums, total);
    if (b <= n) {
      bin_offsets[b] = (int32_t)a;
      int i = at;
      for (int64_t p = a; p < e; p += tile) list[i++] = make_int2((int)p, b < n ? b : -1);
    }
    done += total;
  }
  if (threadIdx.x == 0) {
    bin_offsets[n + 1] = (int32_t)rows;
    tiles[0] = done;
    list[done] = make_int2((int)rows, -1);
  }
}

// ------------------------------------------------------------------------------------ pairs of a MoE layer
// Pairs (token, choice) sorted by expert and, inside an expert, by bin: the stable routing sort over the pairs in the plan's
// order of tokens does both, since that order is the bins'. A tile starts where the expert or the bin changes and at every
// multiple of the tile height.
__global__ void pair_ids_kernel(const int32_t* __restrict__ ids, const int32_t* __restrict__ order, int64_t pairs, int k, int E,
                                int32_t* __restrict__ permuted) {
  const int64_t q = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (q >= pairs) return;
  const int e = ids[(int64_t)order[q / k] * k + q % k];
  permuted[q] = e >= 0 && e < E ? e : -1;
}

struct PairLists {
  const int64_t* sorted;      // position -> pair in the plan's order of tokens, -1: dropped
  const int32_t* permuted;    // its expert
  const int32_t *order, *bins;
  int64_t pairs;
  int k, E, n, tile;
  int64_t* pair_order;        // position -> token * k + choice, -1: dropped
  int32_t *x_rows, *tiles, *counts;
};

__device__ __forceinline__ int pair_matrix(const PairLists& a, int64_t p, int64_t& pair, int32_t& token) {
  const int64_t q = a.sorted[p];
  pair = -1, token = 0;
  if (q < 0) return -2;
  token = a.order[q / a.k];
  pair = (int64_t)token * a.k + q % a.k;
  const int b = a.bins[q / a.k], e = a.permuted[q];
  return b < a.n ? b * a.E + e : -1 - 2 * (e + 1);  // no adapter: one negative number per expert
}

// PLACE false: the tile starts of each block's positions are counted; true: they are written behind those of the blocks before
template <bool PLACE>
__global__ void __launch_bounds__(PLAN_THREADS) pair_lists_kernel(const PairLists a) {
  __shared__ int sums[32];
  const int64_t p = (int64_t)blockIdx.x * PLAN_THREADS + threadIdx.x;
  bool starts = false;
  int m = -2;
  if (p < a.pairs) {
    int64_t pair, other;
    int32_t token, unused;
    m = pair_matrix(a, p, pair, token);
    const int before = p ? pair_matrix(a, p - 1, other, unused) : -2;
    starts = m != -2 && (m != before || p % a.tile == 0);
    if (!PLACE) a.pair_order[p] = pair, a.x_rows[p] = token;
  }
  int total;
  int at = block_scan(starts, sums, total);
  if (!PLACE) {
    if (threadIdx.x == 0) a.counts[blockIdx.x] = total;
    return;
  }
  int before = 0;
  for (int b = threadIdx.x; b < (int)blockIdx.x; b += PLAN_THREADS) before += a.counts[b];
  int base, unused;
  unused = block_scan(before, sums, base);
  (void)unused;
  at += base;
  int2* list = reinterpret_cast<int2*>(a.tiles + 4);
  if (starts) list[at] = make_int2((int)p, m < 0 ? -1 : m);
  if (blockIdx.x == gridDim.x - 1 && threadIdx.x == 0) {
    a.tiles[0] = base + total;
    list[base + total] = make_int2((int)a.tiles[2], -1);
  }
}

__global__ void pair_count_kernel(const int64_t* __restrict__ offsets, int E, int32_t* __restrict__ tiles) { tiles[2] = (int32_t)offsets[E]; }

size_t align16(size_t v) { return (v + 15) & ~(size_t)15; }

}  // namespace
}  // namespace dst

extern "C" int64_t dst_adapter_tile_capacity(int64_t rows, int64_t bins, int tile) {
  if (rows < 0 || bins <= 0 || tile <= 0) return 0;
  return 4 + 2 * (std::min(rows, dst::cdiv64(rows, tile) + bins) + 1);
}

extern "C" size_t dst_adapter_plan_workspace_bytes(int64_t rows, int64_t n) {
  using namespace dst;
  if (rows <= 0 || n <= 0 || (rows <= PLAN_ROWS && n < PLAN_BINS)) return 0;
  return align16(rows * 4) + align16(rows * 8) + align16((n + 2) * 8) + align16(dst_sort_workspace_bytes(rows, n + 1));
}

extern "C" int dst_adapter_plan(const int32_t* offsets, const int32_t* slots, int64_t requests, int64_t rows, int64_t n, int tile,
                                int32_t* order, int32_t* bins, int32_t* bin_offsets, int32_t* tiles, void* workspace, size_t workspace_bytes,
                                dst_stream_t stream) {
  using namespace dst;
  if (rows < 0 || requests < 0 || n <= 0 || tile <= 0) return DST_ERR_BAD_ARG;
  if (rows > 0x7fffffff || requests > 0x7ffffffe || n > 4095) return DST_ERR_BAD_SHAPE;
  if (!bin_offsets || !tiles || (rows > 0 && (!order || !bins)) || (requests > 0 && !slots)) return DST_ERR_BAD_ARG;
  if ((reinterpret_cast<uintptr_t>(tiles) & 7) != 0) return DST_ERR_ALIGNMENT;
  auto st = static_cast<cudaStream_t>(stream);
  if (rows <= PLAN_ROWS && n < PLAN_BINS) {
    const size_t smem = ((size_t)PLAN_WARPS * (n + 1) + 2 * (n + 2)) * 4 + (size_t)rows * 2;  // at most 168 KB
    if (smem > 48 * 1024) DST_CUDA_TRY(cudaFuncSetAttribute(plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    plan_kernel<<<1, PLAN_THREADS, smem, st>>>(offsets, slots, requests, (int)rows, (int)n, tile, order, bins, bin_offsets, tiles);
    DST_CUDA_TRY(cudaGetLastError());
    return DST_OK;
  }
  if (rows == 0) {
    DST_CUDA_TRY(cudaMemsetAsync(bin_offsets, 0, (size_t)(n + 2) * sizeof(int32_t), st));
    DST_CUDA_TRY(cudaMemsetAsync(tiles, 0, 6 * sizeof(int32_t), st));  // no tile, the end at position 0
    return DST_OK;
  }
  if (!workspace || workspace_bytes < dst_adapter_plan_workspace_bytes(rows, n)) return DST_ERR_BAD_ARG;
  char* w = static_cast<char*>(workspace);
  int32_t* bin = reinterpret_cast<int32_t*>(w);
  int64_t* order64 = reinterpret_cast<int64_t*>(w += align16(rows * 4));
  int64_t* offsets64 = reinterpret_cast<int64_t*>(w += align16(rows * 8));
  bins_kernel<<<(unsigned)cdiv64(rows, 256), 256, 0, st>>>(offsets, slots, requests, rows, (int)n, bin);
  DST_CUDA_TRY(cudaGetLastError());
  const int rc = sort_rows(bin, 1, rows, n + 1, order64, offsets64, nullptr, w + align16((n + 2) * 8), nullptr, st);
  if (rc != DST_OK) return rc;
  lists_kernel<<<(unsigned)std::min<int64_t>(cdiv64(rows, PLAN_THREADS), 296), PLAN_THREADS, 0, st>>>(order64, offsets64, bin, rows, (int)n, tile,
                                                                                                    order, bins, bin_offsets, tiles);
  DST_CUDA_TRY(cudaGetLastError());
  return DST_OK;
}

extern "C" size_t dst_adapter_plan_experts_workspace_bytes(int64_t pairs, int64_t E) {
  using namespace dst;
  if (pairs <= 0 || E <= 0) return 0;
  return align16(pairs * 4) + align16(pairs * 8) + align16(cdiv64(pairs, PLAN_THREADS) * 4) + align16(dst_sort_workspace_bytes(pairs, E));
}

extern "C" int dst_adapter_plan_experts(const int32_t* ids, int64_t T, int top_k, int64_t E, const int32_t* order, const int32_t* bins, int64_t n,
                                        int tile, int64_t* pair_order, int64_t* offsets, int32_t* x_rows, int32_t* tiles, void* workspace,
                                        size_t workspace_bytes, dst_stream_t stream) {
  using namespace dst;
  if (T < 0 || top_k <= 0 || E <= 0 || n <= 0 || tile <= 0) return DST_ERR_BAD_ARG;
  if (T > 0x7fffffff / top_k || E > 4096 || n * E > 0x3fffffff) return DST_ERR_BAD_SHAPE;
  if (!offsets || !tiles) return DST_ERR_BAD_ARG;
  if ((reinterpret_cast<uintptr_t>(tiles) & 7) != 0) return DST_ERR_ALIGNMENT;
  auto st = static_cast<cudaStream_t>(stream);
  const int64_t pairs = T * top_k;
  if (pairs == 0) {
    DST_CUDA_TRY(cudaMemsetAsync(tiles, 0, 6 * sizeof(int32_t), st));  // no tile, the end at position 0
    DST_CUDA_TRY(cudaMemsetAsync(offsets, 0, (size_t)(E + 1) * sizeof(int64_t), st));
    return DST_OK;
  }
  if (!ids || !order || !bins || !pair_order || !x_rows || !workspace || workspace_bytes < dst_adapter_plan_experts_workspace_bytes(pairs, E))
    return DST_ERR_BAD_ARG;
  const unsigned blocks = (unsigned)cdiv64(pairs, PLAN_THREADS);
  char* w = static_cast<char*>(workspace);
  PairLists a{};
  int32_t* permuted = reinterpret_cast<int32_t*>(w);
  int64_t* sorted = reinterpret_cast<int64_t*>(w += align16(pairs * 4));
  a.counts = reinterpret_cast<int32_t*>(w += align16(pairs * 8));
  w += align16((size_t)blocks * 4);
  pair_ids_kernel<<<(unsigned)cdiv64(pairs, 256), 256, 0, st>>>(ids, order, pairs, top_k, (int)E, permuted);
  DST_CUDA_TRY(cudaGetLastError());
  const int rc = sort_rows(permuted, 1, pairs, E, sorted, offsets, nullptr, w, nullptr, st);
  if (rc != DST_OK) return rc;
  pair_count_kernel<<<1, 1, 0, st>>>(offsets, (int)E, tiles);
  a.sorted = sorted, a.permuted = permuted, a.order = order, a.bins = bins, a.pairs = pairs, a.k = top_k, a.E = (int)E, a.n = (int)n, a.tile = tile;
  a.pair_order = pair_order, a.x_rows = x_rows, a.tiles = tiles;
  pair_lists_kernel<false><<<blocks, PLAN_THREADS, 0, st>>>(a);
  pair_lists_kernel<true><<<blocks, PLAN_THREADS, 0, st>>>(a);
  DST_CUDA_TRY(cudaGetLastError());
  return DST_OK;
}
