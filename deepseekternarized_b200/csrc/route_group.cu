// Routing to experts in groups. For a token with logits l_e over E experts in G groups of E / G consecutive ids:
//
//   s_e = f(l_e / temp)          f: softmax over the E logits, sigmoid or sqrt(softplus)
//   key_e = s_e + bias_e         the selection; the weights come from s_e
//   group score                  the largest key of the group, or the sum of its two largest
//   kept                         the topk_groups groups of the largest scores (equal scores: the lower group)
//   picks                        the top_k largest keys among the kept groups' experts (equal keys: the lower id), in that order
//   weight_i = s of pick i, divided by the picks' sum + 1e-20 when renormalised (top_k > 1), times route_scale
//
// The picks are those of exact arithmetic: keys closer than the rounding of their scores are compared in 64 bits. A NaN ranks
// above every number, so a token's ids are distinct and inside [0, E) whatever the logits hold.
#include <type_traits>

#include "dst_common.cuh"

namespace dst {
namespace {

// A key as an unsigned number of the same order; NaNs above everything and equal among themselves, 0 below every key.
__device__ __forceinline__ uint64_t order_of(double v) {
  if (v != v) return ~0ull;
  const uint64_t u = (uint64_t)__double_as_longlong(v + 0.0);
  return (u >> 63) ? ~u : (u | (1ull << 63));
}
__device__ __forceinline__ double value_of(uint64_t r) {
  if (r == ~0ull) return __longlong_as_double(0x7ff8000000000000ll);
  return __longlong_as_double((long long)((r >> 63) ? (r & ~(1ull << 63)) : ~r));
}

struct GroupRoute {
  const void* logits;
  int64_t stride;
  const float* bias;
  int64_t T;
  int E, groups, size, lanes, chunk, kept, two, top_k, score, renorm;  // lanes: of the warp for one group; chunk: experts per lane
  float temp, scale;
  float* weights;
  int32_t* ids;
};

template <typename T>
__device__ __forceinline__ float logit(const T* p) {
  if constexpr (sizeof(T) == 4) return *p;
  else if constexpr (std::is_same<T, __half>::value) return __half2float(*p);
  else return __bfloat162float(*p);
}

__device__ __forceinline__ uint64_t shfl64(uint64_t v, int src) { return __shfl_sync(0xffffffffu, v, src); }
__device__ __forceinline__ uint64_t shfl64_xor(uint64_t v, int m) { return __shfl_xor_sync(0xffffffffu, v, m); }

// One token by one warp in 64 bits. A group belongs to `lanes` neighbouring lanes (a power of two), a lane to `chunk`
// consecutive experts of it, so ids rise with the lane and with j.
template <int PL, typename T>
__device__ __forceinline__ void route_token(const GroupRoute& a, int64_t t, int lane) {
  const T* row = static_cast<const T*>(a.logits) + t * a.stride;
  const int group = lane / a.lanes, first = (lane % a.lanes) * a.chunk;
  int n = group < a.groups ? min(a.chunk, a.size - first) : 0;
  const int id0 = group * a.size + first;
  double s[PL];
  double mx = -INFINITY;
#pragma unroll
  for (int j = 0; j < PL; ++j) {
    s[j] = j < n ? (double)logit(row + id0 + j) / (double)a.temp : -INFINITY;
    mx = fmax(mx, s[j]);
  }
  if (a.score == DST_SCORE_SOFTMAX) {
    for (int off = 16; off > 0; off >>= 1) mx = fmax(mx, __shfl_xor_sync(0xffffffffu, mx, off));
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < PL; ++j) {
      s[j] = exp(s[j] - mx);
      if (j < n) sum += s[j];
    }
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
#pragma unroll
    for (int j = 0; j < PL; ++j) s[j] = s[j] / sum;
  } else if (a.score == DST_SCORE_SIGMOID) {
#pragma unroll
    for (int j = 0; j < PL; ++j) s[j] = 1.0 / (1.0 + exp(-s[j]));
  } else {
#pragma unroll
    for (int j = 0; j < PL; ++j) s[j] = sqrt(fmax(s[j], 0.0) + log1p(exp(-fabs(s[j]))));
  }
  uint64_t rank[PL], m1 = 0, m2 = 0;
#pragma unroll
  for (int j = 0; j < PL; ++j) {
    rank[j] = j < n ? order_of(a.bias ? s[j] + (double)a.bias[id0 + j] : s[j]) : 0ull;
    if (rank[j] > m1) m2 = m1, m1 = rank[j];
    else if (rank[j] > m2) m2 = rank[j];
  }
  for (int off = 1; off < a.lanes; off <<= 1) {
    const uint64_t o1 = shfl64_xor(m1, off), o2 = shfl64_xor(m2, off);
    if (o1 > m1) m2 = m1 > o2 ? m1 : o2, m1 = o1;
    else m2 = m2 > o1 ? m2 : o1;
  }
  uint64_t g = m1;
  if (a.two && m2) g = order_of(value_of(m1) + value_of(m2));
  int better = 0;
  for (int h = 0; h < a.groups; ++h) {
    const uint64_t o = shfl64(g, h * a.lanes);
    better += o > g || (o == g && h < group);
  }
  if (better >= a.kept) {
#pragma unroll
    for (int j = 0; j < PL; ++j) rank[j] = 0;
  }
  double my_w = 0.0, wsum = 0.0;
  int my_id = 0;
  for (int r = 0; r < a.top_k; ++r) {
    uint64_t best = 0;
    int at = 0;
    double w = 0.0;
#pragma unroll
    for (int j = 0; j < PL; ++j)
      if (rank[j] > best) best = rank[j], at = j, w = s[j];
    uint64_t top = best;
    for (int off = 16; off > 0; off >>= 1) {
      const uint64_t o = shfl64_xor(top, off);
      top = o > top ? o : top;
    }
    const int win = __ffs(__ballot_sync(0xffffffffu, best == top)) - 1;
    if (lane == win) {
#pragma unroll
      for (int j = 0; j < PL; ++j)
        if (j == at) rank[j] = 0;
    }
    w = __shfl_sync(0xffffffffu, w, win);
    const int id = __shfl_sync(0xffffffffu, id0 + at, win);
    if (lane == r) my_w = w, my_id = id;
    wsum += w;
  }
  if (lane < a.top_k) {
    a.weights[t * a.top_k + lane] = (float)((a.renorm && a.top_k > 1 ? my_w / (wsum + 1e-20) : my_w) * (double)a.scale);
    a.ids[t * a.top_k + lane] = my_id;
  }
}

template <int PL, typename T>
__global__ void __launch_bounds__(128) route_group_kernel(const GroupRoute a) {
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (t < a.T) route_token<PL, T>(a, t, threadIdx.x & 31);
}

template <typename T>
int launch(const GroupRoute& a, cudaStream_t st) {
  const unsigned grid = (unsigned)cdiv64(a.T, 4);
  if (a.chunk <= 4) route_group_kernel<4, T><<<grid, 128, 0, st>>>(a);
  else if (a.chunk <= 8) route_group_kernel<8, T><<<grid, 128, 0, st>>>(a);
  else if (a.chunk <= 16) route_group_kernel<16, T><<<grid, 128, 0, st>>>(a);
  else route_group_kernel<64, T><<<grid, 128, 0, st>>>(a);
  DST_CUDA_TRY(cudaGetLastError());
  return DST_OK;
}

}  // namespace
}  // namespace dst

extern "C" int dst_route_group_topk(const void* logits, int logits_dtype, int64_t row_stride, const float* bias, int64_t T, int64_t E,
                                    int n_groups, int topk_groups, int group_score, int top_k, int score_func, float gate_temp, int renorm,
                                    float route_scale, float* weights, int32_t* ids, dst_stream_t stream) {
  using namespace dst;
  if (T < 0 || E <= 0 || top_k <= 0 || n_groups <= 0 || topk_groups <= 0 || score_func < DST_SCORE_SOFTMAX ||
      score_func > DST_SCORE_SQRTSOFTPLUS || (group_score != DST_GROUP_MAX && group_score != DST_GROUP_TOP2) || !(gate_temp < 0.f || gate_temp > 0.f) ||
      logits_dtype < DST_OUT_F32 || logits_dtype > DST_OUT_F16)
    return DST_ERR_BAD_ARG;
  if (E % n_groups != 0 || topk_groups > n_groups || row_stride < E || T > 0x7fffffff) return DST_ERR_BAD_SHAPE;
  const int size = (int)(E / n_groups);
  if (E > 1024 || n_groups > 32 || top_k > 8 || (int64_t)top_k > (int64_t)topk_groups * size) return DST_ERR_UNSUPPORTED;
  if (T == 0) return DST_OK;
  if (!logits || !weights || !ids) return DST_ERR_BAD_ARG;
  GroupRoute a{};
  a.logits = logits, a.stride = row_stride, a.bias = bias, a.T = T, a.E = (int)E, a.groups = n_groups, a.size = size;
  a.lanes = 32;
  while (a.lanes * n_groups > 32) a.lanes >>= 1;
  a.chunk = (size + a.lanes - 1) / a.lanes;  // at most 60: 17 groups of 60 on a lane each
  a.kept = topk_groups, a.two = group_score == DST_GROUP_TOP2, a.top_k = top_k, a.score = score_func, a.renorm = renorm;
  a.temp = gate_temp, a.scale = route_scale, a.weights = weights, a.ids = ids;
  auto st = static_cast<cudaStream_t>(stream);
  if (logits_dtype == DST_OUT_F32) return launch<float>(a, st);
  return logits_dtype == DST_OUT_BF16 ? launch<__nv_bfloat16>(a, st) : launch<__half>(a, st);
}
