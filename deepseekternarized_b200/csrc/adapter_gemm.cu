// Low-rank adapters of many requests beside a projection:
//
//   out[r, :] = round( base[r, :] + scale_a * B_m (A_m x[x(r), :]) )      rows of an adapter a with matrices m
//   out[r, :] = round( base[r, :] )                                       rows without one
//
// A_m [parts * rank, K], B_m [N, rank]: part p of the output's N / parts columns takes its own rank rows of A (the gate and up
// matrices of an expert stacked, projections that share their input). h = A x is a sum of exact 16-bit products in fp32; it is
// split into 16-bit pieces (bf16: two for 16-bit outputs, three for float32 ones, 2^-17 and 2^-25 of h; fp16: two, 2^-22, after a
// power of two per row that keeps h in range), so that B h runs on the matrix instructions too without a rounding of h that the
// result would show. base is added in fp32 and the sum rounded once.
//
// A tile (up to 16 rows of one matrix) belongs to a cluster of CTAs: they share K for h, add their parts through the cluster's
// shared memory in a fixed order (results do not depend on scheduling), and share the N columns after that.
#include <cooperative_groups.h>

#include <algorithm>

#include "dst_common.cuh"

namespace dst {
namespace {

namespace cg = cooperative_groups;

struct AdapterCall {
  const void* x;
  int64_t x_stride;
  const int32_t *x_rows, *rows, *tiles;  // x row and base / out row of a position; null: the position itself
  const uint16_t *a, *b;
  const float* scale;
  const int32_t* ranks;
  int64_t per_slot;  // matrices of one adapter
  int64_t K, Kp, Np; // Kp: columns of A as stored; Np: columns of a part
  int parts;
  const void* base;
  int64_t base_stride, out_stride;
  void* out;
  int base_dtype, out_dtype;  // DST_OUT_*; base null: zeros
  int x_vec, out_vec;         // rows of x / of base and out can be read 16 bytes at a time
};

__device__ __forceinline__ void mma16(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, __nv_bfloat16) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, __half) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Eight 16-bit values of a row at element i of n, zeros behind its end
__device__ __forceinline__ uint4 load8(const uint16_t* p, int64_t i, int64_t n, bool vec) {
  if (vec && i + 8 <= n) return *reinterpret_cast<const uint4*>(p + i);
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t lo = i + 2 * j < n ? p[i + 2 * j] : 0u, hi = i + 2 * j + 1 < n ? p[i + 2 * j + 1] : 0u;
    w[j] = lo | (hi << 16);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ float to_float(uint16_t v, __nv_bfloat16) { return __uint_as_float((uint32_t)v << 16); }
__device__ __forceinline__ float to_float(uint16_t v, __half) { return __half2float(__ushort_as_half(v)); }

// The nearest 16-bit value below infinity in magnitude where v is finite, and what is left of v
__device__ __forceinline__ uint16_t piece(float& v, __nv_bfloat16) {
  const uint16_t h = __bfloat16_as_ushort(__float2bfloat16_rn(v));
  v = isfinite(v) ? v - __uint_as_float((uint32_t)h << 16) : 0.f;
  return h;
}
__device__ __forceinline__ uint16_t piece(float& v, __half) {
  const float c = isfinite(v) ? fminf(fmaxf(v, -65504.f), 65504.f) : v;
  const uint16_t h = __half_as_ushort(__float2half_rn(c));
  v = isfinite(v) ? v - __half2float(__ushort_as_half(h)) : 0.f;
  return h;
}

__device__ __forceinline__ float element(const void* p, int64_t i, int dtype) {
  if (dtype == DST_OUT_F32) return static_cast<const float*>(p)[i];
  if (dtype == DST_OUT_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}

// base + v for eight neighbouring columns of a row, rounded and stored
__device__ __forceinline__ void finish8(const AdapterCall& c, int64_t row, int64_t col, int n, float* v) {
  const int64_t bi = row * c.base_stride + col, oi = row * c.out_stride + col;
  if (c.out_vec && n == 8) {
    if (c.base) {
      if (c.base_dtype == DST_OUT_F32) {
        const float4 p = *reinterpret_cast<const float4*>(static_cast<const float*>(c.base) + bi);
        const float4 q = *reinterpret_cast<const float4*>(static_cast<const float*>(c.base) + bi + 4);
        v[0] += p.x, v[1] += p.y, v[2] += p.z, v[3] += p.w, v[4] += q.x, v[5] += q.y, v[6] += q.z, v[7] += q.w;
      } else {
        const uint4 p = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(c.base) + bi);
        const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint16_t u = (uint16_t)(w[j >> 1] >> (16 * (j & 1)));
          v[j] += c.base_dtype == DST_OUT_BF16 ? to_float(u, __nv_bfloat16()) : to_float(u, __half());
        }
      }
    }
    if (c.out_dtype == DST_OUT_F32) {
      float* o = static_cast<float*>(c.out) + oi;
      *reinterpret_cast<float4*>(o) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>(o + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (c.out_dtype == DST_OUT_BF16) {
          const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
          w[j] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
          const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
          w[j] = *reinterpret_cast<const uint32_t*>(&h);
        }
      }
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(c.out) + oi) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < n) {
      const float r = c.base ? v[j] + element(c.base, bi + j, c.base_dtype) : v[j];
      if (c.out_dtype == DST_OUT_F32) static_cast<float*>(c.out)[oi + j] = r;
      else if (c.out_dtype == DST_OUT_BF16) static_cast<__nv_bfloat16*>(c.out)[oi + j] = __float2bfloat16_rn(r);
      else static_cast<__half*>(c.out)[oi + j] = __float2half_rn(r);
    }
}

constexpr int ROWS = 16, WARPS = 8;

// RP: rank as stored (16, 32, 64 or 128), P: parts; RP * P rows of A
template <typename T, int RP, int P>
__global__ void __launch_bounds__(WARPS * 32) adapter_kernel(const AdapterCall c) {
  constexpr int R = RP * P, NT = R / 8, HS = R + 8;  // HS: row stride of the pieces of h, shifted banks
  extern __shared__ char smem[];
  float* red = reinterpret_cast<float*>(smem);        // [WARPS][ROWS][R] each warp's part of h, the first becomes the CTA's
  uint16_t* pieces = reinterpret_cast<uint16_t*>(red + WARPS * ROWS * R);  // [3][ROWS][HS]
  __shared__ float factor[ROWS];
  __shared__ int out_row[ROWS], x_row[ROWS];
  const cg::cluster_group cluster = cg::this_cluster();
  const int ctas = (int)cluster.num_blocks(), cta = (int)cluster.block_rank();
  const int tile = (int)(blockIdx.x / ctas);
  if (tile >= c.tiles[0]) return;
  const int2* list = reinterpret_cast<const int2*>(c.tiles + 4);
  const int first = list[tile].x, matrix = list[tile].y, rows = min(list[tile + 1].x - first, ROWS);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q = lane & 3;
  const int worker = cta * WARPS + warp, workers = ctas * WARPS;
  if (tid < ROWS) {
    const int at = first + (tid < rows ? tid : 0);
    out_row[tid] = c.rows ? c.rows[at] : at;
    x_row[tid] = c.x_rows ? c.x_rows[at] : at;
  }
  __syncthreads();
  const int n_pieces = c.out_dtype == DST_OUT_F32 && std::is_same<T, __nv_bfloat16>::value ? 3 : 2;

  if (matrix >= 0) {
    // h: the warp's share of K, 32 values a step; a lane's eight neighbouring values feed two instructions (the order of k
    // inside a step is the same for both operands, so it does not matter)
    float acc[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
    const uint16_t* xa = static_cast<const uint16_t*>(c.x) + x_row[g] * c.x_stride;
    const uint16_t* xb = static_cast<const uint16_t*>(c.x) + x_row[g + 8] * c.x_stride;
    const uint16_t* a = c.a + (int64_t)matrix * R * c.Kp + (int64_t)g * c.Kp;
    const bool va = g < rows, vb = g + 8 < rows;
    for (int64_t k = (int64_t)worker * 32 + q * 8; k < c.Kp; k += (int64_t)workers * 32) {
      const uint4 u = va ? load8(xa, k, c.K, c.x_vec) : make_uint4(0, 0, 0, 0);
      const uint4 v = vb ? load8(xb, k, c.K, c.x_vec) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const uint4 w = *reinterpret_cast<const uint4*>(a + (int64_t)i * 8 * c.Kp + k);
        mma16(acc[i], u.x, v.x, u.y, v.y, w.x, w.y, T());
        mma16(acc[i], u.z, v.z, u.w, v.w, w.z, w.w, T());
      }
    }
    float* mine = red + warp * ROWS * R;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      *reinterpret_cast<float2*>(mine + g * R + i * 8 + 2 * q) = make_float2(acc[i][0], acc[i][1]);
      *reinterpret_cast<float2*>(mine + (g + 8) * R + i * 8 + 2 * q) = make_float2(acc[i][2], acc[i][3]);
    }
    __syncthreads();
    for (int i = tid; i < ROWS * R; i += WARPS * 32) {
      float s = red[i];
#pragma unroll
      for (int w = 1; w < WARPS; ++w) s += red[w * ROWS * R + i];
      red[i] = s;
    }
    cluster.sync();
    // h of all CTAs, times the adapter's scale, in pieces; sixteen threads a row
    const float scale = c.scale[matrix / c.per_slot];
    const int rank = c.ranks[matrix / c.per_slot];
    float h[R / 16];
    const int row = tid >> 4, col = tid & 15;
    float big = 0.f;
#pragma unroll
    for (int j = 0; j < R / 16; ++j) {
      float s = 0.f;
      for (int b = 0; b < ctas; ++b) s += cluster.map_shared_rank(red, b)[row * R + j * 16 + col];
      h[j] = (j * 16 + col) % RP < rank ? s * scale : 0.f;
      big = fmaxf(big, fabsf(h[j]));
    }
    if (std::is_same<T, __half>::value) {
      for (int off = 8; off > 0; off >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, off));
      int ex = 0;
      if (big > 0.f && isfinite(big)) {
        (void)frexpf(big, &ex);
        ex -= 8;  // the largest in [128, 256)
      }
      if (col == 0) factor[row] = ldexpf(1.f, ex);
#pragma unroll
      for (int j = 0; j < R / 16; ++j) h[j] = ldexpf(h[j], -ex);
    } else if (col == 0) {
      factor[row] = 1.f;
    }
#pragma unroll
    for (int j = 0; j < R / 16; ++j)
      for (int p = 0; p < n_pieces; ++p) pieces[(p * ROWS + row) * HS + j * 16 + col] = piece(h[j], T());
    cluster.sync();  // also: every CTA has read the others' parts
  }

  // the columns, 32 a step: the eight B rows of instruction j are columns 8 (g / 2) + 2 j + g % 2, so that a lane ends with eight
  // neighbouring columns of its two rows
  const int per_part = (int)((c.Np + 31) / 32);
  for (int block = worker; block < per_part * P; block += workers) {
    const int part = block / per_part;
    const int64_t col0 = (int64_t)(block - part * per_part) * 32;
    float d[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) d[j][0] = d[j][1] = d[j][2] = d[j][3] = 0.f;
    if (matrix >= 0) {
      const uint16_t* b = c.b + ((int64_t)matrix * P + part) * c.Np * RP;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t col = col0 + 8 * (g >> 1) + 2 * j + (g & 1);
        const bool in = col < c.Np;
        const uint16_t* br = b + col * RP;
        if constexpr (RP == 16) {
          const uint2 w = in ? *reinterpret_cast<const uint2*>(br + q * 4) : make_uint2(0, 0);
          for (int p = 0; p < n_pieces; ++p) {
            const uint2 u = *reinterpret_cast<const uint2*>(pieces + (p * ROWS + g) * HS + part * RP + q * 4);
            const uint2 v = *reinterpret_cast<const uint2*>(pieces + (p * ROWS + g + 8) * HS + part * RP + q * 4);
            mma16(d[j], u.x, v.x, u.y, v.y, w.x, w.y, T());
          }
        } else {
#pragma unroll
          for (int k = 0; k < RP; k += 32) {
            const uint4 w = in ? *reinterpret_cast<const uint4*>(br + k + q * 8) : make_uint4(0, 0, 0, 0);
            for (int p = 0; p < n_pieces; ++p) {
              const uint4 u = *reinterpret_cast<const uint4*>(pieces + (p * ROWS + g) * HS + part * RP + k + q * 8);
              const uint4 v = *reinterpret_cast<const uint4*>(pieces + (p * ROWS + g + 8) * HS + part * RP + k + q * 8);
              mma16(d[j], u.x, v.x, u.y, v.y, w.x, w.y, T());
              mma16(d[j], u.z, v.z, u.w, v.w, w.z, w.w, T());
            }
          }
        }
      }
    }
    const int64_t col = col0 + 8 * q;
    const int n = (int)min((int64_t)8, c.Np - col);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int r = g + 8 * half;
      if (r < rows && n > 0) {
        const float f = matrix >= 0 ? factor[r] : 0.f;
        float v[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[2 * j] = d[j][2 * half] * f, v[2 * j + 1] = d[j][2 * half + 1] * f;
        finish8(c, out_row[r], part * c.Np + col, n, v);
      }
    }
  }
}

template <typename T, int RP, int P>
int launch(const AdapterCall& c, int64_t max_tiles, cudaStream_t st) {
  constexpr int R = RP * P;
  constexpr int smem = WARPS * ROWS * R * 4 + 3 * ROWS * (R + 8) * 2;
  auto kernel = adapter_kernel<T, RP, P>;
  if (smem > 48 * 1024) DST_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  const unsigned ctas = 8;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)max_tiles * ctas);
  cfg.blockDim = dim3(WARPS * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr, cfg.numAttrs = 1;
  DST_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, c));
  return DST_OK;
}

template <typename T>
int launch_for(const AdapterCall& c, int rank_padded, int64_t max_tiles, cudaStream_t st) {
  if (c.parts == 1) {
    if (rank_padded == 16) return launch<T, 16, 1>(c, max_tiles, st);
    if (rank_padded == 32) return launch<T, 32, 1>(c, max_tiles, st);
    if (rank_padded == 64) return launch<T, 64, 1>(c, max_tiles, st);
    if (rank_padded == 128) return launch<T, 128, 1>(c, max_tiles, st);
  } else if (c.parts == 2) {
    if (rank_padded == 16) return launch<T, 16, 2>(c, max_tiles, st);
    if (rank_padded == 32) return launch<T, 32, 2>(c, max_tiles, st);
    if (rank_padded == 64) return launch<T, 64, 2>(c, max_tiles, st);
  }
  return DST_ERR_UNSUPPORTED;
}

}  // namespace
}  // namespace dst

extern "C" int dst_adapter_apply(const dst_adapters* w, const dst_adapter_rows* plan, const void* x, int64_t x_stride, const void* base,
                                 int base_dtype, int64_t base_stride, void* out, int out_dtype, int64_t out_stride, dst_stream_t stream) {
  using namespace dst;
  if (!w || !plan || base_dtype < DST_OUT_F32 || base_dtype > DST_OUT_F16 || out_dtype < DST_OUT_F32 || out_dtype > DST_OUT_F16 ||
      (w->dtype != DST_ACT_BF16 && w->dtype != DST_ACT_F16) || w->K <= 0 || w->N <= 0 ||
      w->matrices_per_slot <= 0 || plan->max_tiles < 0)
    return DST_ERR_BAD_ARG;
  if (w->parts < 1 || w->N % w->parts != 0 || w->K_padded < w->K || w->K_padded % 32 != 0 || x_stride < w->K || out_stride < w->N ||
      (base && base_stride < w->N) || plan->max_tiles > 0x0fffffff || plan->tile != ROWS)
    return DST_ERR_BAD_SHAPE;
  if (plan->max_tiles == 0) return DST_OK;
  if (!w->a || !w->b || !w->scale || !w->ranks || !plan->tiles || !x || !out) return DST_ERR_BAD_ARG;
  if (((reinterpret_cast<uintptr_t>(w->a) | reinterpret_cast<uintptr_t>(w->b)) & 15) != 0 || (reinterpret_cast<uintptr_t>(plan->tiles) & 7) != 0)
    return DST_ERR_ALIGNMENT;
  AdapterCall c{};
  c.x = x, c.x_stride = x_stride, c.x_rows = plan->x_rows, c.rows = plan->rows, c.tiles = plan->tiles;
  c.a = static_cast<const uint16_t*>(w->a), c.b = static_cast<const uint16_t*>(w->b), c.scale = w->scale, c.ranks = w->ranks;
  c.per_slot = w->matrices_per_slot, c.K = w->K, c.Kp = w->K_padded, c.Np = w->N / w->parts, c.parts = w->parts;
  c.base = base, c.base_dtype = base_dtype, c.base_stride = base_stride, c.out = out, c.out_dtype = out_dtype, c.out_stride = out_stride;
  const auto rows_of_16 = [](const void* p, int64_t stride, int size) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride * size % 16 == 0; };
  c.x_vec = rows_of_16(x, x_stride, 2);
  c.out_vec = c.Np % 8 == 0 && rows_of_16(out, out_stride, out_dtype == DST_OUT_F32 ? 4 : 2) &&
              (!base || rows_of_16(base, base_stride, base_dtype == DST_OUT_F32 ? 4 : 2));
  auto st = static_cast<cudaStream_t>(stream);
  return w->dtype == DST_ACT_BF16 ? launch_for<__nv_bfloat16>(c, w->rank_padded, plan->max_tiles, st)
                                  : launch_for<__half>(c, w->rank_padded, plan->max_tiles, st);
}
