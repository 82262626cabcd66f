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
  int ctas;                   // of a cluster
  int kind;                   // base and result of the fast forms: 0 float32 / 16 bits, 1 float32 / float32, 2 16 / 16, 3 none / 16; -1: others
  int x_vec;                  // rows of x can be read eight values at a time
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

// Four values of a row and their sum with what `base` holds of it
template <typename T>
__device__ __forceinline__ uint2 pack4(const float* v) {
  uint32_t w[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
      w[j] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
      w[j] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  return make_uint2(w[0], w[1]);
}

// base + v for up to four neighbouring columns, of any types and alignment
__device__ __forceinline__ void finish_single(const AdapterCall& c, int64_t row, int64_t col, int n, const float* v) {
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (j < n) {
      const int64_t bi = row * c.base_stride + col + j, oi = row * c.out_stride + col + j;
      const float r = c.base ? v[j] + element(c.base, bi, c.base_dtype) : v[j];
      if (c.out_dtype == DST_OUT_F32) static_cast<float*>(c.out)[oi] = r;
      else if (c.out_dtype == DST_OUT_BF16) static_cast<__nv_bfloat16*>(c.out)[oi] = __float2bfloat16_rn(r);
      else static_cast<__half*>(c.out)[oi] = __float2half_rn(r);
    }
}

// Asynchronous copies into a lane's own slots: no other thread reads them, so waiting for the lane's own groups is enough. A slot
// is refilled after the instructions that used its values.
__device__ __forceinline__ void copy16(uint32_t to, const void* from, int bytes) {  // the rest of the 16 are zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy8(uint32_t to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void wait_but() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 slot(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}

constexpr int WARPS = 8, MAX_CTAS = 8;
constexpr int XS = 4, BS = 3;  // steps of x and of base on the way

// RP: rank as stored (16, 32, 64 or 128), P: parts, MW: blocks of 16 rows in a tile, each a matter of WARPS / MW warps, which
// share K first and the columns then
template <typename T, int RP, int P, int MW>
struct Shape {
  static constexpr int R = RP * P, NT = R / 8, HS = R + 8;  // HS: row stride of the pieces of h, shifted banks
  static constexpr int ROWS = 16 * MW, KW = WARPS / MW;
  static constexpr int XPART = XS * 1024 > 16 * R * 4 ? XS * 1024 : 16 * R * 4;  // bytes of a warp: steps of x, then its part of h
  static constexpr int BPART = BS * 2048;                                        // steps of base: 16 rows of 32 columns
  static constexpr int BASE = WARPS * XPART, PIECES = BASE + WARPS * BPART, SMEM = PIECES + 3 * ROWS * HS * 2;
};

// What a step of the second product meets: base float32 or of the 16-bit type or none, the result of the 16-bit type or float32
enum { BASE_F32, BASE_T, BASE_NONE };
template <int V>
using Int = std::integral_constant<int, V>;

template <typename T, int RP, int P, int MW>
__global__ void __launch_bounds__(WARPS * 32, RP* P <= 64 ? 2 : 1) adapter_kernel(const AdapterCall c) {
  using S = Shape<T, RP, P, MW>;
  constexpr bool BF = std::is_same<T, __nv_bfloat16>::value;
  constexpr int R = S::R, NT = S::NT, HS = S::HS, ROWS = S::ROWS, KW = S::KW, KB = RP == 16 ? 1 : RP / 32;
  extern __shared__ __align__(16) char smem[];
  uint16_t* pieces = reinterpret_cast<uint16_t*>(smem + S::PIECES);  // [3][ROWS][HS]
  __shared__ float factor[ROWS];
  const cg::cluster_group cluster = cg::this_cluster();
  const int ctas = (int)cluster.num_blocks(), cta = (int)cluster.block_rank();
  const int tile = (int)(blockIdx.x / ctas);
  if (tile >= c.tiles[0]) return;
  const int2* list = reinterpret_cast<const int2*>(c.tiles + 4);
  const int2 head = list[tile];
  const int first = head.x, matrix = head.y, rows = min(list[tile + 1].x - first, ROWS);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q = lane & 3;
  const int mw = warp % MW, kw = warp / MW, worker = cta * KW + kw, workers = ctas * KW;
  const int ra = mw * 16 + g, rb = ra + 8;  // the lane's two rows of the tile
  const bool va = ra < rows, vb = rb < rows;
  const int pa = first + (va ? ra : 0), pb = first + (vb ? rb : 0);

  // A of the warp's first step, before anything that depends on the rows
  const uint16_t* a = c.a + (int64_t)(matrix < 0 ? 0 : matrix) * R * c.Kp + g * 32 + q * 8;
  const int k_steps = matrix < 0 ? 0 : (int)(c.Kp / 32);
  uint4 aw[NT];
  const auto load_a = [&](int step, uint4 (&w)[NT]) {
#pragma unroll
    for (int i = 0; i < NT; ++i) w[i] = __ldg(reinterpret_cast<const uint4*>(a + (int64_t)step * (R * 32) + i * 256));
  };
  if (worker < k_steps) load_a(worker, aw);

  // Steps of 32 columns, those of the second part behind those of the first. A lane has four neighbouring columns and the four 16
  // further on: quads of lanes then read and write whole 32-byte sectors whatever the types.
  const int Np = (int)c.Np, N = Np * P, per_part = (Np + 31) / 32, steps = per_part * P;
  const auto column = [&](int step) { return step * 32 + (P == 2 && step >= per_part ? Np - per_part * 32 : 0); };
  const auto behind = [&](int step, int col) { return (P == 2 && step < per_part ? Np : N) - col; };
  const int64_t oa = c.rows ? c.rows[pa] : pa, ob = c.rows ? c.rows[pb] : pb;
  const uint32_t base_slots = (uint32_t)__cvta_generic_to_shared(smem + S::BASE + warp * S::BPART) + lane * 16;
  const int es = c.base_dtype == DST_OUT_F32 ? 4 : 2;
  const char* base_a = static_cast<const char*>(c.base) + (oa * c.base_stride + 4 * q) * es;
  const char* base_b = static_cast<const char*>(c.base) + (ob * c.base_stride + 4 * q) * es;
  const int kind = c.kind;  // of what the fast form covers, else -1
  const auto fetch_base = [&](auto base_kind, int step, int stage) {
    if (decltype(base_kind)::value != BASE_NONE && step < steps) {
      constexpr int ES = decltype(base_kind)::value == BASE_F32 ? 4 : 2;
      const int col = column(step), left = behind(step, col) - 4 * q;
      const char *fa = base_a + (int64_t)col * ES, *fb = base_b + (int64_t)col * ES;
      const uint32_t to = base_slots + stage * 2048;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (left > 16 * i) {
          if constexpr (ES == 4) {
            if (va) copy16(to + i * 512, fa + 16 * ES * i, 16);
            if (vb) copy16(to + 1024 + i * 512, fb + 16 * ES * i, 16);
          } else {
            if (va) copy8(to + i * 512, fa + 16 * ES * i);
            if (vb) copy8(to + 1024 + i * 512, fb + 16 * ES * i);
          }
        }
    }
    commit();
  };
#pragma unroll
  for (int s = 0; s < BS; ++s) {
    if (kind == 0 || kind == 1) fetch_base(Int<BASE_F32>(), worker + s * workers, s);
    else if (kind == 2) fetch_base(Int<BASE_T>(), worker + s * workers, s);
  }
  // B of a step. The eight rows of instruction j are columns 16 (j / 2) + 4 (g / 2) + 2 (j % 2) + g % 2, which gives a lane its
  // own. Up to 31 rows behind the part's last one are read and not used.
  const uint16_t* b = c.b + ((int64_t)(matrix < 0 ? 0 : matrix) * N + 4 * (g >> 1) + (g & 1)) * RP + q * (RP == 16 ? 4 : 8);
  uint4 bw[KB][4];
  const auto load_b = [&](int step, uint4 (&w)[KB][4]) {
    if (matrix < 0 || step >= steps) return;
    const uint16_t* p = b + (int64_t)column(step) * RP;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint16_t* br = p + (16 * (j >> 1) + 2 * (j & 1)) * RP;
      if constexpr (RP == 16) {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(br));
        w[0][j].x = v.x, w[0][j].y = v.y;
      } else {
#pragma unroll
        for (int k = 0; k < KB; ++k) w[k][j] = __ldg(reinterpret_cast<const uint4*>(br + k * 32));
      }
    }
  };
  constexpr bool EARLY_B = RP <= 32 && R <= 64;  // the first step's B before anything is waited for, where registers allow
  if (EARLY_B) load_b(worker, bw);

  if (matrix >= 0) {
    // h: the warp's share of K, 32 values a step; a lane's eight neighbouring values feed two instructions (the order of k
    // inside a step is the same for both operands, so it does not matter). A is stored step by step.
    float acc[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
    const uint16_t* xa = static_cast<const uint16_t*>(c.x) + (c.x_rows ? c.x_rows[pa] : pa) * c.x_stride + q * 8;
    const uint16_t* xb = static_cast<const uint16_t*>(c.x) + (c.x_rows ? c.x_rows[pb] : pb) * c.x_stride + q * 8;
    const uint32_t x_slots = (uint32_t)__cvta_generic_to_shared(smem + warp * S::XPART) + lane * 16;
    const int K = (int)c.K;
    const int full_a = va ? 16 : 0, full_b = vb ? 16 : 0;
    const auto fetch_x = [&](int step, int stage) {
      const uint32_t to = x_slots + stage * 1024;
      if (step < k_steps) {
        const int k = step * 32;
        if (c.x_vec) {
          const bool whole = k + 32 <= K;
          const int bytes = whole ? 16 : min(16, max(0, (K - k - q * 8) * 2));
          const int at = bytes > 0 ? k : 0;  // a copy of nothing still wants an address
          copy16(to, xa + at, min(bytes, full_a));
          copy16(to + 512, xb + at, min(bytes, full_b));
        } else {
          const uint4 u = va ? load8(xa, k, K - q * 8, false) : make_uint4(0, 0, 0, 0);
          const uint4 v = vb ? load8(xb, k, K - q * 8, false) : make_uint4(0, 0, 0, 0);
          asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(to), "r"(u.x), "r"(u.y), "r"(u.z), "r"(u.w) : "memory");
          asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(to + 512), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
        }
      }
      commit();
    };
#pragma unroll
    for (int s = 0; s < XS; ++s) fetch_x(worker + s * workers, s);
    int stage = 0;
    for (int step = worker; step < k_steps; step += workers) {
      uint4 an[NT];
      if (R <= 64 && step + workers < k_steps) load_a(step + workers, an);
      wait_but<XS - 1>();
      const uint4 u = slot(x_slots + stage * 1024), v = slot(x_slots + stage * 1024 + 512);
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        mma16(acc[i], u.x, v.x, u.y, v.y, aw[i].x, aw[i].y, T());
        mma16(acc[i], u.z, v.z, u.w, v.w, aw[i].z, aw[i].w, T());
      }
      fetch_x(step + XS * workers, stage);
      stage = (stage + 1) % XS;
      if (R <= 64) {
#pragma unroll
        for (int i = 0; i < NT; ++i) aw[i] = an[i];
      } else if (step + workers < k_steps) {
        load_a(step + workers, aw);
      }
    }
    if (!EARLY_B) load_b(worker, bw);  // on the way while the parts of h are added up
    float* mine = reinterpret_cast<float*>(smem + warp * S::XPART);  // over the warp's own x, which is used up
    __syncwarp();
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      *reinterpret_cast<float2*>(mine + g * R + i * 8 + 2 * q) = make_float2(acc[i][0], acc[i][1]);
      *reinterpret_cast<float2*>(mine + (g + 8) * R + i * 8 + 2 * q) = make_float2(acc[i][2], acc[i][3]);
    }
    // element i of the tile's h: row i / R, in the part of the row's first warp
    const auto place = [&](int i) { return (i / (16 * R)) * (S::XPART / 4) + i % (16 * R); };
    float* parts = reinterpret_cast<float*>(smem);
    if (KW > 1) {
      __syncthreads();
      for (int i = tid * 4; i < ROWS * R; i += WARPS * 32 * 4) {
        float4 s = *reinterpret_cast<float4*>(parts + place(i));
#pragma unroll
        for (int w = 1; w < KW; ++w) {
          const float4 o = *reinterpret_cast<float4*>(parts + w * MW * (S::XPART / 4) + place(i));
          s.x += o.x, s.y += o.y, s.z += o.z, s.w += o.w;
        }
        *reinterpret_cast<float4*>(parts + place(i)) = s;
      }
    }
    cluster.sync();
    // h of all CTAs, times the adapter's scale, in pieces: four neighbouring values a thread
    const float scale = c.scale[matrix / c.per_slot];
    const int rank = c.ranks[matrix / c.per_slot];
    const int n_pieces = BF && (c.out_dtype == DST_OUT_F32 || kind < 0) ? 3 : 2;
    const float* from[MAX_CTAS];
#pragma unroll
    for (int i = 0; i < MAX_CTAS; ++i) from[i] = cluster.map_shared_rank(parts, i < ctas ? i : 0);
    for (int i = tid * 4; i < ROWS * R; i += WARPS * 32 * 4) {
      const int row = i / R, col = i % R;
      float4 o[MAX_CTAS];
#pragma unroll
      for (int k = 0; k < MAX_CTAS; ++k) o[k] = k < ctas ? *reinterpret_cast<const float4*>(from[k] + place(i)) : make_float4(0.f, 0.f, 0.f, 0.f);
      float h[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < MAX_CTAS; ++k) h[0] += o[k].x, h[1] += o[k].y, h[2] += o[k].z, h[3] += o[k].w;
#pragma unroll
      for (int j = 0; j < 4; ++j) h[j] = (col + j) % RP < rank ? h[j] * scale : 0.f;
      if (!BF) {  // a row is R / 4 lanes of a warp
        float big = fmaxf(fmaxf(fabsf(h[0]), fabsf(h[1])), fmaxf(fabsf(h[2]), fabsf(h[3])));
#pragma unroll
        for (int off = R / 8; off > 0; off >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, off));
        int ex = 0;
        if (big > 0.f && isfinite(big)) {
          (void)frexpf(big, &ex);
          ex -= 8;  // the largest in [128, 256)
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) h[j] = ldexpf(h[j], -ex);
        if (col == 0) factor[row] = ldexpf(1.f, ex);
      }
#pragma unroll
      for (int p = 0; p < 3; ++p)
        if (p < n_pieces) {
          const uint32_t h0 = piece(h[0], T()), h1 = piece(h[1], T()), h2 = piece(h[2], T()), h3 = piece(h[3], T());
          *reinterpret_cast<uint2*>(pieces + (p * ROWS + row) * HS + col) = make_uint2(h0 | (h1 << 16), h2 | (h3 << 16));
        }
    }
    cluster.sync();  // also: every CTA has read the others' parts
  }

  const float fa = !BF && matrix >= 0 ? factor[ra] : 1.f, fb = !BF && matrix >= 0 ? factor[rb] : 1.f;
  // d = the pieces of h times B of a step (NP pieces)
  const auto product = [&](auto np, int part, float (&d)[4][4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) d[j][0] = d[j][1] = d[j][2] = d[j][3] = 0.f;
    if (matrix < 0) return;
#pragma unroll
    for (int p = 0; p < decltype(np)::value; ++p) {
      const uint16_t* ha = pieces + (p * ROWS + ra) * HS + part * RP;
      const uint16_t* hb = pieces + (p * ROWS + rb) * HS + part * RP;
      if constexpr (RP == 16) {
        const uint2 u = *reinterpret_cast<const uint2*>(ha + q * 4), v = *reinterpret_cast<const uint2*>(hb + q * 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) mma16(d[j], u.x, v.x, u.y, v.y, bw[0][j].x, bw[0][j].y, T());
      } else {
#pragma unroll
        for (int k = 0; k < KB; ++k) {
          const uint4 u = *reinterpret_cast<const uint4*>(ha + k * 32 + q * 8), v = *reinterpret_cast<const uint4*>(hb + k * 32 + q * 8);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            mma16(d[j], u.x, v.x, u.y, v.y, bw[k][j].x, bw[k][j].y, T());
            mma16(d[j], u.z, v.z, u.w, v.w, bw[k][j].z, bw[k][j].w, T());
          }
        }
      }
    }
    if (!BF) {
#pragma unroll
      for (int j = 0; j < 4; ++j) d[j][0] *= fa, d[j][1] *= fa, d[j][2] *= fb, d[j][3] *= fb;
    }
  };
  const auto next_b = [&](const uint4 (&w)[KB][4]) {
#pragma unroll
    for (int k = 0; k < KB; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) bw[k][j] = w[k][j];
  };
  const auto columns = [&](auto base_kind, auto out_f32) {
    constexpr int BK = decltype(base_kind)::value;
    constexpr bool OF = decltype(out_f32)::value != 0;
    char* out_a = static_cast<char*>(c.out) + (oa * c.out_stride + 4 * q) * (OF ? 4 : 2);
    char* out_b = static_cast<char*>(c.out) + (ob * c.out_stride + 4 * q) * (OF ? 4 : 2);
    int stage = 0;
    for (int step = worker; step < steps; step += workers) {
      uint4 bn[KB][4];
      load_b(step + workers, bn);
      float d[4][4];
      product(Int<OF && BF ? 3 : 2>(), P == 2 && step >= per_part, d);
      if (BK != BASE_NONE) wait_but<BS - 1>();
      const int col = column(step), left = behind(step, col) - 4 * q;
      const uint32_t at = base_slots + stage * 2048;
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if ((half ? vb : va) && left > 16 * i) {
            float v[4] = {d[2 * i][2 * half], d[2 * i][2 * half + 1], d[2 * i + 1][2 * half], d[2 * i + 1][2 * half + 1]};
            if (BK == BASE_F32) {
              const uint4 w = slot(at + half * 1024 + i * 512);
              v[0] += __uint_as_float(w.x), v[1] += __uint_as_float(w.y), v[2] += __uint_as_float(w.z), v[3] += __uint_as_float(w.w);
            } else if (BK == BASE_T) {
              const uint4 w = slot(at + half * 1024 + i * 512);
              v[0] += to_float((uint16_t)w.x, T()), v[1] += to_float((uint16_t)(w.x >> 16), T());
              v[2] += to_float((uint16_t)w.y, T()), v[3] += to_float((uint16_t)(w.y >> 16), T());
            }
            char* o = (half ? out_b : out_a) + (int64_t)(col + 16 * i) * (OF ? 4 : 2);
            if (OF) *reinterpret_cast<float4*>(o) = make_float4(v[0], v[1], v[2], v[3]);
            else *reinterpret_cast<uint2*>(o) = pack4<T>(v);
          }
      if (BK != BASE_NONE) fetch_base(base_kind, step + BS * workers, stage);
      stage = stage + 1 == BS ? 0 : stage + 1;
      next_b(bn);
    }
  };
  if (kind == 0) columns(Int<BASE_F32>(), Int<0>());
  else if (kind == 1) columns(Int<BASE_F32>(), Int<1>());
  else if (kind == 2) columns(Int<BASE_T>(), Int<0>());
  else if (kind == 3) columns(Int<BASE_NONE>(), Int<0>());
  else
    for (int step = worker; step < steps; step += workers) {
      uint4 bn[KB][4];
      load_b(step + workers, bn);
      float d[4][4];
      product(Int<BF ? 3 : 2>(), P == 2 && step >= per_part, d);
      const int col = column(step), left = behind(step, col) - 4 * q;
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if ((half ? vb : va) && left > 16 * i) {
            const float v[4] = {d[2 * i][2 * half], d[2 * i][2 * half + 1], d[2 * i + 1][2 * half], d[2 * i + 1][2 * half + 1]};
            finish_single(c, half ? ob : oa, col + 4 * q + 16 * i, min(4, left - 16 * i), v);
          }
      next_b(bn);
    }
}

template <typename T, int RP, int P, int MW>
int launch(const AdapterCall& c, int64_t max_tiles, cudaStream_t st) {
  using S = Shape<T, RP, P, MW>;
  auto kernel = adapter_kernel<T, RP, P, MW>;
  if (S::SMEM > 48 * 1024) DST_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM));
  const unsigned ctas = c.ctas;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)max_tiles * ctas);
  cfg.blockDim = dim3(WARPS * 32);
  cfg.dynamicSmemBytes = S::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr, cfg.numAttrs = 1;
  DST_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, c));
  return DST_OK;
}

template <typename T, int RP, int P>
int launch_tile(const AdapterCall& c, int tile, int64_t max_tiles, cudaStream_t st) {
  if (tile == 16) return launch<T, RP, P, 1>(c, max_tiles, st);
  if (tile == 32) return launch<T, RP, P, 2>(c, max_tiles, st);
  return launch<T, RP, P, 4>(c, max_tiles, st);
}

template <typename T>
int launch_for(const AdapterCall& c, int rank_padded, int tile, int64_t max_tiles, cudaStream_t st) {
  if (c.parts == 1) {
    if (rank_padded == 16) return launch_tile<T, 16, 1>(c, tile, max_tiles, st);
    if (rank_padded == 32) return launch_tile<T, 32, 1>(c, tile, max_tiles, st);
    if (rank_padded == 64) return launch_tile<T, 64, 1>(c, tile, max_tiles, st);
    if (rank_padded == 128) return launch_tile<T, 128, 1>(c, tile, max_tiles, st);
  } else if (c.parts == 2) {
    if (rank_padded == 16) return launch_tile<T, 16, 2>(c, tile, max_tiles, st);
    if (rank_padded == 32) return launch_tile<T, 32, 2>(c, tile, max_tiles, st);
    if (rank_padded == 64) return launch_tile<T, 64, 2>(c, tile, max_tiles, st);
  }
  return DST_ERR_UNSUPPORTED;
}

}  // namespace
}  // namespace dst

// Taller tiles read A and B less often, once there are enough of them for all SMs. Measured, us in tiles of 16 / 32 / 64 with the
// best number of CTAs: 333 rows 8.0 / 8.7 / 12; 4000 rows (rank 64) 55 / 54 / 56; 16 384 rows 123 / 118 / 112
extern "C" int dst_adapter_tile(int64_t rows) {
  const int64_t sms = dst::sm_count();
  return rows >= 64 * sms ? 64 : rows >= 20 * sms ? 32 : 16;
}

extern "C" int dst_adapter_apply(const dst_adapters* w, const dst_adapter_rows* plan, const void* x, int64_t x_stride, const void* base,
                                 int base_dtype, int64_t base_stride, void* out, int out_dtype, int64_t out_stride, dst_stream_t stream) {
  using namespace dst;
  if (!w || !plan || base_dtype < DST_OUT_F32 || base_dtype > DST_OUT_F16 || out_dtype < DST_OUT_F32 || out_dtype > DST_OUT_F16 ||
      (w->dtype != DST_ACT_BF16 && w->dtype != DST_ACT_F16) || w->K <= 0 || w->N <= 0 ||
      w->matrices_per_slot <= 0 || plan->max_tiles < 0)
    return DST_ERR_BAD_ARG;
  if (w->parts < 1 || w->N % w->parts != 0 || w->K_padded < w->K || w->K_padded % 32 != 0 || x_stride < w->K || out_stride < w->N ||
      (base && base_stride < w->N) || plan->max_tiles > 0x0fffffff || w->N > (1 << 24) || w->K_padded > (1 << 24) || (plan->tile != 16 && plan->tile != 32 && plan->tile != 64))
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
  const auto aligned = [](const void* p, int64_t stride, int n, int size) { return reinterpret_cast<uintptr_t>(p) % (n * size) == 0 && stride % n == 0; };
  c.x_vec = aligned(x, x_stride, 8, 2);
  const int own = w->dtype == DST_ACT_BF16 ? DST_OUT_BF16 : DST_OUT_F16;
  c.kind = -1;
  if (c.Np % 4 == 0 && aligned(out, out_stride, 4, out_dtype == DST_OUT_F32 ? 4 : 2) &&
      (!base || aligned(base, base_stride, 4, base_dtype == DST_OUT_F32 ? 4 : 2))) {
    if (base && base_dtype == DST_OUT_F32 && (out_dtype == own || out_dtype == DST_OUT_F32)) c.kind = out_dtype == own ? 0 : 1;
    else if (out_dtype == own && (!base || base_dtype == own)) c.kind = base ? 2 : 3;
  }
  // As many CTAs to a tile as run at once (two an SM), up to a portable cluster. Measured, us with 1 / 2 / 4 / 8 CTAs: one row of
  // 4096 x 4096 11.9 / 7.6 / 5.4 / 4.4; 64 rows of 37 adapters through 11008 x 4096 38 / 22 / 14.7 / 15.0; 4000 rows in tiles of 32,
  // rank 64 56 / 54 / 59 / 73; 16 384 rows in tiles of 64 112 / 118 / 126 / 145
  c.ctas = 1;
  while (c.ctas < MAX_CTAS && plan->max_tiles * c.ctas * 2 <= 2 * (int64_t)sm_count()) c.ctas *= 2;
  auto st = static_cast<cudaStream_t>(stream);
  return w->dtype == DST_ACT_BF16 ? launch_for<__nv_bfloat16>(c, w->rank_padded, plan->tile, plan->max_tiles, st)
                                  : launch_for<__half>(c, w->rank_padded, plan->tile, plan->max_tiles, st);
}
