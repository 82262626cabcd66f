// Low-rank adapters: what a call of the library hands to the kernels of a type (adapter_gemm.cuh).
#pragma once

#include "dst_common.cuh"

namespace dst {

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
  int ctas, splits;           // of a cluster; of K (h) or of the columns between the CTAs of a tile
  float* h;                   // [splits of K][positions][rows of A]
  int64_t positions;
  int k_splits, share, sub;  // shares of K in the workspace; warps of a row block for h; row blocks of a tile
  int shared_a, shared_b;     // the row blocks of a tile share A, B
  int kind;                   // base and result of the fast forms: 0 float32 / 16 bits, 1 float32 / float32, 2 16 / 16, 3 none / 16; -1: others
  int x_vec;                  // rows of x can be read eight values at a time
};

int adapter_launch_bf16(const AdapterCall& c, int rank_padded, int64_t max_tiles, cudaStream_t st);
int adapter_launch_f16(const AdapterCall& c, int rank_padded, int64_t max_tiles, cudaStream_t st);

constexpr int ADAPTER_MAX_CTAS = 8;  // of a cluster

}  // namespace dst
