// C-ABI entry points of the low-rank adapters: argument checks and how a call is cut.
#include <algorithm>

#include "adapter_call.cuh"

namespace dst {
namespace {

// How a call is cut: CTAs of a cluster (0: two kernels); warps of 16 rows for h inside a CTA and CTAs of them; those for the columns;
// whether the row blocks of a tile share A and B
struct Cut {
  int ctas, share, k_splits, columns, shared_a, shared_b;
};
Cut cut_of(int64_t max_tiles, int tile, int64_t K_padded, int64_t N, int rank_padded) {
  const int64_t sms = sm_count(), blocks = max_tiles * (tile / 16);
  Cut cut{0, 8, 1, 1, 0, 0};
  // Up to 48 blocks the cluster's one launch costs the host 5 us less (11 against 16 a call) and the device as much: 1 row of 4096 x
  // 4096 4.2 us against 4.1, 333 rows 8.0 against 8.2, 48 pairs (rank 16 twice) 13.1 against 14.4 with their plan; 64 rows of 37
  // adapters (53 blocks) through 4096 x 11008 14.9 against 10.8. A cluster takes tiles of 16 rows only.
  if (tile == 16 && blocks <= 48) {
    cut.ctas = 1;
    while (cut.ctas < ADAPTER_MAX_CTAS && max_tiles * cut.ctas * 2 <= 2 * sms) cut.ctas *= 2;
    return cut;
  }
  // Tiles of 128 rows share B from rank 64 on, and A where there are many: 4000 rows of 2048 x 4096, rank 64, 37.2 us with B shared
  // against 39.8, rank 128 53 against 60; A shared 37.7 against 37.2, rank 128 57.7 against 54.4, 12 000 rows of 4096 x 4096 98 against
  // 105 and 190 against 196.
  cut.shared_b = tile == 128 && rank_padded >= 64, cut.shared_a = cut.shared_b && blocks >= 4 * sms;
  // Warps of a block: doubled as long as those of the machine are few or their steps many enough to pay for a warp's start. Measured,
  // us for 1, 2, 4 ... warps with the other product at its best: 64 rows of 37 adapters, 4096 x 11008, rank 32, columns - / 64.7 / 36.4 /
  // 22.7 / 15.9 / 14.1 / 12.1 (64) / 15.2, h 36.3 / 23.4 / 16.7 / 13.8 / 12.1 / 11.4 (32) / 13.9; 281 rows of 6488 x 1904, rank 128, columns
  // 67.6 / 44.4 / 32.5 / 26.9 / 23.3 / 21.5 (32) / 24.5, h 74.7 / 46.0 / 32.3 / 24.3 / 21.6 (16) / 24.4; 2000 rows of 1024 x 1024, rank 16,
  // columns 17.4 / 11.6 / 9.0 / 7.8 / 7.5 (16) / 9.2, h 10.1 / 8.5 / 7.5 / 7.2 (8) / 7.3; 12 000 rows of 4096 x 4096, rank 64, columns
  // - / 115.6 / 112.2 / 103.2 (8) / 106.6, h 109.1 / 99.4 / 98.0 (4) / 102.6
  const auto doubled = [](auto more) {
    int n = 1;
    while (more((int64_t)n * 2)) n *= 2;
    return n;
  };
  const int h = doubled([&](int64_t n) {  // steps of 64 values of K; long sums count twice
    const int64_t steps = K_padded / 64, all = blocks * n * (rank_padded >= 64 ? 2 : 1);
    return all <= 22 * sms ? steps >= n * (all <= 4 * sms ? 1 : all <= 12 * sms ? 2 : 4) : n <= 4 && steps >= 16 * n;
  });
  cut.columns = doubled([&](int64_t n) {  // steps of 32 columns; the widest shared ones count twice
    const int64_t steps = (N + 31) / 32, weight = cut.shared_b && rank_padded > 64 ? 2 : 1, all = blocks * n * weight;
    return all <= 32 * sms ? 10 * steps >= n * (all <= 8 * sms ? 10 : all <= 16 * sms ? 18 : 50) : n <= 8 && steps >= 16 * weight * n;
  });
  cut.share = cut.shared_a ? 1 : std::min(h, 8), cut.k_splits = std::min(cut.shared_a ? h : std::max(h / 8, 1), 16);
  return cut;
}

}  // namespace
}  // namespace dst

// Tiles of 128 rows let eight warps share A and B where the rank is 64 or more, once requests fill them (lower ranks take their
// row blocks apart). Rank 64: 4000 rows, float32 results 37 us against 41 in tiles of 16, 1654 rows 30 against 21.
extern "C" int dst_adapter_tile(int64_t rows, int64_t bins) { return rows >= 20 * (int64_t)dst::sm_count() && rows >= 128 * bins ? 128 : 16; }

extern "C" size_t dst_adapter_workspace_bytes(const dst_adapters* w, const dst_adapter_rows* plan) {
  using namespace dst;
  if (!w || !plan || plan->max_tiles <= 0 || plan->positions <= 0 || w->parts < 1 || w->rank_padded < 1 || w->K_padded < 1 || w->N < 1)
    return 0;
  const Cut cut = cut_of(plan->max_tiles, plan->tile, w->K_padded, w->N, w->rank_padded);
  return cut.ctas ? 0 : (size_t)cut.k_splits * plan->positions * w->parts * w->rank_padded * sizeof(float);
}

extern "C" int dst_adapter_apply(const dst_adapters* w, const dst_adapter_rows* plan, const void* x, int64_t x_stride, const void* base,
                                 int base_dtype, int64_t base_stride, void* out, int out_dtype, int64_t out_stride, void* workspace,
                                 size_t workspace_bytes, dst_stream_t stream) {
  using namespace dst;
  if (!w || !plan || base_dtype < DST_OUT_F32 || base_dtype > DST_OUT_F16 || out_dtype < DST_OUT_F32 || out_dtype > DST_OUT_F16 ||
      (w->dtype != DST_ACT_BF16 && w->dtype != DST_ACT_F16) || w->K <= 0 || w->N <= 0 ||
      w->matrices_per_slot <= 0 || plan->max_tiles < 0)
    return DST_ERR_BAD_ARG;
  if (w->parts < 1 || w->N % w->parts != 0 || w->N > (1 << 24) || w->K > (1 << 24) || w->K_padded != cdiv64(w->K, 64) * 64 || x_stride < w->K ||
      out_stride < w->N || (base && base_stride < w->N) || plan->max_tiles > 0x00ffffff || plan->positions < 0 ||
      (plan->tile != 16 && plan->tile != 128))
    return DST_ERR_BAD_SHAPE;
  if (plan->max_tiles == 0) return DST_OK;
  if (!w->a || !w->b || !w->scale || !w->ranks || !plan->tiles || !x || !out) return DST_ERR_BAD_ARG;
  const auto off = [](const void* p, int size) { return reinterpret_cast<uintptr_t>(p) % size != 0; };
  if (off(w->a, 16) || off(w->b, 16) || off(plan->tiles, 8) || off(w->scale, 4) || off(w->ranks, 4) || off(plan->rows, 4) ||
      off(plan->x_rows, 4) || off(x, 2) || off(base, base_dtype == DST_OUT_F32 ? 4 : 2) || off(out, out_dtype == DST_OUT_F32 ? 4 : 2))
    return DST_ERR_ALIGNMENT;
  AdapterCall c{};
  c.x = x, c.x_stride = x_stride, c.x_rows = plan->x_rows, c.rows = plan->rows, c.tiles = plan->tiles;
  c.a = static_cast<const uint16_t*>(w->a), c.b = static_cast<const uint16_t*>(w->b), c.scale = w->scale, c.ranks = w->ranks;
  c.per_slot = w->matrices_per_slot, c.K = w->K, c.Kp = w->K_padded, c.Np = w->N / w->parts, c.parts = w->parts;
  c.base = base, c.base_dtype = base_dtype, c.base_stride = base_stride, c.out = out, c.out_dtype = out_dtype, c.out_stride = out_stride;
  const auto aligned = [](const void* p, int64_t stride, int size) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * size % 16 == 0; };
  c.x_vec = aligned(x, x_stride, 2);
  const int own = w->dtype == DST_ACT_BF16 ? DST_OUT_BF16 : DST_OUT_F16, out_size = out_dtype == DST_OUT_F32 ? 4 : 2;
  c.kind = -1;
  if (c.Np % (w->parts == 1 ? 16 / out_size : 32) == 0 && aligned(out, out_stride, out_size) &&
      (!base || aligned(base, base_stride, base_dtype == DST_OUT_F32 ? 4 : 2))) {
    if (base && base_dtype == DST_OUT_F32 && (out_dtype == own || out_dtype == DST_OUT_F32)) c.kind = out_dtype == own ? 0 : 1;
    else if (out_dtype == own && (!base || base_dtype == own)) c.kind = base ? 2 : 3;
  }
  const Cut cut = cut_of(plan->max_tiles, plan->tile, w->K_padded, w->N, w->rank_padded);
  c.sub = plan->tile / 16, c.shared_a = cut.shared_a, c.shared_b = cut.shared_b, c.ctas = cut.ctas, c.share = cut.share, c.k_splits = cut.k_splits, c.splits = cut.columns;
  c.positions = plan->positions, c.h = static_cast<float*>(workspace);
  if (!cut.ctas) {
    if (!workspace || workspace_bytes < dst_adapter_workspace_bytes(w, plan)) return DST_ERR_BAD_ARG;
    if ((reinterpret_cast<uintptr_t>(workspace) & 15) != 0) return DST_ERR_ALIGNMENT;
  }
  auto st = static_cast<cudaStream_t>(stream);
  return w->dtype == DST_ACT_BF16 ? adapter_launch_bf16(c, w->rank_padded, plan->max_tiles, st)
                                  : adapter_launch_f16(c, w->rank_padded, plan->max_tiles, st);
}
