// One element type's instances of the dense product (compiled once per type: -DBNPVI_T=0 fp32, 1 bf16, 2 fp16).
#include "dense_kernels.h"

namespace bnpvi {

#if BNPVI_T == 0
typedef float elem_t;
#define BNPVI_GEMM_LAUNCH launch_gemm_f32
#elif BNPVI_T == 1
typedef bf16_t elem_t;
#define BNPVI_GEMM_LAUNCH launch_gemm_bf16
#else
typedef f16_t elem_t;
#define BNPVI_GEMM_LAUNCH launch_gemm_f16
#endif

template <int KIND, int BR, int BC, int WR, int WC, bool DIRECT, bool PAIR>
static int launch_one(const GemmArgs& a, const bnpvi_ctx* ctx, int64_t tiles, hipStream_t s) {
  static LdsLimit limit;
  constexpr int threads = (BR / WR) * (BC / WC) * 64, lds = Rings<BR, BC, WR, WC, 128, KIND, DIRECT, PAIR>::kBytes;
  auto kernel = gemm_kernel<elem_t, KIND, BR, BC, WR, WC, 128, DIRECT, PAIR>;
  if (lds > 64 * 1024) BNPVI_HIP(limit.raise((const void*)kernel, ctx->device));
  // as many workgroups as fit a CU (LDS; two waves a SIMD of the larger tiles fill the registers), no more than tiles
  const int64_t per_cu = std::min(kMaxLdsBytes / lds, 1024 / threads);
  kernel<<<(unsigned)std::min<int64_t>(tiles, per_cu * ctx->num_cu), threads, lds, s>>>(a, (uint32_t)tiles);
  BNPVI_LAUNCH_CHECK();
  return BNPVI_OK;
}

template <int KIND, bool DIRECT, bool PAIR>
static int launch_tile(const GemmArgs& a, int tile, const bnpvi_ctx* ctx, int64_t tiles, hipStream_t s) {
  switch (tile) {
    case kTile256:
      if constexpr (DIRECT && sizeof(elem_t) == 2) return launch_one<KIND, 256, 256, 128, 64, DIRECT, PAIR>(a, ctx, tiles, s);
      return BNPVI_EINVAL;
    case kTile128:
      return launch_one<KIND, 128, 128, 64, 64, DIRECT, PAIR>(a, ctx, tiles, s);
    case kTile64:
      return launch_one<KIND, 64, 64, 32, 32, DIRECT, PAIR>(a, ctx, tiles, s);
    case kTileFlat:
      return launch_one<KIND, 32, 128, 32, 32, DIRECT, PAIR>(a, ctx, tiles, s);
    default:
      // 32 columns of a half-long stage are less than a piece a lane
      if constexpr (PAIR) return BNPVI_EINVAL;
      else return launch_one<KIND, 128, 32, 32, 32, DIRECT, PAIR>(a, ctx, tiles, s);
  }
}

int BNPVI_GEMM_LAUNCH(int kind, int tile, bool direct, bool pair, const GemmArgs& a, const bnpvi_ctx* ctx, hipStream_t s) {
  const int64_t tiles = (int64_t)a.row_tiles * a.col_tiles * (kind == kDw && a.map != nullptr ? a.entries : a.splits);
  if (tiles <= 0) return BNPVI_OK;
  BNPVI_REQUIRE(tiles < (int64_t(1) << 31), "dense: %lld tiles", (long long)tiles);
  if (pair) {
    if constexpr (sizeof(elem_t) == 2) {
      if (kind == kDx) return direct ? launch_tile<kDx, true, true>(a, tile, ctx, tiles, s) : launch_tile<kDx, false, true>(a, tile, ctx, tiles, s);
      if (kind == kDw) return direct ? launch_tile<kDw, true, true>(a, tile, ctx, tiles, s) : launch_tile<kDw, false, true>(a, tile, ctx, tiles, s);
    }
    return BNPVI_EINVAL;
  }
  if (direct) {
    if (kind == kFwd) return launch_tile<kFwd, true, false>(a, tile, ctx, tiles, s);
    if (kind == kDx) return launch_tile<kDx, true, false>(a, tile, ctx, tiles, s);
    return launch_tile<kDw, true, false>(a, tile, ctx, tiles, s);
  }
  if (kind == kFwd) return launch_tile<kFwd, false, false>(a, tile, ctx, tiles, s);
  if (kind == kDx) return launch_tile<kDx, false, false>(a, tile, ctx, tiles, s);
  return launch_tile<kDw, false, false>(a, tile, ctx, tiles, s);
}

}  // namespace bnpvi
