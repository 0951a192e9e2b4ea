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

template <int KIND, int BR, int BC, int WR, int WC, bool DIRECT>
static int launch_one(const GemmArgs& a, int device, int64_t grid, hipStream_t s) {
  static LdsLimit limit;
  constexpr int lds = gemm_lds_bytes<BR, BC>();
  auto kernel = gemm_kernel<elem_t, KIND, BR, BC, WR, WC, DIRECT>;
  if (lds > 64 * 1024) BNPVI_HIP(limit.raise((const void*)kernel, device));
  kernel<<<(unsigned)grid, (BR / WR) * (BC / WC) * 64, lds, s>>>(a);
  BNPVI_LAUNCH_CHECK();
  return BNPVI_OK;
}

template <int KIND, bool DIRECT>
static int launch_tile(const GemmArgs& a, int tile, int device, int64_t grid, hipStream_t s) {
  switch (tile) {
    case kTile128:
      return launch_one<KIND, 128, 128, 64, 64, DIRECT>(a, device, grid, s);
    case kTile256:
      if constexpr (DIRECT && sizeof(elem_t) == 2) return launch_one<KIND, 256, 256, 128, 64, DIRECT>(a, device, grid, s);
      return BNPVI_EINVAL;
    case kTile64:
      return launch_one<KIND, 64, 64, 32, 32, DIRECT>(a, device, grid, s);
    case kTileFlat:
      return launch_one<KIND, 32, 128, 32, 32, DIRECT>(a, device, grid, s);
    default:
      return launch_one<KIND, 128, 32, 32, 32, DIRECT>(a, device, grid, s);
  }
}

int BNPVI_GEMM_LAUNCH(int kind, int tile, bool direct, const GemmArgs& a, int device, hipStream_t s) {
  const int64_t z = kind == kDw ? (int64_t)a.G * a.splits : a.splits;
  const int64_t grid = a.row_tiles * a.col_tiles * z;
  if (grid <= 0) return BNPVI_OK;
  BNPVI_REQUIRE(grid < (int64_t(1) << 31), "dense: %lld workgroups", (long long)grid);
  if (direct) {
    if (kind == kFwd) return launch_tile<kFwd, true>(a, tile, device, grid, s);
    if (kind == kDx) return launch_tile<kDx, true>(a, tile, device, grid, s);
    return launch_tile<kDw, true>(a, tile, device, grid, s);
  }
  if (kind == kFwd) return launch_tile<kFwd, false>(a, tile, device, grid, s);
  if (kind == kDx) return launch_tile<kDx, false>(a, tile, device, grid, s);
  return launch_tile<kDw, false>(a, tile, device, grid, s);
}

}  // namespace bnpvi
