// Tiles of int8 linears (gemm_tile.h).
#include "gemm_tile.h"

namespace mi355 {
namespace {

constexpr TileSpec kTiles[] = {{G256X256, 256, 256, 1, true, 1.85f},   {G128X256, 128, 256, 1, true, 1.14f},
                               {G128X128X2, 128, 128, 2, true, 1.16f}, {G128X128, 128, 128, 1, true, 0.66f},
                               {G64X128, 64, 128, 1, true, 0.42f},     {G64X64, 64, 64, 1, false, 0.31f}};

TilePlan plan(const LinArgs& a) {
  return gemm_plan(kTiles, a.M, a.N, lin_rows(a), static_cast<int>(cdiv(a.K * kind_bytes(kind_of(a)), GSB)));
}

}  // namespace

int launch_linear_keep(const LinArgs& a, const TilePlan& p, hipStream_t st);

int linear_gemm_splits(const LinArgs& a) { return plan(a).splits; }

int launch_linear_gemm(const LinArgs& a0, const LinArgs& a, hipStream_t st) {
  const TilePlan p = plan(a0);
  if (a0.z) return launch_linear_keep(a, p, st);
  if (p.splits > 1) return launch_gemm_shape<K_I8, false, false, false, E_RAW>(a, p, st);
  if (lin_gated(a.activation)) return launch_gemm_shape<K_I8, false, false, true, E_LINEAR>(a, p, st);
  return launch_gemm_shape<K_I8, false, false, false, E_LINEAR>(a, p, st);
}

}  // namespace mi355
