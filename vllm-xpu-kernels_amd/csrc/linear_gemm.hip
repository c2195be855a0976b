// Tiles of int8 linears, and the choice of tiles of linears that keep their sums (gemm_tile.h).
#include "gemm_tile.h"

namespace mi355 {

int launch_linear_keep(const LinArgs& a, const TilePlan& p, hipStream_t st);

namespace {

constexpr TileSpec kTiles[] = {{G256X128, 256, 128, 1, 1.05f, 5.f}, {G128X256, 128, 256, 1, 1.10f, 5.f},
                               {G128X128X2, 128, 128, 2, 1.09f, 5.f}, {G128X128, 128, 128, 1, 0.64f, 4.f},
                               {G64X128, 64, 128, 1, 0.42f, 3.f}, {G64X64, 64, 64, 1, 0.31f, 2.5f}};
constexpr TileSpec kTilesGated[] = {{G256X256, 256, 256, 1, 2.0f, 8.f}, {G256X128, 256, 128, 1, 0.98f, 5.f},
                                    {G128X256, 128, 256, 1, 1.02f, 5.f}, {G128X128X2, 128, 128, 2, 1.03f, 5.f},
                                    {G128X128, 128, 128, 1, 0.60f, 4.f}, {G64X128, 64, 128, 1, 0.41f, 3.f},
                                    {G64X64, 64, 64, 1, 0.31f, 2.5f}};
constexpr TileSpec kTilesKeep[] = {{G256X256, 256, 256, 1, 1.8f, 12.f}, {G256X128, 256, 128, 1, 0.93f, 7.f},
                                   {G128X256, 128, 256, 1, 0.96f, 7.f}, {G128X128X2, 128, 128, 2, 1.02f, 7.f},
                                   {G128X128, 128, 128, 1, 0.58f, 5.f}, {G64X128, 64, 128, 1, 0.40f, 4.f},
                                   {G64X64, 64, 64, 1, 0.31f, 2.5f}};

TilePlan plan(const LinArgs& a) {
  const int nk = static_cast<int>(cdiv(a.K * kind_bytes(kind_of(a)), GSB));
  if (a.z) return gemm_plan(kTilesKeep, a.M, a.N, lin_rows(a), nk);
  if (lin_gated(a.activation)) return gemm_plan(kTilesGated, a.M, a.N, lin_rows(a), nk);
  return gemm_plan(kTiles, a.M, a.N, lin_rows(a), nk);
}

}  // namespace

int linear_gemm_splits(const LinArgs& a) { return plan(a).splits; }

int launch_linear_gemm(const LinArgs& a0, const LinArgs& a, hipStream_t st) {
  const TilePlan p = plan(a0);
  if (a0.z) return launch_linear_keep(a, p, st);
  if (p.splits > 1) return launch_gemm_shape<K_I8, false, false, false, E_RAW, true>(a, p, st);
  if (lin_gated(a.activation)) return launch_gemm_shape<K_I8, false, false, true, E_LINEAR, true>(a, p, st);
  return launch_gemm_shape<K_I8, false, false, false, E_LINEAR, true>(a, p, st);
}

}  // namespace mi355
