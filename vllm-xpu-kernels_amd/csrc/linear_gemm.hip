// Tiles of int8 linears, and the choice of tiles of linears that keep their sums (gemm_tile.h).
#include "gemm_tile.h"

namespace mi355 {

int launch_linear_keep(const LinArgs& a, const TilePlan& p, hipStream_t st);

namespace {

// Times of a stage and of the rest of a round, from 8192 x 4096 x 8192 (gated 8192 x 8192 x 8192,
// kept 8192 x 7168 x 4096) and products of 1003 and 300 rows on every shape (rows x K x weight
// rows).  Shapes for the fill of 256 CUs: int8 1003 x 2880 x 2880 96 x 128 21.0 us, 128 x 128 with
// two workgroups to a CU 26.8, 192 x 128 33.5; kept 1003 x 2880 x 5760 128 x 192 42.6, 256 x 128
// 48.3.  A gated product's last shapes are those of its split one, which has no gates.
constexpr TileSpec kTiles[] = {
    {G256X128, 256, 128, 1, 1.0f, 6.0f},
    {G128X256, 128, 256, 1, 1.0f, 5.0f},
    {G192X128, 192, 128, 1, 0.86f, 5.0f},
    {G128X128X2, 128, 128, 2, 0.97f, 6.0f},
    {G128X128, 128, 128, 1, 0.58f, 3.0f},
    {G96X128, 96, 128, 1, 0.49f, 2.6f},
    {G64X128X2, 64, 128, 2, 0.68f, 2.0f},
    {G64X64X3, 64, 64, 3, 0.7f, 1.5f}};
constexpr TileSpec kTilesGated[] = {
    {G256X256, 256, 256, 1, 1.78f, 7.0f},
    {G256X128, 256, 128, 1, 0.98f, 5.0f},
    {G128X256, 128, 256, 1, 0.98f, 5.0f},
    {G128X192, 128, 192, 1, 0.76f, 5.0f},
    {G128X128X2, 128, 128, 2, 0.97f, 6.0f},
    {G128X128, 128, 128, 1, 0.55f, 3.0f},
    {G64X128X2, 64, 128, 2, 0.65f, 2.0f},
    {G192X128, 192, 128, 1, 0.86f, 5.0f},
    {G96X128, 96, 128, 1, 0.49f, 2.6f},
    {G64X64X3, 64, 64, 3, 0.7f, 1.5f}};
constexpr TileSpec kTilesKeep[] = {
    {G256X256, 256, 256, 1, 1.77f, 12.0f},
    {G256X128, 256, 128, 1, 0.99f, 6.0f},
    {G128X256, 128, 256, 1, 0.99f, 6.0f},
    {G128X192, 128, 192, 1, 0.77f, 5.0f},
    {G128X128X2, 128, 128, 2, 1.05f, 6.0f},
    {G128X128, 128, 128, 1, 0.6f, 3.5f},
    {G64X128X2, 64, 128, 2, 0.68f, 2.5f},
    {G192X192, 192, 192, 1, 0.95f, 5.0f},
    {G192X128, 192, 128, 1, 0.69f, 4.0f},
    {G96X128, 96, 128, 1, 0.45f, 2.0f},
    {G64X64X3, 64, 64, 3, 0.7f, 1.5f}};

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
  if (p.splits > 1) return launch_gemm_shape<K_I8, false, false, false, E_RAW>(a, p, st);
  if (lin_gated(a.activation)) return launch_gemm_shape<K_I8, false, false, true, E_LINEAR>(a, p, st);
  return launch_gemm_shape<K_I8, false, false, false, E_LINEAR>(a, p, st);
}

}  // namespace mi355
