// Tiles of the products of a backward pass (product.h, gemm_tile.h).
#include "gemm_tile.h"

namespace mi355 {
namespace {

// Times of a stage and of the rest of a round, from dx 8192 x 4096 x 7168 and dW 4096 x 8192 x 7168
// (I x R x J) on every shape.  Shapes for the fill of 256 CUs: 1003 x 5760 x 2880 96 x 128 43 us,
// 128 x 128 49; 5760 x 1003 x 2880 192 x 192 42 us, 128 x 128 44 to 52, 256 x 256 77.
constexpr TileSpec kTiles[] = {
    {G256X256, 256, 256, 1, 1.51f, 7.0f},
    {G256X128, 256, 128, 1, 0.9f, 5.0f},
    {G128X256, 128, 256, 1, 0.9f, 5.0f},
    {G192X192, 192, 192, 1, 0.98f, 4.5f},
    {G192X128, 192, 128, 1, 0.7f, 3.5f},
    {G128X128X2, 128, 128, 2, 0.99f, 5.0f},
    {G128X128, 128, 128, 1, 0.56f, 3.0f},
    {G96X128, 96, 128, 1, 0.44f, 1.5f},
    {G64X128X2, 64, 128, 2, 0.65f, 1.5f},
    {G64X64X3, 64, 64, 3, 0.7f, 1.5f}};

TilePlan plan(const Product& p) {
  return gemm_plan(kTiles, p.I, p.J, p.J, static_cast<int>(cdiv(p.R, GSB / 2)));
}

template <int KIND>
int launch(const LinArgs& a, bool transposed, const TilePlan& n, hipStream_t st) {
  if (n.splits > 1)
    return transposed ? launch_gemm_shape<KIND, true, true, false, E_RAW>(a, n, st)
                      : launch_gemm_shape<KIND, false, true, false, E_RAW>(a, n, st);
  return transposed ? launch_gemm_shape<KIND, true, true, false, E_PLAIN>(a, n, st)
                    : launch_gemm_shape<KIND, false, true, false, E_PLAIN>(a, n, st);
}

}  // namespace

bool product_tile_supported(const Product& p, bool padded) {
  const int64_t lim = int64_t(1) << 32;
  auto rows16 = [](const void* b, int64_t ld) {
    return ((reinterpret_cast<uintptr_t>(b) | static_cast<uintptr_t>(ld * 2)) & 15) == 0;
  };
  return p.R > 0 && rows16(p.q, p.ldq) && rows16(p.p, p.ldp) && (p.J % 8 == 0 || padded) &&
         256 * p.ldq * 2 < lim && 256 * p.ldp * 2 < lim && p.R < (int64_t(1) << 30) &&
         cdiv(p.I, 64) * cdiv(p.J, 64) < (int64_t(1) << 24);  // tiles are counted in 32 bits
}
int product_tile_splits(const Product& p) { return plan(p).splits; }
int launch_product_tile(const Product& p, float* part, hipStream_t st) {
  const TilePlan n = plan(p);
  LinArgs a{};
  a.x_dtype = a.out_dtype = p.dtype;
  a.activation = MI355MOE_LINEAR_NONE;
  a.M = p.I;
  a.N = p.J;
  a.K = p.R;
  a.x = p.q;
  a.ldx = p.ldq;
  a.weight = p.p;
  a.ldw = p.ldp;
  a.out = n.splits > 1 ? static_cast<void*>(part) : p.out;
  a.ldo = p.ldo;
  return p.dtype == MI355MOE_F16 ? launch<K_F16>(a, p.transposed, n, st)
                                 : launch<K_BF16>(a, p.transposed, n, st);
}

}  // namespace mi355
