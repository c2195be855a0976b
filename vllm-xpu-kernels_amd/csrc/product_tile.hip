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

template <int KIND, bool TQ, bool TP, bool GATED, int EPI, int BI, int BJ, int WI, int WJ, int NSTAGE, typename Walk,
          int BYTES>
__device__ __forceinline__ void gemm_tiles(const LinArgs& a, int tiles_i, int tiles_j, int stages_per_split,
                                           Walk walk, uint8_t (&lds)[BYTES]) {
#include "gemm_tile_body.h"
}
// Two products in one launch, 256 x 256 tiles on 256 workgroups: those of w, then those of x
// (tile_walk.h).
template <int KIND>
__global__ __launch_bounds__(512, gemm_waves_per_simd(8, 256, 256, 2)) void product_pair_kernel(
    const LinArgs w, const LinArgs x, int wi, int wj, int wn, int xi, int xj, int xn, int extra) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * 512 * GSB];
  const int block = static_cast<int>(blockIdx.x), blocks = static_cast<int>(gridDim.x);
  gemm_tiles<KIND, true, true, false, E_PLAIN, 256, 256, 2, 4, 2>(w, wi, wj, wn, XcdWalk(wi * wj, block, blocks),
                                                                  lds);
  gemm_tiles<KIND, false, true, false, E_PLAIN, 256, 256, 2, 4, 2>(
      x, xi, xj, xn, SecondWalk(wi * wj, xi * xj, extra, block, blocks), lds);
}

// How many tiles of x the light workgroups take first, or -1 where two launches take as
// long: by the last workgroup's tiles, in stages and their rounds (a whole backward pass in us, two
// launches / one: 8192 x 7168 x 4096 847 / 813, 4323 x 8456 x 1368 238 / 217, 3216 x 8960 x 4078
// 479 / 433, 7431 x 8200 x 1362 367 / 351).
int pair_extra(const Product& x, const Product& w) {
  // (small ones have no such tiles: their plans, 0.4 us each, are not made again)
  if (static_cast<double>(x.I) * x.J * x.R < 1e10) return -1;
  const TilePlan px = plan(x), pw = plan(w);
  if (px.shape != G256X256 || pw.shape != G256X256 || px.splits > 1 || pw.splits > 1) return -1;
  const int64_t nx = cdiv(cdiv(x.I, 256) * cdiv(x.J, 256), 8), nw = cdiv(cdiv(w.I, 256) * cdiv(w.J, 256), 8);
  const double cx = kTiles[0].us * px.per + kTiles[0].round, cw = kTiles[0].us * pw.per + kTiles[0].round;
  const int64_t heavy = nw % 32, light = 32 - heavy;
  if (!heavy) return -1;
  int64_t extra = static_cast<int64_t>(cw / cx + 0.5);
  extra = extra < nx / light ? extra : nx / light;
  const double first = nw / 32 * cw + (extra * cx > cw ? extra * cx : cw);
  const double one = first + cdiv(nx - light * extra, 32) * cx;
  return extra && one < 0.98 * (cdiv(nw, 32) * cw + cdiv(nx, 32) * cx) ? static_cast<int>(extra) : -1;
}

LinArgs args_of(const Product& p) {
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
  a.out = p.out;
  a.ldo = p.ldo;
  return a;
}

}  // namespace

bool product_pair_supported(const Product& x, const Product& w) {
  return !x.transposed && w.transposed && product_tile_supported(x) && product_tile_supported(w) &&
         pair_extra(x, w) > 0;
}
int launch_product_pair(const Product& x, const Product& w, hipStream_t st) {
  const int extra = pair_extra(x, w);
  auto go = [&](auto kind) {
    product_pair_kernel<decltype(kind)::value><<<dim3(256), dim3(512), 0, st>>>(
        args_of(w), args_of(x), static_cast<int>(cdiv(w.I, 256)), static_cast<int>(cdiv(w.J, 256)), plan(w).per,
        static_cast<int>(cdiv(x.I, 256)), static_cast<int>(cdiv(x.J, 256)), plan(x).per, extra);
  };
  if (x.dtype == MI355MOE_F16) go(std::integral_constant<int, K_F16>{});
  else go(std::integral_constant<int, K_BF16>{});
  MI_LAUNCH_CHECK();
  return MI355MOE_OK;
}

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
  LinArgs a = args_of(p);
  if (n.splits > 1) a.out = part;
  return p.dtype == MI355MOE_F16 ? launch<K_F16>(a, p.transposed, n, st)
                                 : launch<K_BF16>(a, p.transposed, n, st);
}

}  // namespace mi355
