// The products of a backward pass (product.h) for any size, stride and alignment:
// 64 x 64 output tiles, 4 waves of 16 columns each, both operands' stages of 64 r copied
// through registers into LDS with zeros past the edges.  Operands that lie along r
// are read as they are, those that lie across r by the transposing LDS read (each
// lane's 8 values of a matrix instruction are a column's).
#include "product.h"

namespace mi355 {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int PT = 64;           // tile side, and r of a stage
constexpr int PITCH = 2 * PT + 16;

// Stages [split * per, ...); the next stage is in registers while this one's products run.
template <bool F16, bool TQ>
__global__ __launch_bounds__(256) void product_any_kernel(const Product a, float* __restrict__ part,
                                                          int per) {
  __shared__ __attribute__((aligned(16))) uint8_t sq[PT * PITCH];
  __shared__ __attribute__((aligned(16))) uint8_t sp[PT * PITCH];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int l16 = lane & 15, g = lane >> 4;
  const int64_t j0 = static_cast<int64_t>(blockIdx.x) * PT, i0 = static_cast<int64_t>(blockIdx.y) * PT;
  const int64_t r0 = static_cast<int64_t>(blockIdx.z) * per * PT;
  const int64_t rend = r0 + static_cast<int64_t>(per) * PT < a.R ? r0 + static_cast<int64_t>(per) * PT : a.R;
  const uint8_t* q = static_cast<const uint8_t*>(a.q);
  const uint8_t* p = static_cast<const uint8_t*>(a.p);

  f32x4 acc[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  uint4 pq[2], pp[2];
  auto fetch = [&](int64_t r) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int row = (e * 256 + tid) >> 3, c = ((e * 256 + tid) & 7) * 8;
      pp[e] = row16(p + (r + row) * a.ldp * 2, r + row < rend, (j0 + c) * 2, a.J * 2);
      if constexpr (TQ) pq[e] = row16(q + (r + row) * a.ldq * 2, r + row < rend, (i0 + c) * 2, a.I * 2);
      else pq[e] = row16(q + (i0 + row) * a.ldq * 2, i0 + row < a.I, (r + c) * 2, rend * 2);
    }
  };
  if (r0 < rend) fetch(r0);
  for (int64_t r = r0; r < rend; r += PT) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int at = ((e * 256 + tid) >> 3) * PITCH + ((e * 256 + tid) & 7) * 16;
      *reinterpret_cast<uint4*>(sq + at) = pq[e];
      *reinterpret_cast<uint4*>(sp + at) = pp[e];
    }
    __syncthreads();
    if (r + PT < rend) fetch(r + PT);  // uniform
    // 8 r of column `col`: two transposing reads of 4
    auto column8 = [&](const uint8_t* s, int t, int col) __attribute__((always_inline)) {
      const uint8_t* at = s + (32 * t + 8 * g + (l16 >> 2)) * PITCH + (col + 4 * (l16 & 3)) * 2;
      const uint2 a0 = lds_column4(at), a1 = lds_column4(at + 4 * PITCH);
      return make_uint4(a0.x, a0.y, a1.x, a1.y);
    };
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint4 av = column8(sp, t, 16 * wave);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint4 bv;
        if constexpr (TQ) bv = column8(sq, t, 16 * i);
        else bv = *reinterpret_cast<const uint4*>(sq + (16 * i + l16) * PITCH + 64 * t + 16 * g);
        acc[i] = mfma16_16x16x32<F16>(av, bv, acc[i]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t row = i0 + 16 * i + l16;
    if (row >= a.I) continue;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t col = j0 + 16 * wave + 4 * g + k;
      if (col >= a.J) continue;
      if (part) part[(static_cast<int64_t>(blockIdx.z) * a.I + row) * a.J + col] = acc[i][k];
      else static_cast<uint16_t*>(a.out)[row * a.ldo + col] = st16<F16>(acc[i][k]);
    }
  }
}

// r is split until there are about 1000 workgroups (four per CU), 4 stages each at least
int any_stages(const Product& p) {
  const int64_t n = cdiv(p.R, PT), tiles = cdiv(p.I, PT) * cdiv(p.J, PT);
  const int64_t most = n / 4 > 1 ? n / 4 : 1, want = cdiv(1000, tiles);
  const int64_t per = cdiv(n, want < most ? want : most);
  return static_cast<int>(per > 0 ? per : 1);
}
int any_splits(const Product& p) {
  const int s = static_cast<int>(cdiv(cdiv(p.R, PT), any_stages(p)));
  return s > 0 ? s : 1;
}
size_t partials(const Product& p, int splits) {
  return splits == 1 ? 0 : static_cast<size_t>(splits) * p.I * p.J * sizeof(float);
}

// What runs: the product on p's rows, or on a copy of them (launch_pack_rows) in the workspace,
// before the partial sums.
struct Run {
  Product p;
  bool pack = false, tile = false;
  int splits = 1;
  size_t parts = 0, total = 0;
};
// p's rows that direct copies cannot fetch are copied to rows that they can: x for dW always, the
// weight for dx where 64 rows share the copy (rows x K x weight rows, us through registers /
// copied: dW 1024 x 6709 x 4094 270 / 86, 257 x 1001 x 1030 20.7 / 13.7, 64 x 1001 x 1030 10.8 / 10.3; dx
// 1024 x 6709 x 4094 360 / 92, 64 x 1001 x 1030 18.3 / 15.4, 40 x 7001 x 6002 52.5 / 56.0).
// Products below 10^9 operations stay as they are: the copy's launch costs a caller what it saves.
constexpr int64_t kPackRows = 64;
constexpr double kPackWork = 1e9;
Run run_of(const Product& given, void* workspace) {
  Run r;
  r.p = given;
  r.tile = product_tile_supported(given);
  if (!r.tile && given.R > 0 && (given.transposed || given.I >= kPackRows) &&
      2.0 * given.I * given.J * given.R >= kPackWork) {
    Product b = given;
    b.p = workspace;
    b.ldp = (given.J + 7) / 8 * 8;
    if (product_tile_supported(b, true)) {
      r.p = b;
      r.pack = r.tile = true;
      r.parts = static_cast<size_t>(b.R) * b.ldp * 2;
    }
  }
  r.splits = r.tile ? product_tile_splits(r.p) : any_splits(r.p);
  r.total = r.parts + partials(r.p, r.splits);
  return r;
}

int launch_any(const Product& p, int splits, float* part, hipStream_t st) {
  const int per = any_stages(p);
  const dim3 grid(static_cast<unsigned>(cdiv(p.J, PT)), static_cast<unsigned>(cdiv(p.I, PT)),
                  static_cast<unsigned>(splits));
  if (p.dtype == MI355MOE_F16) {
    if (p.transposed) product_any_kernel<true, true><<<grid, dim3(256), 0, st>>>(p, part, per);
    else product_any_kernel<true, false><<<grid, dim3(256), 0, st>>>(p, part, per);
  } else {
    if (p.transposed) product_any_kernel<false, true><<<grid, dim3(256), 0, st>>>(p, part, per);
    else product_any_kernel<false, false><<<grid, dim3(256), 0, st>>>(p, part, per);
  }
  MI_LAUNCH_CHECK();
  return MI355MOE_OK;
}

}  // namespace

size_t product_workspace(const Product& p) { return p.I ? run_of(p, nullptr).total : 0; }

int launch_product(const Product& given, void* workspace, hipStream_t st) {
  const Run r = run_of(given, workspace);
  const Product& p = r.p;
  if (r.pack)
    if (const int rc = launch_pack_rows(given.p, given.ldp * 2, given.J * 2, workspace, p.R, st)) return rc;
  float* part = r.splits > 1 ? reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + r.parts) : nullptr;
  const int rc = r.tile ? launch_product_tile(p, part, st) : launch_any(p, r.splits, part, st);
  if (rc || r.splits == 1) return rc;
  LinArgs f{};
  f.out_dtype = p.dtype;
  f.activation = MI355MOE_LINEAR_NONE;
  f.M = p.I;
  f.N = p.J;
  f.K = 1;
  f.out = p.out;
  f.ldo = p.ldo;
  return launch_linear_finish(f, part, r.splits, st);
}

}  // namespace mi355
