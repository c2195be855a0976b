// Backward pass of a gated linear (mi355moe_gated_linear_backward).  With z = x W^T + b
// as its forward kept it, gate z1 = z[:, :N], factor z2 = z[:, N:]:
//   dz1 = dout z2 f'(z1),  dz2 = dout f(z1)
//   dx = dz W,  dW = dz^T x,  db = sum_m dz
// Three launches and two more where they are needed: dz (HBM: 8 bytes of z and 2 of
// dout read, 4 written for each of M x N), the two products (matrix cores; one launch
// where large ones then fill the last rounds of the CUs), and the
// sums of split products and of db's parts.
//
// Precision.  z stays fp32 (16-bit z would add its rounding to every factor of dz);
// dz is rounded to the operands' type, which the matrix instructions take: half a
// step of that type for each term of a sum, the size of the one rounding of the
// output.  db sums the fp32 values.
#include "product.h"

namespace mi355 {
namespace {

typedef mi355moe_gated_linear_backward_args GradArgs;

// f(z) and f'(z) of the gate.
//   SiLU, s = sigmoid(z):  f = z s,  f' = s (1 + z (1 - s))
//   GELU, P = (1 + erf(z / sqrt 2)) / 2:  f = z P,  f' = P + z exp(-z^2 / 2) / sqrt(2 pi)
//   its tanh form = z sigmoid(2 t), t = sqrt(2 / pi) (z + 0.044715 z^3):
//     f' = s + z s (1 - s) 2 t'   (z^2 is bounded in t', where s (1 - s) is 0 long before)
template <int ACT>
__device__ __forceinline__ void gate_grad(float z, float& f, float& df) {
  constexpr float kLog2e = 1.4426950408889634f;
  if constexpr (ACT == MI355MOE_LINEAR_SILU_AND_MUL) {
    const float s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -kLog2e));
    f = z * s;
    df = s * (1.f + z * (1.f - s));
  } else if constexpr (ACT == MI355MOE_LINEAR_GELU_AND_MUL) {
    const float p = 0.5f * (1.f + erff(z * 0.70710678118654752f));
    f = z * p;
    df = p + z * (__builtin_amdgcn_exp2f(z * z * (-0.5f * kLog2e)) * 0.3989422804014327f);
  } else {
    const float t2 = 1.5957691216057308f * (z + 0.044715f * (z * z * z));
    const float s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(t2 * -kLog2e));
    f = z * s;
    df = s + f * (1.f - s) * (1.5957691216057308f * (1.f + 0.134145f * fminf(z * z, 1e30f)));
  }
}

constexpr int kRowBlocks = 128;  // db's parts at most

// Rows of x's block y, 8 columns of the gate and of the factor per lane (VEC: consecutive
// ones; else 64 apart, so that a wave's accesses are runs of 64); with DB the
// workgroup's sums of dz in fp32 go to part[y][2N].  ld: dz's row stride, a multiple of
// 8; the columns past 2N are zeros.
template <int ACT, bool F16, bool VEC, bool DB>
__global__ __launch_bounds__(256) void gated_dz_kernel(const GradArgs a, uint16_t* __restrict__ dz,
                                                       int64_t ld, int64_t rows_per_block,
                                                       float* __restrict__ part) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  constexpr int STEP = VEC ? 1 : 64;
  const int64_t n = static_cast<int64_t>(blockIdx.x) * 512 + (VEC ? lane * 8 : lane);
  const int64_t first = static_cast<int64_t>(blockIdx.y) * rows_per_block;
  const int64_t end = first + rows_per_block < a.M ? first + rows_per_block : a.M;
  const bool on = n < a.N;
  float s1[8], s2[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) s1[k] = s2[k] = 0.f;
  if (on) {
    for (int64_t m = first + wave; m < end; m += 4) {
      const float* z = a.z + m * 2 * a.N + n;
      const uint16_t* d = static_cast<const uint16_t*>(a.dout) + m * a.ldd + n;
      float g[8], u[8], e[8], r1[8], r2[8];
      if constexpr (VEC) {
        const float4* zp = reinterpret_cast<const float4*>(z);
        const float4* up = reinterpret_cast<const float4*>(z + a.N);
        const float4 v[4] = {zp[0], zp[1], up[0], up[1]};
        const uint4 w = *reinterpret_cast<const uint4*>(d);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          g[4 * k] = v[k].x; g[4 * k + 1] = v[k].y; g[4 * k + 2] = v[k].z; g[4 * k + 3] = v[k].w;
          u[4 * k] = v[2 + k].x; u[4 * k + 1] = v[2 + k].y;
          u[4 * k + 2] = v[2 + k].z; u[4 * k + 3] = v[2 + k].w;
        }
        const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) unpack16x2<F16>(ww[k], e[2 * k], e[2 * k + 1]);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const bool in = n + k * STEP < a.N;
          g[k] = in ? z[k * STEP] : 0.f;
          u[k] = in ? z[a.N + k * STEP] : 0.f;
          e[k] = in ? ld16<F16>(d[k * STEP]) : 0.f;
        }
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        float f, df;
        gate_grad<ACT>(g[k], f, df);
        r1[k] = e[k] * u[k] * df;
        r2[k] = e[k] * f;
        if constexpr (DB) {
          s1[k] += r1[k];
          s2[k] += r2[k];
        }
      }
      uint16_t* o = dz + m * ld + n;
      if constexpr (VEC) {
        *reinterpret_cast<uint4*>(o) = make_uint4(pack16x2<F16>(r1[0], r1[1]), pack16x2<F16>(r1[2], r1[3]),
                                                  pack16x2<F16>(r1[4], r1[5]), pack16x2<F16>(r1[6], r1[7]));
        *reinterpret_cast<uint4*>(o + a.N) = make_uint4(pack16x2<F16>(r2[0], r2[1]), pack16x2<F16>(r2[2], r2[3]),
                                                        pack16x2<F16>(r2[4], r2[5]), pack16x2<F16>(r2[6], r2[7]));
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (n + k * STEP < a.N) {
            o[k * STEP] = st16<F16>(r1[k]);
            o[a.N + k * STEP] = st16<F16>(r2[k]);
          }
        if (n == 0)
          for (int64_t c = 2 * a.N; c < ld; ++c) dz[m * ld + c] = 0;
      }
    }
  }
  if constexpr (DB) {
    __shared__ float red[4][64][17];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      red[wave][lane][k] = s1[k];
      red[wave][lane][8 + k] = s2[k];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * 16; i += 256) {
      const int l = (i >> 3) & 63, k = (i & 7) + (i >> 9) * 8;
      const int64_t c = static_cast<int64_t>(blockIdx.x) * 512 + (VEC ? l * 8 + (i & 7) : l + (i & 7) * 64);
      if (c >= a.N) continue;
      const float v = (red[0][l][k] + red[1][l][k]) + (red[2][l][k] + red[3][l][k]);
      part[blockIdx.y * 2 * a.N + (i >> 9) * a.N + c] = v;
    }
  }
}

// db: the parts' sums, 64 columns to a workgroup, its 16 waves a share of the parts each
__global__ __launch_bounds__(1024) void gated_db_kernel(const float* __restrict__ part, int parts,
                                                        int64_t cols, void* out, int dtype) {
  __shared__ float red[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 64 + lane;
  float s = 0.f;
  if (c < cols) {
#pragma unroll
    for (int e = 0; e < kRowBlocks / 16; ++e) {
      const int p = wave * (kRowBlocks / 16) + e;
      if (p < parts) s += part[p * cols + c];
    }
  }
  red[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && c < cols) {
#pragma unroll
    for (int w = 1; w < 16; ++w) s += red[w][lane];
    st_any(out, dtype, c, s);
  }
}

template <int ACT, bool F16, bool VEC>
void launch_dz(const GradArgs& a, uint16_t* dz, int64_t ld, float* part, int blocks, int64_t per,
               hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(cdiv(a.N, 512)), static_cast<unsigned>(blocks));
  if (a.dbias) gated_dz_kernel<ACT, F16, VEC, true><<<grid, dim3(256), 0, st>>>(a, dz, ld, per, part);
  else gated_dz_kernel<ACT, F16, VEC, false><<<grid, dim3(256), 0, st>>>(a, dz, ld, per, part);
}
template <int ACT>
void launch_dz(const GradArgs& a, uint16_t* dz, int64_t ld, float* part, int blocks, int64_t per,
               hipStream_t st) {
  const bool vec = a.N % 8 == 0 && (reinterpret_cast<uintptr_t>(a.z) & 15) == 0 &&
                   ((reinterpret_cast<uintptr_t>(a.dout) | static_cast<uintptr_t>(a.ldd * 2)) & 15) == 0;
  if (a.dtype == MI355MOE_F16) {
    if (vec) launch_dz<ACT, true, true>(a, dz, ld, part, blocks, per, st);
    else launch_dz<ACT, true, false>(a, dz, ld, part, blocks, per, st);
  } else {
    if (vec) launch_dz<ACT, false, true>(a, dz, ld, part, blocks, per, st);
    else launch_dz<ACT, false, false>(a, dz, ld, part, blocks, per, st);
  }
}

int check(const GradArgs& a) {
  MI_ARG(a.dtype == MI355MOE_BF16 || a.dtype == MI355MOE_F16,
         "gated_linear_backward: operands must be bfloat16 or float16");
  MI_ARG(a.activation >= MI355MOE_LINEAR_SILU_AND_MUL &&
             a.activation <= MI355MOE_LINEAR_GELU_TANH_AND_MUL,
         "gated_linear_backward: the activation must be a gated one");
  MI_ARG(!a.dbias || a.dbias_dtype == MI355MOE_F32 || a.dbias_dtype == MI355MOE_BF16 ||
             a.dbias_dtype == MI355MOE_F16,
         "gated_linear_backward: dbias must be float32, bfloat16 or float16");
  MI_ARG(a.M >= 0 && a.N > 0 && a.K > 0, "gated_linear_backward: invalid shape");
  MI_ARG(a.M <= 64 * 65535 && a.N <= (1 << 20) && a.K <= (1 << 24),
         "gated_linear_backward: size too large");
  MI_ARG(a.ldx >= 0 && a.ldw >= 0 && a.ldd >= 0 && a.lddx >= 0 && a.lddw >= 0,
         "gated_linear_backward: negative stride");
  MI_ARG(!a.dx || a.M <= 1 || a.lddx >= a.K, "gated_linear_backward: rows of dx overlap");
  MI_ARG(!a.dweight || a.lddw >= a.K, "gated_linear_backward: rows of dweight overlap");
  // (without rows dx has no elements, so it may have no address)
  MI_ARG(a.M == 0 || a.dx || a.dweight || a.dbias, "gated_linear_backward: no gradient is asked for");
  return MI355MOE_OK;
}

size_t up16(size_t n) { return (n + 15) & ~static_cast<size_t>(15); }

// The workspace's parts, each at a multiple of 16 bytes: dz, db's parts, and the
// partial sums of a split product (the two products follow each other on it).
struct Layout {
  int64_t ld, per;
  int blocks;
  size_t part, sums, total;
  Product dx, dw;
};
Layout layout(const GradArgs& a, uintptr_t ws) {
  Layout l{};
  l.ld = (2 * a.N + 7) / 8 * 8;
  // rows of a dz workgroup: 4 to 32, a wave's in turn, for some 1000 workgroups (61 x 1536
  // 6.5 -> 3.4 us, 257 x 1030 29 -> 6.5); db's parts bound their number
  l.per = cdiv(a.M * cdiv(a.N, 512), 1024 * 4) * 4;
  l.per = l.per < 4 ? 4 : l.per > 32 ? 32 : l.per;
  if (a.dbias && cdiv(a.M, l.per) > kRowBlocks) l.per = cdiv(a.M, kRowBlocks);
  if (cdiv(a.M, l.per) > 65535) l.per = cdiv(a.M, 65535);
  l.blocks = static_cast<int>(cdiv(a.M, l.per));
  l.part = up16(static_cast<size_t>(a.M) * l.ld * 2);
  l.sums = l.part + (a.dbias ? up16(static_cast<size_t>(l.blocks) * 2 * a.N * 4) : 0);
  const void* dz = reinterpret_cast<const void*>(ws);
  size_t split = 0;
  if (a.dx) {
    l.dx = Product{a.dtype, false, a.M, a.K, 2 * a.N, dz, l.ld, a.weight, a.ldw, a.dx, a.lddx};
    split = product_workspace(l.dx);
  }
  if (a.dweight) {
    l.dw = Product{a.dtype, true, 2 * a.N, a.K, a.M, dz, l.ld, a.x, a.ldx, a.dweight, a.lddw};
    const size_t s = product_workspace(l.dw);
    split = s > split ? s : split;
  }
  l.total = l.sums + split;
  return l;
}

}  // namespace
}  // namespace mi355

using namespace mi355;

extern "C" size_t mi355moe_gated_linear_backward_workspace_size(
    const mi355moe_gated_linear_backward_args* p) {
  if (!p || check(*p)) return 0;
  return layout(*p, 0).total;
}

extern "C" int mi355moe_gated_linear_backward(const mi355moe_gated_linear_backward_args* p,
                                              void* workspace, size_t workspace_bytes, void* stream) {
  MI_ARG(p, "null pointer");
  const GradArgs a = *p;
  if (const int rc = check(a)) return rc;
  MI_ARG(a.M == 0 || (a.z && a.dout && (a.weight || !a.dx) && (a.x || !a.dweight)), "null pointer");
  hipStream_t st = static_cast<hipStream_t>(stream);
  const Layout l = layout(a, reinterpret_cast<uintptr_t>(workspace));
  MI_CHECK(l.total == 0 || (workspace && workspace_bytes >= l.total), MI355MOE_ERR_WORKSPACE,
           "gated_linear_backward: workspace too small");
  MI_ARG(l.total == 0 || (reinterpret_cast<uintptr_t>(workspace) & 15) == 0,
         "gated_linear_backward: workspace must be 16-byte aligned");
  uint16_t* dz = static_cast<uint16_t*>(workspace);
  float* part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + l.part);
  void* sums = static_cast<uint8_t*>(workspace) + l.sums;
  if (a.M) {
    switch (a.activation) {
      case MI355MOE_LINEAR_SILU_AND_MUL:
        launch_dz<MI355MOE_LINEAR_SILU_AND_MUL>(a, dz, l.ld, part, l.blocks, l.per, st);
        break;
      case MI355MOE_LINEAR_GELU_AND_MUL:
        launch_dz<MI355MOE_LINEAR_GELU_AND_MUL>(a, dz, l.ld, part, l.blocks, l.per, st);
        break;
      default: launch_dz<MI355MOE_LINEAR_GELU_TANH_AND_MUL>(a, dz, l.ld, part, l.blocks, l.per, st);
    }
    MI_LAUNCH_CHECK();
  }
  if (a.dbias) {
    gated_db_kernel<<<dim3(static_cast<unsigned>(cdiv(2 * a.N, 64))), dim3(1024), 0, st>>>(
        part, l.blocks, 2 * a.N, a.dbias, a.dbias_dtype);
    MI_LAUNCH_CHECK();
  }
  if (a.dx && a.dweight && a.M && product_pair_supported(l.dx, l.dw)) return launch_product_pair(l.dx, l.dw, st);
  if (a.dx && a.M)
    if (const int rc = launch_product(l.dx, sums, st)) return rc;
  if (a.dweight) return launch_product(l.dw, sums, st);
  return MI355MOE_OK;
}
