// out[i, j] = sum_r q(i, r) p[r, j] on 16-bit operands, fp32 sums, one rounding: the
// products of a backward pass, whose second operand has its sums' index along the
// rows (a gradient times the weight, or a transposed gradient times the input).
#pragma once

#include "linear.h"

namespace mi355 {

// q is a workspace's: its rows are readable to a multiple of 8 columns, and along r they
// hold zeros there.
struct Product {
  int dtype;          // BF16 or F16
  bool transposed;    // q is [R, I], else [I, R]
  int64_t I, J, R;
  const void* q;
  int64_t ldq;
  const void* p;      // [R, J]
  int64_t ldp;
  void* out;          // [I, J]
  int64_t ldo;
};

typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4_t lds_s16x4_t;

// Four 16-bit values of one column: of 4 x 16 values that a group of 16 lanes points
// at, lane t at row t / 4, columns 4 (t % 4) .. + 3, lane t gets column t.
__device__ __forceinline__ uint2 lds_column4(const uint8_t* at) {
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)at));
}

// operands that direct copies to LDS can fetch (product_tile.hip)
// (padded: p's rows are readable to a multiple of 8 columns)
bool product_tile_supported(const Product& p, bool padded = false);
int product_tile_splits(const Product& p);
int launch_product_tile(const Product& p, float* part, hipStream_t st);

// dx and dW in one launch, where that fills the CUs better than one after the other
bool product_pair_supported(const Product& x, const Product& w);
int launch_product_pair(const Product& x, const Product& w, hipStream_t st);

// bytes of workspace (copied rows, partial sums; 0: neither), 16-byte aligned, that launch_product wants
size_t product_workspace(const Product& p);
int launch_product(const Product& p, void* workspace, hipStream_t st);

}  // namespace mi355
