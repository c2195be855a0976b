// Tiles of 16-bit gated linears whose sums are kept for a backward pass (gemm_tile.h).
#include "gemm_tile.h"

namespace mi355 {

int launch_linear_keep(const LinArgs& a, const TilePlan& p, hipStream_t st) {
  const bool f16 = a.x_dtype == MI355MOE_F16;
  if (p.splits > 1)
    return f16 ? launch_gemm_shape<K_F16, false, false, false, E_RAW>(a, p, st)
               : launch_gemm_shape<K_BF16, false, false, false, E_RAW>(a, p, st);
  return f16 ? launch_gemm_shape<K_F16, false, false, true, E_KEEP>(a, p, st)
             : launch_gemm_shape<K_BF16, false, false, true, E_KEEP>(a, p, st);
}

}  // namespace mi355
