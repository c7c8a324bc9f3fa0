// The Newton-Schulz products of muon.hip (muon_gemm.hip, muon_gemm_kmajor.hip).
#pragma once
#include "gemm_ring.h"

namespace zk {
namespace gemm {

// The products of a group (fp16; first[] of tiles of t), B K-major or along K.
void launch_poly(Tile t, const PolyGroup& g, hipStream_t s);
void launch_poly_kmajor(Tile t, const PolyGroup& g, hipStream_t s);

template <bool BKM>
inline void launch_poly_t(Tile t, const PolyGroup& g, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(g.first[g.n]));
  if (t == k256)
    hipLaunchKernelGGL((gemm_tiled_kernel<f16, 4, false, BKM>), grid, dim3(256), 0, s, g);
  else if (t == k128)
    hipLaunchKernelGGL((gemm_ring_kernel<f16, 4, false, BKM, 4, 4, 2, 2, 1>), grid, dim3(256), 0, s, g);
  else
    hipLaunchKernelGGL((gemm_ring_kernel<f16, 4, false, BKM, 2, 2, 4, 2, 1>), grid, dim3(256), 0, s, g);
}

}  // namespace gemm
}  // namespace zk
