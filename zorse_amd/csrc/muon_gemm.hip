// The Newton-Schulz products with both operands along the reduction.
#include "muon.h"

namespace zk {
namespace gemm {
void launch_poly(Tile t, const PolyGroup& g, hipStream_t s) { launch_poly_t<false>(t, g, s); }
}  // namespace gemm
}  // namespace zk
