// The Newton-Schulz products with the right operand K-major, compiled with the
// register-assignment flag of the other K-major forms (gemm_kernels.h).
#include "muon.h"

namespace zk {
namespace gemm {
void launch_poly_kmajor(Tile t, const PolyGroup& g, hipStream_t s) { launch_poly_t<true>(t, g, s); }
}  // namespace gemm
}  // namespace zk
