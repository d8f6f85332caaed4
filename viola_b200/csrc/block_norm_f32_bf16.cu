// Norms around a block: float stream, __nv_bfloat16 branch.
#include "block_norm.cuh"

namespace vb {
template int launch_shape<float, __nv_bfloat16>(const NormArgs&, const NormShape&, const NormLaunch&);
}  // namespace vb
