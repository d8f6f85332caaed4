// Norms around a block: __nv_bfloat16 stream, __nv_bfloat16 branch.
#include "block_norm.cuh"

namespace vb {
template int launch_shape<__nv_bfloat16, __nv_bfloat16>(const NormArgs&, const NormShape&, const NormLaunch&);
}  // namespace vb
