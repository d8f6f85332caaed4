// Norms around a block: float stream, __half branch.
#include "block_norm.cuh"

namespace vb {
template int launch_shape<float, __half>(const NormArgs&, const NormShape&, const NormLaunch&);
}  // namespace vb
