// Norms around a block: float stream, float branch.
#include "block_norm.cuh"

namespace vb {
template int launch_shape<float, float>(const NormArgs&, const NormShape&, const NormLaunch&);
}  // namespace vb
