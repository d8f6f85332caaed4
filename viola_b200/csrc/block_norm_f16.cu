// Norms around a block: __half stream, __half branch.
#include "block_norm.cuh"

namespace vb {
template int launch_shape<__half, __half>(const NormArgs&, const NormShape&, const NormLaunch&);
}  // namespace vb
