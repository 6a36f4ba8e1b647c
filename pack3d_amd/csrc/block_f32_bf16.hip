#include "block_kernels.hpp"

namespace p3d {
template int launch_block<float, __bf16>(const BlockDev&, const BlockLaunch&);
}
