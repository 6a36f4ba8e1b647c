#include "block_kernels.hpp"

namespace p3d {
template int launch_block<__bf16, __bf16>(const BlockDev&, const BlockLaunch&);
}
