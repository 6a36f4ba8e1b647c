#include "block_kernels.hpp"

namespace p3d {
template int launch_block<float, float>(const BlockDev&, const BlockLaunch&);
}
