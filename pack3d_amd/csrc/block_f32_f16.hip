#include "block_kernels.hpp"

namespace p3d {
template int launch_block<float, _Float16>(const BlockDev&, const BlockLaunch&);
}
