#include "block_kernels.hpp"

namespace p3d {
template int launch_block<_Float16, _Float16>(const BlockDev&, const BlockLaunch&);
}
