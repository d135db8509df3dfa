// The 4-bit stream kernels for groups of 32 columns.
#include "few_token_host.cuh"

namespace gmlp {
int launch_w4_g32(const DeviceInfo* dev, const W4Call& c, bool dual) { return launch_w4_group<0>(dev, c, dual); }
}  // namespace gmlp
