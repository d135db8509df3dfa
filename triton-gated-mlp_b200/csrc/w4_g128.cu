// The 4-bit stream kernels for groups of 128 columns.
#include "few_token_host.cuh"

namespace gmlp {
int launch_w4_g128(const DeviceInfo* dev, const W4Call& c, bool dual) { return launch_w4_group<2>(dev, c, dual); }
}  // namespace gmlp
