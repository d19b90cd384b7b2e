// What the 8-bit tensor-core kernels share with the library's diagnostics.
#pragma once

#include <cuda_runtime.h>

namespace tagi {

// Error word of the 8-bit kernels on the current device (see tagi_device_status).
int int8_device_status(int reset);
// Their part of tagi_set_wait_limit_ns.
cudaError_t int8_set_wait_limit(unsigned long long ns, int force);
// Counts one tcgen05 launch (tagi_tc_launches).
void count_tc_launch();

}  // namespace tagi
