// The error contract of the C ABI (capi.hip) for entry points defined in other
// files of the library.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/phi_qlinear.h"

namespace phi_capi {

// Leaves the message for phi_hip_last_error() and returns st.
phi_status fail(phi_status st, const char* fmt, ...);
// PHI_OK with no message.
phi_status ok();
// What a launch returned, as a phi_status; a fault of the device stays sticky.
phi_status check_hip(hipError_t e, const char* what);
bool device_lost();

}  // namespace phi_capi
