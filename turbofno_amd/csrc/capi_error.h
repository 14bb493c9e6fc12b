// How the entry points of the C ABI report an error: the code they return, and the text behind turbofno_last_error_string().
#pragma once
#include <hip/hip_runtime.h>

namespace tfno {

int fail(int code, const char* fmt, ...);               // returns code
int hip_status(hipError_t e, const char* what);         // TURBOFNO_OK or TURBOFNO_ERR_HIP

}  // namespace tfno
