// What the sources of the C ABI share.
#pragma once
#include <cuda_runtime.h>

namespace ocrvl {

// Stores the calling thread's error text (ocrvl_last_error) and returns `code`.
int api_fail(int code, const char *msg) noexcept;

}  // namespace ocrvl
