// What the C-ABI translation units share on the host side.
#pragma once

#include <cstddef>

namespace flash_hip {

constexpr size_t kErrorBytes = 512;
// sets the text that flash_hip_last_error() gives to the calling thread and returns `code`
__attribute__((visibility("hidden"), format(printf, 2, 3))) int set_error(int code, const char* fmt, ...);

}  // namespace flash_hip
