// What the extern "C" files of the library share: the message of the last failure, the device status word, the launch count.
#pragma once

#include <cstddef>
#include <cstdint>

namespace cs2d {

// Leaves the message for cs2d_last_error() and returns code.
__attribute__((format(printf, 2, 3))) int fail(int code, const char *fmt, ...);
// Device address of the status word on the current device (looked up once per device; NULL: the look-up failed).
int *status_ptr();
void count_launches(int n);

}  // namespace cs2d
