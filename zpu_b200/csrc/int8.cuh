// The error word of int8.cu's bounded waits, for zpucuda_check_device.
#pragma once

namespace zc {

// Reads the word (synchronous); a status.
int int8_device_error(unsigned int *e);

}  // namespace zc
