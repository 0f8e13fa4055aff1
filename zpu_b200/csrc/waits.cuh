// The error words of the language-model head's bounded waits (int8.cu,
// distill.cu), for zpucuda_check_device.
#pragma once

namespace zc {

// Read the word (synchronous); a status.
int int8_device_error(unsigned int *e);
int distill_device_error(unsigned int *e);

}  // namespace zc
