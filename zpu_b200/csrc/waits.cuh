// The error words of the language-model head's bounded waits (int8.cu,
// distill.cu), for zpucuda_check_device.
#pragma once

namespace zc {

// Read the word into *e, left as it is where no kernel that may set it has
// been launched (a synchronous copy less: 12 us); a status.
int int8_device_error(unsigned int *e);
int distill_device_error(unsigned int *e);

}  // namespace zc
