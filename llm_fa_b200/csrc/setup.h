// What the library's translation units share on the host side.
#pragma once

namespace llmfa {

// Device address of the current device's status word (llmfa_device_status), set
// up on the device's first use. Returns an llmfa status code.
__attribute__((visibility("hidden"))) int device_status_ptr(int** out);

// SMs of the current device (same).
__attribute__((visibility("hidden"))) int device_sms(int* out);

// Upper bound on every in-kernel wait (llmfa_set_wait_timeout_ms).
__attribute__((visibility("hidden"))) unsigned long long wait_limit_ns();

}  // namespace llmfa
