// What the library's translation units share on the host side.
#pragma once

namespace llmfa {

// Device address of the current device's status word (llmfa_device_status), set
// up on the device's first use. Returns an llmfa status code.
__attribute__((visibility("hidden"))) int device_status_ptr(int** out);

}  // namespace llmfa
