// ql_host.h — what the translation units of libqlinear.so share on the host.
#pragma once

namespace ql_host {

struct Device {
  int sms = 0;
  unsigned* err_word = nullptr;   // the device error word (ql_device_error)
};

// The current device's properties; a QL_* status.
__attribute__((visibility("hidden"))) int current(Device* out);

}  // namespace ql_host
