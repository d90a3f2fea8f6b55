// status.h — the error text behind fwb_last_error(), for every translation
// unit of the library.
#pragma once

namespace fwb {

// Sets this thread's error text (defined in runtime.cu).
void set_last_error(const char *text) noexcept;

}  // namespace fwb
