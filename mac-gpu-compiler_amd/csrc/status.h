// Error reporting shared by the sources behind the C ABI: every entry point returns a status and
// leaves its message for qe_last_error() (include/qe.h).
#pragma once

#include <cstdint>

namespace qe {
// A range of memory, for checks of what must not overlap.
struct Bytes {
  const void* at;
  uint64_t n;
  bool meets(const Bytes& o) const {
    const uintptr_t a = reinterpret_cast<uintptr_t>(at), b = reinterpret_cast<uintptr_t>(o.at);
    return at && o.at && n && o.n && (a < b ? b - a < n : a - b < o.n);
  }
};
// Stores the printf-formatted message as the calling thread's last error and returns `code`.
int set_error(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
}  // namespace qe
