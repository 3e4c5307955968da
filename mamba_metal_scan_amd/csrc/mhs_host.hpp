// What the library's host units share (defined in mhs_capi.hip).
#pragma once

#include <cstddef>
#include <cstdint>

namespace mhs {

// Sets the calling thread's message; returns `code`.
int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
void clear_error();
// The last launch's error, as MHS_EHIP with `what`, or MHS_OK.
int check_launch(const char* what);
// Compute units of the current device.
int device_cus();

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline size_t round_up(size_t n, size_t m) { return (n + m - 1) / m * m; }

}  // namespace mhs
