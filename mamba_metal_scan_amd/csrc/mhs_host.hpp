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
// mhs_gemm_f32 of alpha[0] (a device scalar, forms NN and TN; null: 1) times the product.
int gemm_f32(int form, const float* a, int64_t lda, const float* b, int64_t ldb, float* c,
             int64_t ldc, int64_t m, int64_t n, int64_t k, int accumulate, const float* alpha,
             void* workspace, size_t workspace_bytes, void* stream);

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline size_t round_up(size_t n, size_t m) { return (n + m - 1) / m * m; }

}  // namespace mhs
