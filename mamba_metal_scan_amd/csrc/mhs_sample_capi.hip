// C ABI of the sampling of tokens (declared in include/mamba_hip_scan.h).
#include <hip/hip_runtime.h>

#include "mamba_hip_scan.h"
#include "mhs_host.hpp"
#include "mhs_sample.hpp"

using mhs::check_launch;
using mhs::fail;

namespace {

// Words up to which a row has 256 threads in the first kernel: its list holds them all then. (207
// rows of 2562 words, k up to 1000: 115 us with 256, rows being left to the search.)
constexpr int64_t kSmallVocab = mhs::ListShared<256>::kList;

// Whether rows may be left: they have more words than the list of 1024 threads holds.
bool may_leave(int64_t vocab) { return vocab > mhs::ListShared<1024>::kList; }

// Whether some row may be looked at by parts: it has more words than a part, and top-k may be off.
bool in_parts(const void* top_k, int64_t top_k_value, int64_t vocab) {
  return vocab > mhs::kPart && (top_k || top_k_value < 1 || top_k_value >= vocab);
}
int64_t part_count(int64_t vocab) { return (vocab + mhs::kPart - 1) / mhs::kPart; }

template <class T>
int launch(const mhs::SampleArgs& a, int64_t rows, bool parts, hipStream_t s) {
  const unsigned grid = (unsigned)rows;
  if (a.vocab <= kSmallVocab) mhs::sample_kernel<T, 256><<<grid, 256, 0, s>>>(a);
  else mhs::sample_kernel<T, 1024><<<grid, 1024, 0, s>>>(a);
  const int rc = check_launch("sample kernel");
  if (rc || !a.state) return rc;
  if (parts) mhs::sample_bins_kernel<T><<<dim3((unsigned)a.parts, grid), 256, 0, s>>>(a);
  mhs::sample_rest_kernel<T><<<grid, 1024, 0, s>>>(a);
  return check_launch("sample kernels of the rows left");
}

int check_sizes(int64_t rows, int64_t vocab) {
  if (rows < 0 || rows >= 1LL << 16 || vocab < 1 || vocab > 1LL << 24)
    return fail(MHS_EINVAL, "rows must be in [0, 2^16), vocab in [1, 2^24]; got %lld, %lld",
                (long long)rows, (long long)vocab);
  if (rows * part_count(vocab) >= 1LL << 24)
    return fail(MHS_EINVAL, "%lld rows x %lld words are too many", (long long)rows,
                (long long)vocab);
  return MHS_OK;
}

}  // namespace

extern "C" {

size_t mhs_sample_workspace_bytes(int64_t rows, int64_t vocab, int top_k_array,
                                  int64_t top_k_value) {
  mhs::clear_error();
  if (check_sizes(rows, vocab) || !may_leave(vocab)) return 0;
  const int64_t parts =
      in_parts(top_k_array ? &rows : nullptr, top_k_value, vocab) ? part_count(vocab) : 0;
  return mhs::round_up((size_t)rows * sizeof(mhs::SampleRow), 256) +
         (size_t)(rows * parts) * mhs::kMassBins * 8;
}

int mhs_sample(int dtype, const void* logits, int64_t ld, const float* uniform,
               const float* temperature, float temperature_value, const void* top_k, int top_k64,
               int64_t top_k_value, const float* top_p, float top_p_value, const float* min_p,
               float min_p_value, int64_t* tokens, float* logprobs, int64_t rows, int64_t vocab,
               void* workspace, size_t workspace_bytes, void* stream) {
  mhs::clear_error();
  if (dtype != MHS_F32 && dtype != MHS_BF16 && dtype != MHS_F16)
    return fail(MHS_EINVAL, "dtype must be MHS_F32, MHS_BF16 or MHS_F16; got %d", dtype);
  const int rc = check_sizes(rows, vocab);
  if (rc) return rc;
  if (rows == 0) return MHS_OK;
  if (!logits || !uniform || !tokens) return fail(MHS_EINVAL, "null pointer argument");
  if (rows > 1 && ld < vocab)
    return fail(MHS_EINVAL, "the rows of logits must be at least vocab elements apart; got %lld",
                (long long)ld);
  const size_t need = mhs_sample_workspace_bytes(rows, vocab, top_k != nullptr, top_k_value);
  if (need && (!workspace || workspace_bytes < need))
    return fail(MHS_EINVAL, "workspace too small: %zu < %zu bytes", workspace_bytes, need);
  if (need && (reinterpret_cast<uintptr_t>(workspace) & 255u))
    return fail(MHS_EINVAL, "workspace must be 256-byte aligned");
  const bool parts = in_parts(top_k, top_k_value, vocab);
  int words = 0;   // 2^words >= vocab
  while ((1LL << words) < vocab) ++words;
  mhs::SampleArgs a{logits, ld, uniform, temperature, top_p, min_p, top_k, top_k64,
                    temperature_value, top_p_value, min_p_value, (long long)top_k_value,
                    reinterpret_cast<long long*>(tokens), logprobs, (int)vocab,
                    words <= 17 ? 45 : 62 - words,
                    need ? static_cast<mhs::SampleRow*>(workspace) : nullptr,
                    reinterpret_cast<unsigned long long*>(
                        static_cast<char*>(workspace) +
                        mhs::round_up((size_t)rows * sizeof(mhs::SampleRow), 256)),
                    parts ? (int)part_count(vocab) : 1};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == MHS_F32) return launch<mhs::F32>(a, rows, parts, s);
  if (dtype == MHS_BF16) return launch<mhs::Bf16>(a, rows, parts, s);
  return launch<mhs::Fp16>(a, rows, parts, s);
}

}  // extern "C"
