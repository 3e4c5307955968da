// C ABI of the sampling of tokens (declared in include/mamba_hip_scan.h).
#include <hip/hip_runtime.h>

#include "mamba_hip_scan.h"
#include "mhs_host.hpp"
#include "mhs_sample.hpp"

using mhs::check_launch;
using mhs::fail;

namespace {

// Threads of a row's block.
constexpr int64_t kSmallVocab = 8192;

template <class T>
void launch(const mhs::SampleArgs& a, int64_t rows, hipStream_t s) {
  const unsigned grid = (unsigned)rows;
  if (a.vocab <= kSmallVocab) mhs::sample_kernel<T, 256><<<grid, 256, 0, s>>>(a);
  else mhs::sample_kernel<T, 1024><<<grid, 1024, 0, s>>>(a);
}

}  // namespace

extern "C" {

int mhs_sample(int dtype, const void* logits, int64_t ld, const float* uniform,
               const float* temperature, float temperature_value, const void* top_k, int top_k64,
               int64_t top_k_value, const float* top_p, float top_p_value, const float* min_p,
               float min_p_value, int64_t* tokens, float* logprobs, int64_t rows, int64_t vocab,
               void* stream) {
  mhs::clear_error();
  if (dtype != MHS_F32 && dtype != MHS_BF16 && dtype != MHS_F16)
    return fail(MHS_EINVAL, "dtype must be MHS_F32, MHS_BF16 or MHS_F16; got %d", dtype);
  if (rows < 0 || rows > 1LL << 21 || vocab < 1 || vocab > 1LL << 24)
    return fail(MHS_EINVAL, "rows must be in [0, 2^21], vocab in [1, 2^24]; got %lld, %lld",
                (long long)rows, (long long)vocab);
  if (rows == 0) return MHS_OK;
  if (!logits || !uniform || !tokens) return fail(MHS_EINVAL, "null pointer argument");
  if (rows > 1 && ld < vocab)
    return fail(MHS_EINVAL, "the rows of logits must be at least vocab elements apart; got %lld",
                (long long)ld);
  int words = 0;   // 2^words >= vocab
  while ((1LL << words) < vocab) ++words;
  mhs::SampleArgs a{logits, ld, uniform, temperature, top_p, min_p, top_k, top_k64,
                    temperature_value, top_p_value, min_p_value, (long long)top_k_value,
                    reinterpret_cast<long long*>(tokens), logprobs, (int)vocab,
                    words <= 17 ? 45 : 62 - words};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == MHS_F32) launch<mhs::F32>(a, rows, s);
  else if (dtype == MHS_BF16) launch<mhs::Bf16>(a, rows, s);
  else launch<mhs::Fp16>(a, rows, s);
  return check_launch("sample kernel");
}

}  // extern "C"
