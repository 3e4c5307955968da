// Sums of the packed scan's gradients over the blocks and pieces, in a fixed order.
#pragma once

#include "mhs_packed.hpp"

namespace mhs {

// dB, dC (total, N): the blocks' partials in order, rounded to T once. Bound by the partials' bytes
// (16 blocks of 32768 x 16 x 2: 67 MB, 19.5 us; 12 of 8192: 12.6 MB, 6.5 us).
template <class T>
__global__ void __launch_bounds__(256)
packed_sum_bc_kernel(const float* part, void* dB, void* dC, int nblk, long long rows, int N) {
  const long long e = (long long)blockIdx.x * 256 + threadIdx.x;   // (row, kind, n)
  if (e >= rows * 2 * N) return;
  const long long all = rows * 2 * N;
  float s = 0.f;
  for (int k = 0; k < nblk; ++k) s += part[(long long)k * all + e];
  const long long row = e / (2 * N);
  const int n = (int)(e % (2 * N));
  st_p<T>(n < N ? dB : dC, (size_t)(row * N + n % N), s);
}

// dAneg (D, N): the pieces' partials. Each of a block's 16 waves adds every sixteenth, in
// four sums, then the block adds the waves': a fixed order. (us with four waves of one
// sum: 30 of 281 pieces x 1536 x 16, the loads one after the other.)
__global__ void __launch_bounds__(1024)
packed_sum_a_kernel(const float* part, float* da, int pieces, int slice) {
  __shared__ float sums[16][64];
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, e = blockIdx.x * 64 + lane;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  if (e < slice) {
    for (int p = w; p < pieces; p += 64) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (p + 16 * k < pieces) s[k] += part[(size_t)(p + 16 * k) * slice + e];
    }
  }
  sums[w][lane] = (s[0] + s[1]) + (s[2] + s[3]);
  __syncthreads();
  if (w || e >= slice) return;
  float total = sums[0][lane];
#pragma unroll
  for (int k = 1; k < 16; ++k) total += sums[k][lane];
  da[e] = total;
}

}  // namespace mhs
