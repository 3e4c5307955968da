// Distillation of given logits from a teacher's top words for gfx950 (formulas
// in mhs_head.hpp): logits (rows, vocab) fp32, bf16 or fp16, per row up to
// kMaxTop words of the teacher with its logits.
//
// HBM-bound: a block per row, 16-byte accesses at any row length and alignment;
// the forward reads the logits once and keeps 4 bytes a row and the teacher's
// probabilities, the backward reads them once more and writes the gradient.
#pragma once

#include "mhs_head.hpp"

namespace mhs {

constexpr int kMaxTop = 1024;   // teacher words per row

// A row of n elements at any alignment of whole elements: up to kVec - 1 single
// ones to the first 16-byte boundary (head), whole vectors, and the rest.
template <class T>
struct RowSplit {
  int head, ends;
  long long vecs;
  __device__ __forceinline__ RowSplit(const elem_t<T>* x, long long n) {
    constexpr int V = kVec<T>;
    const int off = (int)((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(elem_t<T>));
    head = (int)min((long long)((V - off) % V), n);
    vecs = (n - head) / V;
    ends = (int)(n - vecs * V);
  }
  // The index of single element j < ends.
  __device__ __forceinline__ long long end(int j) const {
    return j < head ? j : vecs * kVec<T> + j;
  }
};

// fp32 8192 x 32768 237 us (4.5 TB/s; a large copy takes 4.7), bf16 4096 x 50257 110
// us (3.7, bound by its arithmetic and by rows that start at any element). A row to
// 512 threads takes 2% less there, but forward and backward of 4096 x 4096 66 us
// against 53.
template <class T>
__global__ void __launch_bounds__(kXentThreads)
distill_fwd_kernel(HeadRows g) {
  extern __shared__ float zk[];   // 2 k floats
  __shared__ float red[4];
  constexpr int V = kVec<T>;
  const int r = blockIdx.x;
  const elem_t<T>* x = static_cast<const elem_t<T>*>(g.h) + (long long)r * g.ldh;
  const float c = kLog2e / g.temperature;
  for (int k = threadIdx.x; k < g.k; k += kXentThreads) {
    const long long id = g.ids[(long long)r * g.k + k];
    zk[k] = id >= 0 && id < g.vocab ? T::to(x[id]) : 0.f;
  }
  const RowSplit<T> row(x, g.vocab);
  float m = -INFINITY, s = 0.f;
  if ((int)threadIdx.x < row.ends) lse2_combine(m, s, T::to(x[row.end(threadIdx.x)]) * c, 1.f);
  const Vec<T>* xv = reinterpret_cast<const Vec<T>*>(x + row.head);
  constexpr int U = 16 / V;   // vectors per update of the running maximum
  long long i = threadIdx.x;
  for (; i + (U - 1) * kXentThreads < row.vecs; i += U * kXentThreads) {
    Vec<T> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = xv[i + u * kXentThreads];
    float y[U * V];
#pragma unroll
    for (int k = 0; k < U * V; ++k) y[k] = T::to(v[k / V].v[k % V]);
    float mc = y[0];
#pragma unroll
    for (int k = 1; k < U * V; ++k) mc = fmaxf(mc, y[k]);
    mc *= c;
    const float sh = lse2_shift(mc);
    float sc = 0.f;
#pragma unroll
    for (int k = 0; k < U * V; ++k) sc += exp2_hw(__builtin_fmaf(y[k], c, -sh));
    lse2_combine(m, s, mc, sc);
  }
  for (; i < row.vecs; i += kXentThreads) {
    const Vec<T> v = xv[i];
    float mc = -INFINITY, sc = 0.f;
#pragma unroll
    for (int k = 0; k < V; ++k) mc = fmaxf(mc, T::to(v.v[k]));
    mc *= c;
    const float sh = lse2_shift(mc);
#pragma unroll
    for (int k = 0; k < V; ++k) sc += exp2_hw(__builtin_fmaf(T::to(v.v[k]), c, -sh));
    lse2_combine(m, s, mc, sc);
  }
  block_lse2(m, s);   // (its barrier publishes zk)
  teacher_row(g, r, m + log2f(s), zk, red);
}

// dlogits (rows, vocab) contiguous. The teacher's words are put right after the
// row is written (a word named twice: the same value twice). fp32 8192 x 32768 430
// us (5.0 TB/s), bf16 4096 x 50257 210 us (3.9).
template <class T>
__global__ void __launch_bounds__(kXentThreads)
distill_bwd_kernel(const elem_t<T>* __restrict__ logits, long long ld,
                   const long long* __restrict__ ids, const float* __restrict__ q,
                   const float* __restrict__ lse2, RowScale rs, elem_t<T>* __restrict__ dlogits,
                   long long vocab, int top, float c) {
  constexpr int V = kVec<T>;
  const long long r = blockIdx.x;
  const elem_t<T>* x = logits + r * ld;
  elem_t<T>* dx = dlogits + r * vocab;
  const float cf = rs.at(r), l2 = lse2[r];
  const bool zero = cf == 0.f;
  const RowSplit<T> row(x, vocab);
  const bool same = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(dx)) & 15u) == 0;
  if ((int)threadIdx.x < row.ends) {
    const long long j = row.end(threadIdx.x);
    dx[j] = T::from(zero ? 0.f : cf * exp2_hw(__builtin_fmaf(T::to(x[j]), c, -l2)));
  }
  const Vec<T>* xv = reinterpret_cast<const Vec<T>*>(x + row.head);
  // U vectors at a time, their loads in flight together (16-bit elements are bound
  // by their arithmetic: one, two and four vectors take 328, 344 and 352 us a pass
  // forward and backward at 4096 x 50257; of fp32, two, four and eight 690, 679 and
  // 671 at 8192 x 32768).
  constexpr int U = __is_same(T, Fp32) ? 8 : 1;
  for (long long i0 = threadIdx.x; i0 < row.vecs; i0 += U * kXentThreads) {
    Vec<T> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (!zero && i0 + u * kXentThreads < row.vecs) v[u] = xv[i0 + u * kXentThreads];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long i = i0 + u * kXentThreads;
      if (i >= row.vecs) break;
#pragma unroll
      for (int k = 0; k < V; ++k)
        v[u].v[k] = zero ? elem_t<T>(0)
                         : T::from(cf * exp2_hw(__builtin_fmaf(T::to(v[u].v[k]), c, -l2)));
      if (same) {
        reinterpret_cast<Vec<T>*>(dx + row.head)[i] = v[u];
      } else {
#pragma unroll
        for (int k = 0; k < V; ++k) dx[row.head + i * V + k] = v[u].v[k];
      }
    }
  }
  if (zero) return;
  __syncthreads();   // the row's stores before its words'
  for (int k = threadIdx.x; k < top; k += kXentThreads) {
    const long long id = ids[r * top + k];
    if (id >= 0 && id < vocab)
      dx[id] = T::from(cf * (exp2_hw(__builtin_fmaf(T::to(x[id]), c, -l2)) - q[r * top + k]));
  }
}

}  // namespace mhs
