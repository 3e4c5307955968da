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

// A row's exponents are formed in one step, c z - (the rounded c max z): off by half a
// unit of that product, 2^-12 at 4096 and anything from 2^31 on, where c z may overflow
// besides. A row whose log-sum-exp lies further out (all its logits a mask's -1e9 or the
// type's lowest value, say) goes a second way, by differences of the logits: two more
// passes, here and in the backward (all rows so, fp32 8192 x 32768: 639 and 1392 us
// for 236 and 432). Of other rows the branch takes nothing measurable.
constexpr float kFarLse2 = 4096.f;
__device__ __forceinline__ bool far_row(float lse2) { return !(fabsf(lse2) <= kFarLse2); }

// (M, log2 sum 2^(c (z - M))) of the row, M its largest logit; the sum NaN where a logit
// is NaN or infinity or all are -inf. The same in every thread.
template <class T>
__device__ __forceinline__ float2 far_row_lse2(const elem_t<T>* x, long long n, float c,
                                               float* red) {
  float m = -INFINITY, s = 0.f;
  for (long long i = threadIdx.x; i < n; i += kXentThreads) m = fmaxf(m, T::to(x[i]));
  m = block_max(m, red);
  for (long long i = threadIdx.x; i < n; i += kXentThreads) s += exp2_hw((T::to(x[i]) - m) * c);
  return make_float2(m, log2f(block_sum(s, red)));
}

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
  teacher_row(g, r, m + log2f(s), zk, red, [&](float& lse2) {
    if (!far_row(lse2)) return lse2;
    const float2 far = far_row_lse2<T>(x, g.vocab, c, red);
    for (int k = threadIdx.x; k < g.k; k += kXentThreads) zk[k] -= far.x;
    lse2 = far.y;
    return __builtin_fmaf(far.x, c, far.y);
  });
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
  __shared__ float red[4];
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
  if (far_row(l2)) {   // the row again
    const float2 far = far_row_lse2<T>(x, vocab, c, red);   // (its barriers: the stores above)
    const auto p = [&](long long i) {
      return exp2_hw(__builtin_fmaf(T::to(x[i]) - far.x, c, -far.y));
    };
    for (long long i = threadIdx.x; i < vocab; i += kXentThreads) dx[i] = T::from(cf * p(i));
    __syncthreads();   // the row's stores before its words'
    for (int k = threadIdx.x; k < top; k += kXentThreads) {
      const long long id = ids[r * top + k];
      if (id >= 0 && id < vocab) dx[id] = T::from(cf * (p(id) - q[r * top + k]));
    }
    return;
  }
  __syncthreads();   // the row's stores before its words'
  for (int k = threadIdx.x; k < top; k += kXentThreads) {
    const long long id = ids[r * top + k];
    if (id >= 0 && id < vocab)
      dx[id] = T::from(cf * (exp2_hw(__builtin_fmaf(T::to(x[id]), c, -l2)) - q[r * top + k]));
  }
}

}  // namespace mhs
