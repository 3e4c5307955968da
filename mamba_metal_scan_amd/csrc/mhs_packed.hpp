// What the kernels over packed sequences share: element types and the cut of the
// sequences into pieces.
//
// nseq sequences lie behind each other in the rows of (total, D) tensors: row
// cu[s] is the first of sequence s, cu[s + 1] the first behind it; rows behind
// cu[nseq] belong to none. The lengths are known on the device only, so that
// the grids are sized from total and nseq alone: a sequence is cut into pieces
// of `tc` rows from its own first row, and piece j of sequence s has the
// number cu[s] / tc + s + j. Those numbers never meet: a sequence of n rows
// from row b has max(1, ceil(n / tc)) pieces, and
// (b + n) / tc + 1 - b / tc >= that. The rows of no sequence are cut like a
// sequence nseq. There are at most total / tc + nseq + 1 numbers; those
// between the last piece of a sequence and the first of the next have no rows.
#pragma once

#include <type_traits>
#include <utility>

#include "mhs_common.hpp"
#include "mhs_mm16.hpp"

namespace mhs {

// Elements of activations: Elem<T>::bytes of them are a T (Bf16, Fp16) or a float.
struct F32 {
  static __device__ __forceinline__ float to(float v) { return v; }
};
template <class T>
constexpr int kElem = std::is_same<T, F32>::value ? 4 : 2;

template <class T, int POL = 0>
__device__ __forceinline__ float ld_t(const GBuf& g, unsigned byte_off) {
  if constexpr (kElem<T> == 4) return g.ld<POL>(byte_off);
  else return T::to(__builtin_amdgcn_raw_buffer_load_b16(g.r, byte_off, 0, POL));
}
template <class T, int POL = 0>
__device__ __forceinline__ void st_t(const GBuf& g, float v, unsigned byte_off) {
  if constexpr (kElem<T> == 4) g.st<POL>(v, byte_off);
  else __builtin_amdgcn_raw_buffer_store_b16(T::from(v), g.r, byte_off, 0, POL);
}
// Element idx of a tensor of T's, read or written through its address.
template <class T>
__device__ __forceinline__ float ld_p(const void* p, size_t idx) {
  if constexpr (kElem<T> == 4) return static_cast<const float*>(p)[idx];
  else return T::to(static_cast<const unsigned short*>(p)[idx]);
}
template <class T>
__device__ __forceinline__ void st_p(void* p, size_t idx, float v) {
  if constexpr (kElem<T> == 4) static_cast<float*>(p)[idx] = v;
  else static_cast<unsigned short*>(p)[idx] = T::from(v);
}
template <class T>
__device__ __forceinline__ GBuf buf_t(const void* base, size_t idx, unsigned bytes) {
  return GBuf(elem_at<kElem<T>>(base, idx), bytes);
}

// f(integral_constant<int, 0>), ..., f(integral_constant<int, N - 1>).
template <class F, int... I>
__device__ __forceinline__ void static_for_impl(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void static_for(F&& f) {
  static_for_impl(f, std::make_integer_sequence<int, N>{});
}

// ------------------------------------------------------------------ pieces

struct Seqs {
  const void* cu;   // nseq + 1 ints, or 64-bit ones
  int cu64;
  int nseq;
  int total;        // rows of the tensors
};

// cu[s], within the rows whatever the caller's numbers are.
__device__ __forceinline__ int cu_at(const Seqs& q, int s) {
  const long long v = q.cu64 ? static_cast<const long long*>(q.cu)[s]
                             : (long long)static_cast<const int*>(q.cu)[s];
  return (int)max(0LL, min(v, (long long)q.total));
}

struct Piece {
  int seq;      // -1: the number has no piece; nseq: rows of no sequence
  int begin;    // the sequence's first row
  int j;        // the piece's number in its sequence
  int t0, len;  // its rows
  int last;     // whether the sequence ends with it
};

// The piece of number p: the last sequence whose first piece's number is at
// most p, by 64 probes a round (for any cu the search ends, and the rows it
// gives lie inside the tensors). All lanes of the wave call it; the result is
// uniform.
__device__ __forceinline__ Piece find_piece(const Seqs& q, int tc, int p) {
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = q.nseq + 1;
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) / 64;
    const int s = lo + lane * step;
    const bool at_most = s < hi && cu_at(q, s) / tc + s <= p;
    const int n = __popcll(__ballot(at_most));
    if (n == 0) break;
    lo += (n - 1) * step;
    hi = min(hi, lo + step);
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  Piece r;
  r.seq = -1;
  const int b = __builtin_amdgcn_readfirstlane(cu_at(q, lo));
  const int e = lo == q.nseq ? q.total
                             : max(b, __builtin_amdgcn_readfirstlane(cu_at(q, lo + 1)));
  const int j = p - (b / tc + lo);
  if (j < 0 || (j > 0 && (long long)b + (long long)j * tc >= e)) return r;
  r.seq = lo;
  r.begin = b;
  r.j = j;
  r.t0 = b + j * tc;
  r.len = min(tc, e - r.t0);
  r.last = r.t0 + r.len >= e;
  return r;
}

// The pieces of sequence s and the number of its first one.
__device__ __forceinline__ int seq_pieces(const Seqs& q, int tc, int s, int* first) {
  const int b = cu_at(q, s), e = max(b, cu_at(q, s + 1));
  *first = b / tc + s;
  return e > b ? (e - b - 1) / tc + 1 : 1;   // (e - b may be next to 2^31)
}

}  // namespace mhs
