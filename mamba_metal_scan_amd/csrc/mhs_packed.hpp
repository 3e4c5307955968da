// What the kernels over packed sequences share: element types, the cut of the
// sequences into pieces, and moves between lanes.
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
  return max(1, (e - b + tc - 1) / tc);
}

// ------------------------------------------------------- moves between lanes

// Row r of the wave (its 16 lanes 16 r ..) holds step r in v: o[s] is step s in
// every row.
__device__ __forceinline__ void spread_rows(float v, float (&o)[4]) {
  const unsigned u = __float_as_uint(v);
  const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);   // rows 0101, 2323
  const auto b = __builtin_amdgcn_permlane16_swap(a[0], a[0], false, false);
  const auto c = __builtin_amdgcn_permlane16_swap(a[1], a[1], false, false);
  o[0] = __uint_as_float(b[0]);
  o[1] = __uint_as_float(b[1]);
  o[2] = __uint_as_float(c[0]);
  o[3] = __uint_as_float(c[1]);
}

// The way back: the sum over the four rows of v[s], in row s.
__device__ __forceinline__ float gather_rows(const float (&v)[4]) {
  const auto swap32 = [](float x, float y) {
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(y), false,
                                                    false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
  };
  // rows 0, 1: the two halves' sum of v[0] (v[1]); rows 2, 3: of v[2] (v[3])
  const float a = swap32(v[0], v[2]), b = swap32(v[1], v[3]);
  const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false,
                                                  false);
  return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

// Lane K of each row of b, times v (the compiler folds the broadcast into the
// multiply); y += that (it does not fold it into a multiply-add: by hand. b
// must not come from a VALU instruction less than two instructions before).
template <int K>
__device__ __forceinline__ float row_mul(float b, float v) {
  return dpp_get<0x150 + K>(b) * v;
}
template <int K>
__device__ __forceinline__ void row_fmac(float& y, float b, float v) {
  asm("v_fmac_f32_dpp %0, %1, %2 row_newbcast:%3 row_mask:0xf bank_mask:0xf"
      : "+v"(y)
      : "v"(b), "v"(v), "n"(K));
}
// The two wait states between VALU writes of v and row_fmac's reads of it.
template <int M>
__device__ __forceinline__ void row_fmac_ready(float (&v)[M]) {
  static_assert(M == 1 || M == 2 || M == 4, "one, two or four registers");
  if constexpr (M == 1) asm("s_nop 1" : "+v"(v[0]));
  else if constexpr (M == 2) asm("s_nop 1" : "+v"(v[0]), "+v"(v[1]));
  else asm("s_nop 1" : "+v"(v[0]), "+v"(v[1]), "+v"(v[2]), "+v"(v[3]));
}

// ------------------------------------------------------------- states

// The NPL states n0 .. of channel d in a (D, N) slice: an address of the first
// and how many of them there are; whole vectors where N allows them.
template <int NPL>
struct StateAt {
  size_t off;
  int valid;   // 0 .. NPL
  bool vec;
  __device__ __forceinline__ StateAt(int d, int n0, int D, int N)
      : off((size_t)d * N + n0), valid(d < D ? max(0, min(NPL, N - n0)) : 0),
        vec(N % NPL == 0) {}
  __device__ __forceinline__ void load(float (&v)[NPL], const float* p) const {
#pragma unroll
    for (int j = 0; j < NPL; ++j) v[j] = 0.f;
    if (vec) {
      if (valid) load_vec<NPL>(v, p + off);
    } else {
#pragma unroll
      for (int j = 0; j < NPL; ++j)
        if (j < valid) v[j] = p[off + j];
    }
  }
  __device__ __forceinline__ void store(float* p, const float (&v)[NPL]) const {
    if (vec) {
      if (valid) store_vec<NPL>(p + off, v);
    } else {
#pragma unroll
      for (int j = 0; j < NPL; ++j)
        if (j < valid) p[off + j] = v[j];
    }
  }
};

}  // namespace mhs
