// Selective scan over packed sequences for gfx950 (see mhs_packed.hpp for the
// pieces), forward and backward:
//   h_t = exp(-dt_t Aneg) h_{t-1} + dt_t x_t B_t,   y_t = sum_n C_tn h_tn
// per sequence, from h0 (nseq, D, N) or from zero.
//
// Mapping. The four lanes of a quad split the states of two neighbouring channels, NPL
// each (4 NPL states a wave; a block has WS waves for the states and 4 / WS
// times 32 channels). A register of x, dt or dy holds four steps as loaded, lane q of the
// quad step q. B and C, which all channels share, go through LDS: a lane reads its NPL states of
// a step at once; each wave has its own tiles, so that the waves of a block run without
// barriers (but for sums over waves). So do dt and dt x (dy) in the forward and
// the carry passes, four steps of a channel a read; the backward's main pass
// takes them from its quad within the multiply or multiply-add (DPP). The sums over the
// states are sums over a quad, those over the channels sums over the other four bits of
// the lane, which every step of a reduce-scatter halves without a select.
//
// The vector units bound it: cycles of a wave's instruction, measured with four waves a
// SIMD, multiply 2.9, multiply-add 4.8, exponential 8.3, and with a broadcast of a
// lane of the quad in it 4.4 and 5.0, v_permlane swaps 8.3. Per step, channel and state the
// carry passes need 19 of them, the forward 24 and the backward 70. (Operands by LDS or by DPP,
// us, each pair in one run, 32768 x 2048 x 16 bf16 | 8192 x 1536 x 16 fp32: carry 167 or 190 | 43
// or 44, its adjoint 175 or 185 | 40 or 43, the forward 277 or 282 | 66 or 65; the backward 655
// or 660 | 170 or 146, its registers being full. The quad's sums by LDS too: 280 | 65, 665 | 153.
// What the kernels take now stands at each, at steady clocks; from idle 5 to 10% more.)
//
// A sequence longer than a piece takes three launches: the carry pass walks
// each piece but the last from a zero state and leaves its end state and its
// sum of dt; the fold turns these into the states at the pieces' starts,
// H <- exp(-Aneg sum dt) H + end; the main pass walks every piece from there.
// The exponentials of the pieces that the carry pass walks are so taken twice.
#pragma once

#include "mhs_packed.hpp"

namespace mhs {

constexpr int kCkpt = 8;   // rows between checkpoints, and of a sub-chunk of the backward
constexpr int kSub = 16;   // rows of a sub-chunk of the forward and the carry passes

struct PackedScanArgs {
  Seqs q;
  const void *x, *dt, *B, *C;
  int ld_x, ld_dt, ld_b, ld_c;   // elements between rows
  const float* aneg;
  const float* h0;       // null: zeros
  void* y;               // (total, D)
  float* h_last;         // null: not wanted
  float* ckpt;           // (total / 8, D, N), null: not wanted. Entry begin / 8 + g - 1 is the
                         // state before step 8 g of its sequence, g >= 1
  float* carry;          // (pieces, D, N): the carry pass's states (adjoints) at the pieces' ends
  float* sdt;            // (pieces, D): its sums of dt
  float* start;          // (pieces, D, N): the states (adjoints) that the main pass starts from
  int D, N, tc;
  // backward
  const void* dy;
  int ld_dy;
  const float* dh_last;  // null: zeros
  void *dx, *ddt;        // (total, D)
  float* dh0;            // null: not wanted
  float* part_bc;        // (blocks of channels, total, 2, N): dB, dC of a block's channels
  float* part_a;         // (pieces, D, N): dAneg of a piece
};

// Rows [t0, t0 + len) of the block's channels of out are zeros.
template <class T>
__device__ __forceinline__ void zero_rows(void* out, int t0, int len, int D, int d_lo, int d_hi) {
  const int w = min(D, d_hi) - d_lo;
  for (int i = threadIdx.x; i < w * len; i += blockDim.x)
    st_p<T>(out, (size_t)(t0 + i / w) * D + d_lo + i % w, 0.f);
}

template <int NPL, int WS>
struct ScanLane {
  static constexpr int kStates = 4 * NPL;        // of a wave
  static constexpr int kChans = 32 * (4 / WS);   // of a block
  int wave, lane, q, ws, wc, d, n0;
  bool act[2];
  __device__ __forceinline__ explicit ScanLane(int D) {
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    lane = threadIdx.x & 63;
    q = lane & 3;
    ws = wave % WS;
    wc = wave / WS;
    d = blockIdx.y * kChans + wc * 32 + 2 * (lane >> 2);
    n0 = ws * kStates + q * NPL;
    act[0] = d < D;
    act[1] = d + 1 < D;
  }
};

// The states of a lane's two channels in (D, N) slices. VEC: whole vectors of them (N
// divides by NPL). No access has a branch: what is not there lies past the slice.
template <int NPL, bool VEC>
struct StatePair {
  unsigned bytes, off[2];
  int valid;
  __device__ __forceinline__ StatePair(int d, int n0, int D, int N, const bool (&act)[2])
      : bytes(4u * (unsigned)D * (unsigned)N), valid(N - n0) {
#pragma unroll
    for (int c = 0; c < 2; ++c)
      off[c] = act[c] && valid > 0 ? 4u * ((unsigned)(d + c) * (unsigned)N + n0) : kOOB;
  }
  __device__ __forceinline__ void load(float (&v)[2][NPL], const float* p,
                                       bool there = true) const {
    const GBuf g(p, there ? bytes : 0u);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      if constexpr (VEC && NPL == 4) {
        const auto r = __builtin_amdgcn_raw_buffer_load_b128(g.r, off[c], 0, 0);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[c][j] = __uint_as_float(r[j]);
      } else if constexpr (VEC && NPL == 2) {
        const auto r = __builtin_amdgcn_raw_buffer_load_b64(g.r, off[c], 0, 0);
        v[c][0] = __uint_as_float(r[0]);
        v[c][1] = __uint_as_float(r[1]);
      } else {
#pragma unroll
        for (int j = 0; j < NPL; ++j) v[c][j] = g.ld(j < valid ? off[c] + 4u * j : kOOB);
      }
    }
  }
  __device__ __forceinline__ void store(float* p, const float (&v)[2][NPL],
                                        bool there = true) const {
    const GBuf g(p, there ? bytes : 0u);
    typedef unsigned u4 __attribute__((ext_vector_type(4)));
    typedef unsigned u2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      if constexpr (VEC && NPL == 4) {
        __builtin_amdgcn_raw_buffer_store_b128(
            u4{__float_as_uint(v[c][0]), __float_as_uint(v[c][1]), __float_as_uint(v[c][2]),
               __float_as_uint(v[c][3])}, g.r, off[c], 0, 0);
      } else if constexpr (VEC && NPL == 2) {
        __builtin_amdgcn_raw_buffer_store_b64(
            u2{__float_as_uint(v[c][0]), __float_as_uint(v[c][1])}, g.r, off[c], 0, 0);
      } else {
#pragma unroll
        for (int j = 0; j < NPL; ++j) g.st(v[c][j], j < valid ? off[c] + 4u * j : kOOB);
      }
    }
  }
};

// One operand of the channels, (rows, D): register [c][k] of the S rows from row i S of the
// piece on holds row 4 k + q of channel d + c, 0 behind the piece's end.
// VEC: both channels in one access.
template <class T, int S, bool VEC>
struct ChanLoad {
  static constexpr int E = kElem<T>;
  GBuf g;
  unsigned off[2], step4, sub;
  __device__ __forceinline__ ChanLoad(const void* base, int ld, int t0, int len, int D, int d,
                                      int q, const bool (&act)[2])
      : g(buf_t<T>(base, (size_t)t0 * ld, len > 0 ? E * ((unsigned)(len - 1) * ld + D) : 0u)),
        step4(4 * E * ld), sub(S * E * ld) {
#pragma unroll
    for (int c = 0; c < 2; ++c) off[c] = act[c] ? E * ((unsigned)q * ld + d + c) : kOOB;
  }
  __device__ __forceinline__ void load(float (&v)[2][S / 4], int i) const {
#pragma unroll
    for (int k = 0; k < S / 4; ++k) {
      const unsigned o = (unsigned)i * sub + k * step4;
      if constexpr (!VEC) {
        v[0][k] = ld_t<T>(g, off[0] + o);
        v[1][k] = ld_t<T>(g, off[1] + o);
      } else if constexpr (E == 4) {
        const auto r = __builtin_amdgcn_raw_buffer_load_b64(g.r, off[0] + o, 0, 0);
        v[0][k] = __uint_as_float(r[0]);
        v[1][k] = __uint_as_float(r[1]);
      } else {
        const unsigned r = __builtin_amdgcn_raw_buffer_load_b32(g.r, off[0] + o, 0, 0);
        v[0][k] = T::to((unsigned short)r);
        v[1][k] = T::to((unsigned short)(r >> 16));
      }
    }
  }
  __device__ __forceinline__ void store(float v0, float v1, int i, int k) const {
    const unsigned o = (unsigned)i * sub + k * step4;
    if constexpr (!VEC) {
      st_t<T>(g, v0, off[0] + o);
      st_t<T>(g, v1, off[1] + o);
    } else if constexpr (E == 4) {
      typedef unsigned u2 __attribute__((ext_vector_type(2)));
      __builtin_amdgcn_raw_buffer_store_b64(u2{__float_as_uint(v0), __float_as_uint(v1)}, g.r,
                                            off[0] + o, 0, 0);
    } else {
      __builtin_amdgcn_raw_buffer_store_b32((unsigned)T::from(v0) | (unsigned)T::from(v1) << 16,
                                            g.r, off[0] + o, 0, 0);
    }
  }
};

// S rows of B or C, (rows, N), on their way to LDS: lane (row, q) takes the row's NPL
// states from n0 on (S 8: for the lanes 0 .. 31 of the wave, or the others).
template <class T, int NPL, int S, bool VEC>
struct StateLoad {
  static constexpr int E = kElem<T>;
  GBuf g;
  unsigned off, sub;
  int valid;
  __device__ __forceinline__ StateLoad(const void* base, int ld, int t0, int len, int N, int n0,
                                       int row)
      : g(buf_t<T>(base, (size_t)t0 * ld, len > 0 ? E * ((unsigned)(len - 1) * ld + N) : 0u)),
        off(E * ((unsigned)row * ld + n0)), sub(S * E * ld), valid(N - n0) {}
  __device__ __forceinline__ void load(float (&v)[NPL], int i) const {
    const unsigned o = off + (unsigned)i * sub;
    if constexpr (NPL == 1) {
      v[0] = ld_t<T>(g, valid > 0 ? o : kOOB);
    } else if constexpr (!VEC) {
#pragma unroll
      for (int j = 0; j < NPL; ++j) v[j] = ld_t<T>(g, j < valid ? o + E * j : kOOB);
    } else {
      unsigned r[4] = {0, 0, 0, 0};
      constexpr int W = NPL * E / 4;   // words
      if constexpr (W == 4) {
        const auto l = __builtin_amdgcn_raw_buffer_load_b128(g.r, o, 0, 0);
#pragma unroll
        for (int w = 0; w < 4; ++w) r[w] = l[w];
      } else if constexpr (W == 2) {
        const auto l = __builtin_amdgcn_raw_buffer_load_b64(g.r, o, 0, 0);
        r[0] = l[0];
        r[1] = l[1];
      } else {
        r[0] = __builtin_amdgcn_raw_buffer_load_b32(g.r, o, 0, 0);
      }
      // (states past N are the next row's numbers)
#pragma unroll
      for (int j = 0; j < NPL; ++j) {
        float f;
        if constexpr (E == 4) f = __uint_as_float(r[j]);
        else f = T::to((unsigned short)(r[j / 2] >> (16 * (j & 1))));
        v[j] = j < valid ? f : 0.f;
      }
    }
  }
};

// Lane K of each quad of b, times v; acc += that (b must not come from a VALU
// instruction less than two instructions before: quad_ready).
constexpr int quad_bcast(int k) { return k * 0x55; }
template <int K>
__device__ __forceinline__ float quad_mul(float b, float v) {
  return dpp_get<quad_bcast(K)>(b) * v;
}
template <int K>
__device__ __forceinline__ void quad_fmac(float& acc, float b, float v) {
  asm("v_fmac_f32_dpp %0, %1, %2 quad_perm:[%3,%3,%3,%3] row_mask:0xf bank_mask:0xf"
      : "+v"(acc)
      : "v"(b), "v"(v), "n"(K));
}
__device__ __forceinline__ void quad_ready(float (&v)[2][2]) {
  asm("s_nop 1" : "+v"(v[0][0]), "+v"(v[0][1]), "+v"(v[1][0]), "+v"(v[1][1]));
}

// Rows of R floats per channel of a wave in LDS, channel c of pair p in row 16 c + p: of R =
// 12 and 20 the 16 pairs' float4s lie in distinct banks. Register [c][k] (row 4 k + q of
// channel c) goes to its place; a lane reads four rows of a channel.
template <int S>
struct ChanTile {
  static constexpr int R = S + 4, kFloats = 32 * R;
  static __device__ __forceinline__ void store(float* t, int pair, int q,
                                               const float (&v)[2][S / 4]) {
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int k = 0; k < S / 4; ++k) t[(16 * c + pair) * R + 4 * k + q] = v[c][k];
  }
  static __device__ __forceinline__ float4 rows(const float* t, int pair, int c, int k) {
    return lds4(t + (16 * c + pair) * R + 4 * k);
  }
};
__device__ __forceinline__ float at4(const float4& v, int i) {
  return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}

// Steps behind a piece's rows, in its last sub-chunk, have dt = 0: exp2(0) keeps the state. A rate
// that is infinite would make them NaN. The backward's products are therefore 0 wherever dt is
// (v_mul_legacy_f32: 0 times anything; in a row of the sequence the forward gave NaN there), the
// forward walks the rows of such a sub-chunk once more. (A select of every step is one in 24
// of the forward's instructions; a copy of the loop for the last sub-chunk takes 35 registers,
// in the backward spills.)
__device__ __forceinline__ float zero_mul(float dt, float rate) {
  float v;
  asm("v_mul_legacy_f32 %0, %1, %2" : "=v"(v) : "v"(dt), "v"(rate));
  return v;
}
template <int NPL>
__device__ __forceinline__ bool endless_rate(const float (&a2)[2][NPL]) {   // in any lane
  bool any = false;
#pragma unroll
  for (int j = 0; j < NPL; ++j) any |= __builtin_isinf(a2[0][j]) || __builtin_isinf(a2[1][j]);
  return __any(any);
}

// Sums over the quad of v[s], s < 4: lane q ends with that of v[q].
__device__ __forceinline__ float quad_gather(const float (&v)[4], int q) {
  float a[2], b[1];
  rs_stage_dpp<kDppXor1>(v, a, q & 1);
  rs_stage_dpp<kDppXor2>(a, b, q >> 1);
  return b[0];
}

// Sum of dt over the piece, by channel: the quad's lanes hold each a part.
__device__ __forceinline__ void store_sdt(const PackedScanArgs& a, int q, int d,
                                          const bool (&act)[2], float s0, float s1) {
  s0 = group_sum<4>(s0);
  s1 = group_sum<4>(s1);
  float* p = a.sdt + (size_t)blockIdx.x * a.D + d;
  if (q == 0 && act[0]) p[0] = s0;
  if (q == 0 && act[1]) p[1] = s1;
}

// ----------------------------------------------------------------- forward
//
// CARRY: the carry pass, else the main one. All is branch-free buffer accesses, what is not
// there lying past the buffer: a branch within the loop made the compiler wait for all loads
// in flight (twice the time). 32768 x 2048 x 16 in bf16: 149 and 267 us, 8192 x 1536 x 16 in fp32
// 39 and 66 us, of 129 and 162, 24 and 30 that the vector units need for the formula alone.

template <class T, int NPL, int WS, bool VEC, bool CARRY, bool CKPT>
__global__ void __launch_bounds__(256)
packed_scan_fwd_kernel(PackedScanArgs a) {
  typedef ScanLane<NPL, WS> Lane;
  constexpr int NS = Lane::kStates;
  typedef ChanTile<kSub> Tile;
  // of a wave's sub-chunk: dt, dt x; B, C
  __shared__ __align__(16) float chans[4][2][Tile::kFloats];
  __shared__ __align__(16) float tiles[4][CARRY ? 1 : 2][kSub * NS];
  __shared__ float2 ysum[WS > 1 ? 2 : 1][WS > 1 ? 4 : 1][WS > 1 ? 4 : 1][64];
  const Piece pc = find_piece(a.q, a.tc, blockIdx.x);
  if (pc.seq < 0) return;
  const Lane L(a.D);
  if (pc.seq == a.q.nseq) {
    if (!CARRY)
      zero_rows<T>(a.y, pc.t0, pc.len, a.D, blockIdx.y * Lane::kChans,
                   (blockIdx.y + 1) * Lane::kChans);
    return;
  }
  if (CARRY && pc.last) return;
  const size_t slice = (size_t)a.D * a.N;
  const StatePair<NPL, VEC> at(L.d, L.n0, a.D, a.N, L.act);
  float a2[2][NPL], h[2][NPL];
  at.load(a2, a.aneg);
#pragma unroll
  for (int j = 0; j < NPL; ++j) {
    a2[0][j] *= -kLog2e;
    a2[1][j] *= -kLog2e;
    h[0][j] = h[1][j] = 0.f;
  }
  if constexpr (!CARRY) {
    if (pc.j > 0) at.load(h, a.start + (size_t)blockIdx.x * slice);
    else if (a.h0) at.load(h, a.h0 + (size_t)pc.seq * slice);
  }
  const int row = L.lane >> 2;
  const ChanLoad<T, kSub, VEC> lx(a.x, a.ld_x, pc.t0, pc.len, a.D, L.d, L.q, L.act);
  const ChanLoad<T, kSub, VEC> ldt(a.dt, a.ld_dt, pc.t0, pc.len, a.D, L.d, L.q, L.act);
  const StateLoad<T, NPL, kSub, VEC> lb(a.B, a.ld_b, pc.t0, pc.len, a.N, L.n0, row);
  const StateLoad<T, NPL, kSub, VEC> lc(a.C, a.ld_c, pc.t0, CARRY ? 0 : pc.len, a.N, L.n0, row);
  const ChanLoad<T, kSub, VEC> sy(a.y, a.D, pc.t0, CARRY ? 0 : pc.len, a.D, L.d, L.q, L.act);
  // the checkpoint before row 0 of the piece (not there for a sequence's first)
  float* ck = a.ckpt + ((ptrdiff_t)(pc.begin / kCkpt + pc.j * (a.tc / kCkpt)) - 1) *
                           (ptrdiff_t)slice;
  float* const tb = tiles[L.wave][0];
  float* const tc = tiles[L.wave][CARRY ? 0 : 1];
  float* const td = chans[L.wave][0];
  float* const tx = chans[L.wave][1];
  const int nsub = (pc.len + kSub - 1) / kSub;
  float nx[2][4], nd[2][4], nb[NPL], nc[NPL];   // the next sub-chunk's
  const auto load = [&](int i) {
    ldt.load(nd, i);
    lx.load(nx, i);
    lb.load(nb, i);
    if (!CARRY) lc.load(nc, i);
  };
  load(0);
  float sum_dt[2] = {0.f, 0.f};
  float before[2][NPL];   // the states before the sub-chunk
  for (int i = 0; i < nsub; ++i) {
    if constexpr (!CARRY) {
#pragma unroll
      for (int j = 0; j < NPL; ++j) {
        before[0][j] = h[0][j];
        before[1][j] = h[1][j];
      }
    }
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        nx[c][k] *= nd[c][k];
        if (CARRY) sum_dt[c] += nd[c][k];
      }
    wave_lds_sync();
    Tile::store(td, row, L.q, nd);
    Tile::store(tx, row, L.q, nx);
    store_vec<NPL>(tb + L.lane * NPL, nb);
    if (!CARRY) store_vec<NPL>(tc + L.lane * NPL, nc);
    wave_lds_sync();
    load(i + 1);
    static_for<4>([&](auto kc) {
      constexpr int k = decltype(kc)::value;
      if constexpr (CKPT && (4 * k) % kCkpt == 0)
        at.store(ck + (ptrdiff_t)(i * (kSub / kCkpt) + 4 * k / kCkpt) * (ptrdiff_t)slice, h,
                 (i > 0 || pc.j > 0 || k > 0) && i * kSub + 4 * k < pc.len);
      float y[2][4];
      const float4 dt[2] = {Tile::rows(td, row, 0, k), Tile::rows(td, row, 1, k)};
      const float4 bx[2] = {Tile::rows(tx, row, 0, k), Tile::rows(tx, row, 1, k)};
      static_for<4>([&](auto sc) {
        constexpr int s = decltype(sc)::value;
        float b[NPL], cv[NPL];
        load_vec<NPL>(b, tb + (4 * k + s) * NS + L.q * NPL);
        if (!CARRY) load_vec<NPL>(cv, tc + (4 * k + s) * NS + L.q * NPL);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int j = 0; j < NPL; ++j) {
            const float da = exp2_hw(at4(dt[c], s) * a2[c][j]);
            h[c][j] = __builtin_fmaf(da, h[c][j], at4(bx[c], s) * b[j]);
            if (!CARRY) y[c][s] = j ? __builtin_fmaf(cv[j], h[c][j], y[c][s]) : cv[j] * h[c][j];
          }
        }
      });
      if constexpr (!CARRY) {
        const float y0 = quad_gather(y[0], L.q), y1 = quad_gather(y[1], L.q);
        if constexpr (WS == 1) sy.store(y0, y1, i, k);
        else ysum[i & 1][L.wave][k][L.lane] = make_float2(y0, y1);
      }
    });
    if constexpr (WS > 1 && !CARRY) {
      // the WS waves of the same channels share out the four registers of y
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (k % WS != L.ws) continue;
        float2 v = ysum[i & 1][L.wc * WS][k][L.lane];
#pragma unroll
        for (int w = 1; w < WS; ++w) {
          const float2 o = ysum[i & 1][L.wc * WS + w][k][L.lane];
          v.x += o.x;
          v.y += o.y;
        }
        sy.store(v.x, v.y, i, k);
      }
    }
  }
  if (CARRY) {
    at.store(a.carry + (size_t)blockIdx.x * slice, h);
    if (L.ws == 0) store_sdt(a, L.q, L.d, L.act, sum_dt[0], sum_dt[1]);
  } else if (pc.last && a.h_last) {
    const int rows = pc.len % kSub;
    if (rows && endless_rate<NPL>(a2)) {   // the last sub-chunk's rows again, without those behind
#pragma unroll 1
      for (int r = 0; r < rows; ++r) {
        float b[NPL];
        load_vec<NPL>(b, tb + r * NS + L.q * NPL);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float dt = td[(16 * c + row) * Tile::R + r], bx = tx[(16 * c + row) * Tile::R + r];
#pragma unroll
          for (int j = 0; j < NPL; ++j)
            before[c][j] = __builtin_fmaf(exp2_hw(dt * a2[c][j]), before[c][j], bx * b[j]);
        }
      }
      at.store(a.h_last + (size_t)pc.seq * slice, before);
    } else {
      at.store(a.h_last + (size_t)pc.seq * slice, h);
    }
  }
}

// carry and sdt -> start of the pieces 1 .. of each sequence of several; with BACK
// of the pieces .. n - 2, from the last (dh_last) down. Block (s, channels x states). Bound by the
// states' bytes, read and written once, and by the chain of a sequence's pieces, eight of
// which are loaded at once (8192 x 1536 x 16 fp32 in pieces of 32 rows, 54 MB: 17 us).
template <bool BACK>
__global__ void __launch_bounds__(256)
packed_fold_kernel(PackedScanArgs a) {
  const int e = blockIdx.y * 256 + threadIdx.x;
  const int s = blockIdx.x;
  int p;
  const int n = seq_pieces(a.q, a.tc, s, &p);
  if (n < 2 || e >= a.D * a.N) return;
  const size_t slice = (size_t)a.D * a.N;
  const float a2 = -a.aneg[e] * kLog2e;
  const float* sd = a.sdt + (size_t)p * a.D + e / a.N;
  const float* end = a.carry + (size_t)p * slice + e;
  float* start = a.start + (size_t)p * slice + e;
  const float* from = BACK ? a.dh_last : a.h0;
  float h = from ? from[(size_t)s * slice + e] : 0.f;
  constexpr int U = 8;   // pieces whose loads are in flight together
  for (int i0 = 0; i0 < n - 1; i0 += U) {
    float v[U], sum[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = min(i0 + u, n - 2), j = BACK ? n - 1 - i : i;
      v[u] = end[(size_t)j * slice];
      sum[u] = sd[(size_t)j * a.D];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i0 + u > n - 2) break;
      h = __builtin_fmaf(exp2_hw(sum[u] * a2), h, v[u]);
      start[(size_t)(BACK ? n - 2 - i0 - u : i0 + u + 1) * slice] = h;
    }
  }
}

// ---------------------------------------------------------------- backward
//
// With G_t the adjoint of h_t and u_t = dA_t G_t what it passes to step t - 1:
//   G_t = dy_t C_t + u_{t+1},   q_t = u_t h_{t-1}
//   dx_t = dt_t sum_n G B,  ddt_t = x_t sum_n G B - sum_n Aneg q,  dAneg -= dt_t q
//   dB_tn = sum_d G dt x,  dC_tn = sum_d dy h,  dh0 = u_0
// The main pass walks the sub-chunks (8 rows) of a piece from the last: their dA and h
// are formed again, from the checkpoint before them, in registers, then the rows
// are walked back. The sums over the channels add a lane's two channels in the products,
// then go over the wave's 16 channel pairs, two rows of four states and two kinds at a time
// so that each lane ends with one of them, in LDS over the block's waves, and over the
// blocks in packed_sum_bc_kernel: always in the same order.
// (Checkpoints every 8 rows rather than 16: what the sums over the channels cost falls with
// the channels a lane holds, and registers hold 8 rows of two.) 32768 x 2048 x 16 in bf16: 159
// (carry) and 609 us, 8192 x 1536 x 16 in fp32 36 and 133 us.

// The adjoint's carry pass: each piece but the first from a zero adjoint.
template <class T, int NPL, int WS, bool VEC>
__global__ void __launch_bounds__(256)
packed_scan_back_carry_kernel(PackedScanArgs a) {
  typedef ScanLane<NPL, WS> Lane;
  constexpr int NS = Lane::kStates;
  typedef ChanTile<kSub> Tile;
  // of a wave's sub-chunk: dt, dy; C
  __shared__ __align__(16) float chans[4][2][Tile::kFloats];
  __shared__ __align__(16) float tiles[4][kSub * NS];
  const Piece pc = find_piece(a.q, a.tc, blockIdx.x);
  if (pc.seq < 0 || pc.seq == a.q.nseq || pc.j == 0) return;
  const Lane L(a.D);
  const size_t slice = (size_t)a.D * a.N;
  const StatePair<NPL, VEC> at(L.d, L.n0, a.D, a.N, L.act);
  float a2[2][NPL], u[2][NPL];
  at.load(a2, a.aneg);
#pragma unroll
  for (int j = 0; j < NPL; ++j) {
    a2[0][j] *= -kLog2e;
    a2[1][j] *= -kLog2e;
    u[0][j] = u[1][j] = 0.f;
  }
  const ChanLoad<T, kSub, VEC> ldt(a.dt, a.ld_dt, pc.t0, pc.len, a.D, L.d, L.q, L.act);
  const ChanLoad<T, kSub, VEC> ldy(a.dy, a.ld_dy, pc.t0, pc.len, a.D, L.d, L.q, L.act);
  const StateLoad<T, NPL, kSub, VEC> lc(a.C, a.ld_c, pc.t0, pc.len, a.N, L.n0, L.lane >> 2);
  float* const tc = tiles[L.wave];
  float* const td = chans[L.wave][0];
  float* const ty = chans[L.wave][1];
  const int row = L.lane >> 2;
  float nd[2][4], ny[2][4], nc[NPL];
  const auto load = [&](int i) {   // (of a sub-chunk -1: zeros)
    ldt.load(nd, i);
    ldy.load(ny, i);
    lc.load(nc, i);
  };
  const int nsub = (pc.len + kSub - 1) / kSub;
  load(nsub - 1);
  float sum_dt[2] = {0.f, 0.f};
  for (int i = nsub - 1; i >= 0; --i) {
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int k = 0; k < 4; ++k) sum_dt[c] += nd[c][k];
    wave_lds_sync();
    Tile::store(td, row, L.q, nd);
    Tile::store(ty, row, L.q, ny);
    store_vec<NPL>(tc + L.lane * NPL, nc);
    wave_lds_sync();
    load(i - 1);
    static_for<4>([&](auto kcn) {
      constexpr int k = 3 - decltype(kcn)::value;
      const float4 dt[2] = {Tile::rows(td, row, 0, k), Tile::rows(td, row, 1, k)};
      const float4 dy[2] = {Tile::rows(ty, row, 0, k), Tile::rows(ty, row, 1, k)};
      static_for<4>([&](auto scn) {
        constexpr int s = 3 - decltype(scn)::value;
        float cv[NPL];
        load_vec<NPL>(cv, tc + (4 * k + s) * NS + L.q * NPL);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int j = 0; j < NPL; ++j)
            u[c][j] = __builtin_fmaf(at4(dy[c], s), cv[j], u[c][j]) *
                      exp2_hw(zero_mul(at4(dt[c], s), a2[c][j]));
        }
      });
    });
  }
  at.store(a.carry + (size_t)blockIdx.x * slice, u);
  if (L.ws == 0) store_sdt(a, L.q, L.d, L.act, sum_dt[0], sum_dt[1]);
}

// Sums over the lanes that share lane & 3 of v[i], i < 16: each lane ends with that of
// index chan_sum_index(lane).
__device__ __forceinline__ float chan_sum16(const float (&v)[16]) {
  float a[8], b[4];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[2 * i]),
                                                    __float_as_uint(v[2 * i + 1]), false, false);
    a[i] = __uint_as_float(s[0]) + __uint_as_float(s[1]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(a[2 * i]),
                                                    __float_as_uint(a[2 * i + 1]), false, false);
    b[i] = __uint_as_float(s[0]) + __uint_as_float(s[1]);
  }
  return rs_bits32_shift(b);
}
__device__ __forceinline__ int chan_sum_index(int lane) {
  return (lane >> 5 & 1) + 2 * (lane >> 4 & 1) + 4 * (lane >> 2 & 1) + 8 * (lane >> 3 & 1);
}

template <class T, int NPL, int WS, bool VEC>
__global__ void __launch_bounds__(256, 2)
packed_scan_bwd_kernel(PackedScanArgs a) {
  typedef ScanLane<NPL, WS> Lane;
  constexpr int WC = 4 / WS;
  constexpr int NS = Lane::kStates;
  constexpr int S = kCkpt, K = S / 4;
  // dB, dC of the sub-chunk by wave: [kind][row][state], the kinds apart by half the banks more
  constexpr int KIND = S * NS + 32;
  __shared__ float tiles[4][2][S * NS];   // B, C of a wave's sub-chunk
  __shared__ float tbc[2][4][2 * KIND];
  __shared__ float4 tss[WS > 1 ? 2 : 1][WS > 1 ? 4 : 1][K][WS > 1 ? 64 : 1];
  const Piece pc = find_piece(a.q, a.tc, blockIdx.x);
  const Lane L(a.D);
  const size_t slice = (size_t)a.D * a.N;
  const StatePair<NPL, VEC> at(L.d, L.n0, a.D, a.N, L.act);
  float* part = a.part_bc + ((size_t)blockIdx.y * a.q.total + max(0, pc.t0)) * 2 * a.N;
  if (pc.seq < 0 || pc.seq == a.q.nseq) {
    const float zero[2][NPL] = {};
    at.store(a.part_a + (size_t)blockIdx.x * slice, zero);
    if (pc.seq < 0) return;
    const int d_lo = blockIdx.y * Lane::kChans, d_hi = d_lo + Lane::kChans;
    zero_rows<T>(a.dx, pc.t0, pc.len, a.D, d_lo, d_hi);
    zero_rows<T>(a.ddt, pc.t0, pc.len, a.D, d_lo, d_hi);
    for (size_t i = threadIdx.x; i < (size_t)pc.len * 2 * a.N; i += blockDim.x) part[i] = 0.f;
    return;
  }
  // (sums of -Aneg log2(e) q and of dt q, scaled once at the end)
  float a2[2][NPL], u[2][NPL], acc[2][NPL];
  at.load(a2, a.aneg);
#pragma unroll
  for (int j = 0; j < NPL; ++j) {
    a2[0][j] *= -kLog2e;
    a2[1][j] *= -kLog2e;
    u[0][j] = u[1][j] = acc[0][j] = acc[1][j] = 0.f;
  }
  if (!pc.last) at.load(u, a.start + (size_t)blockIdx.x * slice);
  else if (a.dh_last) at.load(u, a.dh_last + (size_t)pc.seq * slice);
  const ChanLoad<T, S, VEC> lx(a.x, a.ld_x, pc.t0, pc.len, a.D, L.d, L.q, L.act);
  const ChanLoad<T, S, VEC> ldt(a.dt, a.ld_dt, pc.t0, pc.len, a.D, L.d, L.q, L.act);
  const ChanLoad<T, S, VEC> ldy(a.dy, a.ld_dy, pc.t0, pc.len, a.D, L.d, L.q, L.act);
  // lanes 0 .. 31 bring B's rows to LDS, the others C's
  const bool half = L.lane >= 32;
  const int row = L.lane >> 2 & 7;
  const StateLoad<T, NPL, S, VEC> lb(a.B, a.ld_b, pc.t0, pc.len, a.N, L.n0, row);
  const StateLoad<T, NPL, S, VEC> lc(a.C, a.ld_c, pc.t0, pc.len, a.N, L.n0, row);
  const ChanLoad<T, S, VEC> sdx(a.dx, a.D, pc.t0, pc.len, a.D, L.d, L.q, L.act);
  const ChanLoad<T, S, VEC> sddt(a.ddt, a.D, pc.t0, pc.len, a.D, L.d, L.q, L.act);
  const int g0 = pc.j * (a.tc / S);   // the piece's first sub-chunk in its sequence
  const int nsub = (pc.len + S - 1) / S;
  const float* ck = a.ckpt + ((ptrdiff_t)(pc.begin / S + g0) - 1) * (ptrdiff_t)slice;
  const float* h_first = a.h0 + (size_t)pc.seq * slice;
  float nx[2][K], nd[2][K], ny[2][K], nb[NPL], nc[NPL], nh[2][NPL];
  const auto load = [&](int i) {   // (of a sub-chunk -1: zeros)
    ldt.load(nd, i);
    lx.load(nx, i);
    ldy.load(ny, i);
    lb.load(nb, i);
    lc.load(nc, i);
    const bool first = g0 + i <= 0;
    at.load(nh, first ? h_first : ck + (ptrdiff_t)i * (ptrdiff_t)slice,
            i >= 0 && (!first || a.h0 != nullptr));
  };
  load(nsub - 1);
  float* const tb = tiles[L.wave][0];
  float* const tc = tiles[L.wave][1];
  const int ix = chan_sum_index(L.lane);
  // where this lane's sums go: kind ix / 8, row parity ix / 4 % 2, state ix % 4 of its quad's
  const bool sums = (ix & 3) < NPL;
  const int to = (ix >> 3) * KIND + (ix >> 2 & 1) * NS + L.q * NPL + (ix & 3);
  for (int i = nsub - 1; i >= 0; --i) {
    float x[2][K], dt[2][K], dy[2][K], bx[2][K], h0[2][NPL];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        x[c][k] = nx[c][k];
        dt[c][k] = nd[c][k];
        dy[c][k] = ny[c][k];
        bx[c][k] = nd[c][k] * nx[c][k];
      }
#pragma unroll
      for (int j = 0; j < NPL; ++j) h0[c][j] = nh[c][j];
    }
    quad_ready(dt);
    quad_ready(dy);
    quad_ready(bx);
    wave_lds_sync();
    float nbc[NPL];
#pragma unroll
    for (int j = 0; j < NPL; ++j) nbc[j] = half ? nc[j] : nb[j];
    store_vec<NPL>(tb + L.lane * NPL, nbc);   // (C's tile follows B's)
    wave_lds_sync();
    load(i - 1);
    float da[S][2][NPL], hs[S][2][NPL];
    static_for<S>([&](auto tcn) {
      constexpr int t = decltype(tcn)::value, k = t / 4, s = t % 4;
      float b[NPL];
      load_vec<NPL>(b, tb + t * NS + L.q * NPL);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float now = dpp_get<quad_bcast(s)>(dt[c][k]);
#pragma unroll
        for (int j = 0; j < NPL; ++j) {
          da[t][c][j] = exp2_hw(zero_mul(now, a2[c][j]));
          hs[t][c][j] = __builtin_fmaf(da[t][c][j], t ? hs[t ? t - 1 : 0][c][j] : h0[c][j],
                                       quad_mul<s>(bx[c][k], b[j]));
        }
      }
    });
    float* const mine = tbc[i & 1][L.wave] + to;
    static_for<K>([&](auto kcn) {
      constexpr int k = K - 1 - decltype(kcn)::value;
      float s1[2][4], s2[2][4];
      float v[16];   // of two rows: [kind][row parity][state], kinds G dt x, dy h
      static_for<4>([&](auto scn) {
        constexpr int s = 3 - decltype(scn)::value, t = 4 * k + s;
        float b[NPL], cv[NPL];
        load_vec<NPL>(b, tb + t * NS + L.q * NPL);
        load_vec<NPL>(cv, tc + t * NS + L.q * NPL);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int j = 0; j < NPL; ++j) {
            float& vb = v[(s & 1) * 4 + j];
            float& vc = v[8 + (s & 1) * 4 + j];
            quad_fmac<s>(u[c][j], dy[c][k], cv[j]);   // G
            const float g = u[c][j];
            u[c][j] = da[t][c][j] * g;
            const float qv = u[c][j] * (t ? hs[t ? t - 1 : 0][c][j] : h0[c][j]);
            s1[c][s] = j ? __builtin_fmaf(b[j], g, s1[c][s]) : b[j] * g;
            s2[c][s] = j ? __builtin_fmaf(a2[c][j], qv, s2[c][s]) : a2[c][j] * qv;
            quad_fmac<s>(acc[c][j], dt[c][k], qv);
            if (c == 0) {
              vb = quad_mul<s>(bx[c][k], g);
              vc = quad_mul<s>(dy[c][k], hs[t][c][j]);
            } else {
              quad_fmac<s>(vb, bx[c][k], g);
              quad_fmac<s>(vc, dy[c][k], hs[t][c][j]);
            }
          }
        }
        if constexpr ((s & 1) == 0) {
#pragma unroll
          for (int j = NPL; j < 4; ++j) v[j] = v[4 + j] = v[8 + j] = v[12 + j] = 0.f;
          const float sum = chan_sum16(v);
          if (sums) mine[t * NS] = sum;
        }
      });
      float r1[2], r2[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        r1[c] = quad_gather(s1[c], L.q);
        r2[c] = quad_gather(s2[c], L.q);
      }
      if constexpr (WS == 1) {
        sdx.store(dt[0][k] * r1[0], dt[1][k] * r1[1], i, k);
        sddt.store(__builtin_fmaf(x[0][k], r1[0], r2[0] * kLn2),
                   __builtin_fmaf(x[1][k], r1[1], r2[1] * kLn2), i, k);
      } else {
        tss[i & 1][L.wave][k][L.lane] = make_float4(r1[0], r1[1], r2[0], r2[1]);
      }
    });
    __syncthreads();
    if constexpr (WS > 1) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (k % WS != L.ws) continue;
        float4 r = tss[i & 1][L.wc * WS][k][L.lane];
#pragma unroll
        for (int w = 1; w < WS; ++w) {
          const float4 o = tss[i & 1][L.wc * WS + w][k][L.lane];
          r.x += o.x;
          r.y += o.y;
          r.z += o.z;
          r.w += o.w;
        }
        sdx.store(dt[0][k] * r.x, dt[1][k] * r.y, i, k);
        sddt.store(__builtin_fmaf(x[0][k], r.x, r.z * kLn2),
                   __builtin_fmaf(x[1][k], r.y, r.w * kLn2), i, k);
      }
    }
    // the block's sums of dB and dC: over its waves of channels
    const int len = min(S, pc.len - i * S);
#pragma unroll
    for (int r0 = 0; r0 < 2 * S * WS * NS; r0 += 256) {
      const int r = r0 + threadIdx.x;
      const int n = r % (WS * NS), kind = r / (WS * NS) & 1, step = r / (2 * WS * NS);
      if (n >= a.N || step >= len) continue;
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < WC; ++w)
        sum += tbc[i & 1][w * WS + n / NS][kind * KIND + step * NS + n % NS];
      part[((size_t)(i * S + step) * 2 + kind) * a.N + n] = sum;
    }
  }
#pragma unroll
  for (int j = 0; j < NPL; ++j) {
    acc[0][j] = -acc[0][j];
    acc[1][j] = -acc[1][j];
  }
  at.store(a.part_a + (size_t)blockIdx.x * slice, acc);
  if (pc.j == 0 && a.dh0) at.store(a.dh0 + (size_t)pc.seq * slice, u);
}

}  // namespace mhs
