// Selective scan over packed sequences for gfx950 (see mhs_packed.hpp for the
// pieces), forward and backward:
//   h_t = exp(-dt_t Aneg) h_{t-1} + dt_t x_t B_t,   y_t = sum_n C_tn h_tn
// per sequence, from h0 (nseq, D, N) or from zero.
//
// Mapping. A wave holds 16 channels in its four rows of 16 lanes; the rows
// split the states, NPL each (4 NPL states a wave; a block has WS waves for
// the states and 4 / WS times 16 channels). Time goes in sub-chunks of 16
// steps. A register of x or dt is loaded for four steps at once, row r step r,
// and spread to the rows by swaps between them; B and C lie in the lanes of a
// row, 16 / NPL steps of the row's NPL states a register, and are broadcast
// within the multiply that uses them. The waves of a block run without
// barriers (but for the sum of y over WS > 1 waves).
//
// A sequence longer than a piece takes three launches: the carry pass walks
// each piece but the last from a zero state and leaves its end state and its
// sum of dt; the fold turns these into the states at the pieces' starts,
// H <- exp(-Aneg sum dt) H + end; the main pass walks every piece from there.
// The exponentials of the pieces that the carry pass walks are so taken twice.
#pragma once

#include "mhs_packed.hpp"

namespace mhs {

constexpr int kSub = 16;   // steps of a sub-chunk

struct PackedScanArgs {
  Seqs q;
  const void *x, *dt, *B, *C;
  int ld_x, ld_dt, ld_b, ld_c;   // elements between rows
  const float* aneg;
  const float* h0;       // null: zeros
  void* y;               // (total, D)
  float* h_last;         // null: not wanted
  float* ckpt;           // (total / 16, D, N), null: not wanted. Entry begin / 16 + g - 1 is the
                         // state before step 16 g of its sequence, g >= 1
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
  static constexpr int kChans = 16 * (4 / WS);   // of a block
  int wave, lane, row, c, ws, wc, d, n0;
  bool act;
  __device__ __forceinline__ explicit ScanLane(int D) {
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    lane = threadIdx.x & 63;
    row = lane >> 4;
    c = lane & 15;
    ws = wave % WS;
    wc = wave / WS;
    d = blockIdx.y * kChans + wc * 16 + c;
    n0 = ws * kStates + row * NPL;
    act = d < D;
  }
};

// One operand of the channels, (rows, D): register k of sub-chunk i holds step
// 4 k + r of it in row r, 0 behind the piece's end.
template <class T>
struct ChanLoad {
  GBuf g;
  unsigned off, step4, sub;
  __device__ __forceinline__ ChanLoad(const void* base, int ld, int t0, int len, int D, int d,
                                      int row, bool act)
      : g(buf_t<T>(base, (size_t)t0 * ld,
                   len > 0 ? kElem<T> * ((unsigned)(len - 1) * ld + D) : 0u)),
        off(act ? kElem<T> * ((unsigned)row * ld + d) : kOOB), step4(4 * kElem<T> * ld),
        sub(16 * kElem<T> * ld) {}
  __device__ __forceinline__ void load(float (&v)[4], int i) const {
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = ld_t<T>(g, off + (unsigned)i * sub + k * step4);
  }
  __device__ __forceinline__ void store(float v, int i, int k) const {
    st_t<T>(g, v, off + (unsigned)i * sub + k * step4);
  }
};
// B or C, (rows, N): register k holds, in lane l of row r, step
// k * (16 / NPL) + l / NPL of state n0 + l % NPL.
template <class T, int NPL>
struct StateLoad {
  static constexpr int kPer = 16 / NPL;
  GBuf g;
  unsigned off, stepk, sub;
  __device__ __forceinline__ StateLoad(const void* base, int ld, int t0, int len, int N, int n0,
                                       int c)
      : g(buf_t<T>(base, (size_t)t0 * ld,
                   len > 0 ? kElem<T> * ((unsigned)(len - 1) * ld + N) : 0u)),
        off(n0 + c % NPL < N ? kElem<T> * ((unsigned)(c / NPL) * ld + n0 + c % NPL) : kOOB),
        stepk(kPer * kElem<T> * ld), sub(16 * kElem<T> * ld) {}
  __device__ __forceinline__ void load(float (&v)[NPL], int i) const {
#pragma unroll
    for (int k = 0; k < NPL; ++k) v[k] = ld_t<T>(g, off + (unsigned)i * sub + k * stepk);
  }
};

// ----------------------------------------------------------------- forward

template <class T, int NPL, int WS, bool CARRY>
__global__ void __launch_bounds__(256)
packed_scan_fwd_kernel(PackedScanArgs a) {
  typedef ScanLane<NPL, WS> Lane;
  constexpr int PER = 16 / NPL;
  __shared__ float ysum[WS > 1 ? 2 : 1][WS > 1 ? 4 : 1][WS > 1 ? 4 : 1][64];
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
  const StateAt<NPL> at(L.d, L.n0, a.D, a.N);
  float a2[NPL], h[NPL];
  at.load(a2, a.aneg);
#pragma unroll
  for (int j = 0; j < NPL; ++j) {
    a2[j] *= -kLog2e;
    h[j] = 0.f;
  }
  if (!CARRY) {
    if (pc.j > 0) at.load(h, a.start + (size_t)blockIdx.x * slice);
    else if (a.h0) at.load(h, a.h0 + (size_t)pc.seq * slice);
  }
  const ChanLoad<T> lx(a.x, a.ld_x, pc.t0, pc.len, a.D, L.d, L.row, L.act);
  const ChanLoad<T> ldt(a.dt, a.ld_dt, pc.t0, pc.len, a.D, L.d, L.row, L.act);
  const StateLoad<T, NPL> lb(a.B, a.ld_b, pc.t0, pc.len, a.N, L.n0, L.c);
  const StateLoad<T, NPL> lc(a.C, a.ld_c, pc.t0, CARRY ? 0 : pc.len, a.N, L.n0, L.c);
  const ChanLoad<T> sy(a.y, a.D, pc.t0, CARRY ? 0 : pc.len, a.D, L.d, L.row, L.act);
  float* ck = a.ckpt ? a.ckpt + ((size_t)(pc.begin / kSub) + (size_t)pc.j * (a.tc / kSub)) * slice
                     : nullptr;
  const int nsub = (pc.len + kSub - 1) / kSub;
  float nx[4], nd[4], nb[NPL], nc[NPL];   // the next sub-chunk's
  lx.load(nx, 0);
  ldt.load(nd, 0);
  lb.load(nb, 0);
  if (!CARRY) lc.load(nc, 0);
  float sum_dt = 0.f;
  for (int i = 0; i < nsub; ++i) {
    float bx[4], dc[4], b[NPL], cc[NPL];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      dc[k] = nd[k];
      bx[k] = nd[k] * nx[k];
      if (CARRY) sum_dt += nd[k];
    }
#pragma unroll
    for (int k = 0; k < NPL; ++k) {
      b[k] = nb[k];
      if (!CARRY) cc[k] = nc[k];
    }
    if (!CARRY) row_fmac_ready(cc);
    lx.load(nx, i + 1);
    ldt.load(nd, i + 1);
    lb.load(nb, i + 1);
    if (!CARRY) lc.load(nc, i + 1);
    if (!CARRY && ck && (i > 0 || pc.j > 0)) at.store(ck + ((ptrdiff_t)i - 1) * (ptrdiff_t)slice, h);
    static_for<4>([&](auto qc) {
      constexpr int q = decltype(qc)::value;
      float dts[4], bxs[4], y[4];
      spread_rows(dc[q], dts);
      spread_rows(bx[q], bxs);
      static_for<4>([&](auto sc) {
        constexpr int s = decltype(sc)::value, t = 4 * q + s;
        static_for<NPL>([&](auto jc) {
          constexpr int j = decltype(jc)::value, k = (t % PER) * NPL + j;
          const float u = row_mul<k>(b[t / PER], bxs[s]);
          h[j] = __builtin_fmaf(exp2_hw(dts[s] * a2[j]), h[j], u);
          if constexpr (!CARRY) {
            if constexpr (j == 0) y[s] = row_mul<k>(cc[t / PER], h[j]);
            else row_fmac<k>(y[s], cc[t / PER], h[j]);
          }
        });
      });
      if (!CARRY) {
        const float yr = gather_rows(y);
        if constexpr (WS == 1) sy.store(yr, i, q);
        else ysum[i & 1][L.wave][q][L.lane] = yr;
      }
    });
    if constexpr (WS > 1 && !CARRY) {
      // the WS waves of the same channels share out the four registers of y
      __syncthreads();
#pragma unroll
      for (int q = L.ws; q < 4; q += WS) {
        float v = ysum[i & 1][L.wc * WS][q][L.lane];
#pragma unroll
        for (int w = 1; w < WS; ++w) v += ysum[i & 1][L.wc * WS + w][q][L.lane];
        sy.store(v, i, q);
      }
    }
  }
  if (CARRY) {
    at.store(a.carry + (size_t)blockIdx.x * slice, h);
    // the four rows' steps of the channel
    const float s4[4] = {sum_dt, 0.f, 0.f, 0.f};
    const float total = gather_rows(s4);
    if (L.ws == 0 && L.row == 0 && L.act) a.sdt[(size_t)blockIdx.x * a.D + L.d] = total;
  } else if (pc.last && a.h_last) {
    at.store(a.h_last + (size_t)pc.seq * slice, h);
  }
}

// carry and sdt -> start of the pieces 1 .. of each sequence of several; with BACK
// of the pieces .. n - 2, from the last (dh_last) down. Block (s, channels x states).
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
// The main pass walks the sub-chunks of a piece from the last: dA and h of its 16
// steps are formed again, from the checkpoint before it, in registers, then
// the steps are walked back. The sums over the states go over the rows as y's do;
// those over the channels over the 16 lanes of a row, two steps of four states and
// two kinds at a time so that each lane ends with one of them, then in LDS over the
// block's waves, and over the blocks in packed_sum_bc_kernel: always in
// the same order. The adjoint's carry pass and fold mirror the forward's.

// Sum over the 16 lanes of each row of v[i], i < 16: lane l ends with that of
// index row_sum_index(l).
__device__ __forceinline__ float row_sum16(const float (&v)[16], int lane) {
  float b[8], c[4], d[2];
#pragma unroll
  for (int i = 0; i < 8; ++i) b[i] = 0.f;
  rs_stage_dpp<kDppRor8>(v, b, (lane >> 3) & 1);
  rs_stage_dpp<kDppHalfMirror>(b, c, (lane >> 2) & 1);
  rs_stage_dpp<kDppXor2>(c, d, (lane >> 1) & 1);
  float e[1];
  rs_stage_dpp<kDppXor1>(d, e, lane & 1);
  return e[0];
}
__device__ __forceinline__ int row_sum_index(int lane) {
  return 8 * (lane & 1) + 4 * ((lane >> 1) & 1) + 2 * ((lane >> 2) & 1) + ((lane >> 3) & 1);
}

template <class T, int NPL, int WS, bool CARRY>
__global__ void __launch_bounds__(256, 2)
packed_scan_bwd_kernel(PackedScanArgs a) {
  typedef ScanLane<NPL, WS> Lane;
  constexpr int PER = 16 / NPL;
  constexpr int WC = 4 / WS;
  constexpr int NS = Lane::kStates;
  // dB, dC of the sub-chunk by wave [kind][step][state], and s1, s2 by wave
  __shared__ float tbc[CARRY ? 1 : 2][CARRY ? 1 : 4][CARRY ? 1 : 2 * kSub * NS];
  __shared__ float tss[WS > 1 && !CARRY ? 2 : 1][WS > 1 && !CARRY ? 4 : 1][2][4]
                      [WS > 1 && !CARRY ? 64 : 1];
  const Piece pc = find_piece(a.q, a.tc, blockIdx.x);
  const Lane L(a.D);
  const size_t slice = (size_t)a.D * a.N;
  const StateAt<NPL> at(L.d, L.n0, a.D, a.N);
  float zero[NPL] = {};
  if (pc.seq < 0 || pc.seq == a.q.nseq) {
    if (CARRY) return;
    at.store(a.part_a + (size_t)blockIdx.x * slice, zero);
    if (pc.seq < 0) return;
    const int d_lo = blockIdx.y * Lane::kChans, d_hi = d_lo + Lane::kChans;
    zero_rows<T>(a.dx, pc.t0, pc.len, a.D, d_lo, d_hi);
    zero_rows<T>(a.ddt, pc.t0, pc.len, a.D, d_lo, d_hi);
    float* part = a.part_bc + ((size_t)blockIdx.y * a.q.total + pc.t0) * 2 * a.N;
    for (size_t i = threadIdx.x; i < (size_t)pc.len * 2 * a.N; i += blockDim.x) part[i] = 0.f;
    return;
  }
  if (CARRY && pc.j == 0) return;
  float an[NPL], a2[NPL], u[NPL], acc[NPL];
  at.load(an, a.aneg);
#pragma unroll
  for (int j = 0; j < NPL; ++j) {
    a2[j] = -an[j] * kLog2e;
    u[j] = acc[j] = 0.f;
  }
  if (!CARRY) {
    if (!pc.last) at.load(u, a.start + (size_t)blockIdx.x * slice);
    else if (a.dh_last) at.load(u, a.dh_last + (size_t)pc.seq * slice);
  }
  const int xlen = CARRY ? 0 : pc.len;
  const ChanLoad<T> lx(a.x, a.ld_x, pc.t0, xlen, a.D, L.d, L.row, L.act);
  const ChanLoad<T> ldt(a.dt, a.ld_dt, pc.t0, pc.len, a.D, L.d, L.row, L.act);
  const ChanLoad<T> ldy(a.dy, a.ld_dy, pc.t0, pc.len, a.D, L.d, L.row, L.act);
  const StateLoad<T, NPL> lb(a.B, a.ld_b, pc.t0, xlen, a.N, L.n0, L.c);
  const StateLoad<T, NPL> lc(a.C, a.ld_c, pc.t0, pc.len, a.N, L.n0, L.c);
  const ChanLoad<T> sdx(a.dx, a.D, pc.t0, xlen, a.D, L.d, L.row, L.act);
  const ChanLoad<T> sddt(a.ddt, a.D, pc.t0, xlen, a.D, L.d, L.row, L.act);
  const int g0 = pc.j * (a.tc / kSub);   // the piece's first sub-chunk in its sequence
  const int nsub = (pc.len + kSub - 1) / kSub;
  const float* ck = a.ckpt + ((size_t)(pc.begin / kSub) + (size_t)g0) * slice;
  const float* h_first = a.h0 ? a.h0 + (size_t)pc.seq * slice : nullptr;
  auto load_state = [&](float (&v)[NPL], int i) {   // the state before sub-chunk i
    if (i < 0) return;
    if (g0 + i > 0) {
      at.load(v, ck + ((ptrdiff_t)i - 1) * (ptrdiff_t)slice);
    } else if (h_first) {
      at.load(v, h_first);
    } else {
#pragma unroll
      for (int j = 0; j < NPL; ++j) v[j] = 0.f;
    }
  };
  float nx[4], nd[4], ny[4], nb[NPL], nc[NPL], nh[NPL] = {};
  auto load_sub = [&](int i) {
    if (i < 0) return;
    ldt.load(nd, i);
    ldy.load(ny, i);
    lc.load(nc, i);
    if (CARRY) return;
    lx.load(nx, i);
    lb.load(nb, i);
    load_state(nh, i);
  };
  load_sub(nsub - 1);
  float sum_dt = 0.f;
  float* part = a.part_bc + ((size_t)blockIdx.y * a.q.total + pc.t0) * 2 * a.N;
  for (int i = nsub - 1; i >= 0; --i) {
    float xc[4], dc[4], yc[4], b[NPL], cc[NPL], h0[NPL];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      dc[k] = nd[k];
      yc[k] = ny[k];
      if (!CARRY) xc[k] = nx[k];
      if (CARRY) sum_dt += nd[k];
    }
#pragma unroll
    for (int k = 0; k < NPL; ++k) {
      cc[k] = nc[k];
      if (!CARRY) b[k] = nb[k];
      if (!CARRY) h0[k] = nh[k];
    }
    row_fmac_ready(cc);
    if (!CARRY) row_fmac_ready(b);
    load_sub(i - 1);
    float da[kSub][NPL], hs[CARRY ? 1 : kSub][NPL];
    static_for<4>([&](auto qc) {
      constexpr int q = decltype(qc)::value;
      float dts[4], bxs[4];
      spread_rows(dc[q], dts);
      if (!CARRY) spread_rows(dc[q] * xc[q], bxs);
      static_for<4>([&](auto sc) {
        constexpr int s = decltype(sc)::value, t = 4 * q + s;
        static_for<NPL>([&](auto jc) {
          constexpr int j = decltype(jc)::value, k = (t % PER) * NPL + j;
          da[t][j] = exp2_hw(dts[s] * a2[j]);
          if constexpr (!CARRY)
            hs[t][j] = __builtin_fmaf(da[t][j], t == 0 ? h0[j] : hs[t == 0 ? 0 : t - 1][j],
                                      row_mul<k>(b[t / PER], bxs[s]));
        });
      });
    });
    float* const mine = tbc[CARRY ? 0 : i & 1][CARRY ? 0 : L.wave];
    static_for<4>([&](auto qc) {
      constexpr int q = 3 - decltype(qc)::value;
      float dys[4], dts[4], bxs[4], s1[4], s2[4];
      spread_rows(yc[q], dys);
      if (!CARRY) {
        spread_rows(dc[q], dts);
        spread_rows(dc[q] * xc[q], bxs);
      }
      float v[16];   // products of two steps: [kind][step parity][state], kinds G dt x, dy h
      static_for<4>([&](auto sc) {
        constexpr int s = 3 - decltype(sc)::value, t = 4 * q + s;
        static_for<NPL>([&](auto jc) {
          constexpr int j = decltype(jc)::value, k = (t % PER) * NPL + j;
          float g = u[j];
          row_fmac<k>(g, cc[t / PER], dys[s]);
          u[j] = da[t][j] * g;
          if constexpr (!CARRY) {
            const float qv = u[j] * (t == 0 ? h0[j] : hs[t == 0 ? 0 : t - 1][j]);
            if constexpr (j == 0) {
              s1[s] = row_mul<k>(b[t / PER], g);
              s2[s] = an[j] * qv;
            } else {
              row_fmac<k>(s1[s], b[t / PER], g);
              s2[s] = __builtin_fmaf(an[j], qv, s2[s]);
            }
            acc[j] = __builtin_fmaf(dts[s], qv, acc[j]);
            v[(s & 1) * 4 + j] = g * bxs[s];
            v[8 + (s & 1) * 4 + j] = hs[t][j] * dys[s];
          }
        });
        if constexpr (!CARRY && (s & 1) == 0) {
#pragma unroll
          for (int j = NPL; j < 4; ++j) v[j] = v[4 + j] = v[8 + j] = v[12 + j] = 0.f;
          const float sum = row_sum16(v, L.lane);
          const int ix = row_sum_index(L.lane);
          const int j = ix & 3, kind = ix >> 3, step = t + ((ix >> 2) & 1);
          if (j < NPL) mine[(kind * kSub + step) * NS + L.row * NPL + j] = sum;
        }
      });
      if constexpr (!CARRY) {
        const float r1 = gather_rows(s1), r2 = gather_rows(s2);
        if constexpr (WS == 1) {
          sdx.store(dc[q] * r1, i, q);
          sddt.store(__builtin_fmaf(xc[q], r1, -r2), i, q);
        } else {
          tss[i & 1][L.wave][0][q][L.lane] = r1;
          tss[i & 1][L.wave][1][q][L.lane] = r2;
        }
      }
    });
    if constexpr (!CARRY) {
      __syncthreads();
      if constexpr (WS > 1) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if (q % WS != L.ws) continue;
          float r1 = 0.f, r2 = 0.f;
#pragma unroll
          for (int w = 0; w < WS; ++w) {
            r1 += tss[i & 1][L.wc * WS + w][0][q][L.lane];
            r2 += tss[i & 1][L.wc * WS + w][1][q][L.lane];
          }
          sdx.store(dc[q] * r1, i, q);
          sddt.store(__builtin_fmaf(xc[q], r1, -r2), i, q);
        }
      }
      // the block's sums of dB and dC: over its waves of channels
      const int len = min(kSub, pc.len - i * kSub);
      for (int r = threadIdx.x; r < 2 * kSub * WS * NS; r += 256) {
        const int n = r % (WS * NS), kind = r / (WS * NS) & 1, step = r / (2 * WS * NS);
        if (n >= a.N || step >= len) continue;
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < WC; ++w)
          sum += tbc[i & 1][w * WS + n / NS][(kind * kSub + step) * NS + n % NS];
        part[((size_t)(i * kSub + step) * 2 + kind) * a.N + n] = sum;
      }
    }
  }
  if (CARRY) {
    at.store(a.carry + (size_t)blockIdx.x * slice, u);
    const float s4[4] = {sum_dt, 0.f, 0.f, 0.f};
    const float total = gather_rows(s4);
    if (L.ws == 0 && L.row == 0 && L.act) a.sdt[(size_t)blockIdx.x * a.D + L.d] = total;
    return;
  }
#pragma unroll
  for (int j = 0; j < NPL; ++j) acc[j] = -acc[j];
  at.store(a.part_a + (size_t)blockIdx.x * slice, acc);
  if (pc.j == 0 && a.dh0) at.store(a.dh0 + (size_t)pc.seq * slice, u);
}

// dB, dC (total, N): the blocks' partials in order, rounded to T once.
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

// dAneg (D, N): the pieces' partials. Each wave of a block adds every fourth, then the block its
// four sums: a fixed order.
__global__ void __launch_bounds__(256)
packed_sum_a_kernel(const float* part, float* da, int pieces, int slice) {
  __shared__ float sums[4][64];
  const int w = threadIdx.x >> 6, e = blockIdx.x * 64 + (threadIdx.x & 63);
  float s = 0.f;
  if (e < slice)
    for (int p = w; p < pieces; p += 4) s += part[(size_t)p * slice + e];
  sums[w][threadIdx.x & 63] = s;
  __syncthreads();
  if (w == 0 && e < slice)
    da[e] = (sums[0][threadIdx.x] + sums[1][threadIdx.x]) + (sums[2][threadIdx.x] + sums[3][threadIdx.x]);
}

}  // namespace mhs
