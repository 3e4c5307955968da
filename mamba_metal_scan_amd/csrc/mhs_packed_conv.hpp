// Causal depthwise conv1d + SiLU over packed sequences for gfx950 (see
// mhs_packed.hpp for the pieces):
//   pre_t = bias + sum_{k<K} w_k x_{t-K+1+k},   out_t = pre_t sigmoid(pre_t)
// within each sequence; the K - 1 inputs before its first row come from window
// (nseq, D, K - 1) or are zero, its last K - 1 go to window_out.
//
// HBM-bound stencils: a thread owns V neighbouring channels (8 bytes of a row in the forward, two
// channels in the backward; one where the width, a stride or an address is no multiple of that, or
// the address none of 16) and the rows of a piece, the K - 1 rows before each kept in registers. No
// row needs a test of its sequence: a piece belongs to one.
#pragma once

#include "mhs_packed.hpp"

namespace mhs {

constexpr int kPackedMaxTaps = 8;

struct PackedConvArgs {
  Seqs q;
  const void* x;        // (total, D), rows ld_x apart
  long long ld_x;
  const void* w;        // (D, K) of T, or fp32 (wf32)
  const void* bias;     // (D)
  int wf32;
  const void* window;   // (nseq, D, K - 1) or null
  void* out;            // (total, D)
  void* window_out;     // (nseq, D, K - 1) or null
  int D;
  // backward
  const void* dout;     // (total, D), rows ld_g apart
  long long ld_g;
  const void* dwindow_out;   // (nseq, D, K - 1) or null
  void* dx;             // (total, D)
  void* dwindow;        // (nseq, D, K - 1) or null
  float* part;          // (block rows, K + 1, D): dw, dbias
};

// V neighbouring elements of T (4, 8 or 16 bytes, aligned, or one) as they lie in memory.
template <class T, int V>
struct Chans {
  static constexpr int kWords = V == 1 ? 1 : V * kElem<T> / 4;
  struct alignas(4 * kWords) Words { unsigned u[kWords]; };
  Words r;
  __device__ __forceinline__ void load(const void* p, size_t idx) {
    if constexpr (V == 1) r.u[0] = __float_as_uint(ld_p<T>(p, idx));
    else r = *reinterpret_cast<const Words*>(static_cast<const char*>(p) + idx * kElem<T>);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) r.u[i] = 0;
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (V == 1 || kElem<T> == 4) return __uint_as_float(r.u[i]);
    else return T::to((unsigned short)(r.u[i / 2] >> (16 * (i & 1))));
  }
  __device__ __forceinline__ void get(float (&v)[V]) const {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = get(i);
  }
};
template <class T, int V>
__device__ __forceinline__ void store_chans(void* p, size_t idx, const float (&v)[V]) {
  if constexpr (V == 1) {
    st_p<T>(p, idx, v[0]);
  } else {
    typename Chans<T, V>::Words r;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if constexpr (kElem<T> == 4) r.u[i] = __float_as_uint(v[i]);
      else if (i % 2) r.u[i / 2] |= (unsigned)T::from(v[i]) << 16;
      else r.u[i / 2] = (unsigned)T::from(v[i]);
    }
    *reinterpret_cast<typename Chans<T, V>::Words*>(static_cast<char*>(p) + idx * kElem<T>) = r;
  }
}
// N elements of TW from idx on, which W divides; the address is that of whole W's.
template <class TW, int N, int W>
__device__ __forceinline__ void load_run(float (&v)[N], const void* p, size_t idx) {
  if constexpr (W > 1) {
#pragma unroll
    for (int i = 0; i < N; i += W) {
      Chans<TW, W> c;
      c.load(p, idx + i);
#pragma unroll
      for (int e = 0; e < W; ++e) v[i + e] = c.get(e);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = ld_p<TW>(p, idx + i);
  }
}

template <class T, int K, int V>
struct ConvLane {
  float w[K][V], bias[V];
  template <class TW>
  __device__ __forceinline__ void load(const PackedConvArgs& a, int d) {
    float all[V * K];   // (D, K): a channel's taps are neighbours
    constexpr int W = V < 16 / kElem<TW> ? V : 16 / kElem<TW>;
    load_run<TW, V * K, W>(all, a.w, (size_t)d * K);
    load_run<TW, V, W>(bias, a.bias, d);
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int k = 0; k < K; ++k) w[k][v] = all[v * K + k];
  }
  __device__ __forceinline__ ConvLane(const PackedConvArgs& a, int d) {
    if (a.wf32) load<F32>(a, d);
    else load<T>(a, d);
  }
  // The pre-activation of the step whose K inputs are win[0 .. K - 1].
  __device__ __forceinline__ float pre(const float (&win)[K][V], int v) const {
    float s = bias[v];
#pragma unroll
    for (int k = 0; k < K; ++k) s = __builtin_fmaf(w[k][v], win[k][v], s);
    return s;
  }
};

// The input at row t of a sequence that begins at `begin`: x's, the window's
// before it, or zero.
template <class T, int K, int V>
__device__ __forceinline__ void conv_input(float (&v)[V], const PackedConvArgs& a,
                                           const Piece& pc, int t, int d) {
  if (t >= pc.begin) {
    Chans<T, V> c;
    c.load(a.x, (size_t)t * a.ld_x + d);
    c.get(v);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      v[i] = a.window ? ld_p<T>(a.window, ((size_t)pc.seq * a.D + d + i) * (K - 1) + K - 1 -
                                              (pc.begin - t))
                      : 0.f;
  }
}

// Rows of a piece, and those of them whose loads are in flight together.
constexpr int kConvPiece = 16, kConvBackPiece = 16, kConvBackRows = 4;
// Channels of a thread where the layout allows it. (us of 8192 x 1536 in bf16 | fp32 |
// 32768 x 2048 in bf16. Forward with 16 bytes a thread 17.7 | 22.2 | 55.2, with 8 17.5 | 20.6 |
// 55.6, with 4 16.2 | 22.6 | 60.7. Backward, pieces of 32 rows, with 16 bytes 38.2 | 36.5 | 123.6,
// its registers leaving two waves a SIMD and the rows too few of those, with 8 29.9 | 34.0 | 105.0,
// with 4 27.9 | 34.6 | 97.8; so two channels, and in pieces of 16 rows 25.4 | 36.7 | 97.4.)
template <class T> constexpr int kConvVec = 8 / kElem<T>;
constexpr int kConvBackVec = 2;

// Block (pieces / 4, channels / (64 V)): 64 channel lanes by 4 pieces, so that a wave has one
// piece; all its rows are asked for at once (8192 x 1536 bf16: 17.5 us, 2.9 TB/s;
// 24 us four at a time).
template <class T, int K, int V>
__global__ void __launch_bounds__(256)
packed_conv_fwd_kernel(PackedConvArgs a, int pieces) {
  const int p = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (p >= pieces) return;
  const Piece pc = find_piece(a.q, kConvPiece, p);
  if (pc.seq < 0) return;
  const int d = (blockIdx.y * 64 + (threadIdx.x & 63)) * V;
  if (d >= a.D) return;
  float y[V];
  if (pc.seq == a.q.nseq) {
#pragma unroll
    for (int v = 0; v < V; ++v) y[v] = 0.f;
    for (int i = 0; i < pc.len; ++i) store_chans<T, V>(a.out, (size_t)(pc.t0 + i) * a.D + d, y);
    return;
  }
  Chans<T, V> in[kConvPiece];
#pragma unroll
  for (int i = 0; i < kConvPiece; ++i)   // (rows behind the piece: its last one again)
    if (pc.len > 0) in[i].load(a.x, (size_t)(pc.t0 + min(i, pc.len - 1)) * a.ld_x + d);
  float win[K][V];
#pragma unroll
  for (int k = 0; k < K - 1; ++k) conv_input<T, K, V>(win[k], a, pc, pc.t0 - K + 1 + k, d);
  const ConvLane<T, K, V> L(a, d);
#pragma unroll
  for (int i = 0; i < kConvPiece; ++i) {
    if (i < pc.len) {
      in[i].get(win[K - 1]);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float s = L.pre(win, v);
        y[v] = s * sigmoid_f(s);
#pragma unroll
        for (int k = 0; k < K - 1; ++k) win[k][v] = win[k + 1][v];
      }
      store_chans<T, V>(a.out, (size_t)(pc.t0 + i) * a.D + d, y);
    }
  }
  if (pc.last && a.window_out) {
    // the last K - 1 inputs: those kept, x's and the window's exactly
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int k = 0; k < K - 1; ++k)
        st_p<T>(a.window_out, ((size_t)pc.seq * a.D + d + v) * (K - 1) + k, win[k][v]);
  }
}

// Backward. With s_t = dout_t silu'(pre_t):
//   dx_t = sum_k w_k s_{t+K-1-k},  dw_k = sum_t s_t x_{t-K+1+k},  dbias = sum_t s_t
// and, for the inputs that window_out holds, its gradient. A thread walks the
// rows of its piece and the K - 1 behind it, keeping K of s; a block's four pieces
// are summed in LDS for dw and dbias, the blocks by packed_conv_sum_kernel, always in
// the same order. (8192 x 1536 bf16: 24.5 us, 3.1 TB/s; 32768 x 2048 97 us, 4.1 TB/s: then the
// copy's rate nearly, before that the launch's first loads and the sums at its end.)
template <class T, int K, int V>
__global__ void __launch_bounds__(256)
packed_conv_bwd_kernel(PackedConvArgs a, int pieces) {
  constexpr int U = kConvBackRows;
  __shared__ float sums[4][64 * V];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int p = blockIdx.x * 4 + wave;
  const int d = (blockIdx.y * 64 + lane) * V;
  Piece pc;
  pc.seq = -1;
  if (p < pieces) pc = find_piece(a.q, kConvBackPiece, p);
  float dw[K + 1][V];
#pragma unroll
  for (int k = 0; k <= K; ++k)
#pragma unroll
    for (int v = 0; v < V; ++v) dw[k][v] = 0.f;
  if (pc.seq == a.q.nseq && d < a.D) {
    float z[V];
#pragma unroll
    for (int v = 0; v < V; ++v) z[v] = 0.f;
    for (int i = 0; i < pc.len; ++i) store_chans<T, V>(a.dx, (size_t)(pc.t0 + i) * a.D + d, z);
  } else if (pc.seq >= 0 && d < a.D) {
    const int end = pc.last ? pc.t0 + pc.len
                            : max(__builtin_amdgcn_readfirstlane(cu_at(a.q, pc.seq + 1)),
                                  pc.begin);
    const int rows = pc.len + K - 1;   // of the walk
    Chans<T, V> nx[U], ng[U];
    const auto load = [&](int i0) {   // (0 behind the sequence)
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int t = pc.t0 + i0 + u;
        nx[u].zero();
        ng[u].zero();
        if (i0 + u < rows && t < end) {
          nx[u].load(a.x, (size_t)t * a.ld_x + d);
          ng[u].load(a.dout, (size_t)t * a.ld_g + d);
        }
      }
    };
    load(0);
    float win[K][V], s[K][V];   // inputs t - K + 1 .. t; s of the same rows
#pragma unroll
    for (int k = 0; k < K - 1; ++k) conv_input<T, K, V>(win[k], a, pc, pc.t0 - K + 1 + k, d);
    const ConvLane<T, K, V> L(a, d);
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int v = 0; v < V; ++v) s[k][v] = 0.f;
    // The rows t of the piece, and K - 1 behind it for their s (0 behind the sequence).
    for (int i0 = 0; i0 < rows; i0 += U) {
      Chans<T, V> cx[U], cg[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        cx[u] = nx[u];
        cg[u] = ng[u];
      }
      if (i0 + U < rows) load(i0 + U);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u, t = pc.t0 + i;
        if (i >= rows) continue;
        float o[V];
        cx[u].get(win[K - 1]);
#pragma unroll
        for (int v = 0; v < V; ++v) {
#pragma unroll
          for (int k = 0; k < K - 1; ++k) s[k][v] = s[k + 1][v];
          const float pre = L.pre(win, v), sg = sigmoid_f(pre);
          // (behind the sequence dout counts as 0, whatever pre is)
          const float st = t < end ? cg[u].get(v) * sg * __builtin_fmaf(pre, 1.f - sg, 1.f) : 0.f;
          s[K - 1][v] = st;
          if (i < pc.len) {
#pragma unroll
            for (int k = 0; k < K; ++k) dw[k][v] = __builtin_fmaf(st, win[k][v], dw[k][v]);
            dw[K][v] += st;
          }
          // row t - K + 1: s_{t-K+1+m}, m = 0 .. K - 1, meets w_{K-1-m}
          float acc = 0.f;
#pragma unroll
          for (int m = 0; m < K; ++m) acc = __builtin_fmaf(L.w[K - 1 - m][v], s[m][v], acc);
          o[v] = acc;
#pragma unroll
          for (int k = 0; k < K - 1; ++k) win[k][v] = win[k + 1][v];
        }
        const int r = t - K + 1;   // the row that o is the gradient of
        if (a.dwindow_out && r >= end - (K - 1) && r < end) {
#pragma unroll
          for (int v = 0; v < V; ++v)
            o[v] += ld_p<T>(a.dwindow_out,
                            ((size_t)pc.seq * a.D + d + v) * (K - 1) + r - (end - (K - 1)));
        }
        if (r >= pc.t0) {
          store_chans<T, V>(a.dx, (size_t)r * a.D + d, o);
        } else if (pc.j == 0 && a.dwindow) {   // the window's, rows begin - K + 1 .. begin - 1
#pragma unroll
          for (int v = 0; v < V; ++v)
            st_p<T>(a.dwindow, ((size_t)pc.seq * a.D + d + v) * (K - 1) + r - (pc.begin - (K - 1)),
                    o[v]);
        }
      }
    }
  }
#pragma unroll
  for (int k = 0; k <= K; ++k) {
#pragma unroll
    for (int v = 0; v < V; ++v) sums[wave][lane * V + v] = dw[k][v];
    __syncthreads();
    for (int c = threadIdx.x; c < 64 * V; c += 256) {
      const int dc = blockIdx.y * 64 * V + c;
      if (dc < a.D)
        a.part[((size_t)blockIdx.x * (K + 1) + k) * a.D + dc] =
            (sums[0][c] + sums[1][c]) + (sums[2][c] + sums[3][c]);
    }
    __syncthreads();
  }
}

// dw (D, K), dbias (D): the blocks' partials (n, K + 1, D). A wave's lanes are
// channels; each of a block's 16 waves adds every sixteenth partial, in four sums.
template <class T>
__global__ void __launch_bounds__(1024)
packed_conv_sum_kernel(const float* part, void* dw, void* dbias, int wf32, int n, int K, int D) {
  __shared__ float sums[16][64];
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int d = blockIdx.x * 64 + lane, k = blockIdx.y;
  float t[4] = {0.f, 0.f, 0.f, 0.f};
  if (d < D) {
    for (int p = w; p < n; p += 64) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (p + 16 * j < n) t[j] += part[((size_t)(p + 16 * j) * (K + 1) + k) * D + d];
    }
  }
  sums[w][lane] = (t[0] + t[1]) + (t[2] + t[3]);
  __syncthreads();
  if (w || d >= D) return;
  float s = sums[0][lane];
#pragma unroll
  for (int i = 1; i < 16; ++i) s += sums[i][lane];
  void* to = k < K ? dw : dbias;
  const size_t at = k < K ? (size_t)d * K + k : (size_t)d;
  if (wf32) st_p<F32>(to, at, s);
  else st_p<T>(to, at, s);
}

// ---------------------------------------------------------- tokens by slot
//
// Row r advances entry slots[r] of a pool in place. A row whose slot is below 0
// is padding: its output is 0. A slot at or past the pool, and a slot that an
// earlier row has too, make the row's output NaN; no entry is then touched (the
// earlier row's only by that row).

// 0: an entry to advance, at *at; 1: padding; 2: no such entry, or taken. All threads
// of the block call it, for one row.
__device__ __forceinline__ int slot_of(const void* slots, int slots64, int row, int pool,
                                       long long* at) {
  const auto get = [&](int r) {
    return slots64 ? static_cast<const long long*>(slots)[r]
                   : (long long)static_cast<const int*>(slots)[r];
  };
  if (!slots) {   // row r at entry r
    *at = row;
    return row < pool ? 0 : 2;
  }
  const long long mine = get(row);
  *at = mine;
  int taken = 0;
  for (int r = threadIdx.x; r < row; r += blockDim.x) taken |= get(r) == mine;
  taken = __syncthreads_or(taken);
  return mine < 0 ? 1 : mine >= pool || taken ? 2 : 0;
}

struct ConvStepArgs {
  const void* x;        // (rows, D), rows ld_x apart
  long long ld_x;
  const void* w;        // (D, K)
  const void* bias;     // (D)
  int wf32;
  void* window;         // (pool, D, K - 1)
  const void* slots;    // (rows) or null
  int slots64;
  void* out;            // (rows, D)
  int rows, pool, D;
};

// Block (row, channels), a channel a thread: its taps, its window and two numbers are all there
// is, a few scattered elements each. Bound by launch and latency: 4 x 1536 in fp32 3.0 us, 256 x
// 4096 in bf16 9.1 us (1.8 TB/s), as long as the host takes for the call.
template <class T, int K>
__global__ void __launch_bounds__(256)
conv_step_kernel(ConvStepArgs a) {
  const int r = blockIdx.x;
  long long at;
  const int what = slot_of(a.slots, a.slots64, r, a.pool, &at);
  const int d = blockIdx.y * 256 + threadIdx.x;
  if (d >= a.D) return;
  float o;
  if (what) {
    o = what == 1 ? 0.f : __builtin_nanf("");
  } else {
    const size_t base = ((size_t)at * a.D + d) * (K - 1);
    float win[K];
#pragma unroll
    for (int k = 0; k < K - 1; ++k) win[k] = ld_p<T>(a.window, base + k);
    win[K - 1] = ld_p<T>(a.x, (size_t)r * a.ld_x + d);
    float s = a.wf32 ? ld_p<F32>(a.bias, d) : ld_p<T>(a.bias, d);
#pragma unroll
    for (int k = 0; k < K; ++k)
      s = __builtin_fmaf(a.wf32 ? ld_p<F32>(a.w, (size_t)d * K + k)
                                : ld_p<T>(a.w, (size_t)d * K + k), win[k], s);
    o = s * sigmoid_f(s);
#pragma unroll
    for (int k = 0; k < K - 1; ++k) st_p<T>(a.window, base + k, win[k + 1]);
  }
  st_p<T>(a.out, (size_t)r * a.D + d, o);
}

struct StateStepArgs {
  float* h;             // (pool, D, N)
  const void *x, *dt, *B, *C;   // (rows, D), (rows, N), rows ld_* apart
  long long ld_x, ld_dt, ld_b, ld_c;
  const float* aneg;    // (D, N)
  const void* slots;
  int slots64;
  void* y;              // (rows, D)
  int rows, pool, D, N;
};

// h <- exp(-dt Aneg) h + dt x B, y = sum_n C h. Block (row, channels). LPC lanes
// share a channel, V neighbouring states each (V 4: whole float4s; V 1: any N); y is summed over
// them by DPP. Memory-bound: h is read and written once (256 x 4096 x 16 in bf16, 141 MB:
// 34 us, 4.1 TB/s; 27 us where it is cached; 4 x 1536 x 16 in fp32 3.3 us, latency).
template <class T, int V, int LPC>
__global__ void __launch_bounds__(256)
state_step_kernel(StateStepArgs a) {
  const int r = blockIdx.x;
  long long at;
  const int what = slot_of(a.slots, a.slots64, r, a.pool, &at);
  const int d = blockIdx.y * (256 / LPC) + threadIdx.x / LPC, q = threadIdx.x % LPC;
  const bool act = d < a.D;
  float part = 0.f;
  if (act && !what) {
    const float dt = ld_p<T>(a.dt, (size_t)r * a.ld_dt + d);
    const float bx = dt * ld_p<T>(a.x, (size_t)r * a.ld_x + d);
    const float a2 = -dt * kLog2e;
    float* hp = a.h + ((size_t)at * a.D + d) * a.N;
    const float* ap = a.aneg + (size_t)d * a.N;
    for (int n = q * V; n < a.N; n += LPC * V) {
      float hv[V], av[V];
      load_vec<V>(hv, hp + n);
      load_vec<V>(av, ap + n);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        hv[j] = __builtin_fmaf(exp2_hw(a2 * av[j]), hv[j],
                               ld_p<T>(a.B, (size_t)r * a.ld_b + n + j) * bx);
        part = __builtin_fmaf(ld_p<T>(a.C, (size_t)r * a.ld_c + n + j), hv[j], part);
      }
      store_vec<V>(hp + n, hv);
    }
  }
  part = group_sum<LPC>(part);
  if (act && q == 0)
    st_p<T>(a.y, (size_t)r * a.D + d, what == 0 ? part : what == 1 ? 0.f : __builtin_nanf(""));
}

}  // namespace mhs
