// Matrix products of 16-bit operands (bf16, fp16) on gfx950's matrix cores:
//   acc(m, n) = sum_k A(m, k) B(n, k),  fp32 sums,
// a BM x BN tile at a time per block, in 16 x 16 fragments (MFMAs 32 deep); what
// becomes of a tile is up to the kernel's epilogue (mhs_head.hpp).
//
// An operand is K-major ((rows, K), k contiguous) or row-major ((K, rows)); both
// stage a k tile (64 deep) by 16-byte global loads that write LDS directly, and
// differ in how a wave then reads its fragments: K-major with 16-byte LDS
// reads, row-major with the transposing 8-byte reads (within 16 lanes, lane i
// gives the address of row i / 4, columns 4 (i % 4) .. + 3 and receives column
// i of those four rows).
//
// Two k tiles lie in LDS. A wave reads the fragments of one step (32 deep) while
// it multiplies those of the step before, from two sets of registers; at a k
// tile's last step one wait and barrier publish the next tile and free this one,
// which the loads of the tile after the next then refill. 256 x 256 tiles of 8
// waves, one block per CU: a wave's step is 12 fragments read for 32 MFMAs. Bound by
// the matrix cores at the power limit, 1.5 to 2.0 GHz of 2.4 (a library product of
// 8192^3 reaches 1341 TFLOP/s here, one of 8192 x 16384 x 4096 1618); rates stand at
// the kernels. (TFLOP/s at 8192 x 4096 x 16384, with the sums of exponentials and for
// W's gradient: 1476 and 1334; with 32 x 32 fragments 1358 for the first; 256 x 128
// tiles, two blocks per CU and 32 deep, 1148 for the second.)
#pragma once

#include "mhs_common.hpp"
#include "mhs_gemm.hpp"

namespace mhs {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

// Element types: tags with the MFMA and the conversions.
struct Bf16 {
  static __device__ __forceinline__ f32x4 mfma(s16x8 a, s16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ unsigned short from(float v) {
    return __builtin_bit_cast(unsigned short, (__bf16)v);
  }
  static __device__ __forceinline__ float to(unsigned short u) {
    return __uint_as_float((unsigned)u << 16);
  }
};
struct Fp16 {
  static __device__ __forceinline__ f32x4 mfma(s16x8 a, s16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ unsigned short from(float v) {
    return __builtin_bit_cast(unsigned short, (_Float16)v);
  }
  static __device__ __forceinline__ float to(unsigned short u) {
    return (float)__builtin_bit_cast(_Float16, u);
  }
};

struct MmArgs {
  const void* A;        // K-major: (M, K) rows lda apart; else (K, M) rows lda apart
  const void* B;        // K-major: (N, K) rows ldb apart; else (K, N) rows ldb apart
  long long lda, ldb;   // multiples of 8; both operands 16-byte aligned
  int M, N, K;          // a K-major operand's K, a row-major one's rows: multiples of 8
  int kt_per_split;     // k tiles per split (blockIdx.y)
  int grid_m, grid_n;
  int group_m;          // tiles of a group share the operands' tiles in L2 (see mm_tile)
};

// The resource of a direct load from p on (offsets below kOOB).
__device__ __forceinline__ i32x4 mm_resource(const void* p) {
  const unsigned long long a = reinterpret_cast<unsigned long long>(p);
  return i32x4{__builtin_amdgcn_readfirstlane((int)(unsigned)a),
               __builtin_amdgcn_readfirstlane((int)(unsigned)(a >> 32)), (int)(kOOB - 1u),
               0x00020000};
}

// 64 lanes x 16 bytes from memory straight into LDS at `lds` + 16 lane; lanes at
// or past the resource's end write zeros. Not tracked by the compiler: the
// kernel waits for it with mm_wait, and no register is written.
__device__ __forceinline__ void mm_load_lds(i32x4 rsrc, unsigned voff, unsigned lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(lds), "v"(voff), "s"(rsrc)
               : "m0");
}

// The wave's LDS reads done, all but its last N direct loads done, then the
// block's barrier.
template <int N>
__device__ __forceinline__ void mm_wait() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(N) : "memory");
}

// The row of the tile that a transposing epilogue's LDS row x holds: within 64
// rows (4 fragments i of 16 rows x % 16) the first halves of the fragments follow
// each other, then the second halves. After the epilogue has exchanged fragments
// and groups of 16 lanes, a lane then holds 8 neighbours, and the 4 groups 32.
__device__ __forceinline__ constexpr int mm_perm(int x) {
  return (x & ~63) + (x & 8) * 4 + ((x >> 4) & 3) * 8 + (x & 7);
}

constexpr int kMmK = 64;        // k's of a k tile
constexpr int kMmStages = 2;    // k tiles in LDS
// What a stream's tiles have beside their k tiles (mm_stream's side) lies in as many
// slots, a tile's number modulo them. The loads run kMmStages k tiles ahead: of tiles
// of a single k tile as many whole tiles, whose sides come in before the epilogue of
// the tile at hand has read its own.
constexpr int kMmSlots = kMmStages + 1;

// One operand of a block of WAVES waves: R rows from r0 of `rows`. PERM: its rows
// lie in LDS in mm_perm's order (K-major).
template <int R, bool KMAJOR, int WAVES, bool PERM = false>
struct MmOperand {
  static constexpr int kBytes = R * kMmK * 2;                // of a k tile
  static constexpr int kLoads = kBytes / 1024 / WAVES;     // direct loads per wave and k tile
  static constexpr int kLanes = (KMAJOR ? kMmK : R) / 8;     // lanes per row (K-major) or k row
  static_assert(kLoads * 1024 * WAVES == kBytes, "whole loads");
  unsigned voff[kLoads];                       // byte offset of load j at a k tile, or kOOB
  int kpos[kLoads];                            // the k it starts at within the tile
  const char* base;                            // the block's rows at the next k tile to load
  long long step;                              // bytes per k tile
  unsigned frag;                               // byte offset of the lane's first fragment

  // Chunk c (16 bytes) of row r (K-major) or k row r lies at place c ^ swz(r).
  // K-major: the 16 lanes of a pass of a 16-byte read, lanes 0-3, 12-15 and 20-27
  // (rows of 128 bytes, the last eight a chunk further) or their like, then hit all
  // 64 banks, and so do 16 neighbours; row-major: the k rows that one pass of the
  // transposing reads meets (4 in a row and those 8 further) do.
  // SQ_LDS_BANK_CONFLICT is 0.
  static __device__ __forceinline__ constexpr int swz(int r) {
    return KMAJOR ? (r >> 1) & 7 : ((r & 3) << 2) ^ ((r >> 3) & 1) << 1;
  }

  // wrow: the wave's first row within the tile.
  __device__ __forceinline__ MmOperand(const void* p, long long ld, int r0, int rows, int k_first,
                                       int wave, int lane, int wrow) {
    place(p, ld, r0, rows, k_first, wave, lane);
    if constexpr (KMAJOR) {
      step = kMmK * 2;
      frag = (wrow + (lane & 15)) * (2 * kMmK) + ((lane >> 4 ^ swz(lane & 15)) << 4);
    } else {
      step = ld * (2 * kMmK);
      // Fragment element (row, k) of a lane: row lane % 16, k 8 (lane / 16) + 0..7;
      // the transposing read's own address: k row 8 (lane / 16) + (lane % 16) / 4
      // (+ 4 for its second half), 4 rows from 4 (lane % 4).
      const int k = 8 * (lane >> 4) + ((lane & 15) >> 2);
      const int row = wrow + 4 * (lane & 3);
      frag = k * (2 * R) + ((2 * row) ^ (swz(k) << 4));
    }
  }
  // The loads at rows r0 .., k's k_first ...
  __device__ __forceinline__ void place(const void* p, long long ld, int r0, int rows, int k_first,
                                        int wave, int lane) {
    const int first = wave * kLoads * (64 / kLanes) + lane / kLanes;   // (k) row of load 0
    base = static_cast<const char*>(p) +
           (KMAJOR ? (long long)r0 * ld + k_first : (long long)k_first * ld + r0) * 2;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int row = first + j * (64 / kLanes);   // (row-major: k)
      const int c = (lane % kLanes) ^ swz(row);
      const int at = PERM ? mm_perm(row) : row;
      voff[j] = (KMAJOR ? r0 + at : r0 + 8 * c) < rows
                    ? 2u * ((unsigned)at * (unsigned)ld + 8u * c) : kOOB;
      kpos[j] = KMAJOR ? 8 * c : row;
    }
  }
  // The resource over the next k tile to load, and on to the one after it.
  __device__ __forceinline__ i32x4 next() {
    const i32x4 r = mm_resource(base);
    base += step;
    return r;
  }
  // Load j of that tile (`left` k's remain from its start) into LDS at byte
  // address `lds`, the operand's buffer.
  __device__ __forceinline__ void load(i32x4 r, int j, unsigned lds, int left, int wave) const {
    mm_load_lds(r, kpos[j] < left ? voff[j] : kOOB, lds + (wave * kLoads + j) * 1024);
  }
  // Fragment f (16 rows, 32 deep) of step kk, from the operand's buffer.
  __device__ __forceinline__ s16x8 read(const char* buf, int f, int kk) const {
    if constexpr (KMAJOR) {
      return *reinterpret_cast<const s16x8*>(buf + f * (32 * kMmK) + (frag ^ (kk * 64)));
    } else {
      typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
      // (16 rows are 32 bytes, bits that the swizzle flips and wrow leaves 0 where
      // there is more than one fragment; a step's k rows are 0 mod 16)
      const char* p = buf + kk * (64 * R) + (frag ^ (f * 32));
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 4 * 2 * R));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
};

// Tile `index` of grid_m x grid_n. Blocks go round the 8 XCDs: each takes a
// contiguous run of tiles, so that the rows of A and B it shares stay in its own
// L2; a run goes through groups of group_m tiles in m, n after n.
__device__ __forceinline__ void mm_tile(const MmArgs& g, int index, int& tm, int& tn) {
  const int tiles = g.grid_m * g.grid_n;
  const int xcd = index & 7, per = tiles >> 3, rem = tiles & 7;
  const int t = xcd * per + min(xcd, rem) + (index >> 3);
  const int in_group = g.group_m * g.grid_n;
  const int first = t / in_group * g.group_m;
  const int size = min(g.group_m, g.grid_m - first);
  const int i = t % in_group;
  tm = first + i % size;
  tn = i / size;
}

// A block's shape: BM x BN tile, WM x WN waves of FM x FN fragments.
template <int BM_, int BN_, int WM_, int WN_>
struct MmShape {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;
  static constexpr int kWaves = WM * WN, kThreads = 64 * kWaves;
  static constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
  static constexpr int kLds = kMmStages * (BM + BN) * kMmK * 2;
  // A wave's place in the tile. Waves w and w + 4, which share a SIMD, lie half a
  // tile apart in m, so that in a tile half past the end there each SIMD has one
  // wave at work (640 x 8192 x 16384, its third tile of 256 rows a half one: 184 us,
  // against 196 with two of the half's waves to a SIMD).
  static __device__ __forceinline__ int wave_m(int wave) { return wave / WN; }
  static __device__ __forceinline__ int wave_n(int wave) { return wave % WN; }
};

// acc = the tile's sums over k's k_first .. k_first + k_len - 1. A fragment's
// element e of lane l: row 4 (l / 16) + e, column l % 16. Ends on a barrier, the LDS
// free.
template <class T, class S, bool AK, bool BK>
__device__ __forceinline__ void mm_products(f32x4 (&acc)[S::FM][S::FN], const MmArgs& g, int m0,
                                            int n0, int k_first, int k_len, char* lds) {
  constexpr int FM = S::FM, FN = S::FN, ST = kMmStages, PH = kMmK / 32;
  static_assert(ST == 2 && PH % 2 == 0, "the register sets alternate over whole k tiles");
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  typedef MmOperand<S::BM, AK, S::kWaves> OA;
  typedef MmOperand<S::BN, BK, S::kWaves> OB;
  constexpr int LA = OA::kLoads, LB = OB::kLoads, L = LA + LB;
  constexpr int TA = OA::kBytes, BUF = TA + OB::kBytes;
  OA a(g.A, g.lda, m0, g.M, k_first, wave, lane, S::wave_m(wave) * (FM * 16));
  OB b(g.B, g.ldb, n0, g.N, k_first, wave, lane, S::wave_n(wave) * (FN * 16));
  const unsigned at = (unsigned)(unsigned long long)(__attribute__((address_space(3))) char*)lds;
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int nk = (k_len + kMmK - 1) / kMmK;
#pragma unroll
  for (int s = 0; s < ST; ++s) {
    const i32x4 ra = a.next(), rb = b.next();
#pragma unroll
    for (int j = 0; j < LA; ++j) a.load(ra, j, at + s * BUF, k_len - s * kMmK, wave);
#pragma unroll
    for (int j = 0; j < LB; ++j) b.load(rb, j, at + s * BUF + TA, k_len - s * kMmK, wave);
  }
  mm_wait<(ST - 1) * L>();
  if (m0 + S::wave_m(wave) * (FM * 16) >= g.M || n0 + S::wave_n(wave) * (FN * 16) >= g.N) {
    // Nothing of this wave's is within the product: its share of the loads alone.
    for (int kt = 0, cur = 0; kt < nk; ++kt, cur ^= 1) {
      mm_wait<0>();
      const i32x4 ra = a.next(), rb = b.next();
      const int left = k_len - (kt + ST) * kMmK;
#pragma unroll
      for (int j = 0; j < LA; ++j) a.load(ra, j, at + cur * BUF, left, wave);
#pragma unroll
      for (int j = 0; j < LB; ++j) b.load(rb, j, at + cur * BUF + TA, left, wave);
    }
    mm_wait<0>();
    return;
  }
  s16x8 fa[2][FM], fb[2][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i) fa[0][i] = a.read(lds, i, 0);
#pragma unroll
  for (int j = 0; j < FN; ++j) fb[0][j] = b.read(lds + TA, j, 0);
  // cur: the buffer of the k tile.
  for (int kt = 0, cur = 0; kt < nk; ++kt, cur ^= 1) {
    const int left = k_len - (kt + ST) * kMmK;
    i32x4 ra, rb;
#pragma unroll
    for (int p = 0; p < PH; ++p) {
      if (p == PH - 1) {
        // The next tile has landed, and every wave holds its last fragments of
        // this one: its buffer takes the tile ST further.
        mm_wait<0>();
        ra = a.next();
        rb = b.next();
      }
      const char* nb = lds + (p == PH - 1 ? cur ^ 1 : cur) * BUF;
      // A row of fragments' products at a time, with each its share of the next
      // step's fragments and of the direct loads: the wave issues them while the
      // matrix core works.
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        constexpr int F = FM + FN;
#pragma unroll
        for (int f = i * F / FM; f < (i + 1) * F / FM; ++f) {
          if (f < FM) fa[1 - p % 2][f] = a.read(nb, f, (p + 1) % PH);
          else fb[1 - p % 2][f - FM] = b.read(nb + TA, f - FM, (p + 1) % PH);
        }
        if (p == PH - 1) {
#pragma unroll
          for (int l = i * L / FM; l < (i + 1) * L / FM; ++l) {
            if (l < LA) a.load(ra, l, at + cur * BUF, left, wave);
            else b.load(rb, l - LA, at + cur * BUF + TA, left, wave);
          }
        }
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = T::mfma(fa[p % 2][i], fb[p % 2][j], acc[i][j]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
  mm_wait<0>();
}

// v, without the compiler's knowledge of it: what is computed from it within a
// loop is computed there, not kept in registers across the loop.
__device__ __forceinline__ int mm_opaque(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

// The tiles blockIdx.x, + gridDim.x, ... of a product of two K-major operands as
// one stream of k tiles: the direct loads run on into the next tile while this
// one's last k tiles are multiplied and while epi(acc, m0, n0) works on its sums
// (without the stages' LDS), so that only the first tile waits for memory. side(n0,
// slot) issues direct loads into a slot when a tile's own loads begin, epi(acc, m0, n0,
// slot) reads it: between a slot's last reads and its next loads lies a k tile's
// barrier, from one tile to the third after it at least one (kMmSlots). A's rows
// lie in mm_perm's order: a fragment's element e of lane l in fragment i is row
// 64 (i / 4) + 32 (l / 32) + 8 (i % 4) + 4 (l / 16 % 2) + e of the wave's.
template <class T, class S, class Side, class Epi>
__device__ __forceinline__ void mm_stream(const MmArgs& g, char* lds, const Side& side,
                                          const Epi& epi) {
  constexpr int FM = S::FM, FN = S::FN, ST = kMmStages, PH = kMmK / 32;
  static_assert(ST == 2, "every k tile waits for all loads before it: side's too");
  static_assert(kMmSlots > ST, "a slot for every tile that loads run ahead, and the one at hand");
  static_assert(PH % 2 == 0 && FM % 4 == 0, "the shape streams");
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  typedef MmOperand<S::BM, true, S::kWaves, true> OA;
  typedef MmOperand<S::BN, true, S::kWaves> OB;
  constexpr int LA = OA::kLoads, LB = OB::kLoads, L = LA + LB;
  constexpr int TA = OA::kBytes, BUF = TA + OB::kBytes;
  const unsigned at = (unsigned)(unsigned long long)(__attribute__((address_space(3))) char*)lds;
  const int tiles = g.grid_m * g.grid_n, nk = (g.K + kMmK - 1) / kMmK;
  // Where the loads are: k tile load_kt of tile load_tile.
  int load_tile = blockIdx.x, load_kt = 0, load_slot = 0, tm, tn;
  mm_tile(g, load_tile, tm, tn);
  OA a(g.A, g.lda, tm * S::BM, g.M, 0, wave, lane, S::wave_m(wave) * (FM * 16));
  OB b(g.B, g.ldb, tn * S::BN, g.N, 0, wave, lane, S::wave_n(wave) * (FN * 16));
  side(tn * S::BN, 0);
  // The resources of the next k tile to load, and the k's from its start.
  auto next = [&](i32x4& ra, i32x4& rb) {
    if (load_kt == nk) {
      load_kt = 0;
      load_tile += gridDim.x;
      load_slot = load_slot == kMmSlots - 1 ? 0 : load_slot + 1;
      if (load_tile < tiles) {
        mm_tile(g, load_tile, tm, tn);
        const int l = mm_opaque(lane);
        a.place(g.A, g.lda, tm * S::BM, g.M, 0, wave, l);
        b.place(g.B, g.ldb, tn * S::BN, g.N, 0, wave, l);
        side(tn * S::BN, load_slot);
      }
    }
    ra = a.next();
    rb = b.next();
    return load_tile < tiles ? g.K - load_kt++ * kMmK : 0;
  };
#pragma unroll
  for (int s = 0; s < ST; ++s) {
    i32x4 ra, rb;
    const int left = next(ra, rb);
#pragma unroll
    for (int j = 0; j < LA; ++j) a.load(ra, j, at + s * BUF, left, wave);
#pragma unroll
    for (int j = 0; j < LB; ++j) b.load(rb, j, at + s * BUF + TA, left, wave);
  }
  mm_wait<(ST - 1) * L>();
  s16x8 fa[2][FM], fb[2][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i) fa[0][i] = a.read(lds, i, 0);
#pragma unroll
  for (int j = 0; j < FN; ++j) fb[0][j] = b.read(lds + TA, j, 0);
  int cur = 0, slot = 0;   // the buffer of the k tile; the tile's slot
  for (int tile = blockIdx.x; tile < tiles;
       tile += gridDim.x, slot = slot == kMmSlots - 1 ? 0 : slot + 1) {
    f32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int kt = 0; kt < nk; ++kt) {
      const int next_buf = cur ^ 1;
      i32x4 ra, rb;
      int left = 0;
#pragma unroll
      for (int p = 0; p < PH; ++p) {
        if (p == PH - 1) {   // (as in mm_products)
          mm_wait<0>();
          left = next(ra, rb);
        }
        const char* nb = lds + (p == PH - 1 ? next_buf : cur) * BUF;
#pragma unroll
        for (int i = 0; i < FM; ++i) {
          constexpr int F = FM + FN;
#pragma unroll
          for (int f = i * F / FM; f < (i + 1) * F / FM; ++f) {
            if (f < FM) fa[1 - p % 2][f] = a.read(nb, f, (p + 1) % PH);
            else fb[1 - p % 2][f - FM] = b.read(nb + TA, f - FM, (p + 1) % PH);
          }
          if (p == PH - 1) {
#pragma unroll
            for (int l = i * L / FM; l < (i + 1) * L / FM; ++l) {
              if (l < LA) a.load(ra, l, at + cur * BUF, left, wave);
              else b.load(rb, l - LA, at + cur * BUF + TA, left, wave);
            }
          }
#pragma unroll
          for (int j = 0; j < FN; ++j)
            acc[i][j] = T::mfma(fa[p % 2][i], fb[p % 2][j], acc[i][j]);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      cur = next_buf;
    }
    int em, en;
    mm_tile(g, tile, em, en);
    epi(acc, em * S::BM, en * S::BN, slot);
  }
  mm_wait<0>();   // (no load may outlive the block)
}

// LDS written before by any wave of the block is visible after (without a wait
// for the direct loads, as __syncthreads would have).
__device__ __forceinline__ void mm_lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory");
}

}  // namespace mhs
