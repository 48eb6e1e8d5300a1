// The tile loop shared by the linear-Categorical kernels (csrc/class_logits.hip)
// and the 8-bit products (csrc/int8_linear.hip): one workgroup of four waves
// accumulates a BM x BN block of C[m, n] = sum_k A[m, k] B[n, k] on the matrix
// cores, with operands of 128 bytes of k per step.
//
// Both operands travel global -> LDS by DMA (buffer_load ... lds, 16 bytes a
// lane).  The buffer descriptor carries the bounds: rows past the operand's end
// and, through the lane's own offset, columns past its k range arrive as zeros,
// so odd sizes need no other code.  An operand is stored in one of two ways:
//   k-contiguous ("kc"): row m holds its k's side by side.  LDS row m is 128
//     bytes; its eight 16-byte chunks are rotated by XOR with (m >> 1) & 7, so
//     that the 16 lanes that a ds_read_b128 serves at a time (rows {0-3, 12-15,
//     20-27} / {4-11, 16-19, 28-31} of a 32-row block) touch all 64 banks once.
//   k-major ("km"): row k holds the m's side by side.  The LDS row k is BM (BN)
//     elements.  2-byte elements: the fragment is taken by the transposing
//     read ds_read_b64_tr_b16, 4 k's x 16 m's per group of 16 lanes; chunks are
//     XORed with 4 (k & 3) so that the four k rows of a read sit in different
//     quarters of the banks.  4-byte elements: four ds_read_b32, the lane
//     halves' rows (4 apart) in different halves of the banks by XOR with 8.  The gradient products contract over rows this
//     way and no operand is ever transposed in memory.
// A step's four MFMA k-slices (kk) are software-pipelined over two register
// sets; the one barrier of a step sits in front of its LAST slice, whose
// operands are in registers by then.  Every slice is written in issue order: the
// next slice's LDS reads in front of its first MFMAs, and the DMA of the step
// NBUF ahead -- into the buffer that the barrier has just freed -- one piece at a
// time between the MFMAs of the three slices behind the barrier (issued in one
// burst, four waves' 64 pieces hold the memory pipe for ~1000 clocks and every
// wave's in-order issue behind it).  Steps past the last are issued with an empty
// descriptor (zeros, no memory traffic), so that the waits count the same
// everywhere.  32768 x 4096 x 4096 bf16, 256 x 256 tiles: burst 1090 TFLOP/s, even
// over all four slices 1130, over three with the MFMA waves' priority raised
// 1385; eight waves of 128 x 64 each 1345, 64-byte steps in four buffers 1280,
// two workgroups of 128 x 128 a CU 1105.
//
// `terms`: float32 operands may come as three bfloat16 planes of x / 2^e: the nearest
// one, the nearest to what it leaves, and the rest, 24 bits in all.  A product is the six
// of nine plane products that are not below 2^-25 of it.  2^e is an operand's own, its
// largest magnitude near 2^48, so that a product of 2^28 terms stays inside float32 and
// all 24 bits of what is 2^-158 of the largest are still there.  The loop runs over the
// pairs, smallest first, into the same float32 accumulators.  One pair otherwise.
#pragma once
#include <type_traits>
#include <utility>

#include "common.h"

namespace zshmc {

typedef unsigned int tu4 __attribute__((ext_vector_type(4)));
typedef unsigned int tu2 __attribute__((ext_vector_type(2)));
typedef int ti4 __attribute__((ext_vector_type(4)));
typedef short ts4 __attribute__((ext_vector_type(4)));
typedef float tf4 __attribute__((ext_vector_type(4)));
typedef float tf16 __attribute__((ext_vector_type(16)));
typedef int ti16 __attribute__((ext_vector_type(16)));
typedef __bf16 tb8 __attribute__((ext_vector_type(8)));
#define ZS_TLDS __attribute__((address_space(3)))

// One operand as it lies in memory: rows x row_bytes, `pitch` bytes apart
// (both multiples of 16, base too), `plane` bytes from one plane to the next.
struct TileOperand {
  const unsigned char* base;
  int64_t pitch, plane;
  int64_t rows, row_bytes;
};

// plane pairs, two bits each, smallest products first (one term: pair 0 0):
// 1 1, 2 0, 0 2, 1 0, 0 1, 0 0
constexpr int kPlanes = 3, kTermsSplit = 6;
constexpr uint32_t kTermsA = 1u | 2u << 2 | 0u << 4 | 1u << 6 | 0u << 8 | 0u << 10;
constexpr uint32_t kTermsB = 1u | 0u << 2 | 2u << 4 | 0u << 6 | 1u << 8 | 0u << 10;

// two float32 -> bfloat16 (to nearest even) in one register
__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
  typedef __bf16 pair __attribute__((ext_vector_type(2)));
  const pair p = {(__bf16)a, (__bf16)b};
  return __builtin_bit_cast(uint32_t, p);
}

// what bfloat16 leaves of x (nothing of an infinity)
__device__ __forceinline__ float bf16_rest(float x) {
  const float h = (float)(__bf16)x;
  return fabsf(h) == __builtin_inff() ? 0.f : x - h;
}
// the planes of two values
__device__ __forceinline__ void bf16_planes(float a, float b, uint32_t (&plane)[kPlanes]) {
#pragma unroll
  for (int k = 0; k < kPlanes; ++k) {
    plane[k] = bf16_pair(a, b);
    a = bf16_rest(a);
    b = bf16_rest(b);
  }
}

// kBytes: of an element of a k-major operand
struct MmaBf16 {
  typedef tf16 Acc;
  static constexpr int kBytes = 2;
  static __device__ __forceinline__ Acc mma(const tu4& a, const tu4& b, const Acc& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(
        __builtin_bit_cast(tb8, a), __builtin_bit_cast(tb8, b), c, 0, 0, 0);
  }
};
// float32 as it is: a lane's four elements of a chunk one MFMA each (k is a dummy
// index; both operands hold the same four)
struct MmaF32 {
  typedef tf16 Acc;
  static constexpr int kBytes = 4;
  static __device__ __forceinline__ Acc mma(const tu4& a, const tu4& b, Acc c) {
    const tf4 x = __builtin_bit_cast(tf4, a), y = __builtin_bit_cast(tf4, b);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[e], y[e], c, 0, 0, 0);
    return c;
  }
};
struct MmaI8 {
  typedef ti16 Acc;
  static constexpr int kBytes = 1;
  static __device__ __forceinline__ Acc mma(const tu4& a, const tu4& b, const Acc& c) {
    return __builtin_amdgcn_mfma_i32_32x32x32_i8(
        __builtin_bit_cast(ti4, a), __builtin_bit_cast(ti4, b), c, 0, 0, 0);
  }
};

// 16 bytes of a row that may start anywhere (global memory takes such accesses
// at its elements' alignment)
typedef unsigned int tu4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned int tu2_any __attribute__((ext_vector_type(2), aligned(2)));

// 16 bytes a lane, global -> LDS at lds + 16 * lane
__device__ __forceinline__ void tile_dma16(const tu4& srd, uint32_t voff, uint32_t lds) {
  asm volatile(
      "s_mov_b32 m0, %2\n\t"
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %0, %1, 0 offen lds"
      :
      : "v"(voff), "s"(srd), "s"(lds)
      : "memory");
}
template <int N>
__device__ __forceinline__ void tile_wait_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}
template <typename F, int... I>
__device__ __forceinline__ void tile_for_impl(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
// a value that is the same in every lane, in scalar registers
__device__ __forceinline__ uint64_t tile_uniform(uint64_t v) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
  return (uint64_t)hi << 32 | lo;
}
// f(0), ..., f(N - 1) with the index a constant
template <int N, typename F>
__device__ __forceinline__ void tile_for(F&& f) {
  tile_for_impl(f, std::make_integer_sequence<int, N>{});
}

// WGM x WGN waves (four), each WM x WN blocks of 32 x 32
template <typename MMA_, int WGM_, int WGN_, int WM_, int WN_, bool A_KM_, bool B_KM_>
struct TileCfg {
  typedef MMA_ MMA;
  static constexpr int WGM = WGM_, WGN = WGN_, WM = WM_, WN = WN_;
  static constexpr bool A_KM = A_KM_, B_KM = B_KM_;
  static constexpr int BM = WGM * WM * 32, BN = WGN * WN * 32;
  static constexpr int kLds = (3 * BM + 2 * BN) * 128;
  static_assert(WGM * WGN == 4, "four waves");
  static_assert(!A_KM || BM == 128 || BM == 256, "whole rows per DMA piece");
  static_assert(!B_KM || BN == 128 || BN == 256, "whole rows per DMA piece");
};

// One operand's side of a step: its DMA lane offsets and its LDS fragments.
// ROWS: BM or BN; OFF: its place in a stage; NB: 32-blocks of the wave.
template <bool KM, int ROWS, int OFF, int NB, int ES>
struct TileSide {
  static constexpr int kPieces = ROWS / 8 / 4;     // 1 KB pieces per wave
  static constexpr int kStepRows = 128 / ES;       // km: rows of a step
  uint32_t voff[kPieces];
  uint32_t chunk16;          // kc: the lane's chunk offset within 128 bytes
  uint32_t frag[KM ? NB : 4];
  tu4 srd;                   // the step that dma() fetches
  // The step after it: where it starts, the bytes from there to the end of what
  // the tile may touch, the bytes of k left in a row (kc), how many steps have
  // been aimed at and how many of them in this plane, and the buffer it goes to
  uint64_t ptr;
  int64_t remain, step_bytes;
  int left, issued, ik;
  uint32_t planes, buf;
  // ... and what a new plane starts from
  uint64_t ptr0;
  int64_t remain0, plane;

  // row0: first m (n) of the tile; k0: first step
  __device__ __forceinline__ void init(const TileOperand& o, int64_t row0, int k0,
                                       int lane, int wave, int blk0, uint32_t planes_) {
    const int64_t pitch = o.pitch;
    int64_t at, end;           // of the first step; of the tile's rows
    if constexpr (!KM) {
      const int sub = lane >> 3;
      const int f = (4 * (wave & 1) + (sub >> 1)) & 7;
      chunk16 = (uint32_t)(((lane & 7) ^ f) * 16);
#pragma unroll
      for (int j = 0; j < kPieces; ++j)
        voff[j] = (uint32_t)((8 * (wave + 4 * j) + sub) * pitch) + chunk16;
      at = row0 * pitch + (int64_t)k0 * 128;
      end = ((o.rows - row0 < ROWS ? o.rows : row0 + ROWS) - 1) * pitch + o.row_bytes;
      left = (int)(o.row_bytes - (int64_t)k0 * 128);
      step_bytes = 128;
      const uint32_t r = OFF + (blk0 * 32 + (lane & 31)) * 128;
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
        frag[kk] = r + (uint32_t)(((2 * kk + (lane >> 5)) ^ ((lane >> 1) & 7)) * 16);
    } else {
      constexpr int CR = ROWS * ES / 16;           // chunks per LDS row
      constexpr int RP = 64 / CR;                  // rows per piece
      chunk16 = 0;
#pragma unroll
      for (int j = 0; j < kPieces; ++j) {
        const int row = RP * (wave + 4 * j) + lane / CR;
        const int swap = ES == 2 ? 4 * (row & 3) : 8 * ((row >> 2) & 1);
        voff[j] = (uint32_t)(row * pitch) + (uint32_t)((lane % CR) ^ swap) * 16;
      }
      at = (int64_t)k0 * kStepRows * pitch + row0 * ES;
      end = (o.rows - 1) * pitch + o.row_bytes;
      left = 0;
      step_bytes = kStepRows * pitch;
      const int k3 = (lane & 15) >> 2, half = lane >> 5;
      const uint32_t kr = OFF + (ES == 2 ? (uint32_t)((half * 8 + k3) * (ROWS * 2) + (lane & 1) * 8)
                                         : (uint32_t)(half * 4 * (ROWS * 4) + (lane & 3) * 4));
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int ch = ES == 2 ? (blk0 + b) * 4 + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1)
                               : (blk0 + b) * 8 + ((lane & 31) >> 2);
        frag[b] = kr + (uint32_t)((ch ^ (ES == 2 ? 4 * k3 : 8 * half)) * 16);
      }
    }
    plane = o.plane;
    planes = planes_;
    ptr0 = tile_uniform(reinterpret_cast<uint64_t>(o.base) + (uint64_t)at);
    remain0 = (int64_t)tile_uniform((uint64_t)(end - at));
    ptr = ptr0 + (planes & 3) * plane;
    remain = remain0;
    issued = ik = 0;
    buf = 0;
    srd[3] = 0x00020000u;
  }
  // The next step, into the next of `bufs` buffers (returned); an empty
  // descriptor behind the last one.  A handful of scalar instructions: they sit
  // between MFMAs, and what does not fit under one delays the next.
  template <int BUFS>
  __device__ __forceinline__ uint32_t aim(int steps, int total) {
    srd[0] = (uint32_t)ptr;
    srd[1] = (uint32_t)(ptr >> 32);
    srd[2] = issued < total ? (remain >> 32 ? 0xffffffffu : (uint32_t)remain) : 0u;
    if constexpr (!KM) {
      // the last step of an operand whose rows end inside it (never one of
      // several planes: those are padded)
      if (left < 128) {
#pragma unroll
        for (int j = 0; j < kPieces; ++j) voff[j] = chunk16 >= (uint32_t)left ? 0xffffff00u : voff[j];
      }
      left -= 128;
    }
    ptr += step_bytes;
    remain -= step_bytes;
    ++issued;
    if (++ik == steps) {
      ik = 0;
      planes >>= 2;
      ptr = ptr0 + (planes & 3) * plane;
      remain = remain0;
      if constexpr (!KM) left += steps * 128;
    }
    const uint32_t dst = buf * (ROWS * 128);
    if (++buf == BUFS) buf = 0;
    return dst;
  }
  // its j-th piece of this wave, into the buffer at `lds` (the operand's first)
  __device__ __forceinline__ void dma(int j, uint32_t lds, int wave) const {
    tile_dma16(srd, voff[j], lds + (uint32_t)(OFF + (wave + 4 * j) * 1024));
  }
  // block b's fragment of slice kk
  __device__ __forceinline__ void read(tu4& f, uint32_t stage, int kk, int b) const {
    if constexpr (!KM) {
      f = *reinterpret_cast<const ZS_TLDS tu4*>(
          (uintptr_t)(stage + frag[kk] + (uint32_t)(b * 4096)));
    } else if constexpr (ES == 4) {
      const uint32_t at = stage + frag[b] + (uint32_t)(kk * 8 * ROWS * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        f[e] = *reinterpret_cast<const ZS_TLDS uint32_t*>((uintptr_t)(at + e * ROWS * 4));
    } else {
      const uint32_t at = stage + frag[b] + (uint32_t)(kk * 16 * ROWS * 2);
      const tu2 lo = __builtin_bit_cast(
          tu2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                   reinterpret_cast<ZS_TLDS ts4*>((uintptr_t)at)));
      const tu2 hi = __builtin_bit_cast(
          tu2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                   reinterpret_cast<ZS_TLDS ts4*>((uintptr_t)(at + 4 * ROWS * 2))));
      f = tu4{lo[0], lo[1], hi[0], hi[1]};
    }
  }
};

// acc = sum over `terms` plane pairs and `steps` k-steps from k0 on.  Leaves
// with every DMA landed and every wave past its last LDS read.
template <typename C>
__device__ __forceinline__ void tile_loop(const TileOperand& A, const TileOperand& B,
                                          int64_t m0, int64_t n0, int k0, int steps, int terms,
                                          uint32_t lds, int lane, int wave,
                                          typename C::MMA::Acc (&acc)[C::WM][C::WN]) {
  typedef TileSide<C::A_KM, C::BM, 0, C::WM, C::MMA::kBytes> SideA;
  typedef TileSide<C::B_KM, C::BN, 3 * C::BM * 128, C::WN, C::MMA::kBytes> SideB;
  constexpr int PA = SideA::kPieces, PB = SideB::kPieces;
  constexpr int M = C::WM * C::WN, R = C::WM + C::WN;
  SideA sa;
  SideB sb;
  sa.init(A, m0, k0, lane, wave, (wave / C::WGN) * C::WM, terms > 1 ? kTermsA : 0u);
  sb.init(B, n0, k0, lane, wave, (wave % C::WGN) * C::WN, terms > 1 ? kTermsB : 0u);
#pragma unroll
  for (int i = 0; i < C::WM; ++i)
#pragma unroll
    for (int j = 0; j < C::WN; ++j) acc[i][j] = typename C::MMA::Acc{};

  const int total = terms * steps;
  uint32_t adst = lds, bdst = lds;
  auto aim_a = [&]() { adst = lds + sa.template aim<3>(steps, total); };
  auto aim_b = [&]() { bdst = lds + sb.template aim<2>(steps, total); };
  auto aim_none = []() {};
  tu4 fa[2][C::WM], fb[2][C::WN];
  // The MFMAs of register set S, in between the reads of slice KK into the other
  // set and the pieces [D0, D1) of the step that A (B) is aimed at
  uint32_t acur = lds, bcur = lds;
  // `then`: what is aimed at next, under the slice's last MFMAs
  auto slice = [&](auto S, auto KK, auto IS_A, auto D0, auto D1, auto&& then) {
    constexpr int s = decltype(S)::value, kk = decltype(KK)::value;
    constexpr int d0 = decltype(D0)::value, nd = decltype(D1)::value - d0;
    tile_for<M>([&](auto M_) {
      constexpr int m = decltype(M_)::value;
      tile_for<R>([&](auto Q) {
        constexpr int q = decltype(Q)::value;
        if constexpr (q * M / R == m) {
          if constexpr (q < C::WN)
            sb.read(fb[s ^ 1][q], bcur, kk, q);
          else
            sa.read(fa[s ^ 1][q - C::WN], acur, kk, q - C::WN);
        }
      });
      tile_for<nd>([&](auto Q) {
        constexpr int q = decltype(Q)::value;
        if constexpr (q * M / nd == m) {
          if constexpr (decltype(IS_A)::value)
            sa.dma(d0 + q, adst, wave);
          else
            sb.dma(d0 + q, bdst, wave);
        }
      });
      constexpr int i = m / C::WN, j = m % C::WN;
      if constexpr (m == M - 1) then();
      if constexpr (m == 0) __builtin_amdgcn_s_setprio(1);
      acc[i][j] = C::MMA::mma(fa[s][i], fb[s][j], acc[i][j]);
      if constexpr (m == M - 1) __builtin_amdgcn_s_setprio(0);
      __builtin_amdgcn_sched_barrier(0);
    });
  };
#define ZS_IC(x) std::integral_constant<int, (x)>{}
  aim_a();
#pragma unroll
  for (int j = 0; j < PA; ++j) sa.dma(j, adst, wave);
  aim_b();
#pragma unroll
  for (int j = 0; j < PB; ++j) sb.dma(j, bdst, wave);
  aim_a();
#pragma unroll
  for (int j = 0; j < PA; ++j) sa.dma(j, adst, wave);
  aim_b();
#pragma unroll
  for (int j = 0; j < PB / 2; ++j) sb.dma(j, bdst, wave);
  tile_wait_barrier<PA + PB / 2>();
  tile_for<C::WN>([&](auto Q) { sb.read(fb[0][decltype(Q)::value], bcur, 0, decltype(Q)::value); });
  tile_for<C::WM>([&](auto Q) { sa.read(fa[0][decltype(Q)::value], acur, 0, decltype(Q)::value); });
  uint32_t abuf = 0;
  for (int t = 0; t < total; ++t) {
    // B of step t + 1
    slice(ZS_IC(0), ZS_IC(1), ZS_IC(0), ZS_IC(PB / 2), ZS_IC(PB), aim_a);
    // A of step t + 2
    slice(ZS_IC(1), ZS_IC(2), ZS_IC(1), ZS_IC(0), ZS_IC(PA / 2), aim_none);
    slice(ZS_IC(0), ZS_IC(3), ZS_IC(1), ZS_IC(PA / 2), ZS_IC(PA), aim_b);
    // step t + 1 has landed (A of step t + 2 may be in flight), and every wave
    // has its last slice of step t in registers: its buffers are free
    tile_wait_barrier<PA>();
    if (++abuf == 3) abuf = 0;
    acur = lds + abuf * (C::BM * 128);
    bcur = lds + ((t + 1) & 1) * (C::BN * 128);
    // B of step t + 2
    slice(ZS_IC(1), ZS_IC(0), ZS_IC(0), ZS_IC(0), ZS_IC(PB / 2), aim_none);
  }
#undef ZS_IC
  tile_wait_barrier<0>();
  // for acc_get: every MFMA is in front of these statements, and its 16 passes
  // and the read's wait states behind the last
#pragma unroll
  for (int i = 0; i < C::WM; ++i)
#pragma unroll
    for (int j = 0; j < C::WN; ++j) asm volatile("" : "+a"(acc[i][j]));
  asm volatile("s_nop 15\n\ts_nop 7" ::: "memory");
}

// Workgroup -> tile.  Workgroups go round-robin over the eight XCDs, each with
// an L2 of its own: every XCD takes a contiguous share of the tiles, ordered
// in bands of eight tile rows, so that the ~32 tiles an XCD runs at a time
// share eight row blocks and four column blocks of the operands.
__device__ __forceinline__ void tile_of_block(uint32_t bid, uint32_t n_wg, uint32_t tiles_m,
                                              uint32_t tiles_n, int& tm, int& tn) {
  const uint32_t x = bid & 7u, idx = bid >> 3;
  const uint32_t per = n_wg >> 3, rem = n_wg & 7u;
  const uint32_t id = x * per + (x < rem ? x : rem) + idx;
  const uint32_t band = id / (8u * tiles_n);
  const uint32_t in = id - band * 8u * tiles_n;
  const uint32_t rows = tiles_m - band * 8u < 8u ? tiles_m - band * 8u : 8u;
  const uint32_t c = in / rows;
  tm = __builtin_amdgcn_readfirstlane((int)(band * 8u + (in - c * rows)));
  tn = __builtin_amdgcn_readfirstlane((int)c);
}

// HIP launches fewer than 2^32 threads along a dimension of the grid
constexpr int64_t kMaxWorkgroups = (1ll << 24) - 1;

// 256 x 256 tiles (one workgroup a CU) or 128 x 128 (two)?  And, for a product whose
// k may be split with the parts joined afterwards, over how many workgroups?  What
// takes the fewest of a large tile's steps (1.6 us): a CU's two small tiles take 0.58
// of a large one's time (1140 against 1330 TFLOP/s); a tile's start and end cost eight
// steps, 5.5 where the CU's other tile multiplies meanwhile (5000 rows bfloat16 over
// 50 000 classes, 128 against 256: 201 against 218 us at 256 features, 304 / 302 at
// 512, 513 / 484 at 1024), and no share is shorter than that; parts are written and
// read by a launch of their own.
struct TilePlan {
  bool big;
  int splits;
};
inline TilePlan plan_tiles(int64_t m, int64_t n, int64_t steps, bool may_split, int cus) {
  TilePlan best{false, 1};
  double least = 0;
  for (int big = 0; big < 2; ++big) {
    const int64_t b = big ? 256 : 128, slots = big ? cus : 2ll * cus;
    const int64_t tiles = ((m + b - 1) / b) * ((n + b - 1) / b);
    int64_t most = 1;
    if (may_split) {
      most = slots / (tiles > 0 ? tiles : 1);
      most = most > steps / 8 ? steps / 8 : most;
      most = most < 1 ? 1 : most > 64 ? 64 : most;
    }
    for (int64_t s = 1; s <= most; s = s < most && 2 * s > most ? most : 2 * s) {
      const double rounds = (double)((tiles * s + slots - 1) / slots);
      const double t = rounds * (big ? 1.0 : 0.58) * ((double)((steps + s - 1) / s) + (big ? 8.0 : 5.5)) +
                       (s > 1 ? 3.0 + 1.1e-6 * (double)(m * n * s) : 0.0);
      if ((big == 0 && s == 1) || t < least) {
        least = t;
        best = TilePlan{big != 0, (int)s};
      }
    }
  }
  return best;
}

// row of a 32 x 32 accumulator block held in register r of lane half h
__device__ __forceinline__ constexpr int acc_row(int r, int h) {
  return (r & 3) + 8 * (r >> 2) + 4 * h;
}

// One accumulator element for the vector unit.  The accumulators of the large
// tiles fill the AGPRs; read through the compiler, all of them move to VGPRs at
// the loop's end, which spills.  This read names the AGPR in place.  tile_loop
// ends with the wait states that such a read needs behind the last MFMA.
__device__ __forceinline__ float acc_get(const tf16& v, int r) {
  float x;
  asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(x) : "a"(v[r]));
  return x;
}
__device__ __forceinline__ int acc_get(const ti16& v, int r) {
  int x;
  asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(x) : "a"(v[r]));
  return x;
}

// The result's rows leave through the LDS.  A lane holds ONE n and, in groups of
// four registers, runs of four m: the caller picks its operands so that m is
// the contiguous direction of the output.  Per block column j, the workgroup's
// WGN x 32 rows of BM values are written as elements T (float, or bfloat16 bits),
// 16 bytes between rows so that they start in different banks, and read back
// in 16-byte pieces; two regions alternate, one barrier a block column.
// As: how a value is written (AsF32, AsBf16).
//   value(i, j, q, v): the four values of registers 4 q .. 4 q + 3 of block (i, j)
//   emit(n, m, piece): 16 bytes of row n (of the tile) from column m on
struct AsF32 {
  typedef float T;
  static __device__ __forceinline__ void put(char* to, const float (&v)[4]) {
    *reinterpret_cast<tf4*>(to) = tf4{v[0], v[1], v[2], v[3]};
  }
};
struct AsBf16 {
  typedef uint16_t T;
  static __device__ __forceinline__ void put(char* to, const float (&v)[4]) {
    *reinterpret_cast<tu2*>(to) = tu2{bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3])};
  }
};
template <typename C, typename As>
constexpr int kTileRowsLds = 2 * C::WGN * 32 * (C::BM * (int)sizeof(typename As::T) + 16);

template <typename C, typename As, typename V, typename E>
__device__ __forceinline__ void tile_rows(char* smem, int lane, int wave, V&& value, E&& emit) {
  typedef typename As::T T;
  constexpr int kRows = C::WGN * 32, kPitch = C::BM * (int)sizeof(T) + 16;
  constexpr int kPer = 16 / (int)sizeof(T), kPieces = C::BM / kPer;
  const int half = lane >> 5, col = lane & 31;
  char* const mine = smem + ((wave % C::WGN) * 32 + col) * kPitch +
                     ((wave / C::WGN) * C::WM * 32 + 4 * half) * (int)sizeof(T);
  tile_for<C::WN>([&](auto J) {
    constexpr int j = decltype(J)::value;
    constexpr int region = (j & 1) * kRows * kPitch;
    tile_for<C::WM>([&](auto I) {
      constexpr int i = decltype(I)::value;
      tile_for<4>([&](auto Q) {
        constexpr int q = decltype(Q)::value;
        float v[4];
        value(I, J, Q, v);
        As::put(mine + region + (i * 32 + 8 * q) * (int)sizeof(T), v);
      });
    });
    __syncthreads();
    for (int c = threadIdx.x; c < kRows * kPieces; c += 256) {
      const int row = c / kPieces, piece = c % kPieces;
      emit((row >> 5) * C::WN * 32 + j * 32 + (row & 31), piece * kPer,
           *reinterpret_cast<const tu4*>(smem + region + row * kPitch + piece * 16));
    }
  });
}

// `piece` (16 bytes) to out[0 ..], `left` elements of T still inside the row
template <typename T>
__device__ __forceinline__ void store_piece(T* out, int64_t left, const tu4& piece) {
  constexpr int N = 16 / (int)sizeof(T);
  if (left >= N) {
    *reinterpret_cast<tu4_any*>(out) = piece;
    return;
  }
#pragma unroll
  for (int e = 0; e < N; ++e)
    if (e < left) {
      if constexpr (sizeof(T) == 4) {
        const uint32_t u = piece[e];
        out[e] = __builtin_bit_cast(T, u);
      } else {
        out[e] = (T)(piece[e / 2] >> (16 * (e & 1)));
      }
    }
}

}  // namespace zshmc
