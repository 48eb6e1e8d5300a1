// Categorical log-probabilities under a linear output layer with many classes
// (reference distributions/univariate.py:496-548 on logits X w^T + b), and
// their gradients, with the classes taken in pieces: the [rows, classes]
// logits are never kept.
//
//   l[n, v] = sum_d x[n, d] w[v, d] + b[v]
//   log_prob[n] = l[n, y_n] - M_n - log S_n,   M_n = max_v l,  S_n = sum_v e^(l - M_n)
//   r[n, v] = g_n ([v == y_n] - e^(l[n, v] - M_n) / S_n)
//   dX = r w,   dw = r^T X,   db[v] = sum_n r[n, v]
//
// Forward: one tile product (tile_gemm.h) whose epilogue leaves, per 256
// classes, each row's maximum and sum (8 bytes per row instead of 512 of
// logits), and one pass that joins them.  Gradient: per piece of classes, the
// logits again, turned into r in the epilogue (bfloat16, or for float32 operands
// float32 or its planes), then the two products over that piece; dX is
// accumulated in float32 over the pieces.  8 N V D flop for both directions,
// six of them unavoidable.  M and S are float32; r is rounded to the operands'
// precision because it is an operand of the matrix cores.
//
// float32 operands go one of two ways.  Few rows: as they are, on
// v_mfma_f32_32x32x2_f32.  More: as three bfloat16 planes each (tile_gemm.h), which
// hold every bit of them; six products on the 16-bit matrix cores are 1.3 times as fast.
#include "tile_gemm.h"

namespace zshmc {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
typedef float cf2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float fast_exp(float x) {
  return __builtin_amdgcn_exp2f(x * kLog2e);
}
__device__ __forceinline__ float only(uint32_t keep, float x) {
  return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, x) & keep);
}
__device__ __forceinline__ uint16_t bf16_bits(float x) {
  return __builtin_bit_cast(uint16_t, (__bf16)x);
}

// ---- operands as the tile loop wants them ------------------------------------
// An operand's unit 2^e: its largest magnitude x is near 2^48 units (see tile_gemm.h).
// With ldexp every exponent can be applied; 0 for zeros.
__device__ __forceinline__ int unit_of(float x) {
  const int e = (int)(__builtin_bit_cast(uint32_t, x) >> 23);
  return x == 0.f ? 0 : (e == 0 ? 1 : e) - 127 - 48;
}

// Rows to be packed, and the largest finite magnitudes that their units come from: of X,
// w and g per workgroup, without the rows (of X and g) that are ignored.  Bound by
// memory: 12 419 + 1021 rows of 784 float32 10 us, 4.0 TB/s.
constexpr int kMaxParts = 1024;
struct PackJob {
  const void* src;
  int64_t rows, cols, ld;
  unsigned char* dst;
  const int64_t* labels;           // rows labelled `ignore` become zeros; or NULL
};
struct PackArgs {
  PackJob job[2];                  // X, w (in planes both, else any that need it)
  int64_t pitch, ignore;
  const float* part;               // [3][kMaxParts]: of X, w, g
  int* unit;                       // [3]
  int has_g;
};

__global__ __launch_bounds__(256) void part_max_kernel(PackArgs a, const float* __restrict__ g,
                                                       float* __restrict__ part) {
  const int k = blockIdx.y;
  // X, w, g: the third has one column
  const PackJob& j = a.job[k == 1 ? 1 : 0];
  const float* src = k == 2 ? g : static_cast<const float*>(j.src);
  const int64_t rows = k == 2 && !g ? 0 : j.rows, cols = k == 2 ? 1 : j.cols;
  const int64_t ld = k == 2 ? 1 : j.ld, groups = (cols + 3) / 4, total = rows * groups;
  float mx = 0.f;
  auto widen = [&](float v) {
    v = fabsf(v);
    mx = v <= 3.402823466e38f ? fmaxf(mx, v) : mx;
  };
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / groups, c = (i - r * groups) * 4;
    if (j.labels && j.labels[r] == a.ignore) continue;
    const float* from = src + r * ld + c;
    if (c + 4 <= cols) {
      typedef float any __attribute__((ext_vector_type(4), aligned(4)));
      const any v = *reinterpret_cast<const any*>(from);
#pragma unroll
      for (int e = 0; e < 4; ++e) widen(v[e]);
    } else {
      for (int e = 0; e < cols - c; ++e) widen(from[e]);
    }
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off, 64));
  __shared__ float s[4];
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = mx;
  __syncthreads();
  if (threadIdx.x == 0)
    part[k * kMaxParts + blockIdx.x] = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
}

// the parts' maximum, by a workgroup
__device__ __forceinline__ float join_max(const float* __restrict__ part) {
  __shared__ float s[4];
  float mx = 0.f;
  for (int i = threadIdx.x; i < kMaxParts; i += 256) mx = fmaxf(mx, part[i]);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = mx;
  __syncthreads();
  return fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
}

// blockIdx.y's rows of `cols` elements -> rows of `pitch` bytes, zero behind the
// last column: elements as they are, or (SPLIT) float32 as three bfloat16 planes of x /
// 2^e.  Rows whose label is `ignore` become zeros (whatever they hold, NaN included,
// reaches no product).  An infinite weight stands in the lowest plane alone, which meets
// only the other operand's highest: in the highest it would meet the rest of x, of any
// sign or 0.  (An infinite x makes its row NaN in either.)  Bound by memory: 12 419 + 1021
// rows of 784 21 us, 5.0 TB/s of 4 bytes in and 6 out.
template <typename T, bool SPLIT>
__global__ __launch_bounds__(256) void pack_rows_kernel(PackArgs a) {
  constexpr int N = SPLIT ? 8 : 16 / (int)sizeof(T);     // elements per 16 bytes out
  const PackJob& j = a.job[blockIdx.y];
  const int64_t groups = a.pitch / 16, total = j.rows * groups, plane = j.rows * a.pitch;
  if ((int64_t)blockIdx.x * 256 >= total) return;
  int unit = 0;
  if (SPLIT) {
    unit = unit_of(join_max(a.part + blockIdx.y * kMaxParts));
    if (blockIdx.x == 0) {
      if (threadIdx.x == 0) a.unit[blockIdx.y] = unit;
      if (a.has_g && blockIdx.y == 0) {
        const int unit_g = unit_of(join_max(a.part + 2 * kMaxParts));
        if (threadIdx.x == 0) a.unit[2] = unit_g;
      }
    }
  }
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / groups, c = (i - r * groups) * N;
    const bool out = j.labels && j.labels[r] == a.ignore;
    const T* const from = static_cast<const T*>(j.src) + r * j.ld + c;
    T v[N] = {};
    if (!out && c + N <= j.cols) {
      typedef T any __attribute__((ext_vector_type(N), aligned(sizeof(T))));
      const any w = *reinterpret_cast<const any*>(from);
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] = w[e];
    } else if (!out) {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (c + e < j.cols) v[e] = from[e];
    }
    unsigned char* const to = j.dst + r * a.pitch + (i - r * groups) * 16;
    if constexpr (SPLIT) {
      tu4 p[kPlanes];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float x = ldexpf(v[2 * q], -unit), y = ldexpf(v[2 * q + 1], -unit);
        uint32_t w[kPlanes];
        bf16_planes(x, y, w);
        if (blockIdx.y == 1) {     // w
          const uint32_t low = (fabsf(x) == __builtin_inff() ? 0xffffu : 0u) |
                               (fabsf(y) == __builtin_inff() ? 0xffff0000u : 0u);
          w[kPlanes - 1] |= w[0] & low;
          w[0] &= ~low;
        }
#pragma unroll
        for (int k = 0; k < kPlanes; ++k) p[k][q] = w[k];
      }
#pragma unroll
      for (int k = 0; k < kPlanes; ++k) *reinterpret_cast<tu4*>(to + k * plane) = p[k];
    } else {
      typedef T whole __attribute__((ext_vector_type(N)));
      whole w;
#pragma unroll
      for (int e = 0; e < N; ++e) w[e] = v[e];
      *reinterpret_cast<whole*>(to) = w;
    }
  }
}

// (maximum, sum of exponentials) of two sets of classes together
__device__ __forceinline__ cf2 join(const cf2& t, const cf2& u) {
  const float mx = fmaxf(t[0], u[0]);
  const float off = mx == -__builtin_inff() ? 0.f : mx;
  return cf2{mx, t[1] * fast_exp(t[0] - off) + u[1] * fast_exp(u[0] - off)};
}

// ---- the tile kernels ----------------------------------------------------------
enum { kEpiStats, kEpiResidual, kEpiStore };

struct ClassArgs {
  TileOperand a, b;
  int64_t m, n;                    // extent of the output
  int steps, terms, splits;
  uint32_t tiles_m, tiles_n;
  // kEpiStats / kEpiResidual: m = classes (of the piece), n = rows of X
  const float* bias;               // of the piece's first class, or NULL
  const int64_t* labels;
  int64_t class0;                  // first class of the piece
  int64_t n_classes, ignore;
  int has_ignore;
  cf2* part;                       // [tiles_m][n] (max, sum)
  float* label_logit;              // [n]
  const cf2* stats;                // [n] (M, S)
  const float* g;                  // [n] upstream gradient
  unsigned char* resid;            // r: [plane][n][pitch]
  int64_t resid_pitch, resid_plane;
  float* bias_part;                // [tiles_n][bias_ld], or NULL
  int64_t bias_ld;
  // kEpiStore: out[n, m]
  void* out;
  int64_t out_ld, out_split;       // elements; split s at out + s * out_split
  int out_bf16, accumulate;
  // float32 in planes: the operands' units (their exponents); r is in units of g
  const int *unit_a, *unit_b, *unit_g;
};

// how r leaves through the LDS
template <int F32>
using ResidAs = typename std::conditional<F32 == 0, AsBf16, AsF32>::type;

// LDS behind the tile loop: what the epilogue exchanges; behind that the tile's
// biases and their gradient's column sums
template <typename C, int EPI, int F32>
constexpr int kEpiLds = EPI == kEpiStats      ? C::WGM * C::BN * 8
                        : EPI == kEpiResidual ? kTileRowsLds<C, ResidAs<F32>>
                                              : kTileRowsLds<C, AsF32>;

// F32: 0 bfloat16, 1 float32 as it is, 2 float32 in planes
//
// Bound by the tile loop (tile_gemm.h) and, the fewer its steps, by what lies around
// it: a workgroup's start, and an epilogue that takes e^x of every accumulator while
// no MFMA runs (4 us of a 256 x 256 tile each).  bfloat16, 256 x 256 tiles:
//   statistics  5000 x 1024 over 50 000 classes      542 us   945 TFLOP/s
//               8192 x 4096 over 131 072            6610 us  1331
//   r           4096 x 2048 over 32 768              570 us   965
//   dw / dX     8192 x 4096, 16 384 classes a piece  832 / 908 us, 1322 / 1211
// float32 in planes, 1021 x 784 over 12 419 classes (six products): statistics 131 us,
// 913 TFLOP/s; r 154 us, dw 166 us, dX 161 us.  One row of bfloat16 against
// 32 768 x 4096 (tiles of 128 classes x 32 rows): 40 us, 6.7 TB/s; 100 rows of float32,
// 12 419 x 128: 11 us, 28 TFLOP/s of the float32 matrix cores.
template <typename C, int EPI, int F32>
__global__ __launch_bounds__(256, C::kLds > 80 * 1024 ? 1 : 2) void class_tile_kernel(
    ClassArgs p) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const uint32_t lds = (uint32_t)reinterpret_cast<uintptr_t>(smem);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int tm, tn;
  tile_of_block(blockIdx.x, gridDim.x, p.tiles_m, p.tiles_n, tm, tn);
  const int64_t m0 = (int64_t)tm * C::BM, n0 = (int64_t)tn * C::BN;
  int k0 = 0, steps = p.steps;
  if (EPI == kEpiStore && p.splits > 1) {
    // blockIdx.y's share of the k-steps; a share may be empty
    const int per = (p.steps + p.splits - 1) / p.splits;
    k0 = (int)blockIdx.y * per;
    steps = p.steps - k0 < per ? p.steps - k0 : per;
  }
  const int wm = wave / C::WGN, wn = wave % C::WGN;
  const int half = lane >> 5, col = lane & 31;
  const int mw = wm * C::WM * 32, nw = wn * C::WN * 32;

  // What the epilogue needs of its rows of X (a lane each per block column),
  // fetched in front of the loop: the label's class counted from the wave's
  // first (or -1), M, g and -g / S
  int yl[C::WN];
  float mx[C::WN], g[C::WN], ginv[C::WN], bias_here = 0.f;
  const bool biased = EPI != kEpiStore && (p.bias || p.bias_part || m0 + C::BM > p.m);
  if constexpr (EPI != kEpiStore) {
#pragma unroll
    for (int j = 0; j < C::WN; ++j) {
      const int64_t n = n0 + nw + j * 32 + col;
      yl[j] = -1;
      // (a row behind the last one, or one that is ignored: r = 0)
      mx[j] = 3e38f;
      g[j] = ginv[j] = 0.f;
      if (n < p.n) {
        const int64_t label = p.labels[n];
        const int64_t y = label - p.class0 - m0 - mw;
        if (y >= 0 && y < C::WM * 32 && y + m0 + mw < p.m) yl[j] = (int)y;
        if (EPI == kEpiResidual && !(p.has_ignore && label == p.ignore)) {
          const cf2 st = p.stats[n];
          mx[j] = st[0];
          g[j] = F32 == 2 ? ldexpf(p.g[n], -*p.unit_g) : p.g[n];
          // (a label outside counts only where the caller lets the row count)
          if ((label < 0 || label >= p.n_classes) && g[j] != 0.f) g[j] = __builtin_nanf("");
          ginv[j] = -g[j] / st[1];
        }
      }
    }
    // thread t: the bias of the tile's class t, -inf behind the last class
    const int64_t v = m0 + threadIdx.x;
    if (threadIdx.x < C::BM)
      bias_here = v < p.m ? (p.bias ? p.bias[v] : 0.f) : -__builtin_inff();
  }

  typename C::MMA::Acc acc[C::WM][C::WN];
  if (steps > 0) {
    tile_loop<C>(p.a, p.b, m0, n0, k0, steps, p.terms, lds, lane, wave, acc);
  } else {
#pragma unroll
    for (int i = 0; i < C::WM; ++i)
#pragma unroll
      for (int j = 0; j < C::WN; ++j) acc[i][j] = typename C::MMA::Acc{};
  }

  // what an accumulator counts in
  const int unit = F32 == 2 ? *p.unit_a + *p.unit_b : 0;
  if constexpr (EPI == kEpiStore) {
    auto value = [&](auto I, auto J, auto Q, float (&v)[4]) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        v[r] = acc_get(acc[decltype(I)::value][decltype(J)::value], 4 * decltype(Q)::value + r);
        if (F32 == 2) v[r] = ldexpf(v[r], unit);
      }
    };
    if (F32 == 0 && p.out_bf16) {
      tile_rows<C, AsBf16>(smem, lane, wave, value, [&](int n, int m, const tu4& piece) {
        if (n0 + n < p.n && m0 + m < p.m)
          store_piece(static_cast<uint16_t*>(p.out) + (n0 + n) * p.out_ld + m0 + m,
                      p.m - m0 - m, piece);
      });
    } else {
      float* out = static_cast<float*>(p.out) + (int64_t)blockIdx.y * p.out_split;
      tile_rows<C, AsF32>(smem, lane, wave, value, [&](int n, int m, const tu4& piece) {
        if (n0 + n >= p.n || m0 + m >= p.m) return;
        float* o = out + (n0 + n) * p.out_ld + m0 + m;
        tu4 sum = piece;
        if (p.accumulate) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (e < p.m - m0 - m) {
              const uint32_t u = piece[e];
              sum[e] = __builtin_bit_cast(uint32_t, o[e] + __builtin_bit_cast(float, u));
            }
        }
        store_piece(o, p.m - m0 - m, sum);
      });
    }
    return;
  } else {
    float* sbias = reinterpret_cast<float*>(smem + kEpiLds<C, EPI, F32>);
    // the lane's 16 WM classes' biases stay in registers (read per use, the LDS'
    // latency shows between the accumulator reads)
    tf4 bias[C::WM][4] = {};
    if (biased) {
      if (threadIdx.x < C::BM) sbias[threadIdx.x] = bias_here;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < C::WM; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          bias[i][q] = *reinterpret_cast<const tf4*>(sbias + mw + 4 * half + i * 32 + 8 * q);
    }
    // the logits of registers 4 q .. 4 q + 3 of block (i, j)
    auto logits = [&](auto I, auto J, auto Q, auto BIASED, float (&l)[4]) {
      constexpr int i = decltype(I)::value, j = decltype(J)::value, q = decltype(Q)::value;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        l[r] = acc_get(acc[i][j], 4 * q + r);
        if (F32 == 2) l[r] = ldexpf(l[r], unit);
        if (decltype(BIASED)::value) l[r] += bias[i][q][r];
      }
    };
    auto blocks = [&](auto&& f) {
      tile_for<C::WM>([&](auto I) { tile_for<4>([&](auto Q) { f(I, Q); }); });
    };
    // is some row's label in the wave's classes?
    bool near[C::WN];
#pragma unroll
    for (int j = 0; j < C::WN; ++j) near[j] = __any(yl[j] >= 0);
    if constexpr (EPI == kEpiStats) {
      cf2* red = reinterpret_cast<cf2*>(smem);               // [WGM][BN]
      auto sweep = [&](auto BIASED) {
        tile_for<C::WN>([&](auto J) {
          constexpr int j = decltype(J)::value;
          float l[C::WM][4][4];            // one read of the accumulators
          float most = -__builtin_inff();
          blocks([&](auto I, auto Q) {
            float(&v)[4] = l[decltype(I)::value][decltype(Q)::value];
            logits(I, J, Q, BIASED, v);
            most = fmaxf(fmaxf(most, fmaxf(v[0], v[1])), fmaxf(v[2], v[3]));
          });
          if (near[j]) {
            float picked = 0.f;
            blocks([&](auto I, auto Q) {
              constexpr int i = decltype(I)::value, q = decltype(Q)::value;
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (yl[j] == i * 32 + acc_row(4 * q + r, half)) picked = l[i][q][r];
            });
            if (yl[j] >= 0 && ((yl[j] >> 2) & 1) == half)
              p.label_logit[n0 + nw + j * 32 + col] = picked;
          }
          most = fmaxf(most, __shfl_xor(most, 32, 64));
          const float off = most == -__builtin_inff() ? 0.f : most;
          float s[4] = {0.f, 0.f, 0.f, 0.f};
          blocks([&](auto I, auto Q) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              s[r] += fast_exp(l[decltype(I)::value][decltype(Q)::value][r] - off);
          });
          float sum = (s[0] + s[1]) + (s[2] + s[3]);
          sum += __shfl_xor(sum, 32, 64);
          if (half == 0) red[wm * C::BN + nw + j * 32 + col] = cf2{most, sum};
        });
      };
      if (biased)
        sweep(std::true_type{});
      else
        sweep(std::false_type{});
      __syncthreads();
      for (int i = threadIdx.x; i < C::BN; i += 256) {
        if (n0 + i >= p.n) continue;
        cf2 t = red[i];
#pragma unroll
        for (int k = 1; k < C::WGM; ++k) t = join(t, red[k * C::BN + i]);
        p.part[(int64_t)tm * p.n + n0 + i] = t;
      }
    } else {
      float sum[C::WM][16];                // over the wave's rows, for the bias
      float* scol = sbias + C::BM;         // [WGN][BM]
      // all bits, or none of a row that has no part: its logits need not be numbers (a
      // row of zeros has NaN where a weight is infinite)
      uint32_t keep[C::WN];
#pragma unroll
      for (int j = 0; j < C::WN; ++j) keep[j] = ginv[j] == 0.f ? 0u : ~0u;
      auto write = [&](auto BIASED) {
        auto value = [&](auto I, auto J, auto Q, float (&v)[4]) {
          constexpr int i = decltype(I)::value, j = decltype(J)::value, q = decltype(Q)::value;
          logits(I, J, Q, BIASED, v);
#pragma unroll
          for (int r = 0; r < 4; ++r) v[r] = only(keep[j], ginv[j] * fast_exp(v[r] - mx[j]));
          if (near[j]) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (yl[j] == i * 32 + acc_row(4 * q + r, half)) v[r] += g[j];
          }
          if (decltype(BIASED)::value && p.bias_part) {
#pragma unroll
            for (int r = 0; r < 4; ++r) sum[i][4 * q + r] = j ? sum[i][4 * q + r] + v[r] : v[r];
          }
        };
        tile_rows<C, ResidAs<F32>>(smem, lane, wave, value, [&](int n, int m, const tu4& piece) {
          constexpr int kBytes = F32 == 1 ? 4 : 2;       // of a value in a plane
          const int64_t byte = (m0 + m) * kBytes;
          if (n0 + n >= p.n || byte >= p.resid_pitch) return;
          unsigned char* const to = p.resid + (n0 + n) * p.resid_pitch + byte;
          if constexpr (F32 == 2) {
            const tf4 x = __builtin_bit_cast(tf4, piece);
            uint32_t front[kPlanes], back[kPlanes];
            bf16_planes(x[0], x[1], front);
            bf16_planes(x[2], x[3], back);
#pragma unroll
            for (int k = 0; k < kPlanes; ++k)
              *reinterpret_cast<tu2*>(to + k * p.resid_plane) = tu2{front[k], back[k]};
          } else {
            *reinterpret_cast<tu4*>(to) = piece;
          }
        });
      };
      if (biased)
        write(std::true_type{});
      else
        write(std::false_type{});
      if (p.bias_part) {
        blocks([&](auto I, auto Q) {
          constexpr int i = decltype(I)::value, q = decltype(Q)::value;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float s = group_sum<32>(sum[i][4 * q + r]);
            if (col == 0) scol[wn * C::BM + mw + i * 32 + acc_row(4 * q + r, half)] = s;
          }
        });
        __syncthreads();
        for (int i = threadIdx.x; i < C::BM; i += 256) {
          float s = 0.f;
#pragma unroll
          for (int k = 0; k < C::WGN; ++k) s += scol[k * C::BM + i];
          if (F32 == 2) s = ldexpf(s, *p.unit_g);
          if (m0 + i < p.m) p.bias_part[(int64_t)tn * p.bias_ld + p.class0 + m0 + i] = s;
        }
      }
    }
  }
}

// ---- joins ---------------------------------------------------------------------
// ROWS rows x 256 / ROWS lanes of parts per workgroup: few rows leave the chip empty
// otherwise (1021 rows of 49 parts: two rows a workgroup 1.5 us less than 16); 5000 of 196
// parts 7.5 us, 1.0 TB/s.
template <int ROWS>
__global__ __launch_bounds__(256) void join_stats_kernel(
    const cf2* __restrict__ part, int parts, const float* __restrict__ label_logit,
    const int64_t* __restrict__ labels, int64_t n, int64_t n_classes, int has_ignore,
    int64_t ignore, float* __restrict__ log_prob, cf2* __restrict__ stats) {
  constexpr int kLanes = 256 / ROWS;
  const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x % ROWS;
  const int k = threadIdx.x / ROWS;
  cf2 t{-__builtin_inff(), 0.f};
  if (row < n)
    for (int i = k; i < parts; i += kLanes) t = join(t, part[(int64_t)i * n + row]);
  __shared__ cf2 s[256];
  s[threadIdx.x] = t;
#pragma unroll
  for (int left = kLanes / 2; left > 0; left /= 2) {
    __syncthreads();
    if (k < left) {
      t = join(t, s[threadIdx.x + left * ROWS]);
      s[threadIdx.x] = t;
    }
  }
  if (k || row >= n) return;
  const int64_t y = labels[row];
  float lp = __builtin_nanf("");
  if (has_ignore && y == ignore)
    lp = 0.f;
  else if (y >= 0 && y < n_classes)
    lp = (label_logit[row] - t[0]) - logf(t[1]);
  log_prob[row] = lp;
  if (stats) stats[row] = t;
}

// Logits in `splits` parts [n][classes] each, joined: per row and kStatClasses classes
// (blockIdx.y, .x) their maximum and sum, and the label's logit.
constexpr int kStatClasses = 1024;
__global__ __launch_bounds__(256) void part_stats_kernel(
    const float* __restrict__ parts, int splits, int64_t n_classes,
    const float* __restrict__ bias, const int64_t* __restrict__ labels, cf2* __restrict__ part,
    float* __restrict__ label_logit) {
  const int64_t row = blockIdx.y, rows = gridDim.y, stride = rows * n_classes;
  const int64_t y = labels[row];
  float l[kStatClasses / 256];
  float most = -__builtin_inff();
#pragma unroll
  for (int e = 0; e < kStatClasses / 256; ++e) {
    const int64_t v = (int64_t)blockIdx.x * kStatClasses + e * 256 + threadIdx.x;
    l[e] = -__builtin_inff();
    if (v < n_classes) {
      l[e] = sum_parts8(parts + row * n_classes + v, stride, splits);
      if (bias) l[e] += bias[v];
      if (v == y) label_logit[row] = l[e];
    }
    most = fmaxf(most, l[e]);
  }
  const float off = most == -__builtin_inff() ? 0.f : most;
  cf2 t{most, 0.f};
#pragma unroll
  for (int e = 0; e < kStatClasses / 256; ++e) t[1] += fast_exp(l[e] - off);
#pragma unroll
  for (int step = 32; step > 0; step >>= 1) {
    const float mx = __shfl_xor(t[0], step, 64), sum = __shfl_xor(t[1], step, 64);
    t = join(t, cf2{mx, sum});
  }
  __shared__ cf2 red[4];
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = t;
  __syncthreads();
  if (threadIdx.x == 0)
    part[blockIdx.x * rows + row] = join(join(red[0], red[1]), join(red[2], red[3]));
}

// out[i] = sum of `parts` rows of x, in order; bound by memory (4096 x 2048 of two
// parts to bfloat16: 23 us, 3.6 TB/s)
template <bool BF16>
__global__ __launch_bounds__(256) void sum_rows_kernel(const float* __restrict__ x, int parts,
                                                       int64_t stride, int64_t n,
                                                       void* __restrict__ out) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n;
       i += (int64_t)gridDim.x * 256) {
    const float s = sum_parts8(x + i, stride, parts);
    if (BF16)
      static_cast<uint16_t*>(out)[i] = bf16_bits(s);
    else
      static_cast<float*>(out)[i] = s;
  }
}
__global__ void fill_kernel(uint16_t* __restrict__ out, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n;
       i += (int64_t)gridDim.x * blockDim.x)
    out[i] = 0;
}

// ---- host side -------------------------------------------------------------------
int64_t round_up(int64_t x, int64_t k) { return (x + k - 1) / k * k; }
unsigned grid_for(int64_t items) {
  const int64_t b = (items + 255) / 256;
  return (unsigned)(b < 1 ? 1 : b > 16384 ? 16384 : b);
}

// logits of one piece of classes: r is written, then read by two products (2 bytes a
// logit, 6 in planes).  8192 x 4096, 131 072 classes, bfloat16, training: 2^25 31.2 ms,
// 2^27 27.6, 2^29 27.5; float32 over 65 536 classes: 2^25.4 93.2, 2^26.4 89.2, 2^27 84.3.
constexpr int64_t kPieceLogits = 1ll << 27;
constexpr int64_t kMaxPitch = 4ll << 20;

struct ClassProblem {
  const void *x, *w;
  int64_t n, d, v, ldx, ldw;
  int dtype;                       // ZSHMC_F32 / ZSHMC_BF16
  bool f32() const { return dtype == ZSHMC_DTYPE_F32; }
  int64_t esize() const { return f32() ? 4 : 2; }
};

// rows that the tile loop can read where they lie
bool direct(const void* p, int64_t ld, const ClassProblem& q, bool whole) {
  const int64_t e = q.esize();
  return (whole || !q.f32()) && q.d * e % 16 == 0 && ld * e % 16 == 0 &&
         (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld * e <= kMaxPitch;
}

// Up to how many rows float32 operands are multiplied as they are, 2 N V D flop a
// product at 140 TFLOP/s, rather than packed into planes: 14 bytes an element of w, then
// six products at 1200.  As they are / in planes, us, D x V: forward, 784 x 12 419 of 512
// rows 110 / 105, of 700 201 / 141; 4096 x 32 768 963 / 1006 and 1457 / 1688.  With the
// gradients, 784 x 12 419 of 256 rows 243 / 283, of 400 423 / 379; 4096 x 32 768 2069 /
// 2503 and 3803 / 3180.  (As they are, the matrix cores take what is below 2^-126 for 0.)
constexpr int64_t kWholeRows = 512, kWholeRowsGrad = 256;

// the logits' tiles: classes x rows of X
constexpr int kTileClasses[] = {256, 128, 128, 128}, kTileRows[] = {256, 128, 64, 32};

// Where everything lies in the workspace
struct ClassLayout {
  int64_t pitch;                   // of packed operands, bytes
  int64_t x_plane, w_plane, planes;
  bool pack_x, pack_w;
  int64_t xp, wp;                  // offsets
  int64_t maxima, units;           // float32 in planes: of X, w, g
  int64_t part, label_logit;       // forward
  int splits;                      // of the features; more than one: the parts
  int64_t split_part;
  int tile;                        // see kTileClasses
  int64_t tiles_v;                 // parts of the statistics
  bool whole;                      // float32 operands as they are, no planes
  int64_t piece, pieces;           // gradient: classes per piece
  int64_t resid_pitch, resid_plane;
  int64_t resid, bias_part;
  int64_t dx_part, dw_part;        // float32 parts, where there is more than one
  int dx_splits, dx_tile, dw_splits, dw_tile;
  int64_t total;
};

int64_t tiles(int64_t n, int64_t b) { return (n + b - 1) / b; }

int clip(int splits, int64_t steps) { return (int)(splits < steps ? splits : steps); }

ClassLayout layout_of(const ClassProblem& q, bool grad, bool has_ignore) {
  ClassLayout l;
  l.whole = q.f32() && q.n <= (grad ? kWholeRowsGrad : kWholeRows);
  l.planes = q.f32() && !l.whole ? kPlanes : 1;
  l.pitch = round_up(q.d * (l.whole ? 4 : 2), 128);
  l.pack_x = !direct(q.x, q.ldx, q, l.whole) || (grad && has_ignore);
  l.pack_w = !direct(q.w, q.ldw, q, l.whole);
  l.x_plane = q.n * l.pitch;
  l.w_plane = q.v * l.pitch;
  const int cus = device_cu_count();
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += round_up(bytes, 1024);
    return here;
  };
  l.maxima = l.planes > 1 ? take(3ll * kMaxParts * 4) : 0;
  l.units = l.planes > 1 ? take(3 * 4) : 0;
  l.xp = l.pack_x ? take(l.planes * l.x_plane) : 0;
  l.wp = l.pack_w ? take(l.planes * l.w_plane) : 0;
  const int64_t element = l.whole ? 4 : 2;       // bytes of a plane's
  l.piece = q.v;
  if (grad) {
    int64_t c = kPieceLogits / (q.n > 0 ? q.n : 1) / 256 * 256;
    if (c < 4096) c = 4096;
    // (a step's rows of r stay within the DMA's 32-bit offsets)
    if (c > kMaxPitch / element) c = kMaxPitch / element;
    if (c < l.piece) l.piece = c;
  }
  l.pieces = tiles(q.v, l.piece);
  const int64_t terms = l.planes > 1 ? kTermsSplit : 1;
  l.tile = q.n <= 32                                            ? 3
           : q.n <= 64                                          ? 2
           : plan_tiles(l.piece, q.n, terms * tiles(q.d * element, 128), false, cus).big ? 0
                                                                                         : 1;
  // (half the chip or more without a tile: halve them.  Forward call, float32, 1065 x
  // 3456, 1122 classes: 81 tiles 196 us, 153 halves 176; 128 x 2048, 4096 classes: 32
  // tiles 139 us, 128 quarters 55)
  while (l.tile > 0 && l.tile < 3 &&
         tiles(l.piece, 128) * tiles(q.n, kTileRows[l.tile]) * 2 <= cus)
    ++l.tile;
  l.tiles_v = tiles(q.v, kTileClasses[l.tile]);
  // Still half the chip or more without one, and many features: logits of a share of
  // the features a workgroup, in parts, which a pass of its own joins.  Forward call,
  // float32 7 x 2816 over 4945 classes (39 tiles): 70 us whole, 30 in 8 parts; 128 x
  // 2048 over 4096: 55, 39 in 4; bfloat16, with half the steps: 24 and 22, 25 and 25
  l.splits = 1;
  l.split_part = 0;
  const int64_t all_tiles = l.tiles_v * tiles(q.n, kTileRows[l.tile]);
  const int64_t all_steps = tiles(q.d * element, 128);
  if (!grad && l.tile == 3 && all_tiles > 0 && all_tiles * 2 <= cus) {
    const int64_t room = 2 * cus / all_tiles;
    l.splits = (int)(room < all_steps / 8 ? room : all_steps / 8);
    if (l.splits < 2) l.splits = 1;
    if (l.splits > 64) l.splits = 64;
  }
  if (l.splits > 1) {
    l.split_part = take(l.splits * q.n * q.v * 4);
    l.tiles_v = tiles(q.v, kStatClasses);
  }
  l.part = l.label_logit = l.resid = l.dx_part = l.dw_part = l.bias_part = 0;
  if (!grad) {
    l.part = take(l.tiles_v * q.n * 8);
    l.label_logit = take(q.n * 4);
  } else {
    l.resid_pitch = round_up(l.piece * element, 128);
    l.resid_plane = q.n * l.resid_pitch;
    l.resid = take(l.planes * l.resid_plane);
    // (planes: shares of three k-steps, 18 steps, at least, or the parts grow past r)
    const int64_t rows_k = tiles(q.n * element, 128), classes_k = tiles(l.piece * element, 128);
    const int64_t least = l.planes > 1 ? 3 : 1;
    const TilePlan dw = plan_tiles(l.piece, q.d, terms * rows_k, true, cus);
    l.dw_tile = dw.big ? 0 : 1;
    l.dw_splits = clip(dw.splits, tiles(rows_k, least));
    const TilePlan dx = plan_tiles(q.n, q.d, terms * classes_k, true, cus);
    l.dx_tile = q.n <= 32 ? 3 : q.n <= 64 ? 2 : dx.big ? 0 : 1;
    l.dx_splits = clip(dx.splits, tiles(classes_k, least));
    const int64_t dw_bytes = l.dw_splits > 1 ? l.dw_splits * l.piece * q.d * 4 : 0;
    const int64_t dx_bytes = l.dx_splits * l.pieces > 1 ? l.dx_splits * q.n * q.d * 4 : 0;
    // (of one piece, dw's parts are joined before dX's are written)
    if (l.pieces == 1) {
      l.dw_part = l.dx_part = take(dw_bytes > dx_bytes ? dw_bytes : dx_bytes);
    } else {
      l.dw_part = take(dw_bytes);
      l.dx_part = take(dx_bytes);
    }
    l.bias_part = take(tiles(q.n, kTileRows[l.tile]) * q.v * 4);
  }
  l.total = at;
  return l;
}

template <typename C, int EPI, int F32>
int launch_tile(const ClassArgs& a, hipStream_t s) {
  constexpr int epi = kEpiLds<C, EPI, F32> + C::BM * 4 * (1 + C::WGN);
  constexpr int lds = C::kLds > epi ? C::kLds : epi;
  static_assert(lds <= 160 * 1024, "LDS of a CU");
  static thread_local int attr_dev = -1;
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) dev = 0;
  if (attr_dev != dev) {
    const hipError_t e = hipFuncSetAttribute(
        reinterpret_cast<const void*>(class_tile_kernel<C, EPI, F32>),
        hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return check_hip(e, "hipFuncSetAttribute(LDS)");
    attr_dev = dev;
  }
  ClassArgs p = a;
  p.tiles_m = (uint32_t)tiles(p.m, C::BM);
  p.tiles_n = (uint32_t)tiles(p.n, C::BN);
  const int64_t wgs = (int64_t)p.tiles_m * p.tiles_n;
  ZS_REQUIRE(wgs <= kMaxWorkgroups, "class logits: %lld tiles", (long long)wgs);
  hipLaunchKernelGGL((class_tile_kernel<C, EPI, F32>), dim3((unsigned)wgs, (unsigned)p.splits),
                     dim3(256), lds, s, p);
  ZS_LAUNCH_CHECK("class_tile_kernel launch");
  return ZSHMC_OK;
}

template <typename M, bool AK, bool BK> using Big = TileCfg<M, 2, 2, 4, 4, AK, BK>;
template <typename M, bool AK, bool BK> using Mid = TileCfg<M, 2, 2, 2, 2, AK, BK>;
template <typename M, int WN, bool AK = false> using Few = TileCfg<M, 4, 1, 1, WN, AK, false>;

template <typename M, int EPI, int F32>
int launch_logits(const ClassArgs& a, int tile, hipStream_t s) {
  switch (tile) {
    case 0: return launch_tile<Big<M, false, false>, EPI, F32>(a, s);
    case 1: return launch_tile<Mid<M, false, false>, EPI, F32>(a, s);
    case 2: return launch_tile<Few<M, 2>, EPI, F32>(a, s);
    default: return launch_tile<Few<M, 1>, EPI, F32>(a, s);
  }
}

// a product with r: k-major X and r (dw) or k-major w and rows of r (dX)
template <bool BK, typename M, int F32>
int launch_gradient_of(const ClassArgs& g, int tile, hipStream_t s) {
  if constexpr (!BK) {             // few rows of r (11 x 254, 26 904 classes: 34 -> 13 us)
    if (tile == 2) return launch_tile<Few<M, 2, true>, kEpiStore, F32>(g, s);
    if (tile == 3) return launch_tile<Few<M, 1, true>, kEpiStore, F32>(g, s);
  }
  return tile == 0 ? launch_tile<Big<M, true, BK>, kEpiStore, F32>(g, s)
                   : launch_tile<Mid<M, true, BK>, kEpiStore, F32>(g, s);
}
template <bool BK>
int launch_gradient(const ClassArgs& g, const ClassLayout& l, int tile, hipStream_t s) {
  return l.planes > 1 ? launch_gradient_of<BK, MmaBf16, 2>(g, tile, s)
         : l.whole    ? launch_gradient_of<BK, MmaF32, 1>(g, tile, s)
                      : launch_gradient_of<BK, MmaBf16, 0>(g, tile, s);
}

int sum_rows(const void* parts, int n_parts, int64_t n, bool f32, void* out, hipStream_t s) {
  const float* x = static_cast<const float*>(parts);
  if (f32)
    hipLaunchKernelGGL(sum_rows_kernel<false>, dim3(grid_for(n)), dim3(256), 0, s, x, n_parts, n,
                       n, out);
  else
    hipLaunchKernelGGL(sum_rows_kernel<true>, dim3(grid_for(n)), dim3(256), 0, s, x, n_parts, n,
                       n, out);
  ZS_LAUNCH_CHECK("sum_rows_kernel launch");
  return ZSHMC_OK;
}

// The operands X and w, packed where they have to be; `labels`: rows of X that are
// ignored are left out (NULL: none); g: whose unit is wanted besides, or NULL.
int operands(const ClassProblem& q, const ClassLayout& l, unsigned char* ws,
             const int64_t* labels, int64_t ignore, const float* g, hipStream_t s, TileOperand* x,
             TileOperand* w) {
  const int64_t e = q.esize();
  *x = TileOperand{static_cast<const unsigned char*>(q.x), q.ldx * e, 0, q.n, q.d * e};
  *w = TileOperand{static_cast<const unsigned char*>(q.w), q.ldw * e, 0, q.v, q.d * e};
  PackArgs a{};
  a.pitch = l.pitch;
  a.ignore = ignore;
  a.part = reinterpret_cast<const float*>(ws + l.maxima);
  a.unit = reinterpret_cast<int*>(ws + l.units);
  a.has_g = g != nullptr;
  int jobs = 0;
  int64_t most = 0;
  auto add = [&](const PackJob& j) {
    a.job[jobs++] = j;
    if (j.rows > most) most = j.rows;
  };
  if (l.pack_x) {
    add({q.x, q.n, q.d, q.ldx, ws + l.xp, labels});
    *x = TileOperand{ws + l.xp, l.pitch, l.x_plane, q.n, l.pitch};
  }
  if (l.pack_w) {
    add({q.w, q.v, q.d, q.ldw, ws + l.wp, nullptr});
    *w = TileOperand{ws + l.wp, l.pitch, l.w_plane, q.v, l.pitch};
  }
  if (!jobs) return ZSHMC_OK;
  const dim3 grid(grid_for(most * (l.pitch / 16)), (unsigned)jobs);
  if (l.planes > 1) {                      // (both are packed)
    hipLaunchKernelGGL(part_max_kernel, dim3(kMaxParts, 3), dim3(256), 0, s, a, g,
                       reinterpret_cast<float*>(ws + l.maxima));
    ZS_LAUNCH_CHECK("part_max_kernel launch");
    hipLaunchKernelGGL((pack_rows_kernel<float, true>), grid, dim3(256), 0, s, a);
  } else if (q.f32()) {
    hipLaunchKernelGGL((pack_rows_kernel<float, false>), grid, dim3(256), 0, s, a);
  } else {
    hipLaunchKernelGGL((pack_rows_kernel<uint16_t, false>), grid, dim3(256), 0, s, a);
  }
  ZS_LAUNCH_CHECK("pack_rows_kernel launch");
  return ZSHMC_OK;
}

int join_stats(const ClassProblem& q, const ClassLayout& l, const ClassArgs& a,
               const int64_t* labels, int has_ignore, int64_t ignore, float* log_prob,
               float* stats, hipStream_t s) {
  cf2* st = reinterpret_cast<cf2*>(stats);
  // two rows a workgroup where 16 leave the chip empty
  if (q.n <= 4ll * device_cu_count())
    hipLaunchKernelGGL(join_stats_kernel<2>, dim3((unsigned)tiles(q.n, 2)), dim3(256), 0, s,
                       a.part, (int)l.tiles_v, a.label_logit, labels, q.n, q.v, has_ignore,
                       ignore, log_prob, st);
  else
    hipLaunchKernelGGL(join_stats_kernel<16>, dim3((unsigned)tiles(q.n, 16)), dim3(256), 0, s,
                       a.part, (int)l.tiles_v, a.label_logit, labels, q.n, q.v, has_ignore,
                       ignore, log_prob, st);
  ZS_LAUNCH_CHECK("join_stats_kernel launch");
  return ZSHMC_OK;
}

int check_problem(const ClassProblem& q, const char* who) {
  ZS_REQUIRE(q.dtype == ZSHMC_DTYPE_F32 || q.dtype == ZSHMC_DTYPE_BF16,
             "%s: dtype must be ZSHMC_DTYPE_F32 or _BF16, got %d", who, q.dtype);
  ZS_REQUIRE(q.n >= 0 && q.d > 0 && q.v > 0, "%s: n_rows >= 0, n_features and n_classes > 0",
             who);
  ZS_REQUIRE(q.n <= (1ll << 27) && q.v < (1ll << 31) && q.d <= (1ll << 20),
             "%s: at most 2^27 rows, 2^31 - 1 classes and 2^20 features", who);
  ZS_REQUIRE(q.ldx >= q.d && q.ldw >= q.d, "%s: rows overlap (ldx / ldw < n_features)", who);
  return ZSHMC_OK;
}

// every launch of a call within what HIP launches, in front of the first one
int check_tiles(const ClassProblem& q, const ClassLayout& l, bool grad, const char* who) {
  int64_t most = tiles(l.piece, kTileClasses[l.tile]) * tiles(q.n, kTileRows[l.tile]);
  if (grad) {
    const int64_t b = l.dw_tile ? 128 : 256, dw = tiles(q.d, b) * tiles(l.piece, b);
    const int64_t dx = tiles(q.d, l.dx_tile ? 128 : 256) * tiles(q.n, kTileRows[l.dx_tile]);
    most = most > dw ? most : dw;
    most = most > dx ? most : dx;
  }
  ZS_REQUIRE(most <= kMaxWorkgroups, "%s: %lld tiles, more than one launch takes", who,
             (long long)most);
  return ZSHMC_OK;
}

}  // namespace
}  // namespace zshmc

using namespace zshmc;

extern "C" int zshmc_class_log_prob_workspace(const void* x, const void* w, int64_t n_rows,
                                              int64_t n_features, int64_t n_classes, int64_t ldx,
                                              int64_t ldw, int dtype, int gradient,
                                              int has_ignore, int64_t* n_bytes_host) {
  const ClassProblem q{x, w, n_rows, n_features, n_classes, ldx, ldw, dtype};
  const int rc = check_problem(q, "zshmc_class_log_prob_workspace");
  if (rc != ZSHMC_OK) return rc;
  ZS_REQUIRE(n_bytes_host, "zshmc_class_log_prob_workspace: null pointer");
  *n_bytes_host = layout_of(q, gradient != 0, has_ignore != 0).total;
  return ZSHMC_OK;
}

extern "C" int zshmc_class_log_prob(const void* x, const void* w, const float* bias,
                                    const int64_t* labels, int64_t n_rows, int64_t n_features,
                                    int64_t n_classes, int64_t ldx, int64_t ldw, int dtype,
                                    int has_ignore, int64_t ignore_label, float* log_prob,
                                    float* stats, void* workspace, int64_t workspace_bytes,
                                    void* stream) {
  const ClassProblem q{x, w, n_rows, n_features, n_classes, ldx, ldw, dtype};
  int rc = check_problem(q, "zshmc_class_log_prob");
  if (rc != ZSHMC_OK || n_rows == 0) return rc;
  ZS_REQUIRE(x && w && labels && log_prob && workspace, "zshmc_class_log_prob: null pointer");
  ZS_REQUIRE((reinterpret_cast<uintptr_t>(stats) & 7) == 0,
             "zshmc_class_log_prob: stats must be 8-byte aligned");
  const ClassLayout l = layout_of(q, false, has_ignore != 0);
  ZS_REQUIRE(workspace_bytes >= l.total && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0,
             "zshmc_class_log_prob: %lld bytes of 16-byte aligned workspace needed, got %lld",
             (long long)l.total, (long long)workspace_bytes);
  rc = check_tiles(q, l, false, "zshmc_class_log_prob");
  if (rc != ZSHMC_OK) return rc;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  ClassArgs a{};
  a.part = reinterpret_cast<cf2*>(ws + l.part);
  a.label_logit = reinterpret_cast<float*>(ws + l.label_logit);
  rc = operands(q, l, ws, has_ignore ? labels : nullptr, ignore_label, nullptr, s, &a.b, &a.a);
  if (rc != ZSHMC_OK) return rc;
  a.m = q.v;
  a.n = q.n;
  a.steps = (int)tiles(q.d * (l.whole ? 4 : 2), 128);
  a.terms = l.planes > 1 ? kTermsSplit : 1;
  a.unit_b = reinterpret_cast<const int*>(ws + l.units);
  a.unit_a = a.unit_b + 1;
  a.splits = 1;
  a.bias = bias;
  a.labels = labels;
  a.n_classes = q.v;
  if (l.splits > 1) {
    a.splits = l.splits;
    a.out = ws + l.split_part;
    a.out_ld = q.v;
    a.out_split = q.n * q.v;
    rc = l.planes > 1 ? launch_tile<Few<MmaBf16, 1>, kEpiStore, 2>(a, s)
         : l.whole    ? launch_tile<Few<MmaF32, 1>, kEpiStore, 1>(a, s)
                      : launch_tile<Few<MmaBf16, 1>, kEpiStore, 0>(a, s);
    if (rc != ZSHMC_OK) return rc;
    hipLaunchKernelGGL(part_stats_kernel, dim3((unsigned)l.tiles_v, (unsigned)q.n), dim3(256), 0,
                       s, static_cast<const float*>(a.out), l.splits, q.v, bias, labels, a.part,
                       a.label_logit);
    ZS_LAUNCH_CHECK("part_stats_kernel launch");
    return join_stats(q, l, a, labels, has_ignore, ignore_label, log_prob, stats, s);
  }
  rc = l.planes > 1 ? launch_logits<MmaBf16, kEpiStats, 2>(a, l.tile, s)
       : l.whole    ? launch_logits<MmaF32, kEpiStats, 1>(a, l.tile, s)
                    : launch_logits<MmaBf16, kEpiStats, 0>(a, l.tile, s);
  if (rc != ZSHMC_OK) return rc;
  return join_stats(q, l, a, labels, has_ignore, ignore_label, log_prob, stats, s);
}

extern "C" int zshmc_class_log_prob_grad(
    const void* x, const void* w, const float* bias, const int64_t* labels, int64_t n_rows,
    int64_t n_features, int64_t n_classes, int64_t ldx, int64_t ldw, int dtype, int has_ignore,
    int64_t ignore_label, const float* stats, const float* grad_log_prob, void* grad_x,
    void* grad_w, float* grad_bias, void* workspace, int64_t workspace_bytes, void* stream) {
  const ClassProblem q{x, w, n_rows, n_features, n_classes, ldx, ldw, dtype};
  int rc = check_problem(q, "zshmc_class_log_prob_grad");
  if (rc != ZSHMC_OK) return rc;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (n_rows == 0) {               // nothing to contract over: zeros
    const int64_t halves = q.v * q.d * q.esize() / 2;
    if (grad_w)
      hipLaunchKernelGGL(fill_kernel, dim3(grid_for(halves)), dim3(256), 0, s,
                         static_cast<uint16_t*>(grad_w), halves);
    if (grad_bias)
      hipLaunchKernelGGL(fill_kernel, dim3(grid_for(q.v * 2)), dim3(256), 0, s,
                         reinterpret_cast<uint16_t*>(grad_bias), q.v * 2);
    ZS_LAUNCH_CHECK("fill_kernel launch");
    return ZSHMC_OK;
  }
  ZS_REQUIRE(x && w && labels && stats && grad_log_prob && workspace,
             "zshmc_class_log_prob_grad: null pointer");
  ZS_REQUIRE((reinterpret_cast<uintptr_t>(stats) & 7) == 0,
             "zshmc_class_log_prob_grad: stats must be 8-byte aligned");
  const ClassLayout l = layout_of(q, true, has_ignore != 0);
  ZS_REQUIRE(workspace_bytes >= l.total && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0,
             "zshmc_class_log_prob_grad: %lld bytes of 16-byte aligned workspace needed, got "
             "%lld", (long long)l.total, (long long)workspace_bytes);
  rc = check_tiles(q, l, true, "zshmc_class_log_prob_grad");
  if (rc != ZSHMC_OK) return rc;
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  TileOperand ox, ow;
  rc = operands(q, l, ws, has_ignore ? labels : nullptr, ignore_label, grad_log_prob, s, &ox,
                &ow);
  if (rc != ZSHMC_OK) return rc;
  const int terms = l.planes > 1 ? kTermsSplit : 1;
  const int64_t pb = l.whole ? 4 : 2;            // bytes of a plane's element
  const int* const unit = reinterpret_cast<const int*>(ws + l.units);    // of X, w, g
  const bool dx_joined = l.dx_splits * l.pieces > 1;
  for (int64_t c0 = 0; c0 < q.v; c0 += l.piece) {
    const int64_t c = q.v - c0 < l.piece ? q.v - c0 : l.piece;
    TileOperand wp = ow;
    wp.base += c0 * wp.pitch;
    wp.rows = c;
    const TileOperand r{ws + l.resid, l.resid_pitch, l.resid_plane, q.n, round_up(c * pb, 128)};
    ClassArgs a{};
    a.a = wp;
    a.b = ox;
    a.m = c;
    a.n = q.n;
    a.steps = (int)tiles(q.d * pb, 128);
    a.terms = terms;
    a.unit_a = unit + 1;
    a.unit_b = unit;
    a.unit_g = unit + 2;
    a.splits = 1;
    a.bias = bias ? bias + c0 : nullptr;
    a.labels = labels;
    a.class0 = c0;
    a.n_classes = q.v;
    a.ignore = ignore_label;
    a.has_ignore = has_ignore;
    a.stats = reinterpret_cast<const cf2*>(stats);
    a.g = grad_log_prob;
    a.resid = ws + l.resid;
    a.resid_pitch = l.resid_pitch;
    a.resid_plane = l.resid_plane;
    a.bias_part = grad_bias ? reinterpret_cast<float*>(ws + l.bias_part) : nullptr;
    a.bias_ld = q.v;
    rc = l.planes > 1 ? launch_logits<MmaBf16, kEpiResidual, 2>(a, l.tile, s)
         : l.whole    ? launch_logits<MmaF32, kEpiResidual, 1>(a, l.tile, s)
                      : launch_logits<MmaBf16, kEpiResidual, 0>(a, l.tile, s);
    if (rc != ZSHMC_OK) return rc;
    if (grad_w) {                  // dw = r^T X over the rows of X
      ClassArgs g{};
      g.a = ox;
      g.b = r;
      g.m = q.d;
      g.n = c;
      g.steps = (int)tiles(q.n * pb, 128);
      g.terms = terms;
      g.unit_a = unit;
      g.unit_b = unit + 2;
      g.splits = l.dw_splits;
      g.out_ld = q.d;
      void* const dw = static_cast<unsigned char*>(grad_w) + c0 * q.d * q.esize();
      if (l.dw_splits > 1) {
        g.out = ws + l.dw_part;
        g.out_split = c * q.d;
      } else {
        g.out = dw;
        g.out_bf16 = !q.f32();
      }
      rc = launch_gradient<true>(g, l, l.dw_tile, s);
      if (rc != ZSHMC_OK) return rc;
      if (l.dw_splits > 1) rc = sum_rows(g.out, l.dw_splits, c * q.d, q.f32(), dw, s);
      if (rc != ZSHMC_OK) return rc;
    }
    if (grad_x) {                  // dX += r w over the piece's classes
      ClassArgs g{};
      g.a = wp;
      g.b = r;
      g.m = q.d;
      g.n = q.n;
      g.steps = (int)tiles(c * pb, 128);
      g.terms = terms;
      g.unit_a = unit + 1;
      g.unit_b = unit + 2;
      g.splits = l.dx_splits;
      g.out_ld = q.d;
      if (dx_joined) {
        g.out = ws + l.dx_part;
        g.out_split = q.n * q.d;
        g.accumulate = c0 > 0;
      } else {
        g.out = grad_x;
        g.out_bf16 = !q.f32();
      }
      rc = launch_gradient<false>(g, l, l.dx_tile, s);
      if (rc != ZSHMC_OK) return rc;
    }
  }
  if (grad_x && dx_joined) {
    rc = sum_rows(ws + l.dx_part, l.dx_splits, q.n * q.d, q.f32(), grad_x, s);
    if (rc != ZSHMC_OK) return rc;
  }
  if (grad_bias)
    rc = sum_rows(ws + l.bias_part, (int)tiles(q.n, kTileRows[l.tile]), q.v, true, grad_bias, s);
  return rc;
}
