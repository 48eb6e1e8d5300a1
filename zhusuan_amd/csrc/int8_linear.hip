// Rows of 8-bit integers with one float32 scale each, and the linear layer on
// them.
//
//   s_r = max_k |x[r, k]| / 127,  q[r, k] = rint(x[r, k] / s_r)      (in [-127, 127])
//   out[m, n] = (sx_m sw_n) sum_k qx[m, k] qw[n, k] + bias[n]
//
// The sum is exact (int32 MFMA, |q| <= 127: up to 131 072 terms); s and the
// quotient are float32 with IEEE division, q the even one of two integers that
// are as near.  A row of zeros has the scale 1; a row that holds an infinity
// or a NaN has the scale NaN (and zeros), so that every value read back from
// it, or product with it, is NaN.
#include "tile_gemm.h"

namespace zshmc {
namespace {

// ---- rows to 8 bits and back ---------------------------------------------------
// Memory-bound: a row is read once (16 bytes a lane, up to kHeld of them stay in
// registers; longer rows are read again) and written once.  TPR threads share a
// row: a wave where there are rows enough to fill the chip, a workgroup
// otherwise.  131 072 x 4096 bfloat16: 455 us, 3.5 TB/s (a copy's rate is 4.9: between a
// row's last load and its first store lies the reduction, and the correction of
// quotients near a half); 10 000 x 784 float32 12 us, 3.4 TB/s.
constexpr int kHeld = 8;

template <typename T>
struct RowVec;
template <>
struct RowVec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(const tu4& v, float (&f)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t u = v[e];     // (hipcc's bit_cast of v[e] itself reads v[0])
      f[e] = __builtin_bit_cast(float, u);
    }
  }
};
template <>
struct RowVec<uint16_t> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const tu4& v, float (&f)[8]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f[2 * e] = __builtin_bit_cast(float, v[e] << 16);
      f[2 * e + 1] = __builtin_bit_cast(float, v[e] & 0xffff0000u);
    }
  }
};

__device__ __forceinline__ float element(const float* row, int c) { return row[c]; }
__device__ __forceinline__ float element(const uint16_t* row, int c) {
  return __builtin_bit_cast(float, (uint32_t)row[c] << 16);
}

// N values -> N / 4 words of rint(f / s), f / s rounded to float32 first.  One
// fma with the reciprocal and 1.5 * 2^23 rounds to the integer in the low byte; it
// says which integer unless the quotient falls within 2^-12 of the middle of two
// (the product's error is below 127 * 3 * 2^-24) or `inv` is NaN: then the division
// does, for all N (|f| / s <= 127 (1 + 2^-23) unless s is subnormal).
template <int N>
__device__ __forceinline__ void quotients(const float (&f)[N], float s, float inv,
                                          uint32_t (&w)[N / 4]) {
  constexpr float kMagic = 12582912.f;
  float y[N];
  bool near = false;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    y[e] = __builtin_fmaf(f[e], inv, kMagic);
    near |= !(fabsf(f[e] * inv - (y[e] - kMagic)) <= 0.5f - 0x1p-12f);
  }
  if (near) {
#pragma unroll 1
    for (int e = 0; e < N; ++e) {
      float d = 0.f;
#pragma unroll
      for (int k = 0; k < N; ++k) d = e == k ? f[k] : d;
      d = fminf(fmaxf(rintf(d / s), -127.f), 127.f) + kMagic;
#pragma unroll
      for (int k = 0; k < N; ++k) y[k] = e == k ? d : y[k];
    }
  }
#pragma unroll
  for (int k = 0; k < N / 4; ++k) {
    uint32_t b[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float v = y[4 * k + e];
      b[e] = __builtin_bit_cast(uint32_t, v);
    }
    const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(b[3], b[2], 0x0c0c0400u);
    w[k] = lo | hi << 16;
  }
}

// One row by TPR threads (thread t).  Thread t's k-th vector is columns c .. c + N - 1,
// c = (k TPR + t) N; one that reaches past the row's end is read from cols - N
// instead, so that every load is a whole vector inside the row and needs no mask
// (a value seen twice changes no maximum).  put(c, words) stores a whole vector's N / 4
// words, put1(c, byte) one column of the last, up to `width` columns with zeros
// from `cols` on.  Returns the scale.
template <typename T, int TPR, typename P, typename P1>
__device__ __forceinline__ float quantize_row(const T* row, int cols, int width, int t,
                                              float* part, P&& put, P1&& put1) {
  constexpr int N = RowVec<T>::N;
  float mx = 0.f;
  // a NaN or an infinity turns into a maximum no finite row reaches
  auto widen = [&](float f) {
    const float a = fabsf(f);
    mx = a <= 3.402823466e38f ? fmaxf(mx, a) : __builtin_inff();
  };
  auto load = [&](int c) -> tu4 {
    return *reinterpret_cast<const tu4_any*>(row + (c + N <= cols ? c : cols - N));
  };
  auto widen_all = [&](const tu4& v) {
    float f[N];
    RowVec<T>::unpack(v, f);
#pragma unroll
    for (int e = 0; e < N; ++e) widen(f[e]);
  };
  tu4 held[kHeld];
  const bool tiny = cols < N;              // less than a vector: element by element
  if (!tiny) {
    tile_for<kHeld>([&](auto K) {
      constexpr int k = decltype(K)::value;
      if (k * TPR * N < cols) held[k] = load((k * TPR + t) * N);
    });
    tile_for<kHeld>([&](auto K) {
      constexpr int k = decltype(K)::value;
      if (k * TPR * N < cols) widen_all(held[k]);
    });
#pragma unroll 1
    for (int c = (kHeld * TPR + t) * N; c < cols; c += TPR * N) widen_all(load(c));
  } else {
    for (int c = 0; c < cols; ++c) widen(element(row, c));
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off, 64));
  if constexpr (TPR == 256) {
    __syncthreads();
    if ((t & 63) == 0) part[t >> 6] = mx;
    __syncthreads();
    mx = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
  }
  const bool bad = mx == __builtin_inff();
  float s = mx / 127.f;
  if (s == 0.f) s = 1.f;
  // (a subnormal scale has no float32 reciprocal: every quotient is divided)
  const float inv = s >= 0x1p-120f ? 1.f / s : __builtin_nanf("");
  auto store = [&](const tu4& v, int c) {
    float f[N];
    uint32_t w[N / 4];
    RowVec<T>::unpack(v, f);
    quotients<N>(f, s, inv, w);
    if (bad || c >= cols)
#pragma unroll
      for (int e = 0; e < N / 4; ++e) w[e] = 0;
    if (c + N <= cols || c >= cols) {
      if (c < width) put(c, w);
      return;
    }
    // the row's end: the vector starts at cols - N
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int col = cols - N + e;
      if (col >= c) put1(col, (uint8_t)(w[e / 4] >> (8 * (e & 3))));
      if (col + N < c + N && col + N >= cols) put1(col + N, (uint8_t)0);
    }
  };
  if (!tiny) {
    tile_for<kHeld>([&](auto K) {
      constexpr int k = decltype(K)::value;
      if (k * TPR * N < width) store(k * TPR * N < cols ? held[k] : tu4{}, (k * TPR + t) * N);
    });
#pragma unroll 1
    for (int c = (kHeld * TPR + t) * N; c < width; c += TPR * N)
      store(c < cols ? load(c) : tu4{}, c);
  } else {
    for (int c = t; c < width; c += TPR) {
      float q = 0.f;
      if (c < cols && !bad) q = fminf(fmaxf(rintf(element(row, c) / s), -127.f), 127.f);
      put1(c, (uint8_t)(int8_t)(int)q);
    }
  }
  return bad ? __builtin_nanf("") : s;
}

// (one row per TPR threads and no loop over rows: hoisted out of one, the columns'
// masks and offsets take 240 registers)
template <typename T, int TPR>
__global__ __launch_bounds__(256) void quantize_rows_kernel(
    const T* __restrict__ x, int64_t rows, int cols, int64_t ldx, int8_t* __restrict__ q,
    int pitch, float* __restrict__ scale) {
  const int t = threadIdx.x % TPR;
  __shared__ float part[4];
  const int64_t r = (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
  if (r >= rows) return;                   // (whole waves; TPR = 256: never)
  int8_t* const out = q + r * pitch;
  const float s = quantize_row<T, TPR>(x + r * ldx, cols, pitch, t, part,
                                       [&](int c, const uint32_t* w) {
    if constexpr (RowVec<T>::N == 4)
      *reinterpret_cast<uint32_t*>(out + c) = w[0];
    else
      *reinterpret_cast<tu2*>(out + c) = tu2{w[0], w[1]};
  }, [&](int c, uint8_t b) { out[c] = (int8_t)b; });
  if (t == 0) scale[r] = s;
}

// Four values a thread, the row's scale beside them; bound by memory: 131 072 x 4096
// to float32 504 us, 5.3 TB/s of 1 byte in and 4 out (a large copy: 4.9); to bfloat16 317
// us, 5.1.
template <bool BF16>
__global__ __launch_bounds__(256) void dequantize_rows_kernel(
    const int8_t* __restrict__ q, int64_t pitch, const float* __restrict__ scale, int64_t rows,
    int64_t cols, void* __restrict__ out, int64_t ldo) {
  const int lane = threadIdx.x & 63;
  for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < rows;
       r += (int64_t)gridDim.x * 4) {
    const float s = scale[r];
    for (int64_t c = lane * 4; c < cols; c += 256) {
      // (values are readable in whole 16 bytes)
      const uint32_t w = *reinterpret_cast<const uint32_t*>(q + r * pitch + c);
      float f[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = (float)(int8_t)(w >> (8 * e)) * s;
      if constexpr (BF16) {
        uint16_t h[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) h[e] = __builtin_bit_cast(uint16_t, (__bf16)f[e]);
        uint16_t* o = static_cast<uint16_t*>(out) + r * ldo + c;
        if (c + 4 <= cols) {
          *reinterpret_cast<tu2_any*>(o) =
              tu2_any{h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16};
        } else {
#pragma unroll
          for (int e = 0; e < 3; ++e)
            if (c + e < cols) o[e] = h[e];
        }
      } else {
        float* o = static_cast<float*>(out) + r * ldo + c;
        if (c + 4 <= cols) {
          *reinterpret_cast<tu4_any*>(o) =
              tu4_any{__builtin_bit_cast(uint32_t, f[0]), __builtin_bit_cast(uint32_t, f[1]),
                      __builtin_bit_cast(uint32_t, f[2]), __builtin_bit_cast(uint32_t, f[3])};
        } else {
#pragma unroll
          for (int e = 0; e < 3; ++e)
            if (c + e < cols) o[e] = f[e];
        }
      }
    }
  }
}

// ---- the product ------------------------------------------------------------------
struct Int8Args {
  TileOperand a, b;                // channels of w, rows of x
  int64_t m, n;
  int steps;
  uint32_t tiles_m, tiles_n;
  const float *sx, *sw, *bias;
  void* out;
  int64_t ldo;
};

template <typename C, bool BF16>
__global__ __launch_bounds__(256, C::kLds > 80 * 1024 ? 1 : 2) void int8_tile_kernel(Int8Args p) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const uint32_t lds = (uint32_t)reinterpret_cast<uintptr_t>(smem);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int tm, tn;
  tile_of_block(blockIdx.x, gridDim.x, p.tiles_m, p.tiles_n, tm, tn);
  const int64_t m0 = (int64_t)tm * C::BM, n0 = (int64_t)tn * C::BN;
  // channel t's scale and bias at thread t, a row's scale at its lane
  const int half = lane >> 5, col = lane & 31;
  const int mw = (wave / C::WGN) * C::WM * 32, nw = (wave % C::WGN) * C::WN * 32;
  float sx[C::WN], sw_here = 0.f, bias_here = 0.f;
#pragma unroll
  for (int j = 0; j < C::WN; ++j) {
    const int64_t n = n0 + nw + j * 32 + col;
    sx[j] = n < p.n ? p.sx[n] : 0.f;
  }
  if (threadIdx.x < C::BM && m0 + threadIdx.x < p.m) {
    sw_here = p.sw[m0 + threadIdx.x];
    if (p.bias) bias_here = p.bias[m0 + threadIdx.x];
  }
  ti16 acc[C::WM][C::WN];
  tile_loop<C>(p.a, p.b, m0, n0, 0, p.steps, 1, lds, lane, wave, acc);
  typedef typename std::conditional<BF16, AsBf16, AsF32>::type As;
  typedef typename As::T T;
  float* ssw = reinterpret_cast<float*>(smem + kTileRowsLds<C, As>);    // [2][BM]
  if (threadIdx.x < C::BM) {
    ssw[threadIdx.x] = sw_here;
    ssw[C::BM + threadIdx.x] = bias_here;
  }
  __syncthreads();
  tf4 sw[C::WM][4], bias[C::WM][4];
#pragma unroll
  for (int i = 0; i < C::WM; ++i)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float* mine = ssw + mw + 4 * half + i * 32 + 8 * q;
      sw[i][q] = *reinterpret_cast<const tf4*>(mine);
      bias[i][q] = *reinterpret_cast<const tf4*>(mine + C::BM);
    }
  auto value = [&](auto I, auto J, auto Q, float (&v)[4]) {
    constexpr int i = decltype(I)::value, j = decltype(J)::value, q = decltype(Q)::value;
#pragma unroll
    for (int r = 0; r < 4; ++r)
      v[r] = (float)acc_get(acc[i][j], 4 * q + r) * (sx[j] * sw[i][q][r]) + bias[i][q][r];
  };
  tile_rows<C, As>(smem, lane, wave, value, [&](int n, int m, const tu4& piece) {
    if (n0 + n < p.n && m0 + m < p.m)
      store_piece(static_cast<T*>(p.out) + (n0 + n) * p.ldo + m0 + m, p.m - m0 - m, piece);
  });
}

template <typename C, bool BF16>
int launch_int8(const Int8Args& a, hipStream_t s) {
  constexpr int epi =
      kTileRowsLds<C, typename std::conditional<BF16, AsBf16, AsF32>::type> + C::BM * 8;
  constexpr int lds = C::kLds > epi ? C::kLds : epi;
  static_assert(lds <= 160 * 1024, "LDS of a CU");
  Int8Args p = a;
  p.tiles_m = (uint32_t)((p.m + C::BM - 1) / C::BM);
  p.tiles_n = (uint32_t)((p.n + C::BN - 1) / C::BN);
  const int64_t wgs = (int64_t)p.tiles_m * p.tiles_n;
  ZS_REQUIRE(wgs <= kMaxWorkgroups, "zshmc_int8_linear: %lld tiles, more than one launch takes",
             (long long)wgs);
  static thread_local int attr_dev = -1;
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) dev = 0;
  if (attr_dev != dev) {
    const hipError_t e = hipFuncSetAttribute(
        reinterpret_cast<const void*>(int8_tile_kernel<C, BF16>),
        hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return check_hip(e, "hipFuncSetAttribute(LDS)");
    attr_dev = dev;
  }
  hipLaunchKernelGGL((int8_tile_kernel<C, BF16>), dim3((unsigned)wgs), dim3(256), lds, s, p);
  ZS_LAUNCH_CHECK("int8_tile_kernel launch");
  return ZSHMC_OK;
}

using BigI8 = TileCfg<MmaI8, 2, 2, 4, 4, false, false>;
using FewI8 = TileCfg<MmaI8, 4, 1, 1, 1, false, false>;
using MidI8 = TileCfg<MmaI8, 2, 2, 2, 2, false, false>;

unsigned rows_grid(int64_t rows) {
  const int64_t b = (rows + 3) / 4;
  return (unsigned)(b > 65536 ? 65536 : b);
}

}  // namespace
}  // namespace zshmc

using namespace zshmc;

namespace {
int launch_quantize(const void* x, int64_t n_rows, int64_t n_cols, int64_t ldx, int dtype,
                    int8_t* values, int64_t pitch, float* scale, hipStream_t s) {
  // a wave per row where that is eight waves a CU or more
  const bool wave = n_rows >= 8ll * device_cu_count();
  // (in launches of at most 2^25 rows, see kMaxWorkgroups)
  constexpr int64_t kRows = 1ll << 25;
  for (int64_t r = 0; r < n_rows; r += kRows) {
    const int64_t rows = n_rows - r < kRows ? n_rows - r : kRows;
    const unsigned grid = (unsigned)(wave ? (rows + 3) / 4 : rows);
    auto launch = [&](auto* f) {
      typedef typename std::remove_cv<typename std::remove_pointer<decltype(f)>::type>::type T;
      if (wave)
        hipLaunchKernelGGL((quantize_rows_kernel<T, 64>), dim3(grid), dim3(256), 0, s,
                           f + r * ldx, rows, (int)n_cols, ldx, values + r * pitch, (int)pitch,
                           scale + r);
      else
        hipLaunchKernelGGL((quantize_rows_kernel<T, 256>), dim3(grid), dim3(256), 0, s,
                           f + r * ldx, rows, (int)n_cols, ldx, values + r * pitch, (int)pitch,
                           scale + r);
    };
    if (dtype == ZSHMC_DTYPE_F32)
      launch(static_cast<const float*>(x));
    else
      launch(static_cast<const uint16_t*>(x));
    ZS_LAUNCH_CHECK("quantize_rows_kernel launch");
  }
  return ZSHMC_OK;
}

int check_linear(int64_t n_rows, int64_t n_features, int64_t n_channels, const int8_t* w,
                 int64_t w_pitch, const void* out, int64_t ldo, int dtype, const char* who) {
  ZS_REQUIRE(dtype == ZSHMC_DTYPE_F32 || dtype == ZSHMC_DTYPE_BF16,
             "%s: dtype must be ZSHMC_DTYPE_F32 or _BF16, got %d", who, dtype);
  ZS_REQUIRE(n_rows >= 0 && n_channels > 0 && n_features > 0 && n_features <= 131072,
             "%s: n_rows >= 0, n_channels > 0, 1 .. 131072 features (an int32 holds the sum), "
             "got %lld", who, (long long)n_features);
  ZS_REQUIRE(w_pitch >= (n_features + 15) / 16 * 16 && w_pitch % 16 == 0 &&
                 w_pitch <= (4ll << 20) && (reinterpret_cast<uintptr_t>(w) & 15) == 0 &&
                 ldo >= n_channels,
             "%s: rows of whole 16 bytes, 16-byte aligned; ldo >= n_channels", who);
  ZS_REQUIRE(n_rows < (1ll << 31) && n_channels < (1ll << 31),
             "%s: at most 2^31 - 1 rows and channels", who);
  return ZSHMC_OK;
}

// the product of 8-bit rows
int product(const int8_t* x, int64_t x_pitch, const float* x_scale, const int8_t* w,
            int64_t w_pitch, const float* w_scale, const float* bias, int64_t n_rows,
            int64_t n_features, int64_t n_channels, void* out, int64_t ldo, bool bf16,
            hipStream_t s) {
  const int64_t bytes = (n_features + 15) / 16 * 16;
  Int8Args a{};
  a.a = TileOperand{reinterpret_cast<const unsigned char*>(w), w_pitch, 0, n_channels, bytes};
  a.b = TileOperand{reinterpret_cast<const unsigned char*>(x), x_pitch, 0, n_rows, bytes};
  a.m = n_channels;
  a.n = n_rows;
  a.steps = (int)((bytes + 127) / 128);
  a.sx = x_scale;
  a.sw = w_scale;
  a.bias = bias;
  a.out = out;
  a.ldo = ldo;
  if (n_rows <= 32)
    return bf16 ? launch_int8<FewI8, true>(a, s) : launch_int8<FewI8, false>(a, s);
  if (plan_tiles(n_channels, n_rows, a.steps, false, device_cu_count()).big)
    return bf16 ? launch_int8<BigI8, true>(a, s) : launch_int8<BigI8, false>(a, s);
  return bf16 ? launch_int8<MidI8, true>(a, s) : launch_int8<MidI8, false>(a, s);
}
}  // namespace

extern "C" int zshmc_quantize_rows(const void* x, int64_t n_rows, int64_t n_cols, int64_t ldx,
                                   int dtype, int8_t* values, int64_t pitch, float* scale,
                                   void* stream) {
  ZS_REQUIRE(dtype == ZSHMC_DTYPE_F32 || dtype == ZSHMC_DTYPE_BF16,
             "zshmc_quantize_rows: dtype must be ZSHMC_DTYPE_F32 or _BF16, got %d", dtype);
  ZS_REQUIRE(n_rows >= 0 && n_rows < (1ll << 31) && n_cols > 0 && n_cols < (1ll << 30) &&
                 pitch < (1ll << 30) && ldx >= n_cols,
             "zshmc_quantize_rows: 0 .. 2^31 - 1 rows, 1 .. 2^30 - 1 columns, ldx >= n_cols");
  ZS_REQUIRE(pitch >= n_cols && pitch % 16 == 0 && (reinterpret_cast<uintptr_t>(values) & 15) == 0,
             "zshmc_quantize_rows: values 16-byte aligned with a pitch of whole 16 bytes");
  if (n_rows == 0) return ZSHMC_OK;
  ZS_REQUIRE(x && values && scale, "zshmc_quantize_rows: null pointer");
  return launch_quantize(x, n_rows, n_cols, ldx, dtype, values, pitch, scale,
                         reinterpret_cast<hipStream_t>(stream));
}

extern "C" int zshmc_dequantize_rows(const int8_t* values, int64_t pitch, const float* scale,
                                     int64_t n_rows, int64_t n_cols, void* out, int64_t ldo,
                                     int dtype, void* stream) {
  ZS_REQUIRE(dtype == ZSHMC_DTYPE_F32 || dtype == ZSHMC_DTYPE_BF16,
             "zshmc_dequantize_rows: dtype must be ZSHMC_DTYPE_F32 or _BF16, got %d", dtype);
  ZS_REQUIRE(n_rows >= 0 && n_cols > 0 && pitch >= n_cols && ldo >= n_cols && pitch % 16 == 0 &&
                 (reinterpret_cast<uintptr_t>(values) & 15) == 0,
             "zshmc_dequantize_rows: n_rows >= 0, n_cols > 0, ldo >= n_cols, values 16-byte "
             "aligned with a pitch of whole 16 bytes");
  if (n_rows == 0) return ZSHMC_OK;
  ZS_REQUIRE(values && scale && out, "zshmc_dequantize_rows: null pointer");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == ZSHMC_DTYPE_F32)
    hipLaunchKernelGGL(dequantize_rows_kernel<false>, dim3(rows_grid(n_rows)), dim3(256), 0, s,
                       values, pitch, scale, n_rows, n_cols, out, ldo);
  else
    hipLaunchKernelGGL(dequantize_rows_kernel<true>, dim3(rows_grid(n_rows)), dim3(256), 0, s,
                       values, pitch, scale, n_rows, n_cols, out, ldo);
  ZS_LAUNCH_CHECK("dequantize_rows_kernel launch");
  return ZSHMC_OK;
}

extern "C" int zshmc_int8_linear(const int8_t* x, int64_t x_pitch, const float* x_scale,
                                 const int8_t* w, int64_t w_pitch, const float* w_scale,
                                 const float* bias, int64_t n_rows, int64_t n_features,
                                 int64_t n_channels, void* out, int64_t ldo, int dtype,
                                 void* stream) {
  const int rc = check_linear(n_rows, n_features, n_channels, w, w_pitch, out, ldo, dtype,
                              "zshmc_int8_linear");
  if (rc != ZSHMC_OK) return rc;
  ZS_REQUIRE(x_pitch >= (n_features + 15) / 16 * 16 && x_pitch % 16 == 0 &&
                 x_pitch <= (4ll << 20) && (reinterpret_cast<uintptr_t>(x) & 15) == 0,
             "zshmc_int8_linear: rows of whole 16 bytes, 16-byte aligned");
  if (n_rows == 0) return ZSHMC_OK;
  ZS_REQUIRE(x && w && x_scale && w_scale && out, "zshmc_int8_linear: null pointer");
  return product(x, x_pitch, x_scale, w, w_pitch, w_scale, bias, n_rows, n_features, n_channels,
                 out, ldo, dtype == ZSHMC_DTYPE_BF16, reinterpret_cast<hipStream_t>(stream));
}

extern "C" int zshmc_quantized_linear(const void* x, int64_t ldx, int x_dtype, const int8_t* w,
                                      int64_t w_pitch, const float* w_scale, const float* bias,
                                      int64_t n_rows, int64_t n_features, int64_t n_channels,
                                      void* out, int64_t ldo, int dtype, void* workspace,
                                      int64_t workspace_bytes, void* stream) {
  const int rc = check_linear(n_rows, n_features, n_channels, w, w_pitch, out, ldo, dtype,
                              "zshmc_quantized_linear");
  if (rc != ZSHMC_OK) return rc;
  ZS_REQUIRE(x_dtype == ZSHMC_DTYPE_F32 || x_dtype == ZSHMC_DTYPE_BF16,
             "zshmc_quantized_linear: x_dtype must be ZSHMC_DTYPE_F32 or _BF16, got %d", x_dtype);
  ZS_REQUIRE(ldx >= n_features, "zshmc_quantized_linear: rows overlap (ldx < n_features)");
  if (n_rows == 0) return ZSHMC_OK;
  ZS_REQUIRE(x && w && w_scale && out, "zshmc_quantized_linear: null pointer");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const bool bf16 = dtype == ZSHMC_DTYPE_BF16;
  const int64_t pitch = (n_features + 127) / 128 * 128;
  ZS_REQUIRE(workspace && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0 &&
                 workspace_bytes >= n_rows * (pitch + 4),
             "zshmc_quantized_linear: n_rows * (n_features rounded up to 128, + 4) bytes of "
             "16-byte aligned workspace needed, got %lld", (long long)workspace_bytes);
  int8_t* q = static_cast<int8_t*>(workspace);
  float* scale = reinterpret_cast<float*>(q + n_rows * pitch);
  const int rq = launch_quantize(x, n_rows, n_features, ldx, x_dtype, q, pitch, scale, s);
  if (rq != ZSHMC_OK) return rq;
  return product(q, pitch, scale, w, w_pitch, w_scale, bias, n_rows, n_features, n_channels, out,
                 ldo, bf16, s);
}
