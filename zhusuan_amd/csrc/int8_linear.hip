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
// otherwise.
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

// the 16 bytes from column c on, zero from `cols` on
template <typename T>
__device__ __forceinline__ tu4 load_row(const T* row, int64_t c, int64_t cols) {
  constexpr int N = RowVec<T>::N;
  if (c + N <= cols) return *reinterpret_cast<const tu4_any*>(row + c);
  tu4 v{};
#pragma unroll
  for (int e = 0; e < N; ++e)
    if (c + e < cols) {
      if constexpr (N == 4)
        v[e] = __builtin_bit_cast(uint32_t, row[c + e]);
      else
        v[e / 2] |= (uint32_t)row[c + e] << (16 * (e & 1));
    }
  return v;
}

// rint(x / s), x / s rounded to float32 first: a product with the reciprocal
// says which integer unless it falls within 2^-12 of the middle of two (its error
// is below 127 * 3 * 2^-24), then the division does.
__device__ __forceinline__ float quotient(float x, float s, float inv) {
  const float t = x * inv;
  float q = rintf(t);
  if (fabsf(t - q) > 0.5f - 0x1p-12f) q = rintf(x / s);
  return fminf(fmaxf(q, -127.f), 127.f);
}

template <typename T, int TPR>
__global__ __launch_bounds__(256) void quantize_rows_kernel(
    const T* __restrict__ x, int64_t rows, int64_t cols, int64_t ldx, int8_t* __restrict__ q,
    int64_t pitch, float* __restrict__ scale) {
  constexpr int N = RowVec<T>::N, RPB = 256 / TPR;
  const int t = threadIdx.x % TPR;
  __shared__ float part[4];
  for (int64_t r = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR; r < rows;
       r += (int64_t)gridDim.x * RPB) {
    const T* row = x + r * ldx;
    tu4 held[kHeld];
    float mx = 0.f;
    auto widen = [&](const tu4& v) {
      float f[N];
      RowVec<T>::unpack(v, f);
      // a NaN or an infinity turns into a maximum no finite row reaches
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float a = fabsf(f[e]);
        mx = a <= 3.402823466e38f ? fmaxf(mx, a) : __builtin_inff();
      }
    };
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
      held[k] = tu4{};
      const int64_t c = (int64_t)(k * TPR + t) * N;
      if (c < cols) held[k] = load_row(row, c, cols);
    }
#pragma unroll
    for (int k = 0; k < kHeld; ++k) widen(held[k]);
    for (int64_t c = (int64_t)(kHeld * TPR + t) * N; c < cols; c += TPR * N)
      widen(load_row(row, c, cols));
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
    if (t == 0) scale[r] = bad ? __builtin_nanf("") : s;
    // (a subnormal scale has no float32 reciprocal: every quotient is divided)
    const float inv = s >= 0x1p-120f ? 1.f / s : __builtin_nanf("");
    auto store = [&](const tu4& v, int64_t c) {
      float f[N];
      RowVec<T>::unpack(v, f);
      uint32_t w[N / 4];
#pragma unroll
      for (int e = 0; e < N; ++e) {
        float n = inv == inv ? quotient(f[e], s, inv)
                             : fminf(fmaxf(rintf(f[e] / s), -127.f), 127.f);
        n = bad ? 0.f : n;
        const uint32_t b = (uint32_t)(int)n & 0xffu;
        w[e / 4] = e % 4 == 0 ? b : w[e / 4] | b << (8 * (e % 4));
      }
      if constexpr (N == 4)
        *reinterpret_cast<uint32_t*>(q + r * pitch + c) = w[0];
      else
        *reinterpret_cast<tu2*>(q + r * pitch + c) = tu2{w[0], w[1]};
    };
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
      const int64_t c = (int64_t)(k * TPR + t) * N;
      if (c < pitch) store(held[k], c);
    }
    for (int64_t c = (int64_t)(kHeld * TPR + t) * N; c < pitch; c += TPR * N)
      store(c < cols ? load_row(row, c, cols) : tu4{}, c);
  }
}

// 8 values per thread
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
  typedef typename std::conditional<BF16, uint16_t, float>::type T;
  float* ssw = reinterpret_cast<float*>(smem + kTileRowsLds<C, T>);     // [2][BM]
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
  tile_rows<C, T>(smem, lane, wave, value, [&](int n, int m, const tu4& piece) {
    if (n0 + n < p.n && m0 + m < p.m)
      store_piece(static_cast<T*>(p.out) + (n0 + n) * p.ldo + m0 + m, p.m - m0 - m, piece);
  });
}

template <typename C, bool BF16>
int launch_int8(const Int8Args& a, hipStream_t s) {
  constexpr int epi =
      kTileRowsLds<C, typename std::conditional<BF16, uint16_t, float>::type> + C::BM * 8;
  constexpr int lds = C::kLds > epi ? C::kLds : epi;
  static_assert(lds <= 160 * 1024, "LDS of a CU");
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
  Int8Args p = a;
  p.tiles_m = (uint32_t)((p.m + C::BM - 1) / C::BM);
  p.tiles_n = (uint32_t)((p.n + C::BN - 1) / C::BN);
  const int64_t wgs = (int64_t)p.tiles_m * p.tiles_n;
  ZS_REQUIRE(wgs < (1ll << 31), "zshmc_int8_linear: %lld tiles", (long long)wgs);
  hipLaunchKernelGGL((int8_tile_kernel<C, BF16>), dim3((unsigned)wgs), dim3(256), lds, s, p);
  ZS_LAUNCH_CHECK("int8_tile_kernel launch");
  return ZSHMC_OK;
}

using BigI8 = TileCfg<MmaI8, 2, 2, 4, 4, false, false>;
using MidI8 = TileCfg<MmaI8, 2, 2, 2, 2, false, false>;
using FewI8 = TileCfg<MmaI8, 4, 1, 1, 1, false, false>;

unsigned rows_grid(int64_t rows) {
  const int64_t b = (rows + 3) / 4;
  return (unsigned)(b > 65536 ? 65536 : b);
}

}  // namespace
}  // namespace zshmc

using namespace zshmc;

extern "C" int zshmc_quantize_rows(const void* x, int64_t n_rows, int64_t n_cols, int64_t ldx,
                                   int dtype, int8_t* values, int64_t pitch, float* scale,
                                   void* stream) {
  ZS_REQUIRE(dtype == ZSHMC_DTYPE_F32 || dtype == ZSHMC_DTYPE_BF16,
             "zshmc_quantize_rows: dtype must be ZSHMC_DTYPE_F32 or _BF16, got %d", dtype);
  ZS_REQUIRE(n_rows >= 0 && n_cols > 0 && ldx >= n_cols,
             "zshmc_quantize_rows: n_rows >= 0, n_cols > 0, ldx >= n_cols");
  ZS_REQUIRE(pitch >= n_cols && pitch % 16 == 0 && (reinterpret_cast<uintptr_t>(values) & 15) == 0,
             "zshmc_quantize_rows: values 16-byte aligned with a pitch of whole 16 bytes");
  if (n_rows == 0) return ZSHMC_OK;
  ZS_REQUIRE(x && values && scale, "zshmc_quantize_rows: null pointer");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  // a wave per row where that is eight waves a CU or more
  const bool wave = n_rows >= 8ll * device_cu_count();
  const unsigned grid = wave ? rows_grid(n_rows)
                             : (unsigned)n_rows;
  if (dtype == ZSHMC_DTYPE_F32) {
    const float* f = static_cast<const float*>(x);
    if (wave)
      hipLaunchKernelGGL((quantize_rows_kernel<float, 64>), dim3(grid), dim3(256), 0, s, f, n_rows,
                         n_cols, ldx, values, pitch, scale);
    else
      hipLaunchKernelGGL((quantize_rows_kernel<float, 256>), dim3(grid), dim3(256), 0, s, f,
                         n_rows, n_cols, ldx, values, pitch, scale);
  } else {
    const uint16_t* f = static_cast<const uint16_t*>(x);
    if (wave)
      hipLaunchKernelGGL((quantize_rows_kernel<uint16_t, 64>), dim3(grid), dim3(256), 0, s, f,
                         n_rows, n_cols, ldx, values, pitch, scale);
    else
      hipLaunchKernelGGL((quantize_rows_kernel<uint16_t, 256>), dim3(grid), dim3(256), 0, s, f,
                         n_rows, n_cols, ldx, values, pitch, scale);
  }
  ZS_LAUNCH_CHECK("quantize_rows_kernel launch");
  return ZSHMC_OK;
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
  ZS_REQUIRE(dtype == ZSHMC_DTYPE_F32 || dtype == ZSHMC_DTYPE_BF16,
             "zshmc_int8_linear: dtype must be ZSHMC_DTYPE_F32 or _BF16, got %d", dtype);
  ZS_REQUIRE(n_rows >= 0 && n_channels > 0 && n_features > 0 && n_features <= 131072,
             "zshmc_int8_linear: n_rows >= 0, n_channels > 0, 1 .. 131072 features (an int32 "
             "holds the sum), got %lld", (long long)n_features);
  const int64_t bytes = (n_features + 15) / 16 * 16;
  ZS_REQUIRE(x_pitch >= bytes && w_pitch >= bytes && x_pitch % 16 == 0 && w_pitch % 16 == 0 &&
                 x_pitch <= (4ll << 20) && w_pitch <= (4ll << 20) &&
                 (reinterpret_cast<uintptr_t>(x) & 15) == 0 &&
                 (reinterpret_cast<uintptr_t>(w) & 15) == 0 && ldo >= n_channels,
             "zshmc_int8_linear: rows of whole 16 bytes, 16-byte aligned; ldo >= n_channels");
  ZS_REQUIRE(n_rows < (1ll << 31) && ldo < (1ll << 22),
             "zshmc_int8_linear: at most 2^31 - 1 rows and 2^22 - 1 channels");
  if (n_rows == 0) return ZSHMC_OK;
  ZS_REQUIRE(x && w && x_scale && w_scale && out, "zshmc_int8_linear: null pointer");
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
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const bool bf16 = dtype == ZSHMC_DTYPE_BF16;
  const int64_t big = ((n_rows + 255) / 256) * ((n_channels + 255) / 256);
  if (n_rows <= 32)
    return bf16 ? launch_int8<FewI8, true>(a, s) : launch_int8<FewI8, false>(a, s);
  if (big >= device_cu_count())
    return bf16 ? launch_int8<BigI8, true>(a, s) : launch_int8<BigI8, false>(a, s);
  return bf16 ? launch_int8<MidI8, true>(a, s) : launch_int8<MidI8, false>(a, s);
}
