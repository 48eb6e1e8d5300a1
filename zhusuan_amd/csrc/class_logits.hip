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
// logits again, turned into r in the epilogue (bfloat16, or three bfloat16
// planes for float32 operands), then the two products over that piece; dX is
// accumulated in float32 over the pieces.  8 N V D flop for both directions,
// six of them unavoidable.  M and S are float32; r is rounded to the operands'
// precision because it is an operand of the matrix cores.
#include "tile_gemm.h"

namespace zshmc {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
typedef float cf2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float fast_exp(float x) {
  return __builtin_amdgcn_exp2f(x * kLog2e);
}
__device__ __forceinline__ uint16_t bf16_bits(float x) {
  return __builtin_bit_cast(uint16_t, (__bf16)x);
}
__device__ __forceinline__ float bf16_value(uint16_t b) {
  return __builtin_bit_cast(float, (uint32_t)b << 16);
}

// ---- operands as the tile loop wants them ------------------------------------
// rows of `cols` elements -> bfloat16 rows of `pitch` bytes, zero behind the
// last column; float32 becomes three planes.  Rows whose label is `ignore`
// become zeros (whatever they hold, NaN included, reaches no product).
template <bool F32>
__global__ void pack_rows_kernel(const void* __restrict__ src, int64_t rows, int64_t cols,
                                 int64_t ld, unsigned char* __restrict__ dst, int64_t pitch,
                                 int64_t plane, const int64_t* __restrict__ labels,
                                 int64_t ignore) {
  const int64_t groups = pitch / 16;
  const int64_t total = rows * groups;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / groups, c = (i - r * groups) * 8;
    const bool out = labels && labels[r] == ignore;
    uint16_t p[3][8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const bool in = !out && c + e < cols;
      if constexpr (F32) {
        const float v = in ? static_cast<const float*>(src)[r * ld + c + e] : 0.f;
        p[0][e] = bf16_bits(v);
        const float v1 = v - bf16_value(p[0][e]);
        p[1][e] = bf16_bits(v1);
        p[2][e] = bf16_bits(v1 - bf16_value(p[1][e]));
      } else {
        p[0][e] = in ? static_cast<const uint16_t*>(src)[r * ld + c + e] : (uint16_t)0;
      }
    }
#pragma unroll
    for (int k = 0; k < (F32 ? 3 : 1); ++k) {
      tu4 v;
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] = p[k][2 * q] | (uint32_t)p[k][2 * q + 1] << 16;
      *reinterpret_cast<tu4*>(dst + k * plane + r * pitch + c * 2) = v;
    }
  }
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
  unsigned char* resid;            // r: [plane][n][ld] bfloat16
  int64_t resid_pitch, resid_plane;
  float* bias_part;                // [tiles_n][bias_ld], or NULL
  int64_t bias_ld;
  // kEpiStore
  void* out;
  int64_t out_ld, out_split;       // elements; split s at out + s * out_split
  int out_bf16, accumulate;
};

// LDS that the epilogue's exchange takes (the biases and their column sums sit
// behind it)
template <typename C, int EPI>
constexpr int kEpiLds = EPI == kEpiResidual ? C::BN * (C::BM * 2 + 16)
                        : EPI == kEpiStats  ? C::WGM * C::BN * 8
                                            : 0;

template <typename C, int EPI, bool F32>
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
  typename C::MMA::Acc acc[C::WM][C::WN];
  if (steps > 0) {
    tile_loop<C>(p.a, p.b, m0, n0, k0, steps, p.terms, lds, lane, wave, acc);
  } else {
#pragma unroll
    for (int i = 0; i < C::WM; ++i)
#pragma unroll
      for (int j = 0; j < C::WN; ++j) acc[i][j] = typename C::MMA::Acc{};
  }

  const int wm = wave / C::WGN, wn = wave % C::WGN;
  const int half = lane >> 5, col = lane & 31;
  const int mw = wm * C::WM * 32, nw = wn * C::WN * 32;

  if constexpr (EPI == kEpiStore) {
    const int64_t at = (int64_t)blockIdx.y * p.out_split + (m0 + mw) * p.out_ld + n0 + nw;
    const int ld = (int)p.out_ld;
    const int rows = p.m - m0 - mw < C::BM ? (int)(p.m - m0 - mw) : C::BM;
    const int cols = p.n - n0 - nw < C::BN ? (int)(p.n - n0 - nw) : C::BN;
#pragma unroll
    for (int i = 0; i < C::WM; ++i)
#pragma unroll
      for (int j = 0; j < C::WN; ++j) {
        const int c = j * 32 + col;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int m = i * 32 + acc_row(r, half);
          const float v = acc_get(acc[i][j], r);
          if (m >= rows || c >= cols) continue;
          const int o = m * ld + c;
          if (p.out_bf16) {
            (static_cast<uint16_t*>(p.out) + at)[o] = bf16_bits(v);
          } else {
            float* q = static_cast<float*>(p.out) + at + o;
            *q = p.accumulate ? *q + v : v;
          }
        }
      }
    return;
  } else {
    // the tile's biases, -inf behind the last class; they stay in the LDS
    // beside what follows
    float* sbias = reinterpret_cast<float*>(smem + kEpiLds<C, EPI>);
    for (int i = threadIdx.x; i < C::BM; i += 256) {
      const int64_t v = m0 + i;
      sbias[i] = v < p.m ? (p.bias ? p.bias[v] : 0.f) : -__builtin_inff();
    }
    __syncthreads();
    const float* sb = sbias + mw + 4 * half;
    if constexpr (EPI == kEpiStats) {
      cf2* red = reinterpret_cast<cf2*>(smem);               // [WGM][BN]
#pragma unroll
      for (int j = 0; j < C::WN; ++j) {
        const int64_t n = n0 + nw + j * 32 + col;
        int64_t y = -1;
        if (n < p.n) y = p.labels[n] - m0 - mw;
        const int yl = y >= 0 && y < C::WM * 32 && y + m0 + mw < p.m ? (int)y : -1;
        float mx = -__builtin_inff();
        float picked = 0.f;
#pragma unroll
        for (int i = 0; i < C::WM; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const tf4 b = *reinterpret_cast<const tf4*>(sb + i * 32 + 8 * q);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float l = acc_get(acc[i][j], 4 * q + r) + b[r];
              mx = fmaxf(mx, l);
              if (yl == i * 32 + acc_row(4 * q + r, half)) picked = l;
            }
          }
        if (yl >= 0 && ((yl >> 2) & 1) == half) p.label_logit[n] = picked;
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float off = mx == -__builtin_inff() ? 0.f : mx;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < C::WM; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const tf4 b = *reinterpret_cast<const tf4*>(sb + i * 32 + 8 * q);
#pragma unroll
            for (int r = 0; r < 4; ++r) s += fast_exp((acc_get(acc[i][j], 4 * q + r) + b[r]) - off);
          }
        s += __shfl_xor(s, 32, 64);
        if (half == 0) red[wm * C::BN + nw + j * 32 + col] = cf2{mx, s};
      }
      __syncthreads();
      for (int i = threadIdx.x; i < C::BN; i += 256) {
        if (n0 + i >= p.n) continue;
        cf2 t = red[i];
#pragma unroll
        for (int k = 1; k < C::WGM; ++k) {
          const cf2 u = red[k * C::BN + i];
          const float mx = fmaxf(t[0], u[0]);
          const float off = mx == -__builtin_inff() ? 0.f : mx;
          t = cf2{mx, t[1] * fast_exp(t[0] - off) + u[1] * fast_exp(u[0] - off)};
        }
        p.part[(int64_t)tm * p.n + n0 + i] = t;
      }
    } else {
      // what a row of X (a lane) contributes: g, -g / S, M, its label here
      float g[C::WN], ginv[C::WN], mx[C::WN];
      int yl[C::WN];
      bool zero[C::WN];
#pragma unroll
      for (int j = 0; j < C::WN; ++j) {
        const int64_t n = n0 + nw + j * 32 + col;
        g[j] = ginv[j] = mx[j] = 0.f;
        yl[j] = -1;
        zero[j] = true;
        if (n < p.n) {
          const int64_t label = p.labels[n];
          const cf2 st = p.stats[n];
          mx[j] = st[0];
          g[j] = label < 0 || label >= p.n_classes ? __builtin_nanf("") : p.g[n];
          ginv[j] = -g[j] / st[1];
          zero[j] = p.has_ignore && label == p.ignore;
          const int64_t y = label - p.class0 - m0 - mw;
          if (y >= 0 && y < C::WM * 32) yl[j] = (int)y;
        }
      }
      // The tile goes through LDS ([row of X][class], rows 16 bytes apart modulo
      // the banks) so that whole lines of r are written, one plane at a time;
      // the later planes of a float32 r compute it again rather than keep it.
      constexpr int kPitch = C::BM * 2 + 16;
      constexpr int kPlanes = F32 ? 3 : 1;
      constexpr int kChunks = C::BM / 8;
      float* scol = sbias + C::BM;                           // [WGN][BM]
#pragma unroll 1
      for (int pl = 0; pl < kPlanes; ++pl) {
        // (or the compiler keeps every label comparison across the planes)
#pragma unroll
        for (int j = 0; j < C::WN; ++j) asm volatile("" : "+v"(yl[j]));
#pragma unroll
        for (int i = 0; i < C::WM; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const tf4 b = *reinterpret_cast<const tf4*>(sb + i * 32 + 8 * q);
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < C::WN; ++j) {
              uint16_t h[4];
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                // (behind the last class l = -inf and r = 0; where the row's own r
                // is NaN, so is everything that those columns reach)
                const float l = acc_get(acc[i][j], 4 * q + r) + b[r];
                const float hit = yl[j] == i * 32 + acc_row(4 * q + r, half) ? g[j] : 0.f;
                float v = hit + ginv[j] * fast_exp(l - mx[j]);
                v = zero[j] ? 0.f : v;
                if (pl == 0) sum[r] += v;
                if (F32) {
                  const float v1 = v - bf16_value(bf16_bits(v));
                  v = pl == 0 ? v : pl == 1 ? v1 : v1 - bf16_value(bf16_bits(v1));
                }
                h[r] = bf16_bits(v);
              }
              *reinterpret_cast<tu2*>(smem + (nw + j * 32 + col) * kPitch +
                                      (mw + i * 32 + 8 * q + 4 * half) * 2) =
                  tu2{h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16};
            }
            if (pl == 0 && p.bias_part) {
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const float s = group_sum<32>(sum[r]);
                if (col == 0) scol[wn * C::BM + mw + i * 32 + acc_row(4 * q + r, half)] = s;
              }
            }
          }
        __syncthreads();
        for (int c = threadIdx.x; c < C::BN * kChunks; c += 256) {
          const int row = c / kChunks, ch = c % kChunks;
          const int64_t n = n0 + row, byte = (m0 + ch * 8) * 2;
          if (n < p.n && byte < p.resid_pitch)
            *reinterpret_cast<tu4*>(p.resid + pl * p.resid_plane + n * p.resid_pitch + byte) =
                *reinterpret_cast<const tu4*>(smem + row * kPitch + ch * 16);
        }
        if (pl == 0 && p.bias_part)
          for (int i = threadIdx.x; i < C::BM; i += 256) {
            float s = 0.f;
#pragma unroll
            for (int k = 0; k < C::WGN; ++k) s += scol[k * C::BM + i];
            if (m0 + i < p.m) p.bias_part[(int64_t)tn * p.bias_ld + p.class0 + m0 + i] = s;
          }
        if (pl + 1 < kPlanes) __syncthreads();
      }
    }
  }
}

// ---- joins ---------------------------------------------------------------------
// 16 rows x 16 lanes of parts per workgroup
__global__ __launch_bounds__(256) void join_stats_kernel(
    const cf2* __restrict__ part, int parts, const float* __restrict__ label_logit,
    const int64_t* __restrict__ labels, int64_t n, int64_t n_classes, int has_ignore,
    int64_t ignore, float* __restrict__ log_prob, cf2* __restrict__ stats) {
  const int64_t row = (int64_t)blockIdx.x * 16 + (threadIdx.x & 15);
  const int k = threadIdx.x >> 4;
  const float ninf = -__builtin_inff();
  cf2 t{ninf, 0.f};
  if (row < n)
    for (int i = k; i < parts; i += 16) {
      const cf2 u = part[(int64_t)i * n + row];
      const float mx = fmaxf(t[0], u[0]);
      const float off = mx == ninf ? 0.f : mx;
      t = cf2{mx, t[1] * fast_exp(t[0] - off) + u[1] * fast_exp(u[0] - off)};
    }
  __shared__ cf2 s[16][16];
  s[k][threadIdx.x & 15] = t;
  __syncthreads();
  if (k || row >= n) return;
  for (int i = 1; i < 16; ++i) {
    const cf2 u = s[i][threadIdx.x & 15];
    const float mx = fmaxf(t[0], u[0]);
    const float off = mx == ninf ? 0.f : mx;
    t = cf2{mx, t[1] * fast_exp(t[0] - off) + u[1] * fast_exp(u[0] - off)};
  }
  const int64_t y = labels[row];
  float lp = __builtin_nanf("");
  if (has_ignore && y == ignore)
    lp = 0.f;
  else if (y >= 0 && y < n_classes)
    lp = (label_logit[row] - t[0]) - logf(t[1]);
  log_prob[row] = lp;
  if (stats) stats[row] = t;
}

// out[i] = sum of `parts` rows of x, in order
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
  return (unsigned)(b < 1 ? 1 : b > 65536 ? 65536 : b);
}

// bytes of r that one piece of classes may take: it is written, then read by
// two products
constexpr int64_t kPieceBytes = 256ll << 20;
constexpr int64_t kMaxPitch = 4ll << 20;

struct ClassProblem {
  const void *x, *w;
  int64_t n, d, v, ldx, ldw;
  int dtype;                       // ZSHMC_F32 / ZSHMC_BF16
  bool f32() const { return dtype == ZSHMC_DTYPE_F32; }
  int64_t esize() const { return f32() ? 4 : 2; }
};

bool direct(const void* p, int64_t ld, int64_t d, const ClassProblem& q) {
  return !q.f32() && d % 8 == 0 && ld % 8 == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0 &&
         ld * 2 <= kMaxPitch;
}

// Where everything lies in the workspace
struct ClassLayout {
  int64_t pitch;                   // of packed operands, bytes
  int64_t x_plane, w_plane, planes;
  bool pack_x, pack_w;
  int64_t xp, wp;                  // offsets
  int64_t part, label_logit;       // forward
  int tile;                        // 0: 256 x 256, 1: 128 x 128, 2: 128 classes x 32 rows
  int64_t tiles_v;
  int64_t piece, pieces;           // gradient: classes per piece
  int64_t resid_pitch, resid_plane;
  int64_t resid, dx_part, bias_part;
  int dx_splits, dx_tile, dw_tile;
  int64_t total;
};

int64_t tiles(int64_t n, int64_t b) { return (n + b - 1) / b; }

ClassLayout layout_of(const ClassProblem& q, bool grad, bool has_ignore) {
  ClassLayout l;
  l.planes = q.f32() ? 3 : 1;
  l.pitch = round_up(q.d, 64) * 2;
  l.pack_x = !direct(q.x, q.ldx, q.d, q) || (grad && has_ignore);
  l.pack_w = !direct(q.w, q.ldw, q.d, q);
  l.x_plane = q.n * l.pitch;
  l.w_plane = q.v * l.pitch;
  const int cus = device_cu_count();
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += round_up(bytes, 1024);
    return here;
  };
  l.xp = l.pack_x ? take(l.planes * l.x_plane) : 0;
  l.wp = l.pack_w ? take(l.planes * l.w_plane) : 0;
  l.piece = q.v;
  if (grad) {
    int64_t c = kPieceBytes / (l.planes * 2 * (q.n > 0 ? q.n : 1)) / 256 * 256;
    if (c < 4096) c = 4096;
    if (c < l.piece) l.piece = c;
  }
  l.pieces = tiles(q.v, l.piece);
  // large tiles where they fill the chip
  l.tile = q.n <= 32 ? 2 : tiles(l.piece, 256) * tiles(q.n, 256) >= cus ? 0 : 1;
  l.tiles_v = tiles(q.v, l.tile == 0 ? 256 : 128);
  l.part = l.label_logit = l.resid = l.dx_part = l.bias_part = 0;
  if (!grad) {
    l.part = take(l.tiles_v * q.n * 8);
    l.label_logit = take(q.n * 4);
  } else {
    l.resid_pitch = round_up(l.piece, 64) * 2;
    l.resid_plane = q.n * l.resid_pitch;
    l.resid = take(l.planes * l.resid_plane);
    l.dw_tile = tiles(l.piece, 256) * tiles(q.d, 256) >= cus ? 0 : 1;
    l.dx_tile = tiles(q.n, 256) * tiles(q.d, 256) >= cus ? 0 : 1;
    const int64_t b = l.dx_tile == 0 ? 256 : 128;
    const int64_t t = tiles(q.n, b) * tiles(q.d, b);
    const int64_t steps = tiles(l.piece, 64);
    int64_t s = t > 0 ? (2 * cus) / t : 1;
    if (s > steps / 4) s = steps / 4;
    l.dx_splits = (int)(s < 1 ? 1 : s > 64 ? 64 : s);
    l.dx_part = take(l.dx_splits * q.n * q.d * 4);
    const int64_t bn = l.tile == 0 ? 256 : l.tile == 1 ? 128 : 32;
    l.bias_part = take(tiles(q.n, bn) * q.v * 4);
  }
  l.total = at;
  return l;
}

template <typename C, int EPI, bool F32>
int launch_tile(const ClassArgs& a, hipStream_t s) {
  constexpr int epi = kEpiLds<C, EPI> + C::BM * 4 * (1 + C::WGN);
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
  ZS_REQUIRE(wgs < (1ll << 31), "class logits: %lld tiles", (long long)wgs);
  hipLaunchKernelGGL((class_tile_kernel<C, EPI, F32>), dim3((unsigned)wgs, (unsigned)p.splits),
                     dim3(256), lds, s, p);
  ZS_LAUNCH_CHECK("class_tile_kernel launch");
  return ZSHMC_OK;
}

template <bool AK, bool BK> using Big = TileCfg<MmaBf16, 2, 2, 4, 4, AK, BK>;
template <bool AK, bool BK> using Mid = TileCfg<MmaBf16, 2, 2, 2, 2, AK, BK>;
using Few = TileCfg<MmaBf16, 4, 1, 1, 1, false, false>;

template <int EPI, bool F32>
int launch_logits(const ClassArgs& a, int tile, hipStream_t s) {
  switch (tile) {
    case 0: return launch_tile<Big<false, false>, EPI, F32>(a, s);
    case 1: return launch_tile<Mid<false, false>, EPI, F32>(a, s);
    default: return launch_tile<Few, EPI, F32>(a, s);
  }
}

int pack_rows(const void* src, int64_t rows, int64_t ld, const ClassProblem& q,
              unsigned char* dst, int64_t pitch, int64_t plane, const int64_t* labels,
              int64_t ignore, hipStream_t s) {
  const unsigned grid = grid_for(rows * (pitch / 16));
  if (q.f32())
    hipLaunchKernelGGL(pack_rows_kernel<true>, dim3(grid), dim3(256), 0, s, src, rows, q.d, ld,
                       dst, pitch, plane, labels, ignore);
  else
    hipLaunchKernelGGL(pack_rows_kernel<false>, dim3(grid), dim3(256), 0, s, src, rows, q.d, ld,
                       dst, pitch, plane, labels, ignore);
  ZS_LAUNCH_CHECK("pack_rows_kernel launch");
  return ZSHMC_OK;
}

// the operands X and w, packed where they have to be
int operands(const ClassProblem& q, const ClassLayout& l, unsigned char* ws,
             const int64_t* drop_labels, int64_t ignore, hipStream_t s, TileOperand* x,
             TileOperand* w) {
  const unsigned char* px = static_cast<const unsigned char*>(q.x);
  const unsigned char* pw = static_cast<const unsigned char*>(q.w);
  *x = TileOperand{px, q.ldx * 2, 0, q.n, q.d * 2};
  *w = TileOperand{pw, q.ldw * 2, 0, q.v, q.d * 2};
  if (l.pack_x) {
    const int rc = pack_rows(q.x, q.n, q.ldx, q, ws + l.xp, l.pitch, l.x_plane, drop_labels,
                             ignore, s);
    if (rc != ZSHMC_OK) return rc;
    *x = TileOperand{ws + l.xp, l.pitch, l.x_plane, q.n, l.pitch};
  }
  if (l.pack_w) {
    const int rc = pack_rows(q.w, q.v, q.ldw, q, ws + l.wp, l.pitch, l.w_plane, nullptr, 0, s);
    if (rc != ZSHMC_OK) return rc;
    *w = TileOperand{ws + l.wp, l.pitch, l.w_plane, q.v, l.pitch};
  }
  return ZSHMC_OK;
}

int check_problem(const ClassProblem& q, const char* who) {
  ZS_REQUIRE(q.dtype == ZSHMC_DTYPE_F32 || q.dtype == ZSHMC_DTYPE_BF16,
             "%s: dtype must be ZSHMC_DTYPE_F32 or _BF16, got %d", who, q.dtype);
  ZS_REQUIRE(q.n >= 0 && q.d > 0 && q.v > 0, "%s: n_rows >= 0, n_features and n_classes > 0",
             who);
  ZS_REQUIRE(q.n < (1ll << 31) && q.v < (1ll << 31) && q.d <= (1ll << 20),
             "%s: at most 2^31 - 1 rows and classes and 2^20 features", who);
  ZS_REQUIRE(q.ldx >= q.d && q.ldw >= q.d, "%s: rows overlap (ldx / ldw < n_features)", who);
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
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  ClassArgs a{};
  rc = operands(q, l, ws, nullptr, 0, s, &a.b, &a.a);
  if (rc != ZSHMC_OK) return rc;
  a.m = q.v;
  a.n = q.n;
  a.steps = (int)tiles(q.d, 64);
  a.terms = q.f32() ? kTerms3 : 1;
  a.splits = 1;
  a.bias = bias;
  a.labels = labels;
  a.n_classes = q.v;
  a.part = reinterpret_cast<cf2*>(ws + l.part);
  a.label_logit = reinterpret_cast<float*>(ws + l.label_logit);
  rc = launch_logits<kEpiStats, false>(a, l.tile, s);
  if (rc != ZSHMC_OK) return rc;
  hipLaunchKernelGGL(join_stats_kernel, dim3((unsigned)tiles(q.n, 16)), dim3(256), 0, s, a.part,
                     (int)l.tiles_v, a.label_logit, labels, q.n, q.v, has_ignore, ignore_label,
                     log_prob, reinterpret_cast<cf2*>(stats));
  ZS_LAUNCH_CHECK("join_stats_kernel launch");
  return ZSHMC_OK;
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
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  TileOperand ox, ow;
  rc = operands(q, l, ws, has_ignore ? labels : nullptr, ignore_label, s, &ox, &ow);
  if (rc != ZSHMC_OK) return rc;
  const int terms = q.f32() ? kTerms3 : 1;
  for (int64_t c0 = 0; c0 < q.v; c0 += l.piece) {
    const int64_t c = q.v - c0 < l.piece ? q.v - c0 : l.piece;
    TileOperand wp = ow;
    wp.base += c0 * wp.pitch;
    wp.rows = c;
    const TileOperand r{ws + l.resid, l.resid_pitch, l.resid_plane, q.n, round_up(c, 64) * 2};
    ClassArgs a{};
    a.a = wp;
    a.b = ox;
    a.m = c;
    a.n = q.n;
    a.steps = (int)tiles(q.d, 64);
    a.terms = terms;
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
    rc = q.f32() ? launch_logits<kEpiResidual, true>(a, l.tile, s)
                 : launch_logits<kEpiResidual, false>(a, l.tile, s);
    if (rc != ZSHMC_OK) return rc;
    if (grad_w) {                  // dw = r^T X over the rows of X
      ClassArgs g{};
      g.a = r;
      g.b = ox;
      g.m = c;
      g.n = q.d;
      g.steps = (int)tiles(q.n, 64);
      g.terms = terms;
      g.splits = 1;
      g.out = static_cast<unsigned char*>(grad_w) + c0 * q.d * q.esize();
      g.out_ld = q.d;
      g.out_bf16 = !q.f32();
      rc = l.dw_tile == 0 ? launch_tile<Big<true, true>, kEpiStore, false>(g, s)
                          : launch_tile<Mid<true, true>, kEpiStore, false>(g, s);
      if (rc != ZSHMC_OK) return rc;
    }
    if (grad_x) {                  // dX += r w over the piece's classes
      ClassArgs g{};
      g.a = r;
      g.b = wp;
      g.m = q.n;
      g.n = q.d;
      g.steps = (int)tiles(c, 64);
      g.terms = terms;
      g.splits = l.dx_splits;
      g.out = ws + l.dx_part;
      g.out_ld = q.d;
      g.out_split = q.n * q.d;
      g.accumulate = c0 > 0;
      rc = l.dx_tile == 0 ? launch_tile<Big<false, true>, kEpiStore, false>(g, s)
                          : launch_tile<Mid<false, true>, kEpiStore, false>(g, s);
      if (rc != ZSHMC_OK) return rc;
    }
  }
  if (grad_x) {
    const float* parts = reinterpret_cast<const float*>(ws + l.dx_part);
    const int64_t n = q.n * q.d;
    if (q.f32())
      hipLaunchKernelGGL(sum_rows_kernel<false>, dim3(grid_for(n)), dim3(256), 0, s, parts,
                         l.dx_splits, n, n, grad_x);
    else
      hipLaunchKernelGGL(sum_rows_kernel<true>, dim3(grid_for(n)), dim3(256), 0, s, parts,
                         l.dx_splits, n, n, grad_x);
    ZS_LAUNCH_CHECK("sum_rows_kernel launch");
  }
  if (grad_bias) {
    const int64_t bn = l.tile == 0 ? 256 : l.tile == 1 ? 128 : 32;
    hipLaunchKernelGGL(sum_rows_kernel<false>, dim3(grid_for(q.v)), dim3(256), 0, s,
                       reinterpret_cast<const float*>(ws + l.bias_part), (int)tiles(q.n, bn),
                       q.v, q.v, grad_bias);
    ZS_LAUNCH_CHECK("sum_rows_kernel launch");
  }
  return ZSHMC_OK;
}
