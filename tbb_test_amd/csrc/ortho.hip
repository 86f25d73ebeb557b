// Orthogonalised update: the momentum of a weight matrix's gradient, with its singular values driven
// towards one by Newton-Schulz products.  With U [rows x cols] and m = min, n = max of the two:
//
//   X_0 = U / |U|_F (transposed if rows > cols, so that X is m x n)
//   five times or as often as asked:   A = X X^T,   X <- a X + (b A + c A^2) X,   (a, b, c) below
//   W <- (1 - lr decay) W - lr scale O,   O = X (transposed back)
//
// Precision.  The products run on fp16 MFMAs with fp32 accumulation.  bf16 has the same rate and three
// bits less, which this iteration turns into errors of 1e-2 (flat spectra) to 3e-1 (a few strong
// directions over a floor) of |O|; everything here is bounded, so fp16's range is enough: |X|_F = 1 at
// the start and no singular value ever passes 1.21, hence |A_ij| < 1.5 and |b A + c A^2| < 2.9.
// X is kept to 22 bits, because the a X term carries every direction from one iteration to the next and
// grows small ones 3.4 times each: with the fp16 operand in that term its white rounding noise grows along
// (4e-2 for a floor of 1e-2).  The diagonals of A, near 1, and of b A + c A^2, near b + c, stay in fp32 and out of
// the products: their rounding would be most of what is left.  Together, after five steps: 3e-4 of |O| (200 x 2000,
// flat) .. 8e-4 (256 x 256 and 200 x 2000, steep) .. 1.2e-3 (64 x 64, steep).  p(s) = a s + b s^3 + c s^5 has the
// slope -1.6 at its fixed point 0.87, so an error of a singular value near there grows by that with each step until it
// has settled on the cycle around it: fp32 products start from 1e-6 and grow by the same factors.  Many singular values
// average that out, few do not (2 x 2: 1e-3 at the median, 5e-3 .. 2.5e-2 at the 99th of 100, 6e-2 seen), nor do
// many steps (16 steps: 2e-3 .. 5e-3 at the median, 2e-2 .. 3e-1 at the 99th of 100 up to 64 x 64).
// fp16 for fp32 gradients and weights too: fp32 products run at a tenth of the rate, and the direction that a
// stochastic gradient's momentum gives is not known to 1e-3.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "kernels.h"
#include "tile16.h"

namespace mi {

namespace {

constexpr float NS_A = 3.4445f, NS_B = -4.7750f, NS_C = 2.0315f;
constexpr float GRAM_SCALE = 4096.0f;  // A and b A + c A^2 are stored times this: off-diagonal entries start near 1 / (m sqrt n)

inline size_t up(size_t x, size_t a) { return (x + a - 1) / a * a; }
inline bool fours(const void* q, int bytes) { return reinterpret_cast<uintptr_t>(q) % bytes == 0; }  // null too

// ---- U, its norm, X_0 -------------------------------------------------------------------------------

struct GatherArgs {
  int rows, cols;        // of the gradient
  const void* G;         // fp32 or bf16
  int ldg;
  long long strideG;     // between batch entries
  size_t replica_stride;
  int R;
  float* momentum;       // dense, or null
  long long strideM;
  float mu;
  int nesterov;
  float* U;              // [batch][mp x np], in working orientation
  int mp, np;
  int vec;               // rows of G (and momentum) start at whole 16 bytes (bf16: 8)
  double* sumsq;         // [batch][workgroups of an entry]
};

// U in working orientation, zero padded, and the sum of its squares per workgroup.  64 x 64 tiles of the
// gradient, four consecutive elements per thread and row (16-byte loads where rows allow it: `vec`); FLIP
// turns them through LDS.  Bound by HBM: 8192 x 8192 with four replicas and momentum 385 us, 4.9 TB/s.
template <bool BF16, bool FLIP>
__global__ __launch_bounds__(256) void ortho_gather_kernel(GatherArgs p) {
  __shared__ float tile[FLIP ? 64 : 1][65];
  __shared__ double red[256];
  const int tx = (threadIdx.x & 15) * 4, ty = threadIdx.x >> 4;
  const int r0 = blockIdx.y * 64, c0 = blockIdx.x * 64, col = c0 + tx;
  float* U = p.U + (size_t)blockIdx.z * p.mp * p.np;
  double acc = 0.0;
#pragma unroll
  for (int pass = 0; pass < 4; ++pass) {
    const int i = pass * 16 + ty, row = r0 + i;
    f32x4 u = {0.0f, 0.0f, 0.0f, 0.0f};
    const int n = row < p.rows ? min(p.cols - col, 4) : 0;  // elements that are there
    if (n > 0) {
      const size_t at = (size_t)blockIdx.z * p.strideG + (size_t)row * p.ldg + col;
      const bool whole = p.vec && n == 4;
      if constexpr (BF16) {
        const u16* g = static_cast<const u16*>(p.G) + at;
        if (whole) {
          const u32x2 two = *reinterpret_cast<const u32x2*>(g);
          u = f32x4{__uint_as_float(two[0] << 16), __uint_as_float(two[0] & 0xffff0000u), __uint_as_float(two[1] << 16), __uint_as_float(two[1] & 0xffff0000u)};
        } else {
          for (int k = 0; k < n; ++k) u[k] = bf2f(g[k]);
        }
      } else {
        const float* g = static_cast<const float*>(p.G) + at;
        if (whole) {
          u = *reinterpret_cast<const f32x4*>(g);
          for (int r = 1; r < p.R; ++r) u += *reinterpret_cast<const f32x4*>(g + (size_t)r * p.replica_stride);
        } else {
          for (int k = 0; k < n; ++k) {
            u[k] = g[k];
            for (int r = 1; r < p.R; ++r) u[k] += g[(size_t)r * p.replica_stride + k];
          }
        }
      }
      if (p.momentum) {
        float* m = p.momentum + (size_t)blockIdx.z * p.strideM + (size_t)row * p.cols + col;
        f32x4 now = {0.0f, 0.0f, 0.0f, 0.0f};
        if (whole) now = *reinterpret_cast<const f32x4*>(m);
        else for (int k = 0; k < n; ++k) now[k] = m[k];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          now[k] = fmaf(p.mu, now[k], u[k]);
          u[k] = p.nesterov ? fmaf(p.mu, now[k], u[k]) : now[k];
        }
        if (whole) *reinterpret_cast<f32x4*>(m) = now;
        else for (int k = 0; k < n; ++k) m[k] = now[k];
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) acc += (double)u[k] * (double)u[k];
    if constexpr (FLIP) {
#pragma unroll
      for (int k = 0; k < 4; ++k) tile[i][tx + k] = u[k];
    } else {
      *reinterpret_cast<f32x4*>(U + (size_t)row * p.np + col) = u;
    }
  }
  red[threadIdx.x] = acc;
  __syncthreads();
  if constexpr (FLIP) {
#pragma unroll
    for (int pass = 0; pass < 4; ++pass) {
      const int i = pass * 16 + ty;
      *reinterpret_cast<f32x4*>(U + (size_t)(c0 + i) * p.np + r0 + tx) = f32x4{tile[tx][i], tile[tx + 1][i], tile[tx + 2][i], tile[tx + 3][i]};
    }
  }
  for (int off = 128; off > 0; off >>= 1) {
    if ((int)threadIdx.x < off) red[threadIdx.x] += red[threadIdx.x + off];
    __syncthreads();
  }
  if (threadIdx.x == 0) p.sumsq[((size_t)blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x] = red[0];
}

// 1 / |U|_F from the workgroups' sums of squares; 0 for U = 0, NaN where |U|_F is not finite.  For a whole workgroup.
__device__ __forceinline__ double inverse_norm(const double* __restrict__ sumsq, int blocks, double* red) {
  double part[8] = {};
  int i = threadIdx.x;
  for (; i + 7 * 256 < blocks; i += 8 * 256)
#pragma unroll
    for (int k = 0; k < 8; ++k) part[k] += sumsq[i + 256 * k];
  for (; i < blocks; i += 256) part[0] += sumsq[i];
  red[threadIdx.x] = ((part[0] + part[1]) + (part[2] + part[3])) + ((part[4] + part[5]) + (part[6] + part[7]));
  __syncthreads();
  for (int off = 128; off > 0; off >>= 1) {
    if ((int)threadIdx.x < off) red[threadIdx.x] += red[threadIdx.x + off];
    __syncthreads();
  }
  const double q = red[0];
  return q == 0.0 ? 0.0 : __builtin_isfinite(q) ? 1.0 / sqrt(q) : __builtin_nan("");
}

// One launch more, for matrices with so many sums that every workgroup of the next kernel should not add them up.
constexpr int FEW_SUMS = 1024;
__global__ __launch_bounds__(256) void ortho_norm_kernel(const double* __restrict__ sumsq, int blocks, double* __restrict__ inv) {
  __shared__ double red[256];
  const double f = inverse_norm(sumsq + (size_t)blockIdx.x * blocks, blocks, red);
  if (threadIdx.x == 0) inv[blockIdx.x] = f;
}

// X = scale * x is kept as two fp16 numbers, x rounded and 2^11 times what the rounding left: 22 bits, as much
// traffic as fp32, and the first half is the operand of the products.
constexpr float LOW_SCALE = 2048.0f;
__device__ __forceinline__ float joined(float high, float low) { return fmaf(low, 1.0f / LOW_SCALE, high); }

// X_0 = scale * U / |U|_F as two halves, and the first half transposed.  64 x 64 tiles; 8192 x 8192: 126 us, 5.3 TB/s.
__global__ __launch_bounds__(256) void ortho_scale_kernel(const float* __restrict__ U, u16* __restrict__ Xh, u16* __restrict__ Xl,
                                                          u16* __restrict__ XhT, int mp, int np, const double* __restrict__ sumsq,
                                                          int blocks, const double* __restrict__ inv, float scale) {
  __shared__ u16 tile[64][66];
  __shared__ double red[256];
  const size_t base = (size_t)blockIdx.z * mp * np;
  const int tx = (threadIdx.x & 15) * 4, ty = threadIdx.x >> 4, r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;
  const double f = (double)scale * (blocks > FEW_SUMS ? inv[blockIdx.z] : inverse_norm(sumsq + (size_t)blockIdx.z * blocks, blocks, red));
#pragma unroll
  for (int pass = 0; pass < 4; ++pass) {
    const int i = pass * 16 + ty;
    const size_t at = base + (size_t)(r0 + i) * np + c0 + tx;
    const f32x4 u = *reinterpret_cast<const f32x4*>(U + at);
    float x[4];
    u32x2 high, low;
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = (float)((double)u[k] * f);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      high[k] = pack16<true>(x[2 * k], x[2 * k + 1]);
      low[k] = pack16<true>(LOW_SCALE * (x[2 * k] - f16_lo(high[k])), LOW_SCALE * (x[2 * k + 1] - f16_hi(high[k])));
    }
    *reinterpret_cast<u32x2*>(Xh + at) = high;
    *reinterpret_cast<u32x2*>(Xl + at) = low;
    *reinterpret_cast<unsigned*>(&tile[i][tx]) = high[0];
    *reinterpret_cast<unsigned*>(&tile[i][tx + 2]) = high[1];
  }
  __syncthreads();
#pragma unroll
  for (int pass = 0; pass < 4; ++pass) {
    const int i = pass * 16 + ty;
    *reinterpret_cast<u32x2*>(XhT + base + (size_t)(c0 + i) * mp + r0 + tx) =
        u32x2{tile[tx][i] | (unsigned)tile[tx + 1][i] << 16, tile[tx + 2][i] | (unsigned)tile[tx + 3][i] << 16};
  }
}

// ---- the products -----------------------------------------------------------------------------------

// A = X X^T without its diagonal (times GRAM_SCALE, fp16): a tile of the lower triangle and its mirror image; the
// diagonal in fp32.  Bound by the MFMAs: 8192 x 8192 429 us for half of the product, 1280 TFLOP/s; 8 x 1024 x 1024 17.5 us,
// 36 tiles of 128 x 128 on the 32 CUs of an XCD.
struct EpiGram : NoPre {
  static constexpr bool MAY_SPLIT = true;
  struct Args {
    u16* A;
    float* diag;
    int ld;
    long long batch;
    float scale;  // of the products, to GRAM_SCALE * A
  };
  template <int QB, class Get>
  static __device__ __forceinline__ void run(const Args& e, const Tile16& p, const Pre<QB>& pre, Get get, int row0, int colw, int lane,
                                             unsigned char* stage, int entry) {
    u16* A = e.A + (size_t)entry * e.batch;
    const int l16 = lane & 15, col = colw + 8 * (lane >> 4);
    const bool on_diagonal = row0 / p.tile == colw / p.tile;
    u32x4 pk[QB][2];
#pragma unroll
    for (int jq = 0; jq < QB; ++jq)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = row0 + 16 * jq + l16;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = e.scale * get(jq, h, i);
        if (on_diagonal) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (row == col + 32 * h + i) {
              e.diag[(size_t)entry * e.ld + row] = v[i] * (1.0f / GRAM_SCALE);
              v[i] = 0.0f;
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) pk[jq][h][k] = pack16<true>(v[2 * k], v[2 * k + 1]);
        *reinterpret_cast<u32x4*>(A + (size_t)row * e.ld + col + 32 * h) = pk[jq][h];
      }
    if (!on_diagonal) store_transposed<QB>(A + (size_t)colw * e.ld + row0, e.ld, pk, lane, stage);
  }
};

// P = b A + c A A without its diagonal (times GRAM_SCALE, fp16), the diagonal in fp32.  With A = A' + D, D its
// diagonal: P = c A' A' + b A' + c (D A' + A' D) off the diagonal, and b D + c (A' A' + D D) on it.  About as fast
// as the one above (446 and 20 us).
struct EpiPoly {
  static constexpr bool MAY_SPLIT = true;
  struct Args {
    const u16* A;
    const float* diag_a;
    u16* P;
    float* diag;
    int ld;
    long long batch;
  };
  template <int QB>
  struct Pre {
    u32x4 a[QB][2];
    float d_row[QB];
    f32x4 d_col[2][2];
  };
  template <int QB>
  static __device__ __forceinline__ Pre<QB> before(const Args& e, const Tile16&, int row0, int colw, int lane, int entry) {
    const u16* A = e.A + (size_t)entry * e.batch + (size_t)(row0 + (lane & 15)) * e.ld + colw + 8 * (lane >> 4);
    Pre<QB> v;
#pragma unroll
    for (int jq = 0; jq < QB; ++jq)
#pragma unroll
      for (int h = 0; h < 2; ++h) v.a[jq][h] = *reinterpret_cast<const u32x4*>(A + (size_t)(16 * jq) * e.ld + 32 * h);
    const float* d = e.diag_a + (size_t)entry * e.ld;
#pragma unroll
    for (int jq = 0; jq < QB; ++jq) v.d_row[jq] = d[row0 + (lane & 15) + 16 * jq];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int k = 0; k < 2; ++k) v.d_col[h][k] = *reinterpret_cast<const f32x4*>(d + colw + 8 * (lane >> 4) + 32 * h + 4 * k);
    return v;
  }
  template <int QB, class Get>
  static __device__ __forceinline__ void run(const Args& e, const Tile16& p, const Pre<QB>& pre, Get get, int row0, int colw, int lane,
                                             unsigned char* stage, int entry) {
    u16* P = e.P + (size_t)entry * e.batch;
    const int l16 = lane & 15, col = colw + 8 * (lane >> 4);
    u32x4 pk[QB][2];
    const bool on_diagonal = row0 / p.tile == colw / p.tile;
#pragma unroll
    for (int jq = 0; jq < QB; ++jq)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = row0 + 16 * jq + l16;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const unsigned w = pre.a[jq][h][i >> 1];
          const float factor = fmaf(NS_C, pre.d_row[jq] + pre.d_col[h][i >> 2][i & 3], NS_B);
          v[i] = fmaf(NS_C / GRAM_SCALE, get(jq, h, i), factor * ((i & 1) ? f16_hi(w) : f16_lo(w)));
        }
        if (on_diagonal) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (row == col + 32 * h + i) {
              // here A' is zero and v = GRAM_SCALE c (A' A')
              const float d = pre.d_row[jq];
              e.diag[(size_t)entry * e.ld + row] = fmaf(v[i], 1.0f / GRAM_SCALE, d * fmaf(NS_C, d, NS_B));
              v[i] = 0.0f;
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) pk[jq][h][k] = pack16<true>(v[2 * k], v[2 * k + 1]);
        *reinterpret_cast<u32x4*>(P + (size_t)row * e.ld + col + 32 * h) = pk[jq][h];
      }
    if (!on_diagonal) store_transposed<QB>(P + (size_t)colw * e.ld + row0, e.ld, pk, lane, stage);
  }
};

// X <- (a + diag) X + P X, in place, and the first half's transpose for the next iteration (null: last one).  8192 x 8192:
// 902 us, 1220 TFLOP/s, of which the ten bytes an element take 0.1 ms; 8 x 1024 x 1024: 28 us, half of them those bytes:
// one round of 512 workgroups, two per CU, that all load, multiply and store at the same times.
struct EpiStep {
  static constexpr bool MAY_SPLIT = true;
  struct Args {
    const float* diag;
    u16 *Xh, *Xl, *XhT;
    int mp, np;
    float unscale;  // of the products, to scale * x
  };
  template <int QB>
  struct Pre {
    u32x4 high[QB][2], low[QB][2];
    float keep[QB];
  };
  template <int QB>
  static __device__ __forceinline__ Pre<QB> before(const Args& e, const Tile16&, int row0, int colw, int lane, int entry) {
    const int row = row0 + (lane & 15);
    const size_t at = (size_t)entry * e.mp * e.np + (size_t)row * e.np + colw + 8 * (lane >> 4);
    Pre<QB> v;
#pragma unroll
    for (int jq = 0; jq < QB; ++jq) {
      v.keep[jq] = NS_A + e.diag[(size_t)entry * e.mp + row + 16 * jq];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        v.high[jq][h] = *reinterpret_cast<const u32x4*>(e.Xh + at + (size_t)(16 * jq) * e.np + 32 * h);
        v.low[jq][h] = *reinterpret_cast<const u32x4*>(e.Xl + at + (size_t)(16 * jq) * e.np + 32 * h);
      }
    }
    return v;
  }
  template <int QB, class Get>
  static __device__ __forceinline__ void run(const Args& e, const Tile16& p, const Pre<QB>& pre, Get get, int row0, int colw, int lane,
                                             unsigned char* stage, int entry) {
    const size_t base = (size_t)entry * e.mp * e.np;
    const int l16 = lane & 15, col = colw + 8 * (lane >> 4);
    u32x4 high[QB][2];
    // (all of the tile's X is requested before anything is stored: a load behind a store waits for that store)
    asm volatile("" ::: "memory");
#pragma unroll
    for (int jq = 0; jq < QB; ++jq)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const size_t at = base + (size_t)(row0 + 16 * jq + l16) * e.np + col + 32 * h;
        u32x4 low;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const unsigned hi = pre.high[jq][h][k], lo = pre.low[jq][h][k];
          const float x0 = fmaf(pre.keep[jq], joined(f16_lo(hi), f16_lo(lo)), e.unscale * get(jq, h, 2 * k));
          const float x1 = fmaf(pre.keep[jq], joined(f16_hi(hi), f16_hi(lo)), e.unscale * get(jq, h, 2 * k + 1));
          const unsigned now = pack16<true>(x0, x1);
          high[jq][h][k] = now;
          low[k] = pack16<true>(LOW_SCALE * (x0 - f16_lo(now)), LOW_SCALE * (x1 - f16_hi(now)));
        }
        *reinterpret_cast<u32x4*>(e.Xh + at) = high[jq][h];
        *reinterpret_cast<u32x4*>(e.Xl + at) = low;
      }
    if (e.XhT) store_transposed<QB>(e.XhT + base + (size_t)colw * e.mp + row0, e.mp, high, lane, stage);
  }
};

// ---- O out, W updated -------------------------------------------------------------------------------

struct FinishArgs {
  int rows, cols;
  const u16 *Xh, *Xl;  // [batch][mp x np]
  float unscale;       // of X
  int mp, np;
  u16* O;          // bf16 result, or null
  int ldo;
  long long strideO;
  float* W;        // dense [rows x cols] with its bf16 copies (either may be null), or null
  u16 *W16, *Wt16;
  long long strideW;
  float keep, step;  // W <- keep W - step O
  int vec, vec_t;    // rows of O, W and W16 (of Wt16) start at whole 16 or 8 bytes
};

// Bound by HBM: 8192 x 8192 with both copies 200 us, 5.4 TB/s.
template <bool FLIP>
__global__ __launch_bounds__(256) void ortho_finish_kernel(FinishArgs p) {
  __shared__ float turned[FLIP ? 64 : 1][65];
  __shared__ u16 tile[64][66];
  const size_t base = (size_t)blockIdx.z * p.mp * p.np;
  const int tx = (threadIdx.x & 15) * 4, ty = threadIdx.x >> 4, r0 = blockIdx.y * 64, c0 = blockIdx.x * 64, col = c0 + tx;
  auto x_at = [&](size_t at) {  // four elements (X is padded to whole 64 x 64 tiles)
    const u32x2 high = *reinterpret_cast<const u32x2*>(p.Xh + base + at), low = *reinterpret_cast<const u32x2*>(p.Xl + base + at);
    return f32x4{p.unscale * joined(f16_lo(high[0]), f16_lo(low[0])), p.unscale * joined(f16_hi(high[0]), f16_hi(low[0])),
                 p.unscale * joined(f16_lo(high[1]), f16_lo(low[1])), p.unscale * joined(f16_hi(high[1]), f16_hi(low[1]))};
  };
  if constexpr (FLIP) {
#pragma unroll
    for (int pass = 0; pass < 4; ++pass) {
      const f32x4 x = x_at((size_t)(c0 + pass * 16 + ty) * p.np + r0 + tx);
#pragma unroll
      for (int k = 0; k < 4; ++k) turned[pass * 16 + ty][tx + k] = x[k];
    }
    __syncthreads();
  }
#pragma unroll
  for (int pass = 0; pass < 4; ++pass) {
    const int i = pass * 16 + ty, row = r0 + i;
    const int n = row < p.rows ? min(p.cols - col, 4) : 0;
    if (n <= 0) continue;
    const f32x4 o = FLIP ? f32x4{turned[tx][i], turned[tx + 1][i], turned[tx + 2][i], turned[tx + 3][i]} : x_at((size_t)row * p.np + col);
    const bool whole = p.vec && n == 4;
    if (p.O) {
      u16* out = p.O + (size_t)blockIdx.z * p.strideO + (size_t)row * p.ldo + col;
      if (whole) *reinterpret_cast<u32x2*>(out) = u32x2{pack16<false>(o[0], o[1]), pack16<false>(o[2], o[3])};
      else for (int k = 0; k < n; ++k) out[k] = f2bf(o[k]);
    }
    if (p.W) {
      const size_t at = (size_t)blockIdx.z * p.strideW + (size_t)row * p.cols + col;
      f32x4 w = {0.0f, 0.0f, 0.0f, 0.0f};
      if (whole) w = *reinterpret_cast<const f32x4*>(p.W + at);
      else for (int k = 0; k < n; ++k) w[k] = p.W[at + k];
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = fmaf(-p.step, o[k], p.keep * w[k]);
      const u32x2 h = {pack16<false>(w[0], w[1]), pack16<false>(w[2], w[3])};
      if (whole) {
        *reinterpret_cast<f32x4*>(p.W + at) = w;
        if (p.W16) *reinterpret_cast<u32x2*>(p.W16 + at) = h;
      } else {
        for (int k = 0; k < n; ++k) {
          p.W[at + k] = w[k];
          if (p.W16) p.W16[at + k] = f2bf(w[k]);
        }
      }
      *reinterpret_cast<unsigned*>(&tile[i][tx]) = h[0];
      *reinterpret_cast<unsigned*>(&tile[i][tx + 2]) = h[1];
    }
  }
  if (!p.Wt16) return;
  __syncthreads();
#pragma unroll
  for (int pass = 0; pass < 4; ++pass) {
    const int i = pass * 16 + ty;
    const int n = c0 + i < p.cols ? min(p.rows - r0 - tx, 4) : 0;
    if (n <= 0) continue;
    u16* out = p.Wt16 + (size_t)blockIdx.z * p.strideW + (size_t)(c0 + i) * p.rows + r0 + tx;
    if (p.vec_t && n == 4)
      *reinterpret_cast<u32x2*>(out) = u32x2{tile[tx][i] | (unsigned)tile[tx + 1][i] << 16, tile[tx + 2][i] | (unsigned)tile[tx + 3][i] << 16};
    else
      for (int k = 0; k < n; ++k) out[k] = tile[tx + k][i];
  }
}

// ---- sizes ------------------------------------------------------------------------------------------

struct Plan {
  int m, n, mp, np;
  bool flip;
  float scale;  // of X: a power of two near sqrt(n), so that typical entries start near 1 / sqrt(m)
  Tile16Shape gram, poly, step;
  float* U;
  u16 *Xh, *Xl, *XhT[2], *A, *P;
  float *diag_a, *diag, *part;
  double *sumsq, *inv;
  size_t bytes;
};
Plan plan_ortho(char* base, int batch, int rows, int cols) {
  Plan q{};
  q.flip = rows > cols;
  q.m = std::min(rows, cols);
  q.n = std::max(rows, cols);
  // padded to whole tiles of the largest size that wastes little
  auto pad = [](int v) {
    for (int t : {256, 128})
      if (up(v, t) - v <= (size_t)v / 32) return (int)up(v, t);
    return (int)up(v, 64);
  };
  q.mp = pad(q.m);
  q.np = pad(q.n);
  auto largest = [](int v) { return v % 256 == 0 ? 256 : v % 128 == 0 ? 128 : 64; };
  q.gram = tile16_shape(q.mp, q.mp, q.np, true, batch, 64, largest(q.mp), true);
  q.poly = tile16_shape(q.mp, q.mp, q.mp, true, batch, 64, largest(q.mp), true);
  q.step = tile16_shape(q.mp, q.np, q.mp, false, batch, 64, std::min(largest(q.mp), largest(q.np)), true);
  q.scale = 1.0f;
  while (q.scale * q.scale < (float)q.n && q.scale < 256.0f) q.scale *= 2.0f;
  size_t used = 0;
  auto take = [&](size_t bytes) {
    char* at = base ? base + used : nullptr;
    used += up(bytes, 256);
    return at;
  };
  const size_t x = (size_t)batch * q.mp * q.np, a = (size_t)batch * q.mp * q.mp;
  q.U = (float*)take(x * 4);
  q.Xh = (u16*)take(x * 2);
  q.Xl = (u16*)take(x * 2);
  q.XhT[0] = (u16*)take(x * 2);
  q.XhT[1] = (u16*)take(x * 2);
  q.A = (u16*)take(a * 2);
  q.P = (u16*)take(a * 2);
  q.diag_a = (float*)take((size_t)batch * q.mp * 4);
  q.diag = (float*)take((size_t)batch * q.mp * 4);
  q.part = (float*)take(std::max({q.gram.part_floats, q.poly.part_floats, q.step.part_floats}) * 4);
  q.sumsq = (double*)take((size_t)batch * (q.mp / 64) * (q.np / 64) * 8);
  q.inv = (double*)take((size_t)batch * 8);
  q.bytes = used;
  return q;
}

template <class Epi>
hipError_t tiles(const Plan& q, const Tile16Shape& shape, const u16* A, const u16* B, int M, int N, int K, int batch, bool symmetric,
                 const typename Epi::Args& e, hipStream_t s) {
  Tile16 p{};
  p.A = A; p.B = B; p.lda = K; p.ldb = K; p.M = M; p.N = N; p.K = K;
  p.batchA = (long long)M * K; p.batchB = (long long)N * K;
  p.batch = batch;
  p.symmetric = symmetric;
  return launch_tile16<true, Epi>(p, shape, q.part, e, s);
}

#define TRY(call)                          \
  do {                                     \
    hipError_t e_ = (call);                \
    if (e_ != hipSuccess) return e_;       \
  } while (0)

// U (gathered by `g`) -> scale * X of the last iteration, in q.Xh and q.Xl.
hipError_t newton_schulz(const Plan& q, GatherArgs g, bool bf16, int batch, int steps, hipStream_t s) {
  g.U = q.U;
  g.mp = q.mp;
  g.np = q.np;
  g.sumsq = q.sumsq;
  const dim3 tiles64(q.np / 64, q.mp / 64, batch);                                   // in working orientation
  const dim3 source = q.flip ? dim3(q.mp / 64, q.np / 64, batch) : tiles64;         // in the gradient's
  if (q.flip) {
    if (bf16) launch_kernel((ortho_gather_kernel<true, true>), source, dim3(256), 0, s, g);
    else launch_kernel((ortho_gather_kernel<false, true>), source, dim3(256), 0, s, g);
  } else {
    if (bf16) launch_kernel((ortho_gather_kernel<true, false>), source, dim3(256), 0, s, g);
    else launch_kernel((ortho_gather_kernel<false, false>), source, dim3(256), 0, s, g);
  }
  TRY(hipGetLastError());
  const int blocks = (q.mp / 64) * (q.np / 64);
  if (blocks > FEW_SUMS) {
    launch_kernel(ortho_norm_kernel, dim3(batch), dim3(256), 0, s, (const double*)q.sumsq, blocks, q.inv);
    TRY(hipGetLastError());
  }
  launch_kernel(ortho_scale_kernel, tiles64, dim3(256), 0, s, (const float*)q.U, q.Xh, q.Xl, q.XhT[0], q.mp, q.np,
                (const double*)q.sumsq, blocks, (const double*)q.inv, q.scale);
  TRY(hipGetLastError());
  const long long a = (long long)q.mp * q.mp;
  for (int k = 0; k < steps; ++k) {
    const EpiGram::Args gram{q.A, q.diag_a, q.mp, a, GRAM_SCALE / (q.scale * q.scale)};
    TRY(tiles<EpiGram>(q, q.gram, q.Xh, q.Xh, q.mp, q.mp, q.np, batch, true, gram, s));
    const EpiPoly::Args poly{q.A, q.diag_a, q.P, q.diag, q.mp, a};
    TRY(tiles<EpiPoly>(q, q.poly, q.A, q.A, q.mp, q.mp, q.mp, batch, true, poly, s));
    const EpiStep::Args step{q.diag, q.Xh, q.Xl, k + 1 == steps ? nullptr : q.XhT[(k + 1) & 1], q.mp, q.np, 1.0f / GRAM_SCALE};
    TRY(tiles<EpiStep>(q, q.step, q.P, q.XhT[k & 1], q.mp, q.np, q.mp, batch, false, step, s));
  }
  return hipSuccess;
}

hipError_t finish(const Plan& q, FinishArgs f, int batch, hipStream_t s) {
  f.Xh = q.Xh;
  f.Xl = q.Xl;
  f.unscale = 1.0f / q.scale;
  f.mp = q.mp;
  f.np = q.np;
  const dim3 grid((f.cols + 63) / 64, (f.rows + 63) / 64, batch);
  if (q.flip) launch_kernel(ortho_finish_kernel<true>, grid, dim3(256), 0, s, f);
  else launch_kernel(ortho_finish_kernel<false>, grid, dim3(256), 0, s, f);
  return hipGetLastError();
}

}  // namespace

size_t ortho_bytes(int batch, int rows, int cols) { return plan_ortho(nullptr, batch, rows, cols).bytes; }

hipError_t orthogonalize(bool bf16, int batch, int rows, int cols, const void* G, int ldg, long long strideG, u16* O, int ldo,
                         long long strideO, int steps, void* ws, hipStream_t s) {
  const Plan q = plan_ortho(static_cast<char*>(ws), batch, rows, cols);
  GatherArgs g{};
  g.rows = rows; g.cols = cols; g.G = G; g.ldg = ldg; g.strideG = strideG; g.R = 1;
  g.vec = fours(G, bf16 ? 8 : 16) && ldg % 4 == 0 && strideG % 4 == 0;
  TRY(newton_schulz(q, g, bf16, batch, steps, s));
  FinishArgs f{};
  f.rows = rows; f.cols = cols; f.O = O; f.ldo = ldo; f.strideO = strideO;
  f.vec = fours(O, 8) && ldo % 4 == 0 && strideO % 4 == 0;
  return finish(q, f, batch, s);
}

hipError_t ortho_update(int batch, int rows, int cols, float* W, u16* W16, u16* Wt16, float* momentum, const float* G,
                        size_t layer_stride, size_t replica_stride, int R, float lr, float scale, float decay, float mu,
                        int nesterov, int steps, void* ws, hipStream_t s) {
  const Plan q = plan_ortho(static_cast<char*>(ws), batch, rows, cols);
  GatherArgs g{};
  g.rows = rows; g.cols = cols; g.G = G; g.ldg = cols; g.strideG = (long long)layer_stride;
  g.replica_stride = replica_stride; g.R = R;
  g.momentum = momentum; g.strideM = (long long)layer_stride; g.mu = mu; g.nesterov = nesterov;
  const bool strides = (batch == 1 || layer_stride % 4 == 0) && (R == 1 || replica_stride % 4 == 0);
  g.vec = fours(G, 16) && fours(momentum, 16) && cols % 4 == 0 && strides;
  TRY(newton_schulz(q, g, false, batch, steps, s));
  FinishArgs f{};
  f.rows = rows; f.cols = cols; f.W = W; f.W16 = W16; f.Wt16 = Wt16; f.strideW = (long long)layer_stride;
  f.keep = 1.0f - lr * decay;
  f.step = lr * scale;
  f.vec = fours(W, 16) && fours(W16, 8) && cols % 4 == 0 && strides;
  f.vec_t = fours(Wt16, 8) && rows % 4 == 0 && strides;
  return finish(q, f, batch, s);
}

}  // namespace mi
