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
// X is kept in fp32 beside its fp16 copy, because the a X term carries every direction from one
// iteration to the next and grows small ones 3.4 times each: with the fp16 copy in that term its white
// rounding noise grows along (4e-2 for a floor of 1e-2).  The diagonal of b A + c A^2, near b + c once
// X is near its limit, stays in fp32 too and joins the a X term; its rounding would be most of what is
// left.  Together: 2e-4 .. 8e-4 of |O|.
#include <hip/hip_runtime.h>
#include <cstdlib>

#include <algorithm>

#include "kernels.h"
#include "tile16.h"

namespace mi {

namespace {

constexpr float NS_A = 3.4445f, NS_B = -4.7750f, NS_C = 2.0315f;
constexpr float GRAM_SCALE = 4096.0f;  // A and b A + c A^2 are stored times this: off-diagonal entries start near 1 / (m sqrt n)

inline size_t up(size_t x, size_t a) { return (x + a - 1) / a * a; }

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
  float* X;              // [batch][mp x np], in working orientation
  int mp, np;
  double* sumsq;         // [batch][workgroups of an entry]
};

// U in working orientation, zero padded, and the sum of its squares per workgroup.  64 x 64 tiles of the
// gradient; FLIP turns them through LDS.
template <bool BF16, bool FLIP>
__global__ __launch_bounds__(256) void ortho_gather_kernel(GatherArgs p) {
  __shared__ float tile[FLIP ? 64 : 1][65];
  __shared__ double red[256];
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
  const int r0 = blockIdx.y * 64, c0 = blockIdx.x * 64, col = c0 + tx;
  float* X = p.X + (size_t)blockIdx.z * p.mp * p.np;
  double acc = 0.0;
  for (int i = ty; i < 64; i += 4) {
    const int row = r0 + i;
    float u = 0.0f;
    if (row < p.rows && col < p.cols) {
      const size_t at = (size_t)blockIdx.z * p.strideG + (size_t)row * p.ldg + col;
      if constexpr (BF16) u = bf2f(static_cast<const u16*>(p.G)[at]);
      else {
        const float* g = static_cast<const float*>(p.G) + at;
        u = g[0];
        for (int r = 1; r < p.R; ++r) u += g[(size_t)r * p.replica_stride];
      }
      if (p.momentum) {
        float* m = p.momentum + (size_t)blockIdx.z * p.strideM + (size_t)row * p.cols + col;
        const float now = fmaf(p.mu, *m, u);
        *m = now;
        u = p.nesterov ? fmaf(p.mu, now, u) : now;
      }
    }
    acc += (double)u * (double)u;
    if constexpr (FLIP) tile[i][tx] = u;
    else X[(size_t)row * p.np + col] = u;
  }
  red[threadIdx.x] = acc;
  __syncthreads();
  if constexpr (FLIP) {
    for (int i = ty; i < 64; i += 4) X[(size_t)(c0 + i) * p.np + r0 + tx] = tile[tx][i];
  }
  for (int off = 128; off > 0; off >>= 1) {
    if ((int)threadIdx.x < off) red[threadIdx.x] += red[threadIdx.x + off];
    __syncthreads();
  }
  if (threadIdx.x == 0) p.sumsq[((size_t)blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x] = red[0];
}

// inv[entry] = 1 / |U|_F; 0 for U = 0, NaN where |U|_F is not finite.
__global__ __launch_bounds__(256) void ortho_norm_kernel(const double* __restrict__ sumsq, int blocks, double* __restrict__ inv) {
  __shared__ double red[256];
  double acc = 0.0;
  for (int i = threadIdx.x; i < blocks; i += 256) acc += sumsq[(size_t)blockIdx.x * blocks + i];
  red[threadIdx.x] = acc;
  __syncthreads();
  for (int off = 128; off > 0; off >>= 1) {
    if ((int)threadIdx.x < off) red[threadIdx.x] += red[threadIdx.x + off];
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    const double q = red[0];
    inv[blockIdx.x] = q == 0.0 ? 0.0 : __builtin_isfinite(q) ? 1.0 / sqrt(q) : __builtin_nan("");
  }
}

// X <- X / |U|_F, Xh = fp16(scale X), XhT its transpose.  64 x 64 tiles.
__global__ __launch_bounds__(256) void ortho_scale_kernel(float* __restrict__ X, u16* __restrict__ Xh, u16* __restrict__ XhT, int mp,
                                                          int np, const double* __restrict__ inv, float scale) {
  __shared__ u16 tile[64][66];
  const size_t base = (size_t)blockIdx.z * mp * np;
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6, r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;
  const double f = inv[blockIdx.z];
  for (int i = ty; i < 64; i += 4) {
    const size_t at = base + (size_t)(r0 + i) * np + c0 + tx;
    const float x = (float)((double)X[at] * f);
    X[at] = x;
    const u16 h = __builtin_bit_cast(u16, (_Float16)(scale * x));
    Xh[at] = h;
    tile[i][tx] = h;
  }
  __syncthreads();
  for (int i = ty; i < 64; i += 4) XhT[base + (size_t)(c0 + i) * mp + r0 + tx] = tile[tx][i];
}

// ---- the products -----------------------------------------------------------------------------------

// A = X X^T (times GRAM_SCALE, fp16): a tile of the lower triangle and its mirror image.
struct EpiGram {
  struct Args {
    u16* A;
    int ld;
    long long batch;
    float scale;
  };
  template <int QB, class Get>
  static __device__ __forceinline__ void run(const Args& e, const Tile16& p, Get get, int row0, int colw, int lane,
                                             unsigned char* stage, int entry, int) {
    u16* A = e.A + (size_t)entry * e.batch;
    const int l16 = lane & 15, col = colw + 8 * (lane >> 4);
    u32x4 pk[QB][2];
#pragma unroll
    for (int jq = 0; jq < QB; ++jq)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int k = 0; k < 4; ++k) pk[jq][h][k] = pack16<true>(e.scale * get(jq, h, 2 * k), e.scale * get(jq, h, 2 * k + 1));
        *reinterpret_cast<u32x4*>(A + (size_t)(row0 + 16 * jq + l16) * e.ld + col + 32 * h) = pk[jq][h];
      }
    if (row0 / p.tile != colw / p.tile) store_transposed<QB>(A + (size_t)colw * e.ld + row0, e.ld, pk, lane, stage);
  }
};

// P = b A + c A A without its diagonal (times GRAM_SCALE, fp16), the diagonal in fp32.
struct EpiPoly {
  struct Args {
    const u16* A;
    u16* P;
    float* diag;
    int ld;
    long long batch;
  };
  template <int QB, class Get>
  static __device__ __forceinline__ void run(const Args& e, const Tile16& p, Get get, int row0, int colw, int lane,
                                             unsigned char* stage, int entry, int) {
    const u16* A = e.A + (size_t)entry * e.batch;
    u16* P = e.P + (size_t)entry * e.batch;
    const int l16 = lane & 15, col = colw + 8 * (lane >> 4);
    u32x4 pk[QB][2];
#pragma unroll
    for (int jq = 0; jq < QB; ++jq)
#pragma unroll
      for (int h = 0; h < 2; ++h) pk[jq][h] = *reinterpret_cast<const u32x4*>(A + (size_t)(row0 + 16 * jq + l16) * e.ld + col + 32 * h);
    const bool on_diagonal = row0 / p.tile == colw / p.tile;
#pragma unroll
    for (int jq = 0; jq < QB; ++jq)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = row0 + 16 * jq + l16;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const unsigned w = pk[jq][h][i >> 1];
          v[i] = fmaf(NS_C / GRAM_SCALE, get(jq, h, i), NS_B * ((i & 1) ? f16_hi(w) : f16_lo(w)));
        }
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
        *reinterpret_cast<u32x4*>(P + (size_t)row * e.ld + col + 32 * h) = pk[jq][h];
      }
    if (!on_diagonal) store_transposed<QB>(P + (size_t)colw * e.ld + row0, e.ld, pk, lane, stage);
  }
};

// X <- (a + diag) X + P X; the fp16 copy and its transpose for the next iteration (null: last one).
struct EpiStep {
  struct Args {
    float* X;
    const float* diag;
    u16 *Xh, *XhT;
    int mp, np;
    float unscale, scale;  // accumulator -> X, X -> fp16 copy
  };
  template <int QB, class Get>
  static __device__ __forceinline__ void run(const Args& e, const Tile16& p, Get get, int row0, int colw, int lane,
                                             unsigned char* stage, int entry, int) {
    const size_t base = (size_t)entry * e.mp * e.np;
    const int l16 = lane & 15, col = colw + 8 * (lane >> 4);
    u32x4 pk[QB][2];
#pragma unroll
    for (int jq = 0; jq < QB; ++jq) {
      const int row = row0 + 16 * jq + l16;
      const float keep = NS_A + e.diag[(size_t)entry * e.mp + row];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        f32x4* x = reinterpret_cast<f32x4*>(e.X + base + (size_t)row * e.np + col + 32 * h);
        f32x4 v[2] = {x[0], x[1]};
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i >> 2][i & 3] = fmaf(keep, v[i >> 2][i & 3], e.unscale * get(jq, h, i));
        x[0] = v[0];
        x[1] = v[1];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          pk[jq][h][k] = pack16<true>(e.scale * v[k >> 1][2 * (k & 1)], e.scale * v[k >> 1][2 * (k & 1) + 1]);
        if (e.Xh) *reinterpret_cast<u32x4*>(e.Xh + base + (size_t)row * e.np + col + 32 * h) = pk[jq][h];
      }
    }
    if (e.XhT) store_transposed<QB>(e.XhT + base + (size_t)colw * e.mp + row0, e.mp, pk, lane, stage);
  }
};

// ---- O out, W updated -------------------------------------------------------------------------------

struct FinishArgs {
  int rows, cols;
  const float* X;  // [batch][mp x np]
  int mp, np;
  u16* O;          // bf16 result, or null
  int ldo;
  long long strideO;
  float* W;        // dense [rows x cols] with its bf16 copies (either may be null), or null
  u16 *W16, *Wt16;
  long long strideW;
  float keep, step;  // W <- keep W - step O
};

template <bool FLIP>
__global__ __launch_bounds__(256) void ortho_finish_kernel(FinishArgs p) {
  __shared__ float turned[FLIP ? 64 : 1][65];
  __shared__ u16 tile[64][66];
  const float* X = p.X + (size_t)blockIdx.z * p.mp * p.np;
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6, r0 = blockIdx.y * 64, c0 = blockIdx.x * 64, col = c0 + tx;
  if constexpr (FLIP) {  // X is padded to whole 64 x 64 tiles
    for (int i = ty; i < 64; i += 4) turned[i][tx] = X[(size_t)(c0 + i) * p.np + r0 + tx];
    __syncthreads();
  }
  for (int i = ty; i < 64; i += 4) {
    const int row = r0 + i;
    if (row >= p.rows || col >= p.cols) continue;
    const float o = FLIP ? turned[tx][i] : X[(size_t)row * p.np + col];
    if (p.O) p.O[(size_t)blockIdx.z * p.strideO + (size_t)row * p.ldo + col] = f2bf(o);
    if (p.W) {
      const size_t at = (size_t)blockIdx.z * p.strideW + (size_t)row * p.cols + col;
      const float w = fmaf(-p.step, o, p.keep * p.W[at]);
      p.W[at] = w;
      const u16 h = f2bf(w);
      if (p.W16) p.W16[at] = h;
      tile[i][tx] = h;
    }
  }
  if (!p.Wt16) return;
  __syncthreads();
  for (int i = ty; i < 64; i += 4)
    if (c0 + i < p.cols && r0 + tx < p.rows)
      p.Wt16[(size_t)blockIdx.z * p.strideW + (size_t)(c0 + i) * p.rows + r0 + tx] = tile[tx][i];
}

// ---- sizes ------------------------------------------------------------------------------------------

struct Plan {
  int m, n, mp, np;
  int tile;    // of the products; m and n are padded to multiples of it
  bool flip;
  float scale;  // of the fp16 copies of X: a power of two near sqrt(n), so that typical entries start near 1 / sqrt(m)
  float* X;
  u16 *Xh, *XhT[2], *A, *P;
  float* diag;
  double *sumsq, *inv;
  size_t bytes;
};
Plan plan_ortho(char* base, int batch, int rows, int cols) {
  Plan q{};
  q.flip = rows > cols;
  q.m = std::min(rows, cols);
  q.n = std::max(rows, cols);
  // large matrices: 256 x 256 tiles once even the smallest products (the triangle of m x m) fill the CUs
  const size_t t = up(q.m, 256) / 256;
  q.tile = batch * t * (t + 1) / 2 >= 200 ? 256 : 128;
  { static int t = getenv("TT") ? atoi(getenv("TT")) : 0; if (t) q.tile = t; }
  q.mp = (int)up(q.m, q.tile);
  q.np = (int)up(q.n, q.tile);
  q.scale = 1.0f;
  while (q.scale * q.scale < (float)q.n && q.scale < 256.0f) q.scale *= 2.0f;
  size_t used = 0;
  auto take = [&](size_t bytes) {
    char* at = base ? base + used : nullptr;
    used += up(bytes, 256);
    return at;
  };
  const size_t x = (size_t)batch * q.mp * q.np, a = (size_t)batch * q.mp * q.mp;
  q.X = (float*)take(x * 4);
  q.Xh = (u16*)take(x * 2);
  q.XhT[0] = (u16*)take(x * 2);
  q.XhT[1] = (u16*)take(x * 2);
  q.A = (u16*)take(a * 2);
  q.P = (u16*)take(a * 2);
  q.diag = (float*)take((size_t)batch * q.mp * 4);
  q.sumsq = (double*)take((size_t)batch * (q.mp / 64) * (q.np / 64) * 8);
  q.inv = (double*)take((size_t)batch * 8);
  q.bytes = used;
  return q;
}

template <class Epi>
hipError_t tiles(int tile, const u16* A, const u16* B, int M, int N, int K, long long batchA, long long batchB, int batch, bool symmetric,
                 const typename Epi::Args& e, hipStream_t s) {
  Tile16 p{};
  p.A = A; p.B = B; p.lda = K; p.ldb = K; p.M = M; p.N = N; p.K = K;
  p.batchA = batchA; p.batchB = batchB;
  p.splits = 1;
  p.symmetric = symmetric;
  p.tile = tile;
  return launch_tile16<true, Epi>(p, e, batch, s);
}

#define TRY(call)                          \
  do {                                     \
    hipError_t e_ = (call);                \
    if (e_ != hipSuccess) return e_;       \
  } while (0)

// U (gathered by `g`) -> X of the last iteration, in q.X.
hipError_t newton_schulz(const Plan& q, GatherArgs g, bool bf16, int batch, int steps, hipStream_t s) {
  g.X = q.X;
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
  launch_kernel(ortho_norm_kernel, dim3(batch), dim3(256), 0, s, (const double*)q.sumsq, (q.mp / 64) * (q.np / 64), q.inv);
  TRY(hipGetLastError());
  launch_kernel(ortho_scale_kernel, tiles64, dim3(256), 0, s, q.X, q.Xh, q.XhT[0], q.mp, q.np, (const double*)q.inv, q.scale);
  TRY(hipGetLastError());
  const long long x = (long long)q.mp * q.np, a = (long long)q.mp * q.mp;
  for (int k = 0; k < steps; ++k) {
    const bool last = k + 1 == steps;
    const EpiGram::Args gram{q.A, q.mp, a, GRAM_SCALE / (q.scale * q.scale)};
    TRY(tiles<EpiGram>(q.tile, q.Xh, q.Xh, q.mp, q.mp, q.np, x, x, batch, true, gram, s));
    const EpiPoly::Args poly{q.A, q.P, q.diag, q.mp, a};
    TRY(tiles<EpiPoly>(q.tile, q.A, q.A, q.mp, q.mp, q.mp, a, a, batch, true, poly, s));
    const EpiStep::Args step{q.X, q.diag, last ? nullptr : q.Xh, last ? nullptr : q.XhT[(k + 1) & 1], q.mp, q.np,
                             1.0f / (GRAM_SCALE * q.scale), q.scale};
    TRY(tiles<EpiStep>(q.tile, q.P, q.XhT[k & 1], q.mp, q.np, q.mp, a, x, batch, false, step, s));
  }
  return hipSuccess;
}

hipError_t finish(const Plan& q, FinishArgs f, int batch, hipStream_t s) {
  f.X = q.X;
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
  TRY(newton_schulz(q, g, bf16, batch, steps, s));
  FinishArgs f{};
  f.rows = rows; f.cols = cols; f.O = O; f.ldo = ldo; f.strideO = strideO;
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
  TRY(newton_schulz(q, g, false, batch, steps, s));
  FinishArgs f{};
  f.rows = rows; f.cols = cols; f.W = W; f.W16 = W16; f.Wt16 = Wt16; f.strideW = (long long)layer_stride;
  f.keep = 1.0f - lr * decay;
  f.step = lr * scale;
  return finish(q, f, batch, s);
}

}  // namespace mi
