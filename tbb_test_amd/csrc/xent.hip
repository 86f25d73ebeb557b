// Softmax cross entropy of a linear classifier without keeping its logits.
//
//   z = X W^T + b [M x V]      lse_i = log sum_j exp z_ij      loss_i = lse_i - z_i,t(i)
//   g_ij = d_i (exp(z_ij - lse_i) - [j = t(i)])      dX = g W      dW = g^T X      db_j = sum_i g_ij
//
// Forward, bf16: one pass of MFMA tiles over z.  A tile leaves two numbers per row and 64 columns, the
// maximum m and s = sum exp(z - m) over the columns other than the target, and the target's own logit;
// a fold joins them.  The target is kept apart because lse - z_t cancels where a row is sure of its
// answer; with o = log sum over the others, loss = softplus(o - z_t) does not.
// Backward, bf16: the vocabulary is walked in pieces.  Per piece the tiles of z are computed again and
// leave as g (rounded to bf16, the operand type of the products that follow: at most 2^-8 of each
// term) in both orders that the next two products read, g for dX += g W and g^T for dW = g^T X.
// fp32 models: the same pieces through the framework's fp32 GEMMs, with the softmax between them.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "kernels.h"
#include "tile16.h"

namespace mi {

namespace {

constexpr float LOG2E = 1.44269504088896340736f;

// 16 bytes that start at any element: one load or store where the hardware's alignment rules ask for no more.
template <class Element, class Vector>
struct __attribute__((packed, aligned(sizeof(Element)))) Anywhere {
  Vector v;
};

__device__ __forceinline__ float finite_or_zero(float m) { return __builtin_isinf(m) ? 0.0f : m; }

// (m, s) stands for m' + log s with m' = 0 where m is infinite.  m = -inf: nothing but -inf (s = 0) or
// NaN (s = NaN) so far; m = +inf: s = inf.  NaN travels in s, which every NaN logit reaches.
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
  const float top = fmaxf(m, m2), t = finite_or_zero(top);
  const float w1 = m == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f((finite_or_zero(m) - t) * LOG2E);
  const float w2 = m2 == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f((finite_or_zero(m2) - t) * LOG2E);
  s = s * w1 + s2 * w2;
  m = top;
}

// Loss and lse of a row from the statistics of its other columns and the target's logit.
__device__ __forceinline__ void finish_row(float m, float s, bool counts, float zt, float* loss, float* lse) {
  const float others = finite_or_zero(m) + logf(s);
  if (!counts) {
    *loss = 0.0f;
    *lse = others;
    return;
  }
  const float d = others - zt;
  const float tail = log1pf(expf(-fabsf(d)));
  // d = NaN: the tail is NaN; z_t = inf: lse - z_t is inf - inf, where the other form would make it 0
  *loss = zt == __builtin_inff() ? __builtin_nanf("") : fmaxf(d, 0.0f) + tail;
  *lse = others == zt && __builtin_isinf(zt) ? zt : fmaxf(others, zt) + tail;
}

// ---- bf16 tiles -------------------------------------------------------------------------------------

// Statistics of z, 64 columns of a row at a time: a lane holds 16 of them, the four lanes of a row join by two
// exchanges, one pair of floats is stored.  Bound by the MFMAs: 16384 x 131072 x 4096 in 12.4 ms, 1415 TFLOP/s, what a
// large library product reaches; with K = 2048 (32 steps a tile) the exponentials cost a tenth (1180).
struct EpiStats : NoPre {
  static constexpr bool MAY_SPLIT = false;
  struct Args {
    const float* bias;    // of the first column, or null
    const int* target;
    int first, vocab;     // first column of this launch in the vocabulary, size of the vocabulary
    float* zt;            // [M]
    float2* part;         // [column block of 64][M], from this launch's first block on
  };
  template <int QB, class Get>
  static __device__ __forceinline__ void run(const Args& e, const Tile16& p, const Pre<QB>& pre, Get get, int row0, int colw, int lane,
                                             unsigned char*, int) {
    const int l16 = lane & 15, q = lane >> 4, lane_col = colw + 8 * q;
    if (colw >= p.N) return;
    float bias[2][8];
    const bool edge = colw + 64 > p.N;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int col = lane_col + 32 * h + i;
        bias[h][i] = e.bias && col < p.N ? e.bias[col] : 0.0f;
      }
#pragma unroll
    for (int jq = 0; jq < QB; ++jq) {
      const int row = row0 + 16 * jq + l16;
      int t = row < p.M ? e.target[row] : -1;
      t = t >= 0 && t < e.vocab ? t - e.first - lane_col : -1;  // relative to the lane's first column
      float v[2][8];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 8; ++i) v[h][i] = get(jq, h, i) + bias[h][i];
      if (t >= 0 && t < 40 && (t & 31) < 8) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (t == 32 * h + i) {
              e.zt[row] = v[h][i];
              v[h][i] = -__builtin_inff();
            }
      }
      if (edge) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (lane_col + 32 * h + i >= p.N) v[h][i] = -__builtin_inff();
      }
      float m = v[0][0];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 8; ++i) m = fmaxf(m, v[h][i]);
      m = fmaxf(m, __shfl_xor(m, 16, 64));
      m = fmaxf(m, __shfl_xor(m, 32, 64));
      const float mm = finite_or_zero(m);
      float s = 0.0f;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 8; ++i) s += __builtin_amdgcn_exp2f((v[h][i] - mm) * LOG2E);
      s += __shfl_xor(s, 16, 64);
      s += __shfl_xor(s, 32, 64);
      if (q == 0 && row < p.M) e.part[(size_t)(colw >> 6) * p.M + row] = float2{m, s};
    }
  }
};

// g from z and lse, in both orders, and its column sums.  8192 x 32768 x 4096: 1.79 ms, 1230 TFLOP/s; the 1.07 GB of g
// and g^T take what is missing to the products that store one result (1.58 ms).
struct EpiGrad : NoPre {
  static constexpr bool MAY_SPLIT = false;
  struct Args {
    const float* bias;
    const int* target;
    const float* lse;
    const float* dloss;  // null: 1 for every row
    const float* top;    // g is kept divided by *top, the largest |dloss| (see xent_top_kernel)
    int first, vocab;
    u16* G;              // [rows padded][ldg]
    u16* GT;             // [columns padded][ldgt]
    int ldg, ldgt, lddb;
    float* db_part;      // column sums per wavefront tile of 16 QB rows, [row0 / (16 QB)][lddb], or null
  };
  template <int QB, class Get>
  static __device__ __forceinline__ void run(const Args& e, const Tile16& p, const Pre<QB>& pre, Get get, int row0, int colw, int lane,
                                             unsigned char* stage, int) {
    const int l16 = lane & 15, q = lane >> 4, lane_col = colw + 8 * q;
    float bias[2][8], sums[2][8];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int col = lane_col + 32 * h + i;
        bias[h][i] = e.bias && col < p.N ? e.bias[col] : 0.0f;
        sums[h][i] = 0.0f;
      }
    const bool edge = colw + 64 > p.N;
    const float top = e.dloss ? *e.top : 1.0f;
    u32x4 pk[QB][2];
#pragma unroll
    for (int jq = 0; jq < QB; ++jq) {
      const int row = row0 + 16 * jq + l16;
      int t = row < p.M ? e.target[row] : -1;
      const bool live = t >= 0 && t < e.vocab;
      t = t - e.first - lane_col;
      const float lse = live ? e.lse[row] : 0.0f;
      const float d = live ? (e.dloss ? e.dloss[row] / top : 1.0f) : 0.0f;
      float g[2][8];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float x = __builtin_amdgcn_exp2f((get(jq, h, i) + bias[h][i] - lse) * LOG2E);
          g[h][i] = live ? d * x : 0.0f;
        }
      if (live && t >= 0 && t < 40 && (t & 31) < 8) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (t == 32 * h + i) g[h][i] = d * expm1f(get(jq, h, i) + bias[h][i] - lse);
      }
      if (edge) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (lane_col + 32 * h + i >= p.N) g[h][i] = 0.0f;
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int i = 0; i < 8; ++i) sums[h][i] += g[h][i];
#pragma unroll
        for (int k = 0; k < 4; ++k) pk[jq][h][k] = pack16<false>(g[h][2 * k], g[h][2 * k + 1]);
        *reinterpret_cast<u32x4*>(e.G + (size_t)row * e.ldg + lane_col + 32 * h) = pk[jq][h];
      }
    }
    if (e.db_part) {
      float* dst = e.db_part + (size_t)(row0 / (16 * QB)) * e.lddb + lane_col;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int off = 1; off < 16; off <<= 1) sums[h][i] += __shfl_xor(sums[h][i], off, 64);
        if (l16 == 0) {
          *reinterpret_cast<f32x4*>(dst + 32 * h) = f32x4{sums[h][0], sums[h][1], sums[h][2], sums[h][3]};
          *reinterpret_cast<f32x4*>(dst + 32 * h + 4) = f32x4{sums[h][4], sums[h][5], sums[h][6], sums[h][7]};
        }
      }
    }
    store_transposed<QB>(e.GT + (size_t)colw * e.ldgt + row0, e.ldgt, pk, lane, stage);
  }
};

// C = factor * (base + A B^T), fp32 or bf16; rows and columns behind the result are dropped.  DX: rows that do not count
// become zeros (their g is zero, but zero times an infinity or NaN of W is not); the other results' epilogues are left
// without that (a run-time test takes 4 us of the 27 of dW of 32000 classes x 1024 from one row).
// dW of 32768 classes x 4096 from 8192 rows: 1.59 ms, 1385 TFLOP/s; dX from 32768 classes 1.68 ms (rows of a caller's Wt
// a power of two apart share memory channels).
template <bool OUT_BF16, bool DX = false>
struct EpiOut {
  static constexpr bool MAY_SPLIT = true;
  struct Args {
    void* C;
    int ldc;
    const float* base;    // [M][ld_base] or null; may be C
    int ld_base;          // a multiple of 64
    const float* factor;  // null: 1
    const int* target;    // DX only
    int vocab;
  };
  template <int QB>
  struct Pre {
    int target[DX ? QB : 1];
    f32x4 base[QB][2][2];
  };
  template <int QB>
  static __device__ __forceinline__ Pre<QB> before(const Args& e, const Tile16& p, int row0, int colw, int lane, int) {
    Pre<QB> v;
    if constexpr (DX) {
#pragma unroll
      for (int jq = 0; jq < QB; ++jq) v.target[jq] = e.target[min(row0 + 16 * jq + (lane & 15), p.M - 1)];
    }
    if (!e.base) return v;
#pragma unroll
    for (int jq = 0; jq < QB; ++jq)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int row = row0 + 16 * jq + (lane & 15), col = colw + 8 * (lane >> 4) + 32 * h + 4 * k;
          v.base[jq][h][k] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};  // rows of base have whole groups of 64 columns
          if (row < p.M && col < p.N) v.base[jq][h][k] = *reinterpret_cast<const f32x4*>(e.base + (size_t)row * e.ld_base + col);
        }
    return v;
  }
  template <int QB, class Get>
  static __device__ __forceinline__ void run(const Args& e, const Tile16& p, const Pre<QB>& pre, Get get, int row0, int colw, int lane,
                                             unsigned char*, int) {
    const int l16 = lane & 15, col0 = colw + 8 * (lane >> 4);
    const float factor = e.factor ? *e.factor : 1.0f;
    asm volatile("" ::: "memory");  // (base was requested before the first store)
#pragma unroll
    for (int jq = 0; jq < QB; ++jq) {
      const int row = row0 + 16 * jq + l16;
      if (row >= p.M) continue;
      bool counts = true;
      if constexpr (DX) counts = pre.target[jq] >= 0 && pre.target[jq] < e.vocab;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int col = col0 + 32 * h;
        if (col >= p.N) continue;
        const size_t at = (size_t)row * e.ldc + col;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = get(jq, h, i);
        if (e.base) {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] += pre.base[jq][h][i >> 2][i & 3];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = counts ? v[i] * factor : 0.0f;
        const bool whole = col + 8 <= p.N;
        if constexpr (OUT_BF16) {
          u16* c = reinterpret_cast<u16*>(e.C) + at;
          if (whole) {
            reinterpret_cast<Anywhere<u16, u32x4>*>(c)->v = u32x4{pack16<false>(v[0], v[1]), pack16<false>(v[2], v[3]),
                                                                  pack16<false>(v[4], v[5]), pack16<false>(v[6], v[7])};
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (col + i < p.N) c[i] = f2bf(v[i]);
          }
        } else {
          float* c = reinterpret_cast<float*>(e.C) + at;
          if (whole) {
            reinterpret_cast<Anywhere<float, f32x4>*>(c)[0].v = f32x4{v[0], v[1], v[2], v[3]};
            reinterpret_cast<Anywhere<float, f32x4>*>(c)[1].v = f32x4{v[4], v[5], v[6], v[7]};
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (col + i < p.N) c[i] = v[i];
          }
        }
      }
    }
  }
};

Tile16 product(const u16* A, int lda, const u16* B, int ldb, int M, int N, int K) {
  Tile16 p{};
  p.A = A; p.B = B; p.lda = lda; p.ldb = ldb; p.M = M; p.N = N; p.K = K;
  p.batch = 1;
  return p;
}
template <class Epi>
hipError_t tiles(const Tile16Shape& shape, float* part, const u16* A, int lda, const u16* B, int ldb, int M, int N, int K,
                 const typename Epi::Args& e, hipStream_t s) {
  return launch_tile16<false, Epi>(product(A, lda, B, ldb, M, N, K), shape, part, e, s);
}

// ---- few rows ----------------------------------------------------------------------------------------

// Statistics as EpiStats leaves them, for at most 16 QB rows: W is read once, straight into registers in 16-byte pieces
// that may start at any element (the direct loads into LDS cannot), 16 NB classes per wavefront, AHEAD K chunks (of 32
// elements bf16, 16 fp32) of W and X requested ahead of those being multiplied; X (rows of whole pieces, zeros behind K)
// comes out of the caches.  Wavefronts join to blocks of 64 classes.
// For bf16 classes that the tiles cannot read in place, and for fp32, where tiles of 16 or 32 rows wait for memory:
//   bf16  4 x 30592 x 2956: 47 us, 3.9 TB/s of W, where copying W for the tiles, two more passes over it, makes 164;
//         64 x 49165 x 3501, rows at any 2 bytes: 192 us instead of 422
//   fp32  1 x 32000 x 1024: 32 us, 4.1 TB/s of W, instead of 50; 1 x 44992 x 1944: 82 us, with its copy 337
// More rows want more classes per wavefront (X is read once for each) where that leaves enough wavefronts: 32 rows of
// 50000 x 1002 bf16 52 us with 16 classes and 42 with 32, of 6464 x 1501 30 and 44 us; 64 rows of 49165 x 3501 221 us
// with 32 and 192 with 64.  Few classes leave each wavefront alone with its whole K: 32 rows of 1500 x 1501 bf16 take 32 us
// and through copies and tiles 21 us, of 6464 x 1501 30 and 34 us.
template <class T>
constexpr int FEW_ROWS = sizeof(T) == 2 ? 64 : 32;
template <class T>
struct FewRows {
  const T* X;  // [M][ldx], rows of whole 16-byte pieces, zeros behind K up to whole chunks
  const T* W;  // [V][ldw]
  int M, V, K, ldx, ldw;
  const float* bias;
  const int* target;
  float* zt;
  float2* part;
};
template <class T, int QB, int NB, int AHEAD>
__global__ __launch_bounds__(256) void xent_few_rows_kernel(FewRows<T> p) {
  constexpr int EACH = 16 / sizeof(T), CHUNK = 4 * EACH;  // elements of a piece, and of the four lanes of a class
  using Piece = Anywhere<T, u32x4>;
  __shared__ float2 red[4][16 * QB];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, q = lane >> 4;
  const int c0 = ((int)blockIdx.x * 4 + wave) * 16 * NB;
  const T* w[NB];
  const T* x[QB];
#pragma unroll
  for (int b = 0; b < NB; ++b) w[b] = p.W + (size_t)min(c0 + 16 * b + l16, p.V - 1) * p.ldw + EACH * q;
#pragma unroll
  for (int j = 0; j < QB; ++j) x[j] = p.X + (size_t)min(16 * j + l16, p.M - 1) * p.ldx + EACH * q;
  f32x4 acc[QB][NB];
#pragma unroll
  for (int j = 0; j < QB; ++j)
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[j][b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  struct Chunk {
    u32x4 x[QB], w[NB];
  };
  auto multiply = [&](const Chunk& f) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < QB; ++j)
#pragma unroll
      for (int b = 0; b < NB; ++b)
        if constexpr (sizeof(T) == 2)
          acc[j][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, f.w[b]), __builtin_bit_cast(bf16x8, f.x[j]), acc[j][b], 0, 0, 0);
        else  // one element of each lane's four at a time: which four K elements share a product is the same on both sides
#pragma unroll
          for (int u = 0; u < 4; ++u)
            acc[j][b] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(f.w[b][u]), __uint_as_float(f.x[j][u]), acc[j][b], 0, 0, 0);
  };
  // X is requested as far ahead as W: loads return in order, so one for now would wait for the W of later
  const int whole = p.K / CHUNK;
  Chunk now[AHEAD], next[AHEAD];
  auto request = [&](Chunk(&f)[AHEAD], int t) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
#pragma unroll
      for (int j = 0; j < QB; ++j) f[u].x[j] = *reinterpret_cast<const u32x4*>(x[j] + CHUNK * (t + u));
#pragma unroll
      for (int b = 0; b < NB; ++b) f[u].w[b] = reinterpret_cast<const Piece*>(w[b] + CHUNK * (t + u))->v;
    }
  };
  int t = 0;
  if (t + AHEAD <= whole) request(now, t);
  for (; t + AHEAD <= whole; t += AHEAD) {
    if (t + 2 * AHEAD <= whole) request(next, t + AHEAD);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) multiply(now[u]);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) now[u] = next[u];
  }
  for (; CHUNK * t < p.K; ++t) {  // the chunks left over, the last of them element by element where it is cut
    Chunk f;
#pragma unroll
    for (int j = 0; j < QB; ++j) f.x[j] = *reinterpret_cast<const u32x4*>(x[j] + CHUNK * t);
    const int there = p.K - CHUNK * t - EACH * q;  // elements of the lane's piece that are there
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      f.w[b] = u32x4{0u, 0u, 0u, 0u};
      if (there >= EACH) f.w[b] = reinterpret_cast<const Piece*>(w[b] + CHUNK * t)->v;
      else
#pragma unroll
        for (int i = 0; i < EACH; ++i)
          if (i < there) {
            if constexpr (sizeof(T) == 2) f.w[b][i >> 1] |= (unsigned)w[b][CHUNK * t + i] << (16 * (i & 1));
            else f.w[b][i] = __float_as_uint(w[b][CHUNK * t + i]);
          }
    }
    multiply(f);
  }
  // a lane holds classes c0 + 16 b + 4 q + r of row 16 j + l16
#pragma unroll
  for (int j = 0; j < QB; ++j) {
    const int row = 16 * j + l16;
    int target = row < p.M ? p.target[row] : -1;
    if (target >= p.V) target = -1;
    float top = -__builtin_inff(), sum = 0.0f;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int c = c0 + 16 * b + 4 * q + r;
        float v = acc[j][b][r] + (p.bias && c < p.V ? p.bias[c] : 0.0f);
        if (c == target) p.zt[row] = v;
        if (c == target || c >= p.V) v = -__builtin_inff();
        acc[j][b][r] = v;
        top = fmaxf(top, v);
      }
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const float ref = finite_or_zero(top);
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) sum += __builtin_amdgcn_exp2f((acc[j][b][r] - ref) * LOG2E);
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    if (q == 0) red[wave][row] = float2{top, sum};
  }
  __syncthreads();
  // NB blocks of 64 classes per workgroup, 4 / NB wavefronts each
  for (int i = threadIdx.x; i < NB * 16 * QB; i += 256) {
    const int b = i / (16 * QB), row = i % (16 * QB), block = blockIdx.x * NB + b;
    if (row >= p.M || 64 * block >= p.V) continue;
    float2 all = red[b * (4 / NB)][row];
#pragma unroll
    for (int k = 1; k < 4 / NB; ++k) join(all.x, all.y, red[b * (4 / NB) + k][row].x, red[b * (4 / NB) + k][row].y);
    p.part[(size_t)block * p.M + row] = all;
  }
}

// ---- joins and copies -------------------------------------------------------------------------------

// Joins a row's column-block statistics.  ROWS rows per workgroup, 256 / ROWS lanes on each: a lane takes every
// so-manieth block, the lanes of a row are joined pairwise.  Few rows take many lanes each: one row over 500 blocks
// takes 4 us with 256 lanes and 14 with 16.
template <int ROWS>
__global__ __launch_bounds__(256) void xent_fold_kernel(const float2* __restrict__ part, int blocks, int M, int vocab,
                                                        const int* __restrict__ target, const float* __restrict__ zt,
                                                        float* __restrict__ loss, float* __restrict__ lse) {
  constexpr int LANES = 256 / ROWS;
  __shared__ float2 red[LANES][ROWS + 1];
  const int r = threadIdx.x % ROWS, w = threadIdx.x / ROWS, row = blockIdx.x * ROWS + r;
  float m = -__builtin_inff(), s = 0.0f;
  if (row < M) {
    int c = w;
    for (; c + 3 * LANES < blocks; c += 4 * LANES) {
      float2 v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = part[(size_t)(c + k * LANES) * M + row];
#pragma unroll
      for (int k = 0; k < 4; ++k) join(m, s, v[k].x, v[k].y);
    }
    for (; c < blocks; c += LANES) {
      const float2 v = part[(size_t)c * M + row];
      join(m, s, v.x, v.y);
    }
  }
  red[w][r] = float2{m, s};
  __syncthreads();
  for (int off = LANES / 2; off > 0; off >>= 1) {
    if (w < off) {
      const float2 v = red[w + off][r];
      join(m, s, v.x, v.y);
      red[w][r] = float2{m, s};
    }
    __syncthreads();
  }
  if (w != 0 || row >= M) return;
  const int t = target[row];
  const bool counts = t >= 0 && t < vocab;
  finish_row(m, s, counts, counts ? zt[row] : 0.0f, loss + row, lse + row);
}

// dst[rows][ldd] = src[rows][cols], zeros up to ldd (a multiple of 64).  A wavefront copies 512 elements of a row, eight
// per lane, in one load that may start at any element.
__global__ __launch_bounds__(256) void pack_rows_kernel(u16* __restrict__ dst, const u16* __restrict__ src, int rows, int cols,
                                                        int ld, int ldd) {
  const int c = blockIdx.x * 512 + (threadIdx.x & 63) * 8;
  if (c >= ldd) return;
  for (int r = blockIdx.y * 4 + (threadIdx.x >> 6); r < rows; r += gridDim.y * 4) {
    const u16* from = src + (size_t)r * ld + c;
    u32x4 v = {0u, 0u, 0u, 0u};
    if (c + 8 <= cols) {
      v = reinterpret_cast<const Anywhere<u16, u32x4>*>(from)->v;
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (c + k < cols) v[k >> 1] |= (unsigned)from[k] << (16 * (k & 1));
    }
    *reinterpret_cast<u32x4*>(dst + (size_t)r * ldd + c) = v;
  }
}

// Whether row r counts; target = null: every row does.
__device__ __forceinline__ bool row_counts(const int* __restrict__ target, int vocab, int r) {
  if (!target) return true;
  const int t = target[r];
  return t >= 0 && t < vocab;
}

// dst[c][r] = src[r][c] for c < cols, r < ldd; zeros from row `rows` on, and for rows that do not count (their g is
// zero, but zero times an infinity or NaN would reach every dW).  ldd is a multiple of 64, dst 16-byte
// aligned; vec: src is read in 16-byte pieces where a 64 x 64 tile is whole.
struct Transposition {
  u16* dst;
  const u16* src;
  int rows, cols, ld, ldd, vec;
  int blocks_x, blocks;  // 64 x 64 tiles: across cols, and in all
  const int* target;     // of the rows, or null
  int vocab;
};
__device__ __forceinline__ void transpose_tile(const Transposition& t, int block, u16 (*tile)[72]) {
  const int by = block / t.blocks_x, r0 = by * 64, c0 = (block - by * t.blocks_x) * 64;
  const int part = threadIdx.x & 7, line = threadIdx.x >> 3;
  if (t.vec && r0 + 64 <= t.rows && c0 + 64 <= t.cols) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = line + 32 * i;
      const u32x4 v = *reinterpret_cast<const u32x4*>(t.src + (size_t)(r0 + r) * t.ld + c0 + part * 8);
      *reinterpret_cast<u32x4*>(&tile[r][part * 8]) = row_counts(t.target, t.vocab, r0 + r) ? v : u32x4{0u, 0u, 0u, 0u};
    }
  } else {
    const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
#pragma unroll
    for (int i = ty; i < 64; i += 4)
      tile[i][tx] = r0 + i < t.rows && c0 + tx < t.cols && row_counts(t.target, t.vocab, r0 + i)
                        ? t.src[(size_t)(r0 + i) * t.ld + c0 + tx] : (u16)0;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int c = line + 32 * i;
    if (c0 + c >= t.cols) continue;
    u16 v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = tile[part * 8 + k][c];
    *reinterpret_cast<u32x4*>(t.dst + (size_t)(c0 + c) * t.ldd + r0 + part * 8) =
        u32x4{(unsigned)v[0] | ((unsigned)v[1] << 16), (unsigned)v[2] | ((unsigned)v[3] << 16),
              (unsigned)v[4] | ((unsigned)v[5] << 16), (unsigned)v[6] | ((unsigned)v[7] << 16)};
  }
}

// *top = the largest |dloss| of the rows that count (1 if that is zero).  g is rounded to bf16 divided by it:
// with the mean's weights, all the same, a rounding of 1 / count would shift every term the same way and
// not average out in the sums over rows and classes.  One workgroup.
__device__ __forceinline__ void find_top(const float* __restrict__ dloss, const int* __restrict__ target, int M, int vocab,
                                         float* __restrict__ top, float* red) {
  float m = 0.0f;
#pragma unroll 8
  for (int i = threadIdx.x; i < M; i += 256) {
    const int t = target[i];
    const float d = fabsf(dloss[i]);
    if (t >= 0 && t < vocab && d < __builtin_inff()) m = fmaxf(m, d);
  }
  red[threadIdx.x] = m;
  __syncthreads();
  for (int off = 128; off > 0; off >>= 1) {
    if ((int)threadIdx.x < off) red[threadIdx.x] = fmaxf(red[threadIdx.x], red[threadIdx.x + off]);
    __syncthreads();
  }
  // (below the smallest normal number the quotients could overflow)
  if (threadIdx.x == 0) *top = red[0] >= 1.17549435e-38f ? red[0] : 1.0f;
}

// What the backward call needs before its products, in one launch (50021 x 2048 and 4096 x 2048 turned: 81 us, 5.5 TB/s): the first workgroup finds *top (dloss not null), the
// others transpose X and, where it is needed (w.blocks > 0), the first piece of W.
__global__ __launch_bounds__(256) void xent_prepare_kernel(Transposition x, Transposition w, const float* __restrict__ dloss,
                                                           const int* __restrict__ target, int M, int vocab, float* __restrict__ top) {
  __shared__ __attribute__((aligned(16))) u16 tile[64][72];
  const int block = (int)blockIdx.x - 1;
  if (block < 0) {
    if (dloss) find_top(dloss, target, M, vocab, top, reinterpret_cast<float*>(tile));
  } else if (block < x.blocks) {
    transpose_tile(x, block, tile);
  } else {
    transpose_tile(w, block - x.blocks, tile);
  }
}
__global__ __launch_bounds__(256) void xent_transpose_kernel(Transposition w) {
  __shared__ __attribute__((aligned(16))) u16 tile[64][72];
  transpose_tile(w, blockIdx.x, tile);
}

// C[row][col] = sum over slabs, in slab order, of part[slab][row][col], on top of what C holds where `add`; zeros in rows
// that do not count.  A wavefront takes 512 elements of a row, in 16-byte pieces (part's rows are whole ones, C's may
// start at any element).
__global__ __launch_bounds__(256) void fold_slabs_kernel(float* __restrict__ C, int ldc, const float* __restrict__ part, int ldp,
                                                         long long slab, int slabs, int rows, int cols, int add,
                                                         const int* __restrict__ target, int vocab) {
  using Piece = Anywhere<float, f32x4>;
  for (int r = blockIdx.y * 4 + (threadIdx.x >> 6); r < rows; r += gridDim.y * 4) {
    const bool counts = row_counts(target, vocab, r);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int c = blockIdx.x * 512 + 256 * k + 4 * (threadIdx.x & 63);
      if (c >= cols) break;
      const float* src = part + (size_t)r * ldp + c;
      float* dst = C + (size_t)r * ldc + c;
      const bool whole = c + 4 <= cols;
      f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
      if (add && whole) v = reinterpret_cast<const Piece*>(dst)->v;
      else if (add)
        for (int i = 0; i < 4; ++i)
          if (c + i < cols) v[i] = dst[i];
#pragma unroll 4
      for (int n = 0; n < slabs; ++n) v += *reinterpret_cast<const f32x4*>(src + (size_t)n * slab);
      if (!counts) v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if (whole) reinterpret_cast<Piece*>(dst)->v = v;
      else
        for (int i = 0; i < 4; ++i)
          if (c + i < cols) dst[i] = v[i];
    }
  }
}
// Zeros in the rows of C that do not count: where a GEMM writes dX itself.  C has whole tiles: 16-byte rows, cols a multiple of 32.
__global__ __launch_bounds__(256) void clear_rows_kernel(float* __restrict__ C, int ldc, int rows, int cols, const int* __restrict__ target,
                                                         int vocab) {
  const int r = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= rows || row_counts(target, vocab, r)) return;
  for (int c = 4 * (threadIdx.x & 63); c < cols; c += 256) *reinterpret_cast<f32x4*>(C + (size_t)r * ldc + c) = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
}
// out[c] = factor * sum over lines of part[line][c].  64 columns per workgroup, four groups of lines added up in order.
struct ColumnFold {
  float* out;
  const float* part;
  int ld, lines, cols;
  const float* factor;
  int workgroups;
};
__device__ __forceinline__ void fold_columns(const ColumnFold& f, int workgroup, float (*red)[64]) {
  const int l = threadIdx.x & 63, g = threadIdx.x >> 6, c = workgroup * 64 + l;
  const int each = (f.lines + 3) / 4, from = g * each, to = min(from + each, f.lines);
  float v = 0.0f;
  if (c < f.cols) {
#pragma unroll 8
    for (int b = from; b < to; ++b) v += f.part[(size_t)b * f.ld + c];
  }
  red[g][l] = v;
  __syncthreads();
  if (g != 0 || c >= f.cols) return;
  v = ((red[0][l] + red[1][l]) + red[2][l]) + red[3][l];
  f.out[c] = f.factor ? v * *f.factor : v;
}
__global__ __launch_bounds__(256) void fold_columns_kernel(ColumnFold f) {
  __shared__ float red[4][64];
  fold_columns(f, blockIdx.x, red);
}

// What follows g in a backward call too small to fill the device, in one launch: dX, dW and db do not depend on each
// other.  64 x 64 tiles; workgroups [0, nx) make dX, the next ones dW, the last ones db.
template <class EpiX, class EpiW>
__global__ __launch_bounds__(256) void xent_products_kernel(Tile16 px, typename EpiX::Args ex, int nx, Tile16 pw, typename EpiW::Args ew,
                                                            int nw, ColumnFold db) {
  extern __shared__ __attribute__((aligned(16))) u16 smem_t[];  // the tiles' ring
  const int id = blockIdx.x;
  if (id < nx) tile16_run<false, 64, 64, 4, 1, 4, EpiX>(px, ex, id);
  else if (id < nx + nw) tile16_run<false, 64, 64, 4, 1, 4, EpiW>(pw, ew, id - nx);
  else fold_columns(db, id - nx - nw, reinterpret_cast<float(*)[64]>(smem_t));
}

// ---- fp32 models ------------------------------------------------------------------------------------

// dst[rows_p][cols_p] = src[rows][cols], zeros around it and for rows that do not count.  Whole 16-byte pieces
// where src has them (vec); cols_p is a multiple of 32.
__global__ __launch_bounds__(256) void pad_f32_kernel(float* __restrict__ dst, const float* __restrict__ src, int rows, int cols,
                                                      int ld, int rows_p, int cols_p, const int* __restrict__ target, int vocab, int vec) {
  for (int r = blockIdx.y * 4 + (threadIdx.x >> 6); r < rows_p; r += gridDim.y * 4) {
    const bool there = r < rows && row_counts(target, vocab, r);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int c = blockIdx.x * 512 + 256 * k + 4 * (threadIdx.x & 63);
      if (c >= cols_p) break;
      const float* from = src + (size_t)r * ld + c;
      f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
      if (there && vec && c + 4 <= cols) v = *reinterpret_cast<const f32x4*>(from);
      else if (there)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (c + i < cols) v[i] = from[i];
      *reinterpret_cast<f32x4*>(dst + (size_t)r * cols_p + c) = v;
    }
  }
}

// (1024 x 32000: 24 us, 5.4 TB/s.)  Statistics of one piece of products Z [M x cols] (the bias is added here), joined to those of the pieces
// before (first = 0: none).  One workgroup per row, one pass; `last` turns them into loss and lse.
__global__ __launch_bounds__(256) void xent_rows_f32_kernel(const float* __restrict__ Z, int ldz, int cols, int first, int vocab,
                                                            int last, const float* __restrict__ bias, const int* __restrict__ target,
                                                            float2* __restrict__ part, float* __restrict__ zt,
                                                            float* __restrict__ loss, float* __restrict__ lse, int vec) {
  __shared__ float2 red[256];
  const int row = blockIdx.x, tid = threadIdx.x;
  int t = target[row];
  const bool counts = t >= 0 && t < vocab;
  t = counts ? t - first : -1;
  const float* z = Z + (size_t)row * ldz;
  float m = -__builtin_inff(), s = 0.0f;
  for (int c0 = 4 * tid; c0 < cols; c0 += 4096) {  // sixteen elements at a time, their loads in flight together
    f32x4 four[4], add[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int c = c0 + 1024 * u;
      add[u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if (c >= cols) continue;
      four[u] = *reinterpret_cast<const f32x4*>(z + c);  // rows are padded to whole quadruples
      if (bias && vec && c + 4 <= cols) add[u] = *reinterpret_cast<const f32x4*>(bias + c);
      else if (bias)
        for (int i = 0; i < 4; ++i)
          if (c + i < cols) add[u][i] = bias[c + i];
    }
    float top = -__builtin_inff(), sum = 0.0f;
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = c0 + 1024 * u + i;
        float v = -__builtin_inff();
        if (c < cols && c != t) v = four[u][i] + add[u][i];
        four[u][i] = v;
        top = fmaxf(top, v);
      }
    const float ref = finite_or_zero(top);
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) sum += __builtin_amdgcn_exp2f((four[u][i] - ref) * LOG2E);
    join(m, s, top, sum);
  }
  red[tid] = float2{m, s};
  __syncthreads();
  for (int off = 128; off > 0; off >>= 1) {
    if (tid < off) {
      float2 a = red[tid];
      const float2 b = red[tid + off];
      join(a.x, a.y, b.x, b.y);
      red[tid] = a;
    }
    __syncthreads();
  }
  if (tid != 0) return;
  float2 all = red[0];
  if (first > 0) {
    float2 before = part[row];
    join(before.x, before.y, all.x, all.y);
    all = before;
  }
  if (t >= 0 && t < cols) zt[row] = z[t] + (bias ? bias[t] : 0.0f);
  if (last) finish_row(all.x, all.y, counts, counts ? zt[row] : 0.0f, loss + row, lse + row);
  else part[row] = all;
}

// Products of one piece, class by class, Zt [rows_p x Mp] -> g^T in place, zeros around the rows x M that
// are there; db = its row sums.  One wavefront per class: no sum leaves it.  8192 x 1024: 13 us, 5.2 TB/s.
__global__ __launch_bounds__(256) void xent_grad_f32_kernel(float* __restrict__ Zt, int Mp, int M, int rows, int rows_p, int first,
                                                            int vocab, const float* __restrict__ bias,
                                                            const int* __restrict__ target, const float* __restrict__ lse,
                                                            const float* __restrict__ dloss, float* __restrict__ db, int vec) {
  const int j = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (j >= rows_p) return;
  float* z = Zt + (size_t)j * Mp;
  const float add = bias && j < rows ? bias[j] : 0.0f;
  float sum = 0.0f;
#pragma unroll 2
  for (int i = 4 * lane; i < Mp; i += 256) {
    f32x4 v = *reinterpret_cast<const f32x4*>(z + i);
    int t[4];
    float l[4], d[4];
    if (vec && i + 4 <= M) {  // target, lse and dloss in 16-byte pieces
      const u32x4 t4 = *reinterpret_cast<const u32x4*>(target + i);
      const f32x4 l4 = *reinterpret_cast<const f32x4*>(lse + i), d4 = dloss ? *reinterpret_cast<const f32x4*>(dloss + i) : f32x4{1.0f, 1.0f, 1.0f, 1.0f};
#pragma unroll
      for (int k = 0; k < 4; ++k) t[k] = (int)t4[k], l[k] = l4[k], d[k] = d4[k];
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        t[k] = i + k < M ? target[i + k] : -1;
        l[k] = i + k < M ? lse[i + k] : 0.0f;
        d[k] = i + k < M && dloss ? dloss[i + k] : 1.0f;
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float x = v[k] + add - l[k];
      float g = d[k] * __builtin_amdgcn_exp2f(x * LOG2E);
      if (t[k] == first + j) g = d[k] * expm1f(x);
      if (j >= rows || t[k] < 0 || t[k] >= vocab) g = 0.0f;
      v[k] = g;
      sum += g;
    }
    *reinterpret_cast<f32x4*>(z + i) = v;
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
  if (db && lane == 0 && j < rows) db[j] = sum;
}

// ---- sizes ------------------------------------------------------------------------------------------

inline size_t up(size_t x, size_t a) { return (x + a - 1) / a * a; }
inline bool al16(const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0; }
// Workgroups of four wavefronts, 512 columns of a row each.
inline dim3 row_grid(int rows, int cols) { return dim3((cols + 511) / 512, std::min((rows + 3) / 4, 16384)); }
hipError_t fold_slabs(float* C, int ldc, const float* part, int ldp, long long slab, int slabs, int rows, int cols, bool add,
                      const int* target, int vocab, hipStream_t s) {
  launch_kernel(fold_slabs_kernel, row_grid(rows, cols), dim3(256), 0, s, C, ldc, part, ldp, slab, slabs, rows, cols, (int)add, target,
                vocab);
  return hipGetLastError();
}

// Hands out 256-byte aligned parts of a workspace (or only adds them up, base = null).
struct Carver {
  char* base;
  size_t used = 0;
  template <class T>
  T* take(size_t n) {
    T* q = base ? reinterpret_cast<T*>(base + used) : nullptr;
    used += up(n * sizeof(T), 256);
    return q;
  }
};

// The classes of one product in up to two launches: those that make whole rounds of 256 x 256 tiles on the 256
// CUs, and what is left over on smaller tiles, where that is estimated to be faster than one launch (4096 x 50021
// x 2048: 12 rounds and 869 classes on 128 x 128 tiles instead of 13 rounds).
struct Cut {
  int main;  // classes of the first launch; 0: only the second
  Tile16Shape first, second;
};
Cut cut_classes(int M, int cols, int Kp) {
  const Cut one{0, Tile16Shape{}, tile16_shape(M, cols, Kp, false, 1, 64, 256, false)};
  const long long down = (M + 255) / 256, whole = down * (cols / 256) / 256 * 256;  // tiles of whole rounds
  const int main = (int)(whole / down) * 256;
  if (main == 0 || main == cols) return one;
  const Cut two{main, tile16_shape(M, main, Kp, false, 1, 256, 256, false), tile16_shape(M, cols - main, Kp, false, 1, 64, 128, false)};
  return two.first.us + two.second.us < one.second.us ? two : one;
}

struct ForwardPlan {
  int Kp;          // K rounded up to whole K steps
  int pack_cols;   // columns per launch where W has to be packed
  int rows;        // rows at a time: the statistics of more would not fit 256 MB
  u16 *Xp, *Wp;
  float* zt;
  float2* part;
  size_t bytes;
};
ForwardPlan plan_forward(char* base, int M, int V, int K) {
  ForwardPlan f{};
  Carver c{base};
  f.Kp = (int)up(K, 64);
  f.pack_cols = (int)std::min<size_t>(up(V, 64), std::max<size_t>(((size_t)1 << 24) / f.Kp / 256 * 256, 256));
  f.rows = (int)std::min<size_t>(M, std::max<size_t>(((size_t)1 << 25) / (up(V, 64) / 64) / 256 * 256, 256));
  f.Xp = c.take<u16>((size_t)f.rows * f.Kp);
  f.Wp = c.take<u16>((size_t)std::min(V, f.pack_cols) * f.Kp);
  f.zt = c.take<float>(f.rows);
  f.part = c.take<float2>((size_t)f.rows * (up(V, 64) / 64));
  f.bytes = c.used;
  return f;
}

struct BackwardPlan {
  int Kp, Mp, piece;
  int tile;             // of g's (first) launch; Mp and the pieces are multiples of it
  Tile16Shape x, w;     // the launches that make dX and dW
  int ldg;              // of g: a line more than the piece, so that the rows of a tile do not all start in one memory channel
  u16 *Xp, *Xt, *Wp, *Wt, *G, *GT;
  float *top, *db_part, *x_sum, *part;
  size_t bytes;
};
BackwardPlan plan_backward(char* base, int M, int V, int K) {
  BackwardPlan b{};
  Carver c{base};
  b.Kp = (int)up(K, 64);
  // g and g^T of a piece take 2 x 512 MB, the copies of W's piece 256 MB each, or what 256 classes take where that is
  // more (from 2^20 rows or K = 2^19 on: 2.4 GB of g at 2^21 rows)
  const size_t most = std::min(((size_t)1 << 28) / up(M, 256), ((size_t)1 << 27) / b.Kp) / 256 * 256;
  const size_t widest = std::max<size_t>(most, 256);
  const Cut cut = cut_classes(M, (int)std::min<size_t>(V, widest), b.Kp);
  b.tile = cut.main ? cut.first.tile : cut.second.tile;
  b.Mp = (int)up(M, b.tile);
  b.piece = (int)std::min<size_t>(up(V, b.tile), widest);
  b.ldg = b.piece + 64;
  b.x = tile16_shape(M, K, b.piece, false, 1, 64, 256, true);
  b.w = tile16_shape(b.piece, K, b.Mp, false, 1, 64, 256, true);
  b.top = c.take<float>(1);
  b.Xp = c.take<u16>((size_t)M * b.Kp);
  b.Xt = c.take<u16>((size_t)K * b.Mp);
  b.Wp = c.take<u16>((size_t)std::min(V, b.piece) * b.Kp);
  b.Wt = c.take<u16>((size_t)K * b.piece);
  b.G = c.take<u16>((size_t)b.Mp * b.ldg);
  b.GT = c.take<u16>((size_t)b.Mp * b.piece);
  b.db_part = c.take<float>((size_t)(b.Mp / 16) * b.piece);  // (64 x 64 tiles: a line for every 16 rows)
  b.x_sum = b.piece < V ? c.take<float>((size_t)M * b.Kp) : nullptr;
  b.part = c.take<float>(std::max(b.x.part_floats, b.w.part_floats));
  b.bytes = c.used;
  return b;
}

// fp32: the framework's fp32 GEMMs are fast on whole tiles of aligned operands only, so everything is padded to
// them; what already is whole is used where it stands.
// Backward, 129 to 192 and 257 to 320 rows are padded to whole tiles of 64 only: those are a fifth slower but a quarter or
// a sixth fewer (162 x 80192 x 768 890 and 733 us, 300 x 5000 x 700 126 and 111 us; 400 x 20000 x 1024 528 and 582).
struct F32Plan {
  int Mp, Kp;
  int most, piece;  // classes at a time: at most, and the largest piece in whole tiles
  bool backward;
  int splits;       // of the classes, for dX: at most
  int w_splits;     // of the rows, for dW
  float *Xp, *Wp, *Z, *zt, *x_part, *w_part;
  float2* part;
  size_t bytes;
};
int whole_tiles(int n) { return (int)(n >= 128 ? up(n, 128) : up(n, 32)); }
// K: a dimension of dX and dW too, whose tiles are 64 wide at least; the forward products only need whole K steps.
int whole_k(int K, bool backward) { return !backward ? (int)up(K, 32) : K % 64 == 0 ? K : whole_tiles(K); }
// Which fp32 forward calls take the kernel for few rows: with rows of whole 256 elements the tiles of 32 rows go through the
// LDS and are faster (32 x 50048 x 1536: 98 us, few rows 110), and so are those of few classes that need no copy (16 x 1500
// x 1536: 23 us, few rows 28).
bool few_rows_f32(int M, int V, int K) {
  return M <= FEW_ROWS<float> && (V >= 4096 ? M <= 16 || K % 256 != 0 : M <= 16 && K % 32 != 0);
}
// How many of the `left` classes the next piece takes.  Backward, the products with a row per class run on 128 x 128 tiles,
// one per CU at a time (from 128 rows on): whole rounds of the 256 CUs first, the classes left over as a piece of their own
// on smaller tiles (1024 x 10007 x 1024 in one piece 586 us, in pieces of 8192 and 1815 classes 521).  Where what
// does not make whole tiles would mean copying much, the classes that do are read in place and the others are a piece
// of their own: forward from 8 M elements on (two more passes over them take 13 us, a piece more about as long), backward
// from 32 M (four passes, 110 us; a piece more is six launches, 90 us).  Pieces are multiples of what dX's sum is dealt
// to where they can be.
int next_piece(const F32Plan& f, int left, int K) {
  const int n = std::min(left, f.most), across = f.Mp / 128, deal = 128 * f.splits;  // (f.splits: 0 forward)
  if (f.backward && f.Mp % 128 == 0) {
    const int most = across >= 256 ? 128 : 256 / across * 128, round = most >= deal ? most / deal * deal : most;
    if (n > round) return n / round * round;
  }
  const int unit = f.backward && n > 16384 ? std::min(deal, 1024) : 128;
  const bool large = (size_t)n * K >= (f.backward ? (size_t)1 << 25 : (size_t)1 << 23);
  return n % 128 != 0 && n > 128 && large && K == f.Kp ? n / unit * unit : n;
}
F32Plan plan_f32(char* base, int M, int V, int K, bool backward) {
  F32Plan f{};
  Carver c{base};
  f.Mp = whole_tiles(M);
  f.Kp = whole_k(K, backward);
  // a piece of products and a piece of W take at most 1 GB each
  f.most = (int)std::max<size_t>(((size_t)1 << 28) / std::max(f.Mp, f.Kp) / 128 * 128, 128);
  f.backward = backward;
  if (backward) {
    if (M > 128 && M <= 320) f.Mp = (int)up(M, 64);
    // as many parts of dX's sum as make a round of its 128 x 128 tiles, or four of 64 x 64
    const size_t tiles = up(f.Mp, 128) / 128 * (up(f.Kp, 128) / 128), places = f.Mp % 128 == 0 ? 256 : 512;
    f.splits = (int)std::min<size_t>(std::max<size_t>(places / tiles, 1), 32);
  }
  for (int v0 = 0, n; v0 < V; v0 += n) {
    n = next_piece(f, V - v0, K);
    f.piece = std::max(f.piece, whole_tiles(n));
  }
  f.Xp = c.take<float>((size_t)f.Mp * f.Kp);
  const bool few = !backward && few_rows_f32(M, V, K);
  if (!few) {
    f.Wp = c.take<float>((size_t)f.piece * f.Kp);
    f.Z = c.take<float>((size_t)f.Mp * f.piece);
  }
  if (backward) {
    f.x_part = c.take<float>((size_t)f.splits * f.Mp * f.Kp);
    // Classes so few that dW has not a tile of 128 x 128 for every CU: its sum over the rows is dealt out too (2864 classes x
    // 223 from 13056 rows: 305 -> 200 us).
    const size_t w_tiles = up(f.piece, 128) / 128 * (up(f.Kp, 128) / 128);
    f.w_splits = (int)std::min<size_t>(std::max<size_t>(256 / w_tiles, 1), std::max(f.Mp / 1024, 1));
    while (f.w_splits > 1 && f.Mp % (f.w_splits * 32) != 0) --f.w_splits;
    // Where dW has no whole tiles: in whole tiles here first, or, with a sum over few rows, straight on the slower ragged
    // tiles (64 x 44992 x 1944 700 and 595 us, 300 x 20000 x 1001 538 and 549).
    f.w_part = f.Mp > 128 ? c.take<float>((size_t)f.w_splits * f.piece * f.Kp) : nullptr;
  } else {
    f.zt = c.take<float>(M);
    f.part = c.take<float2>((size_t)M * (few ? up(V, 64) / 64 : 1));
  }
  f.bytes = c.used;
  return f;
}

#define TRY(call)                          \
  do {                                     \
    hipError_t e_ = (call);                \
    if (e_ != hipSuccess) return e_;       \
  } while (0)

// Whether the tiles can read an operand where it is: 16-byte rows, whole K steps, 32-bit offsets in a tile.
bool direct(const u16* q, int ld, int K) { return al16(q) && ld % 8 == 0 && ld <= TILE16_MAX_LD && K % 64 == 0; }

hipError_t pack_rows(u16* dst, const u16* src, int rows, int cols, int ld, int ldd, hipStream_t s) {
  launch_kernel(pack_rows_kernel, row_grid(rows, ldd), dim3(256), 0, s, dst, src, rows, cols, ld, ldd);
  return hipGetLastError();
}
Transposition transposition(u16* dst, const u16* src, int rows, int cols, int ld, int ldd) {
  const int across = (cols + 63) / 64;
  return Transposition{dst, src, rows, cols, ld, ldd, (int)(al16(src) && ld % 8 == 0), across, across * (ldd / 64), nullptr, 0};
}

template <class EpiW>
hipError_t launch_products(const Tile16& px, const EpiOut<true, true>::Args& ex, int nx, const Tile16& pw, const typename EpiW::Args& ew, int nw,
                           const ColumnFold& db, hipStream_t s) {
  using Ring = TileKernel<64, 64, 4, 1, 4>;
  auto kern = xent_products_kernel<EpiOut<true, true>, EpiW>;
  static LdsOptIn opt_in;
  TRY(opt_in.ensure(reinterpret_cast<const void*>(kern), Ring::LDS));
  launch_kernel(kern, dim3(nx + nw + db.workgroups), dim3(256), Ring::LDS, s, px, ex, nx, pw, ew, nw, db);
  return hipGetLastError();
}

}  // namespace

size_t xent_forward_bytes(bool bf16, int M, int V, int K) {
  return bf16 ? plan_forward(nullptr, M, V, K).bytes : plan_f32(nullptr, M, V, K, false).bytes;
}
size_t xent_backward_bytes(bool bf16, int M, int V, int K) {
  return bf16 ? plan_backward(nullptr, M, V, K).bytes : plan_f32(nullptr, M, V, K, true).bytes;
}

template <class T>
static hipError_t launch_few_rows(const FewRows<T>& p, hipStream_t s) {
  auto go = [&](auto kern, int nb) { launch_kernel(kern, dim3((p.V + 64 * nb - 1) / (64 * nb)), dim3(256), 0, s, p); };
  const bool many = p.V >= 1 << 15;
  if (p.M <= 16) go(xent_few_rows_kernel<T, 1, 1, 4>, 1);
  else if (p.M <= 32 && many) go(xent_few_rows_kernel<T, 2, 2, 2>, 2);
  else if (p.M <= 32) go(xent_few_rows_kernel<T, 2, 1, 4>, 1);
  else if constexpr (FEW_ROWS<T> > 32) {
    if (many) go(xent_few_rows_kernel<T, 4, 4, 2>, 4);
    else go(xent_few_rows_kernel<T, 4, 1, 2>, 1);
  }
  return hipGetLastError();
}
static hipError_t launch_fold(const float2* part, int blocks, int M, int V, const int* target, const float* zt, float* loss, float* lse,
                              hipStream_t s) {
  auto fold = [&](auto kern, int rows) {
    launch_kernel(kern, dim3((M + rows - 1) / rows), dim3(256), 0, s, part, blocks, M, V, target, zt, loss, lse);
    return hipGetLastError();
  };
  // whole 128-byte lines of the statistics per workgroup once there are rows for every CU
  return M <= 64 ? fold(xent_fold_kernel<1>, 1) : M <= 1024 ? fold(xent_fold_kernel<4>, 4) : fold(xent_fold_kernel<16>, 16);
}

static hipError_t forward_rows(const ForwardPlan& f, int M, int V, int K, const u16* X, int ldx, const u16* W, int ldw,
                               const float* bias, const int* target, float* loss, float* lse, hipStream_t s) {
  const bool w_direct = direct(W, ldw, K), few = !w_direct && M <= FEW_ROWS<u16> && V >= (M <= 32 ? 4096 : 8192);
  if (few || !direct(X, ldx, K)) {
    TRY(pack_rows(f.Xp, X, M, K, ldx, f.Kp, s));
    X = f.Xp;
    ldx = f.Kp;
  }
  if (few) {
    TRY(launch_few_rows<u16>(FewRows<u16>{X, W, M, V, K, f.Kp, ldw, bias, target, f.zt, f.part}, s));
  }
  const int per = w_direct ? V : f.pack_cols;
  for (int v0 = few ? V : 0; v0 < V; v0 += per) {
    const int cols = std::min(per, V - v0), ld_w = w_direct ? ldw : f.Kp;
    const u16* w = W + (size_t)v0 * ldw;
    if (!w_direct) {
      TRY(pack_rows(f.Wp, w, cols, K, ldw, f.Kp, s));
      w = f.Wp;
    }
    const Cut cut = cut_classes(M, cols, f.Kp);
    for (int c0 = 0; c0 < cols;) {
      const int n = c0 < cut.main ? cut.main : cols - c0, at = v0 + c0;
      const EpiStats::Args e{bias ? bias + at : nullptr, target, at, V, f.zt, f.part + (size_t)(at / 64) * M};
      TRY(tiles<EpiStats>(c0 < cut.main ? cut.first : cut.second, nullptr, X, ldx, w + (size_t)c0 * ld_w, ld_w, M, n, f.Kp, e, s));
      c0 += n;
    }
  }
  return launch_fold(f.part, (int)(up(V, 64) / 64), M, V, target, f.zt, loss, lse, s);
}

hipError_t xent_forward_bf16(int M, int V, int K, const u16* X, int ldx, const u16* W, int ldw, const float* bias,
                             const int* target, float* loss, float* lse, void* ws, hipStream_t s) {
  const ForwardPlan f = plan_forward(static_cast<char*>(ws), M, V, K);
  for (int r0 = 0; r0 < M; r0 += f.rows)
    TRY(forward_rows(f, std::min(f.rows, M - r0), V, K, X + (size_t)r0 * ldx, ldx, W, ldw, bias, target + r0, loss + r0, lse + r0, s));
  return hipSuccess;
}

hipError_t xent_backward_bf16(int M, int V, int K, const u16* X, int ldx, const u16* W, int ldw, const u16* Wt, int ldwt,
                              const float* bias, const int* target, const float* lse, const float* dloss, u16* dX, int lddx,
                              bool dw_bf16, void* dW, int lddw, float* db, void* ws, hipStream_t s) {
  const BackwardPlan b = plan_backward(static_cast<char*>(ws), M, V, K);
  const bool x_direct = direct(X, ldx, K), w_direct = direct(W, ldw, K);
  const float* top = dloss ? b.top : nullptr;
  // the caller's transposed copy serves a piece where whole 16-byte chunks of it can be read
  auto wt_direct = [&](int v0, int cols) { return Wt && direct(Wt + v0, ldwt, cols); };
  auto wt_copy = [&](int v0, int cols) {
    return transposition(b.Wt, W + (size_t)v0 * ldw, cols, K, ldw, (int)up(cols, b.tile));
  };
  const int first = std::min(b.piece, V);
  // One piece and few tiles of 64 x 64: dX, dW and db share a launch (256 x 1000 x 512: 176
  // workgroups in one launch instead of three, the call 24 -> 18.5 us).
  const bool together = b.piece >= V && b.x.tile == 64 && b.w.tile == 64 && b.x.splits == 1 && b.w.splits == 1 &&
                        b.x.full + b.w.full <= 512;
  Transposition xt = transposition(b.Xt, X, M, K, ldx, b.Mp);
  xt.target = target;
  xt.vocab = V;
  const Transposition wt0 = wt_direct(0, first) ? Transposition{} : wt_copy(0, first);
  launch_kernel(xent_prepare_kernel, dim3(1 + xt.blocks + wt0.blocks), dim3(256), 0, s, xt, wt0, dloss, target, M, V, b.top);
  TRY(hipGetLastError());
  if (!x_direct) {
    TRY(pack_rows(b.Xp, X, M, K, ldx, b.Kp, s));
    X = b.Xp;
    ldx = b.Kp;
  }
  for (int v0 = 0; v0 < V; v0 += b.piece) {
    const int cols = std::min(b.piece, V - v0), padded = (int)up(cols, b.tile), steps = (int)up(cols, 64) / 64;
    const u16* w = W + (size_t)v0 * ldw;
    int ld_w = ldw;
    if (!w_direct) {
      TRY(pack_rows(b.Wp, w, cols, K, ldw, b.Kp, s));
      w = b.Wp;
      ld_w = b.Kp;
    }
    // (the rows behind M up to Mp have to be written, as zeros, by either launch: dW sums over them)
    Cut cut = cut_classes(M, cols, b.Kp);
    if (cut.main == 0 || (int)up(M, cut.second.tile) != b.Mp || b.tile != 256) cut = Cut{0, {}, tile16_shape(M, cols, b.Kp, false, 1, b.tile, b.tile, false)};
    ColumnFold fold{};
    for (int c0 = 0; c0 < cols;) {
      const int n = c0 < cut.main ? cut.main : cols - c0, at = v0 + c0;
      const Tile16Shape& shape = c0 < cut.main ? cut.first : cut.second;
      const EpiGrad::Args g{bias ? bias + at : nullptr, target, lse, dloss, top, at, V, b.G + c0, b.GT + (size_t)c0 * b.Mp,
                            b.ldg, b.Mp, b.piece, db ? b.db_part + c0 : nullptr};
      TRY(tiles<EpiGrad>(shape, nullptr, X, ldx, w + (size_t)c0 * ld_w, ld_w, M, n, b.Kp, g, s));
      if (db) {
        const int lines = b.Mp / (shape.tile == 64 ? 16 : shape.tile / 2);  // a wavefront's rows each
        fold = ColumnFold{db + at, b.db_part + c0, b.piece, lines, n, top, (n + 63) / 64};
        if (!together || c0 + n < cols) {  // a part of db each; the shared launch takes the last one along
          launch_kernel(fold_columns_kernel, dim3(fold.workgroups), dim3(256), 0, s, fold);
          TRY(hipGetLastError());
        }
      }
      c0 += n;
    }
    // dX (+)= g W
    const u16* wt = Wt ? Wt + v0 : nullptr;
    int ld_t = ldwt;
    if (!wt_direct(v0, cols)) {
      if (v0 > 0) {
        const Transposition t = wt_copy(v0, cols);
        launch_kernel(xent_transpose_kernel, dim3(t.blocks), dim3(256), 0, s, t);
        TRY(hipGetLastError());
      }
      wt = b.Wt;
      ld_t = padded;
    }
    const float* before = v0 > 0 ? b.x_sum : nullptr;
    const EpiOut<true, true>::Args dx{dX, lddx, before, b.Kp, top, target, V};
    void* dw = static_cast<char*>(dW) + (size_t)v0 * lddw * (dw_bf16 ? 2 : 4);
    const EpiOut<true>::Args dw16{dw, lddw, nullptr, 0, top};
    const EpiOut<false>::Args dw32{dw, lddw, nullptr, 0, top};
    if (together) {
      Tile16 px = product(b.G, b.ldg, wt, ld_t, M, K, steps * 64), pw = product(b.GT, b.Mp, b.Xt, b.Mp, cols, K, b.Mp);
      const int nx = (int)tile16_complete(px, b.x, nullptr), nw = (int)tile16_complete(pw, b.w, nullptr);
      if (nx < 0 || nw < 0) return hipErrorInvalidValue;
      if (dw_bf16) TRY((launch_products<EpiOut<true>>(px, dx, nx, pw, dw16, nw, fold, s)));
      else TRY((launch_products<EpiOut<false>>(px, dx, nx, pw, dw32, nw, fold, s)));
      continue;
    }
    if (v0 + cols < V) {
      const EpiOut<false>::Args sum{b.x_sum, b.Kp, before, b.Kp, nullptr};
      TRY(tiles<EpiOut<false>>(b.x, b.part, b.G, b.ldg, wt, ld_t, M, K, steps * 64, sum, s));
    } else {
      TRY((tiles<EpiOut<true, true>>(b.x, b.part, b.G, b.ldg, wt, ld_t, M, K, steps * 64, dx, s)));
    }
    // dW = g^T X
    if (dw_bf16) TRY(tiles<EpiOut<true>>(b.w, b.part, b.GT, b.Mp, b.Xt, b.Mp, cols, K, b.Mp, dw16, s));
    else TRY(tiles<EpiOut<false>>(b.w, b.part, b.GT, b.Mp, b.Xt, b.Mp, cols, K, b.Mp, dw32, s));
  }
  return hipSuccess;
}

namespace {
// Whether the fp32 GEMMs can read or write a matrix as whole tiles where it is (their byte offsets in a tile have 32 bits).
bool whole(const float* q, int ld, int rows, int rows_p, int cols, int cols_p) {
  return rows == rows_p && cols == cols_p && al16(q) && ld % 4 == 0 && ld <= TILE16_MAX_LD;
}
hipError_t padded_copy(const float*& q, int& ld, float* room, int rows, int cols, int rows_p, int cols_p, const int* target, int vocab,
                       hipStream_t s) {
  launch_kernel(pad_f32_kernel, row_grid(rows_p, cols_p), dim3(256), 0, s, room, q, rows, cols, ld, rows_p, cols_p, target, vocab,
                (int)(al16(q) && ld % 4 == 0));
  q = room;
  ld = cols_p;
  return hipGetLastError();
}
// An operand in whole tiles: where it stands, or copied to `room`.
hipError_t whole_operand(const float*& q, int& ld, float* room, int rows, int cols, int rows_p, int cols_p, hipStream_t s) {
  if (whole(q, ld, rows, rows_p, cols, cols_p)) return hipSuccess;
  return padded_copy(q, ld, room, rows, cols, rows_p, cols_p, nullptr, 0, s);
}
}  // namespace

hipError_t xent_forward_f32(int M, int V, int K, const float* X, int ldx, const float* W, int ldw, const float* bias,
                            const int* target, float* loss, float* lse, void* ws, hipStream_t s) {
  const F32Plan f = plan_f32(static_cast<char*>(ws), M, V, K, false);
  if (few_rows_f32(M, V, K)) {
    if (!whole(X, ldx, M, M, K, f.Kp)) TRY(padded_copy(X, ldx, f.Xp, M, K, M, f.Kp, nullptr, 0, s));
    TRY(launch_few_rows<float>(FewRows<float>{X, W, M, V, K, ldx, ldw, bias, target, f.zt, f.part}, s));
    return launch_fold(f.part, (int)(up(V, 64) / 64), M, V, target, f.zt, loss, lse, s);
  }
  TRY(whole_operand(X, ldx, f.Xp, M, K, f.Mp, f.Kp, s));
  for (int v0 = 0, cols; v0 < V; v0 += cols) {
    cols = next_piece(f, V - v0, K);
    const int cols_p = whole_tiles(cols);
    const float* w = W + (size_t)v0 * ldw;
    int ld_w = ldw;
    TRY(whole_operand(w, ld_w, f.Wp, cols, K, cols_p, f.Kp, s));
    TRY(sgemm_nt(f.Mp, cols_p, f.Kp, X, ldx, w, ld_w, f.Z, cols_p, nullptr, 0, s, 0));
    launch_kernel(xent_rows_f32_kernel, dim3(M), dim3(256), 0, s, (const float*)f.Z, cols_p, cols, v0, V, (int)(v0 + cols == V),
                  bias ? bias + v0 : nullptr, target, f.part, f.zt, loss, lse, (int)al16(bias));
    TRY(hipGetLastError());
  }
  return hipSuccess;
}

// The products are made class by class, Z^T = W X^T, so that g^T is at hand as it is for dW = g^T X and as the
// transposed operand of dX = (g^T)^T W, whose sum over the classes is dealt to `splits` entries of one launch
// where dX has too few tiles to fill the device.
hipError_t xent_backward_f32(int M, int V, int K, const float* X, int ldx, const float* W, int ldw, const float* bias,
                             const int* target, const float* lse, const float* dloss, float* dX, int lddx, float* dW, int lddw,
                             float* db, void* ws, hipStream_t s) {
  const F32Plan f = plan_f32(static_cast<char*>(ws), M, V, K, true);
  // always copied: rows that do not count become zeros, as dW = g^T X needs them (zero times an infinity or NaN is NaN)
  TRY(padded_copy(X, ldx, f.Xp, M, K, f.Mp, f.Kp, target, V, s));
  const bool dx_direct = f.splits == 1 && next_piece(f, V, K) == V && whole(dX, lddx, M, f.Mp, K, f.Kp);
  for (int v0 = 0, cols; v0 < V; v0 += cols) {
    cols = next_piece(f, V - v0, K);
    const int cols_p = whole_tiles(cols);
    const float* w = W + (size_t)v0 * ldw;
    int ld_w = ldw;
    TRY(whole_operand(w, ld_w, f.Wp, cols, K, cols_p, f.Kp, s));
    TRY(sgemm_nt(cols_p, f.Mp, f.Kp, w, ld_w, X, ldx, f.Z, f.Mp, nullptr, 0, s, 0));
    launch_kernel(xent_grad_f32_kernel, dim3((cols_p + 3) / 4), dim3(256), 0, s, f.Z, f.Mp, M, cols, cols_p, v0, V,
                  bias ? bias + v0 : nullptr, target, lse, dloss, db ? db + v0 : nullptr,
                  (int)(al16(target) && al16(lse) && al16(dloss)));
    TRY(hipGetLastError());
    int splits = f.splits;
    while (splits > 1 && (cols_p % (splits * 32) != 0 || cols_p / splits < 256)) --splits;
    float* dx = dx_direct ? dX : f.x_part;
    TRY(sgemm_tn(splits, f.Mp, f.Kp, cols_p / splits, f.Z, f.Mp, w, ld_w, dx, dx_direct ? lddx : f.Kp, (long long)f.Mp * f.Kp,
                 nullptr, 0, s, 0));
    if (dx_direct) {
      launch_kernel(clear_rows_kernel, dim3((M + 3) / 4), dim3(256), 0, s, dX, lddx, M, K, target, V);
      TRY(hipGetLastError());
    } else {
      TRY(fold_slabs(dX, lddx, f.x_part, f.Kp, (long long)f.Mp * f.Kp, splits, M, K, v0 > 0, target, V, s));
    }
    float* dw = dW + (size_t)v0 * lddw;
    if (f.w_splits == 1 && whole(dw, lddw, cols, cols_p, K, f.Kp)) {
      TRY(sgemm_nn(cols_p, f.Kp, f.Mp, f.Z, f.Mp, X, ldx, dw, lddw, nullptr, 0, s, 0));
    } else if (f.w_part == nullptr) {
      TRY(sgemm_nn(cols, K, f.Mp, f.Z, f.Mp, X, ldx, dw, lddw, nullptr, 0, s, 0));
    } else {
      const long long slab = (long long)cols_p * f.Kp;
      TRY(sgemm_nn_parts(f.w_splits, cols_p, f.Kp, f.Mp / f.w_splits, f.Z, f.Mp, X, ldx, f.w_part, f.Kp, slab, s));
      TRY(fold_slabs(dw, lddw, f.w_part, f.Kp, slab, f.w_splits, cols, K, false, nullptr, 0, s));
    }
  }
  return hipSuccess;
}

}  // namespace mi
