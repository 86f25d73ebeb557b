// Building block of the loss and update operators: one tile of C = A[M,K] * B[N,K]^T on 16-bit
// operands (bf16 or fp16), both K-contiguous, fp32 accumulation on v_mfma_f32_16x16x32, handed to an
// epilogue that the operator supplies.  Used by xent.hip and ortho.hip.
//
// K is a multiple of 64 and rows start at multiples of 16 bytes (callers pack operands that do not);
// M and N are arbitrary: tile rows behind the last one read the last one again, and the epilogue drops
// what does not belong to the result.
//
// Orientation, as in gemm_bf16_x32.hip: the register-side index of the 16 x 16 result block is n, the
// lane-side index is m, and the rows of the B tile are dealt to the four n blocks of a wavefront's 64
// columns so that a lane holds two runs of eight consecutive columns of one row:
//   lane (q = lane / 16, l = lane % 16), block row jq, half h, element e
//     ->  row 16 jq + l,  column 32 h + 8 q + e.
#pragma once
#include "gemm_bf16_common.h"
#include "x32w4_loop.h"

namespace mi {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

constexpr int TILE16_MAX_LD = 1 << 22;  // 2 * 256 rows * this many elements: 32-bit byte offsets

struct Tile16 {
  const u16* A;
  const u16* B;
  long long batchA, batchB;  // elements between the operands of consecutive batch entries
  int lda, ldb, M, N, K;
  int batch;
  int symmetric;  // only tiles with tile_m >= tile_n are launched (square results)
  int tile;       // rows and columns of a tile: 64, 128 or 256
  // The tiles of all entries, entry by entry, are numbered through.  The first `full` are one workgroup each; the K
  // steps of each of the others are dealt to `splits` workgroups, whose sums go to `part` and through a second launch.
  int full, joined, splits;  // joined: how many are split
  float* part;
  int tiles_m, tiles_n, tiles;  // set by the launch; tiles: of one entry
};

// Two values rounded to nearest even, packed (low half first).
template <bool F16>
__device__ __forceinline__ unsigned pack16(float lo, float hi) {
  const f32x2 v = {lo, hi};
  if constexpr (F16) return __builtin_bit_cast(unsigned, __builtin_convertvector(v, f16x2));
  else return __builtin_bit_cast(unsigned, __builtin_convertvector(v, bf16x2));
}
__device__ __forceinline__ float f16_lo(unsigned v) { return (float)__builtin_bit_cast(f16x2, v)[0]; }
__device__ __forceinline__ float f16_hi(unsigned v) { return (float)__builtin_bit_cast(f16x2, v)[1]; }

// Number `item` -> batch entry and tile, in an order in which neighbours share operand panels: within an entry
// bands of eight tile rows, walked column by column (32 workgroups of an XCD in flight share eight A panels
// and four B panels), or the rows of the lower triangle one after another.
__device__ __forceinline__ void tile16_of_item(const Tile16& p, int item, int& entry, int& tm, int& tn) {
  entry = __builtin_amdgcn_readfirstlane(item / p.tiles);  // (divisions go through vector registers)
  const int id = item - entry * p.tiles;
  if (p.symmetric) {
    tm = (int)((__builtin_sqrtf(8.0f * (float)id + 1.0f) - 1.0f) * 0.5f);
    while (tm * (tm + 1) / 2 > id) --tm;  // the root is good to a unit only
    while ((tm + 1) * (tm + 2) / 2 <= id) ++tm;
    tm = __builtin_amdgcn_readfirstlane(tm);
    tn = id - tm * (tm + 1) / 2;
    return;
  }
  const int band = __builtin_amdgcn_readfirstlane(id / (8 * p.tiles_n)), within = id - band * 8 * p.tiles_n;
  const int height = p.tiles_m - band * 8 < 8 ? p.tiles_m - band * 8 : 8;
  tn = __builtin_amdgcn_readfirstlane(within / height);
  tm = band * 8 + within - tn * height;
}

// What a workgroup does: its item and the K steps of it.  split < 0: all of them.  Workgroups go to the 8 XCDs
// round-robin; each XCD gets one contiguous range of the items.
struct Tile16Job {
  int item, split, entry, tm, tn, k0, nk;
};
__device__ __forceinline__ Tile16Job tile16_job(const Tile16& p, int id) {
  Tile16Job j;
  const int steps = p.K / 64;
  if (id < p.full) {
    const int xcd = id & 7, rest = p.full & 7;
    j.item = xcd * (p.full >> 3) + (xcd < rest ? xcd : rest) + (id >> 3);
    j.split = -1;
    j.k0 = 0;
    j.nk = steps;
  } else {
    // split by split, so that the workgroups of an XCD share the operands' columns
    id -= p.full;  // (a multiple of 8: id & 7 is still the XCD)
    const int total = p.joined * p.splits, xcd = id & 7, rest = total & 7;
    id = xcd * (total >> 3) + (xcd < rest ? xcd : rest) + (id >> 3);
    j.split = __builtin_amdgcn_readfirstlane(id / p.joined);
    j.item = p.full + id - j.split * p.joined;
    j.k0 = __builtin_amdgcn_readfirstlane((int)((long long)steps * j.split / p.splits));
    j.nk = __builtin_amdgcn_readfirstlane((int)((long long)steps * (j.split + 1) / p.splits)) - j.k0;
  }
  tile16_of_item(p, j.item, j.entry, j.tm, j.tn);
  return j;
}

// Sums of a split: per block of 16 rows x 64 columns of the tile, row blocks first, the four n blocks of each lane.
__device__ __forceinline__ f32x4* tile16_part(const Tile16& p, int item, int split, int row_in_tile, int col_in_tile, int lane) {
  const int block = (row_in_tile >> 4) * (p.tile >> 6) + (col_in_tile >> 6), blocks = (p.tile >> 4) * (p.tile >> 6);
  return reinterpret_cast<f32x4*>(p.part) + (((size_t)(item - p.full) * p.splits + split) * blocks + block) * 256 + lane;
}

// Transposed store of a wavefront's WTM x 64 packed results: dst[col][row], `ld` elements per column,
// dst at the first row and column.  32 columns at a time through `stage` (32 * (2 WTM + 8) bytes of LDS
// private to the wavefront).  Neighbouring lanes hold neighbouring rows: one exchange with lane ^ 1 turns
// a register (columns 2k, 2k+1 of a row) into rows 2p, 2p+1 of one column.
template <int QB>
__device__ __forceinline__ void store_transposed(u16* __restrict__ dst, size_t ld, const u32x4 (&pk)[QB][2], int lane,
                                                 unsigned char* stage) {
  constexpr int COL = QB * 16 * 2 + 8;
  const int l16 = lane & 15, q = lane >> 4;
  const unsigned sel = (lane & 1) ? 0x07060302u : 0x01000504u;  // bytes of {own (4-7), partner (0-3)}
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int jq = 0; jq < QB; ++jq)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const unsigned own = pk[jq][h][k];
        const unsigned partner = (unsigned)__builtin_amdgcn_update_dpp(0, (int)own, 0xB1, 0xf, 0xf, false);  // lane ^ 1
        *reinterpret_cast<unsigned*>(stage + (8 * q + 2 * k + (lane & 1)) * COL + (16 * jq + (l16 & 14)) * 2) =
            __builtin_amdgcn_perm(own, partner, sel);
      }
    constexpr int CHUNKS = QB * 2;  // 16-byte chunks per column
#pragma unroll
    for (int i = lane; i < 32 * CHUNKS; i += 64) {
      const int c = i / CHUNKS, piece = i % CHUNKS;
      const u32x2 lo = *reinterpret_cast<const u32x2*>(stage + c * COL + piece * 16);
      const u32x2 up = *reinterpret_cast<const u32x2*>(stage + c * COL + piece * 16 + 8);
      *reinterpret_cast<u32x4*>(dst + (size_t)(32 * h + c) * ld + piece * 8) = u32x4{lo[0], lo[1], up[0], up[1]};
    }
  }
}

// The tile kernel.  WM x WN wavefronts of (BM / WM) x 64; a ring of STAGES LDS buffers filled by direct
// global -> LDS loads, one barrier per K step of 64.  Step t multiplies buffer t % STAGES in two K chunks;
// between them every wavefront has read what it needs of the buffer and the tile of step t + 1 has landed
// (the counter retires loads in order), then the barrier, then the tile of step t + STAGES is requested
// into the buffer just read out, and the first fragments of step t + 1 are read under the second chunk's
// MFMAs.  A step of 128 x 128 takes 0.31 us alone on a CU (MFMAs alone 0.23, fragment reads alone 0.18, tile loads
// alone 0.14 - 0.32 us), one of 64 x 64 0.17 us; many such tiles at once are bound by the fabric, 12-14 TB/s into the LDS.
template <int BM, int BN, int WM, int WN, int STAGES>
struct TileKernel {
  static constexpr int NW = WM * WN, QB = BM / WM / 16, BK = 64;
  static constexpr int A_ELEMS = BM * BK, B_ELEMS = BN * BK, BUF = A_ELEMS + B_ELEMS;
  static constexpr int NIA = BM / (8 * NW), NIB = BN / (8 * NW), INSTR = NIA + NIB;  // 8 rows of 128 bytes per load instruction
  static constexpr size_t RING = (size_t)STAGES * BUF * 2;
  static constexpr size_t STAGE_REGION = 32 * (QB * 16 * 2 + 8);
  static constexpr size_t LDS = RING > NW * STAGE_REGION ? RING : NW * STAGE_REGION;
  static_assert(BN / WN == 64 && BM % (8 * NW) == 0 && BN % (8 * NW) == 0 && LDS <= 160 * 1024, "tile shape");
};

template <bool F16, int BM, int BN, int WM, int WN, int STAGES, class Epi>
__device__ __forceinline__ void tile16_run(const Tile16& p, const typename Epi::Args& e, int workgroup) {
  using K_ = TileKernel<BM, BN, WM, WN, STAGES>;
  constexpr int NW = K_::NW, QB = K_::QB, BK = K_::BK;
  using frag = std::conditional_t<F16, f16x8, bf16x8>;
  extern __shared__ __attribute__((aligned(16))) u16 smem_t[];
  const unsigned lds_base = __builtin_amdgcn_readfirstlane((unsigned)(size_t)((__attribute__((address_space(3))) const void*)smem_t));
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int l16 = lane & 15, q = lane >> 4;
  const int wm0 = (wave / WN) * (BM / WM), wn0 = (wave % WN) * 64;

  const Tile16Job job = tile16_job(p, workgroup);
  const int m0 = job.tm * BM, n0 = job.tn * BN, nk = job.nk;

  unsigned offa[K_::NIA], offb[K_::NIB];
  const int lrow = lane >> 3, pc = lane & 7;
#pragma unroll
  for (int j = 0; j < K_::NIA; ++j) {
    const int row = (j * NW + wave) * 8 + lrow, real = m0 + row < p.M ? row : p.M - 1 - m0;
    offa[j] = 2u * ((unsigned)real * (unsigned)p.lda + (unsigned)(pc ^ x32::swz_a(row)) * 8u);
  }
#pragma unroll
  for (int j = 0; j < K_::NIB; ++j) {
    const int row = (j * NW + wave) * 8 + lrow, real = n0 + row < p.N ? row : p.N - 1 - n0;
    offb[j] = 2u * ((unsigned)real * (unsigned)p.ldb + (unsigned)(pc ^ x32::swz_b(row)) * 8u);
  }
  // the operand bases as scalar values, advanced with scalar additions
  auto uniform64 = [](const void* q) {
    const unsigned long long v = reinterpret_cast<unsigned long long>(q);
    const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)v), hi = __builtin_amdgcn_readfirstlane((unsigned)(v >> 32));
    return ((unsigned long long)hi << 32) | lo;
  };
  unsigned long long a = uniform64(p.A + (size_t)job.entry * p.batchA + (size_t)m0 * p.lda + (size_t)job.k0 * BK);
  unsigned long long b = uniform64(p.B + (size_t)job.entry * p.batchB + (size_t)n0 * p.ldb + (size_t)job.k0 * BK);
  auto to_lds = [](unsigned long long base, unsigned lane_off, unsigned lds) __attribute__((always_inline)) {
    asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(lds), "v"(lane_off), "s"(base) : "memory", "m0");
  };
  // what the epilogue reads at the result's place, requested ahead of the K loop (older than the tile loads it counts)
  typename Epi::template Pre<QB> pre;
  if (job.split < 0) pre = Epi::template before<QB>(e, p, m0 + wm0, n0 + wn0, lane, job.entry);

  // load i of the tile that goes into buffer buf: A's, then B's; behind the last one on to the next K step
  auto load = [&](auto i_c, int buf) __attribute__((always_inline)) {
    constexpr int i = decltype(i_c)::value;
    if constexpr (i < K_::NIA) to_lds(a, offa[i], lds_base + 2u * (unsigned)(buf * K_::BUF + (i * NW + wave) * 8 * BK));
    else to_lds(b, offb[i - K_::NIA], lds_base + 2u * (unsigned)(buf * K_::BUF + K_::A_ELEMS + ((i - K_::NIA) * NW + wave) * 8 * BK));
    if constexpr (i == K_::INSTR - 1) {
      a += 2 * BK;
      b += 2 * BK;
    }
  };

  unsigned qa[2], pa[2];
#pragma unroll
  for (int kc = 0; kc < 2; ++kc) {
    const int ra = wm0 + l16, rb = wn0 + 8 * (l16 >> 2) + (l16 & 3);
    qa[kc] = lds_base + 2u * (unsigned)(ra * BK + ((kc * 4 + q) ^ x32::swz_a(ra)) * 8);
    pa[kc] = lds_base + 2u * (unsigned)(K_::A_ELEMS + rb * BK + ((kc * 4 + q) ^ x32::swz_b(rb)) * 8);
  }
  f32x4 acc[QB][4];
#pragma unroll
  for (int jq = 0; jq < QB; ++jq)
#pragma unroll
    for (int ip = 0; ip < 4; ++ip) acc[jq][ip] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  // Fragments of one K chunk of 32, two sets: one multiplied while the other is read.  A chunk is written out as
  // volatile asm, which keeps its order: MFMAs that accumulate in place (left to itself the compiler rotates the
  // accumulators through a spare quadruple, four moves and a wait around every MFMA), a fragment read behind each of
  // the first ones, the tile loads behind the later ones.
  frag fq[2][QB], fp[2][4];
  auto read = [&](auto r_c, auto kc_c, unsigned off) __attribute__((always_inline)) {
    constexpr int r = decltype(r_c)::value, kc = decltype(kc_c)::value;
    auto& fq_ = fq; auto& fp_ = fp; auto& qa_ = qa; auto& pa_ = pa;  // (named so that the lambda captures them: operands of asm statements alone do not)
    if constexpr (r < 4)
      asm volatile("ds_read_b128 %0, %1 offset:%2" : "=&v"(fp_[kc][r]) : "v"(pa_[kc] + off), "i"(2 * (32 * (r >> 1) + 4 * (r & 1)) * BK));
    else
      asm volatile("ds_read_b128 %0, %1 offset:%2" : "=&v"(fq_[kc][r - 4]) : "v"(qa_[kc] + off), "i"(2 * (r - 4) * 16 * BK));
  };
  constexpr int READS = QB + 4, MFMAS = QB * 4;
  // multiplies set kc, reads the other set from byte offset `off` and, where asked, requests a tile into buffer `buf`
  auto chunk = [&](auto kc_c, unsigned off, auto fill_c, int buf) __attribute__((always_inline)) {
    constexpr int kc = decltype(kc_c)::value;
    constexpr bool fill = decltype(fill_c)::value;
    auto& fq_ = fq; auto& fp_ = fp; auto& acc_ = acc;
    static_for_h<MFMAS>([&](auto i_c) {
      constexpr int i = decltype(i_c)::value, jq = i / 4, ip = i % 4;
      if constexpr (F16) asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+v"(acc_[jq][ip]) : "v"(fp_[kc][ip]), "v"(fq_[kc][jq]));
      else asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+v"(acc_[jq][ip]) : "v"(fp_[kc][ip]), "v"(fq_[kc][jq]));
      static_for_h<(READS + MFMAS - 1) / MFMAS>([&](auto j_c) {
        constexpr int r = decltype(j_c)::value * MFMAS + i;
        if constexpr (r < READS) read(std::integral_constant<int, r>{}, std::integral_constant<int, kc ^ 1>{}, off);
      });
      if constexpr (fill)
          static_for_h<K_::INSTR>([&](auto l_c) {
            constexpr int l = decltype(l_c)::value;
            if constexpr (l * MFMAS / K_::INSTR == i) load(l_c, buf);
          });
    });
  };
  using C0 = std::integral_constant<int, 0>;
  using C1 = std::integral_constant<int, 1>;
#pragma unroll
  for (int s = 0; s < STAGES; ++s)
    if (s < nk) static_for_h<K_::INSTR>([&](auto l_c) { load(l_c, s); });
  if (nk >= STAGES) __builtin_amdgcn_s_waitcnt(vmcnt_imm((STAGES - 1) * K_::INSTR));
  else __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
  ring_barrier();
  static_for_h<READS>([&](auto r_c) { read(r_c, C0{}, 0u); });
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  int cur = 0;
  auto step = [&](auto fill_c) __attribute__((always_inline)) {
    constexpr bool fill = decltype(fill_c)::value;  // the tile STAGES steps ahead exists
    const int next = cur + 1 == STAGES ? 0 : cur + 1;
    chunk(C0{}, 2u * (unsigned)(cur * K_::BUF), std::false_type{}, 0);
    // the second set is in registers, so this wavefront is done with the buffer, and the next tile has landed
    if constexpr (fill) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "i"((STAGES - 2) * K_::INSTR) : "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    ring_barrier();
    // after the last tile: a harmless read of ring memory
    chunk(C1{}, 2u * (unsigned)(next * K_::BUF), fill_c, cur);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    cur = next;
  };
  int t = 0;
  for (; t + STAGES < nk; ++t) step(std::true_type{});
  for (; t < nk; ++t) step(std::false_type{});
  // what the last step read is used by nothing: kept until it has arrived, lest its registers are given away before
#pragma unroll
  for (int ip = 0; ip < 4; ++ip) asm volatile("" : : "v"(fp[0][ip]));
#pragma unroll
  for (int jq = 0; jq < QB; ++jq) asm volatile("" : : "v"(fq[0][jq]));
  // the compiler does not know that MFMAs have just written the accumulators: wait, then hand them over
  asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
  for (int jq = 0; jq < QB; ++jq)
#pragma unroll
    for (int ip = 0; ip < 4; ++ip) asm volatile("" : "+v"(acc[jq][ip]));
  if constexpr (Epi::MAY_SPLIT)
    if (job.split >= 0) {
#pragma unroll
      for (int jq = 0; jq < QB; ++jq)
#pragma unroll
        for (int ip = 0; ip < 4; ++ip) tile16_part(p, job.item, job.split, wm0 + 16 * jq, wn0, lane)[64 * ip] = acc[jq][ip];
      return;
    }
  __syncthreads();  // every wavefront is done with the operand tiles: the epilogue may use the LDS
  unsigned char* stage = reinterpret_cast<unsigned char*>(smem_t) + (size_t)wave * K_::STAGE_REGION;
  auto get = [&](int jq, int h, int i) __attribute__((always_inline)) { return acc[jq][2 * h + (i >> 2)][i & 3]; };
  Epi::template run<QB>(e, p, pre, get, m0 + wm0, n0 + wn0, lane, stage, job.entry);
}

template <bool F16, int BM, int BN, int WM, int WN, int STAGES, class Epi>
__global__ __launch_bounds__(WM* WN * 64) void tile16_kernel(Tile16 p, typename Epi::Args e) {
  tile16_run<F16, BM, BN, WM, WN, STAGES, Epi>(p, e, blockIdx.x);
}

// The same on tiles of 256 x 256 with four wavefronts of 128 x 128 and the hand-ordered K loop.
template <bool F16, class Epi>
__global__ __launch_bounds__(x32::W4_NW * 64) void tile256_kernel(Tile16 p, typename Epi::Args e) {
  extern __shared__ __attribute__((aligned(16))) u16 smem_t[];
  const unsigned lds_base = __builtin_amdgcn_readfirstlane((unsigned)(size_t)((__attribute__((address_space(3))) const void*)smem_t));
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const Tile16Job job = tile16_job(p, blockIdx.x);
  const int m0 = job.tm * x32::BM, n0 = job.tn * x32::BN;
  f32x4 acc[2][x32::QB][4];
  const x32::W4Operands op{p.A + (size_t)job.entry * p.batchA + (size_t)m0 * p.lda + (size_t)job.k0 * x32::BK,
                           p.B + (size_t)job.entry * p.batchB + (size_t)n0 * p.ldb + (size_t)job.k0 * x32::BK,
                           p.lda, p.ldb, p.M - m0, p.N - n0};
  x32::w4_loop<false, F16, true>(op, job.nk, lds_base, wave, lane, acc);
  // made opaque, so that none of the epilogue's addresses is computed ahead of the K loop and kept through it
  int lane_e = lane, row_e = wave / x32::W4_WN * x32::WTM, col_e = wave % x32::W4_WN * x32::W4_WTN;
  asm volatile("" : "+v"(lane_e), "+s"(row_e), "+s"(col_e));
  // the accumulators are read out of the AGPRs where they are used (one register each, not 256 at once)
  auto value = [&](auto h_c, int jq, int ip, int i) __attribute__((always_inline)) {
    float v;
    asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(v) : "a"(acc[decltype(h_c)::value][jq][ip][i]));
    return v;
  };
  using H0 = std::integral_constant<int, 0>;
  using H1 = std::integral_constant<int, 1>;
  if constexpr (Epi::MAY_SPLIT)
    if (job.split >= 0) {
      auto half = [&](auto h_c) __attribute__((always_inline)) {
#pragma unroll
        for (int jq = 0; jq < x32::QB; ++jq)
#pragma unroll
          for (int ip = 0; ip < 4; ++ip)
            tile16_part(p, job.item, job.split, row_e + 16 * jq, col_e + 64 * decltype(h_c)::value, lane_e)[64 * ip] =
                f32x4{value(h_c, jq, ip, 0), value(h_c, jq, ip, 1), value(h_c, jq, ip, 2), value(h_c, jq, ip, 3)};
      };
      half(H0{});
      half(H1{});
      return;
    }
  __syncthreads();  // every wavefront is done with the operand tiles: the epilogue may use the LDS
  unsigned char* stage = reinterpret_cast<unsigned char*>(smem_t) + (size_t)wave * x32::STAGE_REGION;
  auto half = [&](auto h_c) __attribute__((always_inline)) {
    auto get = [&](int jq, int h, int i) __attribute__((always_inline)) { return value(h_c, jq, 2 * h + (i >> 2), i & 3); };
    const int row = m0 + row_e, col = n0 + col_e + 64 * decltype(h_c)::value;
    const auto pre = Epi::template before<x32::QB>(e, p, row, col, lane_e, job.entry);
    Epi::template run<x32::QB>(e, p, pre, get, row, col, lane_e, stage, job.entry);
  };
  half(H0{});
  half(H1{});
}

// Second launch: the sums of the split tiles, in split order, and their epilogue, a block of 16 x 64 per wavefront.
template <class Epi>
__global__ __launch_bounds__(256) void tile16_join_kernel(Tile16 p, typename Epi::Args e) {
  __shared__ __attribute__((aligned(16))) unsigned char stage[4][32 * (16 * 2 + 8)];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int blocks = (p.tile >> 4) * (p.tile >> 6), groups = blocks / 4;
  const int n = __builtin_amdgcn_readfirstlane((int)blockIdx.x / groups), block = ((int)blockIdx.x - n * groups) * 4 + wave;
  const int row = block / (p.tile >> 6) * 16, col = block % (p.tile >> 6) * 64;
  int entry, tm, tn;
  tile16_of_item(p, p.full + n, entry, tm, tn);
  const f32x4* src = tile16_part(p, p.full + n, 0, row, col, lane);
  f32x4 acc[4];
#pragma unroll
  for (int ip = 0; ip < 4; ++ip) acc[ip] = src[64 * ip];
#pragma unroll 4
  for (int k = 1; k < p.splits; ++k) {
    src += (size_t)blocks * 256;
#pragma unroll
    for (int ip = 0; ip < 4; ++ip) acc[ip] += src[64 * ip];
  }
  auto get = [&](int, int h, int i) __attribute__((always_inline)) { return acc[2 * h + (i >> 2)][i & 3]; };
  const auto pre = Epi::template before<1>(e, p, tm * p.tile + row, tn * p.tile + col, lane, entry);
  Epi::template run<1>(e, p, pre, get, tm * p.tile + row, tn * p.tile + col, lane, stage[wave], entry);
}

// For epilogues that read nothing at the result's place.
struct NoPre {
  template <int QB>
  struct Pre {};
  template <int QB, class Args>
  static __device__ __forceinline__ Pre<QB> before(const Args&, const Tile16&, int, int, int, int) {
    return {};
  }
};

// ---- host side --------------------------------------------------------------------------------------

struct Tile16Shape {
  int tile = 128, full = 0, splits = 1;
  size_t part_floats = 0;
  double us = 0.0;  // the estimate
};
inline long long tile16_count(long long rows, long long cols, int tile, bool symmetric, int batch) {
  const long long m = (rows + tile - 1) / tile, n = (cols + tile - 1) / tile;
  return batch * (symmetric ? m * (m + 1) / 2 : m * n);
}

// Tile and split of a product, from an estimate in microseconds.  largest / smallest: the tiles allowed; may_split: the
// epilogue can run on 16-row blocks in a second launch.  The estimate's constants are measured, on random data: a
// K step of a 256 x 256 tile takes 1.5 us (one workgroup per CU), one of 128 x 128 0.32 us alone on a CU and
// 0.96 us with a second workgroup beside it, one of 64 x 64 0.17 us alone, four together 0.8 us; a launch
// starts and ends in 3-8 us; a join costs 4 us and the sums' way to memory and back at 4 TB/s.
inline Tile16Shape tile16_shape(long long rows, long long cols, int K, bool symmetric, int batch, int smallest, int largest,
                                bool may_split) {
  const int steps = K / 64;
  Tile16Shape best;
  double best_us = 1e30;
  for (int tile = smallest; tile <= largest; tile *= 2) {
    const long long items = tile16_count(rows, cols, tile, symmetric, batch);
    const double step = tile == 256 ? 1.5 : tile == 128 ? 0.32 : 0.17;
    const int at_once = tile == 256 ? 1 : tile == 128 ? 2 : 4;  // workgroups of a CU
    const double crowded = tile == 256 ? 1.5 : tile == 128 ? 0.48 : 0.20;  // a step's share of the CU when it is full
    const double ends = tile == 256 ? 8.0 : tile == 128 ? 5.0 : 3.5;
    auto rounds = [&](long long n, double k) {  // n workgroups of k steps
      if (n <= 0) return 0.0;
      if (n <= 256) return k * step + ends;
      const long long whole = n / (256 * at_once), rest = n - whole * 256 * at_once;
      const double last = rest == 0 ? 0.0 : rest <= 256 ? k * step + ends : k * crowded * (double)((rest + 255) / 256) + ends;
      return (double)whole * (k * crowded * at_once + ends) + last;
    };
    const double plain = rounds(items, steps);
    if (plain < best_us) {
      best_us = plain;
      best = Tile16Shape{tile, (int)items, 1, 0, plain};
    }
    if (!may_split) continue;
    for (const int round : {256, 512}) {  // whole rounds first, split what is left over
      if (round == 512 && at_once == 1) continue;
      const long long full = items / round * round, rest = items - full;
      if (rest == 0) continue;
      for (int splits = 2; splits <= 64; splits += splits < 8 ? 1 : splits < 16 ? 2 : 8) {
        if (steps / splits < 2) break;
        const double few = (double)((steps + splits - 1) / splits), bytes = 8.0 * (double)rest * splits * tile * tile;
        const double us = rounds(full, steps) + rounds(rest * splits, few) + 4.0 + bytes / 4e6;
        if (us < best_us) {
          best_us = us;
          best = Tile16Shape{tile, (int)full, splits, (size_t)rest * splits * tile * tile, us};
        }
      }
    }
  }
  return best;
}

template <bool F16, int BM, int WM, int WN, int STAGES, class Epi>
hipError_t launch_ring(const Tile16& p, const typename Epi::Args& e, unsigned grid, hipStream_t s) {
  using K_ = TileKernel<BM, BM, WM, WN, STAGES>;
  auto kern = tile16_kernel<F16, BM, BM, WM, WN, STAGES, Epi>;
  static LdsOptIn opt_in;
  if (hipError_t err = opt_in.ensure(reinterpret_cast<const void*>(kern), K_::LDS); err != hipSuccess) return err;
  launch_kernel(kern, dim3(grid), dim3(WM * WN * 64), K_::LDS, s, p, e);
  return hipGetLastError();
}

// p.M, N, K, operands, batch and symmetric set; `shape` from tile16_shape for the same sizes, `part` with room for
// its part_floats.  Completes p; the number of workgroups, or -1 where they are too many.
inline long long tile16_complete(Tile16& p, const Tile16Shape& shape, float* part) {
  p.tile = shape.tile;
  p.splits = shape.splits < p.K / 64 ? shape.splits : p.K / 64;  // a K step at least for each (a shorter last piece)
  p.part = part;
  p.tiles_m = (p.M + p.tile - 1) / p.tile;
  p.tiles_n = (p.N + p.tile - 1) / p.tile;
  const long long items = tile16_count(p.M, p.N, p.tile, p.symmetric, p.batch);
  if (items <= 0) return 0;
  p.tiles = (int)(items / p.batch);
  // a smaller product than the one the shape was made for (the last piece of a vocabulary): no more split tiles than it has
  p.full = p.splits <= 1 ? (int)items : (int)(items < shape.full ? items : shape.full);
  const long long joined = items - p.full, total = p.full + joined * p.splits;
  p.joined = (int)joined;
  if (items > (1 << 23) || total > (1 << 23)) return -1;  // (a launch holds less than 2^32 threads)
  if ((size_t)joined * p.splits * p.tile * p.tile > shape.part_floats) return -1;
  return total;
}

// Epi::MAY_SPLIT: the epilogue can run on blocks of 16 rows in a second launch; shapes for others come from tile16_shape
// without splits.
template <bool F16, class Epi>
hipError_t launch_tile16(Tile16 p, const Tile16Shape& shape, float* part, const typename Epi::Args& e, hipStream_t s) {
  const long long total = tile16_complete(p, shape, part);
  if (total <= 0) return total == 0 ? hipSuccess : hipErrorInvalidValue;
  const int joined = p.joined;
  const unsigned grid = (unsigned)total;
  hipError_t err = hipSuccess;
  if (p.tile == 256) {
    auto kern = tile256_kernel<F16, Epi>;
    static LdsOptIn opt_in;
    err = opt_in.ensure(reinterpret_cast<const void*>(kern), x32::LDS_BYTES);
    if (err != hipSuccess) return err;
    launch_kernel(kern, dim3(grid), dim3(x32::W4_NW * 64), x32::LDS_BYTES, s, p, e);
    err = hipGetLastError();
  } else if (p.tile == 128) {
    // more than one workgroup per CU: two buffers (64 KB) let two share it; else four, requested three steps ahead
    // (1000 x 4100, a triangle of 72 workgroups, 66 steps: 24 us instead of 37)
    err = grid > 256 ? launch_ring<F16, 128, 2, 2, 2, Epi>(p, e, grid, s) : launch_ring<F16, 128, 2, 2, 4, Epi>(p, e, grid, s);
  } else {
    err = launch_ring<F16, 64, 4, 1, 4, Epi>(p, e, grid, s);
  }
  if (err != hipSuccess || joined == 0) return err;
  if constexpr (Epi::MAY_SPLIT)
    launch_kernel(tile16_join_kernel<Epi>, dim3((unsigned)(joined * (p.tile / 16) * (p.tile / 64) / 4)), dim3(256), 0, s, p, e);
  return hipGetLastError();
}

}  // namespace mi
