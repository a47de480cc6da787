// Matrix product in 8-bit integers with a scale for every row of either operand, and what makes its operands.
//
//   out[m, n] = (sum over k of a[m, k] * b[n, k]) * (sa[m] * sb[n])
//
// a: states, quantised on the way; b: weights, a row for every output channel.  Sums are exact: v_mfma_i32_16x16x64_i8 adds 64 products at a
// time in 32-bit integers, and K_MOST of the largest stay below 2^31.  The operands are passed with b first: a lane then holds four
// neighbouring columns n of one row m, and the result is stored in pieces of four.
#include "distill_common.hpp"
#include "distill_hip.h"
#include "tiles8.hpp"

#include <algorithm>

namespace dl {

typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int KB = 128;                                        // columns are stored in whole blocks of these
constexpr int64_t K_MOST = 130944;                             // 1023 blocks: 128 * 128 as often stays below 2^31
constexpr float ISCALE = 1.f / 127.f, ISCALE_MIN = 0x1p-100f;

// ---- quantise ---------------------------------------------------------------------------------------
// A workgroup a row, which it holds in registers between the maximum and the codes (up to 16384 columns; wider rows are read twice).
// x / scale, rounded once, is a product with the rounded reciprocal and what that is off by taken off: the remainder is exact but where the code is 0
// whatever it is (scales are 2^-100 or more).
struct RowsQuant {
  const char* x; int64_t row_stride, rows, cols, width;        // width: whole blocks
  signed char* codes; int64_t code_stride;
  float* scales;
};
__device__ __forceinline__ bool not_finite(float f) { return (__float_as_uint(f) & 0x7f800000u) == 0x7f800000u; }
__device__ __forceinline__ u32x2 codes_of_eight(const float* f, float scale, float inverse) {
  u32x2 c = {0u, 0u};
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float q = f[e] * inverse, quotient = fmaf(fmaf(-q, scale, f[e]), inverse, q);
    c[e / 4] |= (unsigned)((int)fminf(fmaxf(rintf(quotient), -127.f), 127.f) & 255) << (e % 4 * 8);
  }
  return c;
}
__device__ __forceinline__ float largest_finite_of_eight(const float* f, float m) {      // infinite where one is not finite
#pragma unroll
  for (int e = 0; e < 8; ++e) m = not_finite(f[e]) ? __builtin_inff() : fmaxf(m, fabsf(f[e]));
  return m;
}
template <class Tag, int NT, int NCH>
__global__ __launch_bounds__(NT) void quantize_whole_rows_kernel(const RowsQuant p) {
  __shared__ float red[NT / WAVE];
  const int64_t row = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
  if (row >= p.rows) return;
  const char* x = p.x + row * p.row_stride * Tag::bytes;
  signed char* to = p.codes + row * p.code_stride;
  const int col = (int)threadIdx.x * 8;
  float f[NCH > 0 ? NCH : 1][8], m = 0.f;
  if constexpr (NCH > 0) {
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[i][e] = 0.f;
      if (col + i * NT * 8 < p.cols) load_eight<Tag>(x, col + i * NT * 8, p.cols, f[i]);
    }
#pragma unroll
    for (int i = 0; i < NCH; ++i) m = largest_finite_of_eight(f[i], m);
  } else {
    for (int64_t c = col; c < p.cols; c += NT * 8) {
      load_eight<Tag>(x, c, p.cols, f[0]);
      m = largest_finite_of_eight(f[0], m);
    }
  }
  m = block_max<NT>(m, red);
  const bool odd = not_finite(m);
  const float scale = odd ? 1.f : fmaxf(m * ISCALE, ISCALE_MIN), inverse = 1.f / scale;
  if (threadIdx.x == 0) p.scales[row] = odd ? __builtin_nanf("") : scale;
  if constexpr (NCH > 0) {
#pragma unroll
    for (int i = 0; i < NCH; ++i)
      if (col + i * NT * 8 < p.width) *reinterpret_cast<u32x2*>(to + col + i * NT * 8) = odd ? u32x2{0u, 0u} : codes_of_eight(f[i], scale, inverse);
  } else {
    for (int64_t c = col; c < p.width; c += NT * 8) {
      load_eight<Tag>(x, c, p.cols, f[0]);
      *reinterpret_cast<u32x2*>(to + c) = odd ? u32x2{0u, 0u} : codes_of_eight(f[0], scale, inverse);
    }
  }
}

// ---- product ----------------------------------------------------------------------------------------
struct RowsParams {
  const unsigned char* a; int64_t a_stride; const float* sa; int64_t M;
  const unsigned char* b; int64_t b_stride; const float* sb; int64_t N;
  int blocks;
  char* out; int64_t out_stride;
  int wide;                                                    // columns of the result that a small tile has, at most its BN
};

// 16 bytes a lane from `base` + `offset` into LDS, from `to` on in lane order (base and to: the wave's).  Said to the compiler as something that touches
// memory and no more: for a load into LDS that it knows it waits before the next access to LDS, and for all that are under way.  (Small tiles then
// drained their own fetches at every step, 128 x 8000 x 4096 17.8 us and with the ring below 23.6, now 12.9; a tile's values waited for the next
// tile's operands and for each other's stores, 8192 x 32000 x 1024 297 us, now 283.)  The waits are the kernels' own, by the count of fetches; those of
// the compiler, which does not count them, can only ask for more.  (m0 holds the place in LDS: it is the operand's register, which the compiler writes ahead of each.)
__device__ __forceinline__ void fetch_to_lds(const unsigned char* base, unsigned offset, unsigned to) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"{m0}"(to), "v"(offset), "s"(base) : "memory");
}

__device__ __forceinline__ void fetch_word_to_lds(const float* base, unsigned offset, unsigned to) {      // 4 bytes a lane
  asm volatile("s_nop 0\n\tglobal_load_lds_dword %1, %2" ::"{m0}"(to), "v"(offset), "s"(base) : "memory");
}

// Tiles of BM x BN, a wave WM x WN of it, a block of 128 columns (two matrix instructions deep) per step.  A step's operands are fetched into LDS by
// loads that bypass the registers, a step ahead of their use; a row of a tile is 128 bytes of LDS, its eight 16-byte pieces permuted
// by piece ^ (row / 2 % 8): the 16 rows x 16 bytes that a quarter of a wave reads then lie on all banks once.  (The loads write LDS in lane
// order, so it is their source addresses that are permuted.)
// Within a step a wave goes through its WM / 16 rows of tiles: the operand of the next row is read while the matrix unit works on this one.  The step's
// barrier sits ahead of the last row, whose operands are in registers by then: what follows it -- the last row's products, the next step's first
// operands, the fetches into what has just become free -- keeps the matrix unit busy.  Workgroups stay: each walks its tiles as one sequence of
// steps, so that the next tile's operands arrive while the last one is stored.
// Measured: 8192 x 128256 x 4096 (bf16 out) 3.42-3.55 ms, 2430-2520 Top/s (a library product with 32-bit results: 4.0-4.3 ms); without its fetches the
// same kernel takes 2.80, without reads of LDS as well 2.47: what is left are the matrix units (2.08 at the 1.98 GHz that the card holds under them) and
// the stores (0.39).  Fetches and reads share LDS with each other.  Tried: 32 x 32 x 32 instructions (3.97 ms), lines asked for ahead into the L2
// (3.88), four waves of 128 x 128 with the next step's b in registers (3.90), a second barrier for earlier fetches (level).
struct Piece { i32x4 lo, hi; };                                // a lane's 32 bytes of a row: 16 columns of either half of the block
__device__ __forceinline__ Piece row_piece(const unsigned char* lds, unsigned lo, unsigned hi, int rows) {
  return Piece{*reinterpret_cast<const i32x4*>(lds + lo + rows * KB), *reinterpret_cast<const i32x4*>(lds + hi + rows * KB)};
}

// The block of columns that a tile begins with (sums are exact: any order gives the same bits).  Tiles that share no operand begin at different ones: in
// step, their rows' places, a row's stride apart, would all lie in the same few channels of memory (1 x 128256 x 4096: 107 us, so 92).  Tiles that
// share operands stay in step, and find them in the L2.
__device__ __forceinline__ int first_block(unsigned tile, unsigned tiles_m, int blocks) { return tiles_m == 1 ? (int)(tile % (unsigned)blocks) : 0; }

// A wave's values, from row m0 and column n0 of the result on, as far as column N.  Two-byte results go through 2 KiB of LDS of the wave's own, `stage`, 16 rows at a
// time, so that a store writes whole 128-byte stretches of 8 rows instead of 32 bytes of 16; a row's 16-byte units are permuted by
// unit ^ (row % 8).
template <class Tag, int TM, int TN>
__device__ __forceinline__ void store_tile(const RowsParams& p, const i32x4 (&acc)[TM][TN], int64_t m0, int64_t n0, int64_t N, int lane, unsigned char* stage,
                                           const float* sa_here = nullptr, const float* sb_here = nullptr) {
  asm volatile("" : "+v"(lane));                               // (keeps the stores' addresses out of the steps' registers)
  const int row = lane % 16, quad = lane / 16;
  f32x4 sb[TN];
#pragma unroll
  for (int j = 0; j < TN; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) sb[j][e] = sb_here ? sb_here[j * 16 + quad * 4 + e] : p.sb[min(n0 + j * 16 + quad * 4 + e, p.N - 1)];
  float sas[TM];                                               // (all ahead of the first store, which a load behind it would wait for)
#pragma unroll
  for (int i = 0; i < TM; ++i) sas[i] = sa_here ? sa_here[i * 16 + row] : p.sa[min(m0 + i * 16 + row, p.M - 1)];
  // (Waited for here, and in all lanes: loads that one without anything to store left unused would be waited for in the next tile's steps, as soon as their
  // registers are written again, and with them the steps' fetches: 64 x 8000 x 4096 11.6 us, so 24.)
#pragma unroll
  for (int i = 0; i < TM; ++i) asm volatile("" : "+v"(sas[i]));
#pragma unroll
  for (int j = 0; j < TN; ++j) asm volatile("" : "+v"(sb[j]));
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const float sa = sas[i];
    f32x4 v[TN];
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[j][e] = (float)acc[i][j][e] * (sa * sb[j][e]);
    if constexpr (Tag::bytes == 2 && TN == 4) {
      const int r8 = lane / 8, unit = lane % 8;
      const int64_t n = n0 + unit * 8;
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const float f[8] = {v[j][0], v[j][1], v[j][2], v[j][3], 0.f, 0.f, 0.f, 0.f};
        const u32x4 c = Chunk<Tag>::pack(f);
        *reinterpret_cast<u32x2*>(stage + row * 128 + ((j * 2 + quad / 2) ^ (row & 7)) * 16 + (quad & 1) * 8) = u32x2{c[0], c[1]};
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int64_t m = m0 + i * 16 + k * 8 + r8;
        const u32x4 c = *reinterpret_cast<const u32x4*>(stage + (k * 8 + r8) * 128 + (unit ^ r8) * 16);
        char* to = p.out + (m * p.out_stride + n) * 2;
        if (m < p.M && n + 8 <= N) store16_stream_any(to, c);
        else if (m < p.M && n < N) store_chunk_elementwise<Tag>(to, 0, (int)(N - n), c);
      }
    } else {
      const int64_t m = m0 + i * 16 + row;
      char* to = p.out + m * p.out_stride * Tag::bytes;
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int64_t n = n0 + j * 16 + quad * 4;
        if (m < p.M && n < N) store_four<Tag>(to, n, N, v[j]);
      }
    }
  }
}

template <class Tag, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__((BM / WM) * (BN / WN) * WAVE, 2) void rows_kernel(const RowsParams p, unsigned tiles_m, unsigned tiles_n) {
  constexpr int WAVES = (BM / WM) * (BN / WN), TM = WM / 16, TN = WN / 16, NA = BM / 8 / WAVES, NB = BN / 8 / WAVES;
  static_assert(TM >= 2 && BM % (8 * WAVES) == 0 && BN % (8 * WAVES) == 0, "whole fetches");
  extern __shared__ __align__(1024) unsigned char lds[];      // two of (a: BM rows, b: BN rows of 128 bytes); two tiles' scales; 2 KiB of each wave's own
  constexpr int STEP = (BM + BN) * KB, SCALES = 2 * STEP, STAGE = SCALES + 2 * (BM + BN) * 4;
  const int lane = threadIdx.x & (WAVE - 1), w = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), i16 = lane % 16;      // (w: known to be the wave's)
  const int wm = (w / (BN / WN)) * WM, wn = (w % (BN / WN)) * WN;
  const TileWalk walk(tiles_m, tiles_n);
  if (walk.first >= walk.end) return;
  const unsigned steps = ((walk.end - walk.first + walk.step - 1) / walk.step) * (unsigned)p.blocks;

  // the fetching side: its tile, its block, this thread's places in them
  unsigned f_tile = walk.first;
  int f_kb, f_left;                                            // the block to fetch, and how many are
  const unsigned char *f_a, *f_b;
  unsigned f_ao[NA], f_bo[NB];
  const auto f_begin = [&]() {
    int64_t m, n;
    walk.origin(f_tile, m, n);
    m *= BM;
    n *= BN;
    f_left = p.blocks;
    f_kb = first_block(f_tile, tiles_m, p.blocks);
    f_a = p.a + m * p.a_stride + (int64_t)f_kb * KB;
    f_b = p.b + n * p.b_stride + (int64_t)f_kb * KB;
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      const int row = (i * WAVES + w) * 8 + lane / 8, piece = (lane & 7) ^ ((row >> 1) & 7);
      f_ao[i] = (unsigned)(min((int64_t)row, p.M - 1 - m) * p.a_stride) + piece * 16;
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int row = (i * WAVES + w) * 8 + lane / 8, piece = (lane & 7) ^ ((row >> 1) & 7);
      f_bo[i] = (unsigned)(min((int64_t)row, p.N - 1 - n) * p.b_stride) + piece * 16;
    }
  };
  const unsigned lds0 = (unsigned)reinterpret_cast<uintptr_t>((lds_words)lds);
  const auto fetch = [&](unsigned step) {
    const unsigned to = lds0 + (step & 1u) * STEP;
#pragma unroll
    for (int i = 0; i < NB; ++i) fetch_to_lds(f_b, f_bo[i], to + BM * KB + (i * WAVES + w) * 1024);
#pragma unroll
    for (int i = 0; i < NA; ++i) fetch_to_lds(f_a, f_ao[i], to + (i * WAVES + w) * 1024);
    f_a += KB;
    f_b += KB;
    if (++f_kb == p.blocks) {
      f_kb = 0;
      f_a -= (int64_t)p.blocks * KB;
      f_b -= (int64_t)p.blocks * KB;
    }
    if (--f_left == 0) {
      f_tile += walk.step;
      if (f_tile < walk.end) f_begin();
    }
  };
  // A tile's scales, BM of a's and BN of b's, 64 at a time: the waves in turn.
  const auto fetch_scales = [&](unsigned tile, unsigned which) {
    int64_t m, n;
    walk.origin(tile, m, n);
    m *= BM;
    n *= BN;
    const unsigned to = lds0 + SCALES + which * (BM + BN) * 4;
    for (int k = w; k < (BM + BN) / WAVE; k += WAVES) {
      const int at = k * WAVE + lane;
      if (k < BM / WAVE) fetch_word_to_lds(p.sa + m, (unsigned)min((int64_t)at, p.M - 1 - m) * 4, to + k * WAVE * 4);
      else fetch_word_to_lds(p.sb + n, (unsigned)min((int64_t)at - BM, p.N - 1 - n) * 4, to + k * WAVE * 4);
    }
  };
  const auto meet = [&]() {                                    // this wave's fetches are there and its reads done, and so are everyone's
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };

  f_begin();
  fetch_scales(walk.first, 0);
  fetch(0);
  meet();
  if (steps > 1) fetch(1);
  // (the permutation of a row depends on its place among 16: the same for all operands of a lane)
  const unsigned lo = i16 * KB + ((lane / 16) ^ (i16 >> 1)) * 16, hi = lo ^ 64u;
  unsigned a_lo = wm * KB + lo, a_hi = wm * KB + hi, b_lo = (BM + wn) * KB + lo, b_hi = (BM + wn) * KB + hi;
  unsigned flip = STEP;                                        // from a place in this step's buffer to the other's
  Piece bf[TN], af[2];
#pragma unroll
  for (int j = 0; j < TN; ++j) bf[j] = row_piece(lds, b_lo, b_hi, j * 16);
  af[0] = row_piece(lds, a_lo, a_hi, 0);
  unsigned step = 0, which = 0;
  for (unsigned tile = walk.first; tile < walk.end; tile += walk.step, which ^= 1u) {
    int64_t m0, n0;
    walk.origin(tile, m0, n0);
    m0 *= BM;
    n0 *= BN;
    i32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
#pragma unroll 1
    for (int kb = 0; kb < p.blocks; ++kb, ++step) {
#pragma unroll
      for (int i = 0; i < TM - 1; ++i) {
        af[(i + 1) & 1] = row_piece(lds, a_lo, a_hi, (i + 1) * 16);
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(bf[j].lo, af[i & 1].lo, acc[i][j], 0, 0, 0);
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(bf[j].hi, af[i & 1].hi, acc[i][j], 0, 0, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);     // the next operand's reads behind the first product
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 2 * TN - 1, 0);
        __builtin_amdgcn_sched_barrier(0);
      }
      meet();
      if (step + 2 < steps) fetch(step);                       // (into this step's buffer)
      if (kb == 0 && tile + walk.step < walk.end) fetch_scales(tile + walk.step, which ^ 1u);      // (all have stored the tile before)
      a_lo += flip;
      a_hi += flip;
      b_lo += flip;
      b_hi += flip;
      flip = 0u - flip;
      // The last row's products, and behind each what the next step begins with, in the order in which that needs it: a's first, b's first
      // halves, b's second halves.  (Behind the last step: what lies there, unused.)
      constexpr int L = TM - 1;
      af[0] = row_piece(lds, a_lo, a_hi, 0);
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        acc[L][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(bf[j].lo, af[L & 1].lo, acc[L][j], 0, 0, 0);
        bf[j].lo = *reinterpret_cast<const i32x4*>(lds + b_lo + j * 16 * KB);
      }
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        acc[L][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(bf[j].hi, af[L & 1].hi, acc[L][j], 0, 0, 0);
        bf[j].hi = *reinterpret_cast<const i32x4*>(lds + b_hi + j * 16 * KB);
      }
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
#pragma unroll
      for (int j = 0; j < 2 * TN; ++j) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
    }
    const float* scales = reinterpret_cast<const float*>(lds + SCALES) + which * (BM + BN);
    store_tile<Tag, TM, TN>(p, acc, m0 + wm, n0 + wn, p.N, lane, lds + STAGE + w * 2048, scales + wm, scales + BM + wn);
  }
}

// The same for small tiles, whose steps are too short to wait for memory with two buffers: a ring of S, S - 1 steps' operands under way, one barrier a step.
template <class Tag, int BM, int BN, int WM, int WN, int S>
__global__ __launch_bounds__((BM / WM) * (BN / WN) * WAVE) void rows_ring_kernel(const RowsParams p, unsigned tiles_m, unsigned tiles_n) {
  constexpr int WAVES = (BM / WM) * (BN / WN), TM = WM / 16, TN = WN / 16, NA = BM / 8 / WAVES, NB = BN / 8 / WAVES;
  static_assert(BM % (8 * WAVES) == 0 && BN % (8 * WAVES) == 0, "whole fetches");
  extern __shared__ __align__(1024) unsigned char lds[];      // S of (a: BM rows, b: BN rows of 128 bytes)
  constexpr int STEP = (BM + BN) * KB;
  const int lane = threadIdx.x & (WAVE - 1), w = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), i16 = lane % 16;
  const int wm = (w / (BN / WN)) * WM, wn = (w % (BN / WN)) * WN;
  const TileWalk walk(tiles_m, tiles_n);
  if (walk.first >= walk.end) return;
  const unsigned steps = ((walk.end - walk.first + walk.step - 1) / walk.step) * (unsigned)p.blocks;
  unsigned f_tile = walk.first, f_step = 0;
  int f_kb, f_left, f_place = 0;
  const unsigned char *f_a, *f_b;
  unsigned f_ao[NA], f_bo[NB];
  const auto f_begin = [&]() {
    int64_t m, n;
    walk.origin(f_tile, m, n);
    m *= BM;
    n *= p.wide;
    f_left = p.blocks;
    f_kb = first_block(f_tile, tiles_m, p.blocks);
    f_a = p.a + m * p.a_stride + (int64_t)f_kb * KB;
    f_b = p.b + n * p.b_stride + (int64_t)f_kb * KB;
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      const int row = (i * WAVES + w) * 8 + lane / 8, piece = (lane & 7) ^ ((row >> 1) & 7);
      f_ao[i] = (unsigned)(min((int64_t)row, p.M - 1 - m) * p.a_stride) + piece * 16;
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int row = (i * WAVES + w) * 8 + lane / 8, piece = (lane & 7) ^ ((row >> 1) & 7);
      f_bo[i] = (unsigned)(min((int64_t)row, min((int64_t)p.wide, p.N - n) - 1) * p.b_stride) + piece * 16;
    }
  };
  const unsigned lds0 = (unsigned)reinterpret_cast<uintptr_t>((lds_words)lds);
  const auto fetch = [&]() {
    const unsigned to = lds0 + f_place * STEP;
#pragma unroll
    for (int i = 0; i < NB; ++i) fetch_to_lds(f_b, f_bo[i], to + BM * KB + (i * WAVES + w) * 1024);
#pragma unroll
    for (int i = 0; i < NA; ++i) fetch_to_lds(f_a, f_ao[i], to + (i * WAVES + w) * 1024);
    f_place = f_place + 1 == S ? 0 : f_place + 1;
    f_a += KB;
    f_b += KB;
    if (++f_kb == p.blocks) {
      f_kb = 0;
      f_a -= (int64_t)p.blocks * KB;
      f_b -= (int64_t)p.blocks * KB;
    }
    ++f_step;
    if (--f_left == 0) {
      f_tile += walk.step;
      if (f_tile < walk.end) f_begin();
    }
  };
  f_begin();
#pragma unroll 1
  for (int s = 0; s < S - 1; ++s)
    if (f_step < steps) fetch();
  const unsigned lo = i16 * KB + ((lane / 16) ^ (i16 >> 1)) * 16, hi = lo ^ 64u;
  int place = 0;
  unsigned step = 0;
  for (unsigned tile = walk.first; tile < walk.end; tile += walk.step) {
    int64_t m0, n0;
    walk.origin(tile, m0, n0);
    m0 *= BM;
    n0 *= p.wide;
    i32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
#pragma unroll 1
    for (int kb = 0; kb < p.blocks; ++kb, ++step) {
      // this step's operands are there: all but the last S - 2 steps' fetches (they come back in order; a tile's stores only add to the count)
      if (step + (S - 2) < steps) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((S - 2) * (NA + NB)) : "memory");
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (f_step < steps) fetch();                             // (into the place of the step before, which all have read)
      const unsigned char* at = lds + place * STEP;
      place = place + 1 == S ? 0 : place + 1;
      Piece af[TM], bf[TN];
#pragma unroll
      for (int j = 0; j < TN; ++j) bf[j] = row_piece(at, (BM + wn) * KB + lo, (BM + wn) * KB + hi, j * 16);
#pragma unroll
      for (int i = 0; i < TM; ++i) af[i] = row_piece(at, wm * KB + lo, wm * KB + hi, i * 16);
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(bf[j].lo, af[i].lo, acc[i][j], 0, 0, 0);
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(bf[j].hi, af[i].hi, acc[i][j], 0, 0, 0);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    store_tile<Tag, TM, TN>(p, acc, m0 + wm, n0 + wn, min(p.N, n0 + p.wide), lane, lds + S * STEP + w * 2048);
  }
}

template <class Tag, int NT, int NCH>
static void launch_quantize(RowsQuant p, hipStream_t st) {
  constexpr int64_t MOST = LAUNCH_THREADS / NT / 65536 * 65536;      // rows of a launch
  for (int64_t all = p.rows; all > 0; all -= MOST) {
    p.rows = std::min(all, MOST);
    const unsigned x = (unsigned)std::min<int64_t>(p.rows, 65536), y = (unsigned)((p.rows + x - 1) / x);
    hipLaunchKernelGGL((quantize_whole_rows_kernel<Tag, NT, NCH>), dim3(x, y), dim3(NT), 0, st, p);
    p.x += MOST * p.row_stride * Tag::bytes;
    p.codes += MOST * p.code_stride;
    p.scales += MOST;
  }
}

static int rows_status() { return hipGetLastError() == hipSuccess ? DL_OK : DL_ERR_LAUNCH; }

template <class Tag, int BM, int BN, int WM, int WN>
static int launch_row_tiles(const RowsParams& p, hipStream_t st) {
  constexpr int threads = (BM / WM) * (BN / WN) * WAVE, bytes = 2 * (BM + BN) * (KB + 4) + threads / WAVE * (WN == 64 && Tag::bytes == 2 ? 2048 : 0), per_cu = 160 * 1024 / bytes;
  const int64_t tm = (p.M + BM - 1) / BM, tn = (p.N + BN - 1) / BN;
  if (tm * tn > 0x7ffffff0LL || p.a_stride * BM > 0xffffffffLL || p.b_stride * BN > 0xffffffffLL) return DL_ERR_LIMIT;
  if (bytes > 64 * 1024 &&
      hipFuncSetAttribute(reinterpret_cast<const void*>(&rows_kernel<Tag, BM, BN, WM, WN>), hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess)
    return DL_ERR_LAUNCH;
  const unsigned grid = (unsigned)std::min<int64_t>((tm * tn + 7) / 8 * 8, 256 * std::min(per_cu, 4));
  hipLaunchKernelGGL((rows_kernel<Tag, BM, BN, WM, WN>), dim3(grid), dim3(threads), bytes, st, p, (unsigned)tm, (unsigned)tn);
  return rows_status();
}

// Columns of a small tile: as many tiles a CU as whole ones make, all of a width, so that no CU has more weights to fetch than others (61 rows, from memory,
// us for whole tiles / even ones: x 32896 x 2048 21.0 / 19.8, x 50257 x 2048 25.4 / 24.0, x 65664 x 2048 34.4 / 30.4; 33 x 40000 x 4096 37.0 / 33.5; 8 x 14336 x 4096 14.6 /
// 13.6).  The places behind them are filled with the last row again: leaving them out costs branches and waits by count (64 x 8000 x 4096 11.5, so 14).
static int ring_wide(int64_t tm, int64_t N, int BN) {
  const int64_t each = (tm * ((N + BN - 1) / BN) + 255) / 256, across = std::max<int64_t>(1, 256 * each / tm);
  return (int)std::min<int64_t>(BN, ((N + across - 1) / across + 7) / 8 * 8);
}

template <class Tag, int BM, int BN, int WM, int WN, int S>
static int launch_row_ring(RowsParams p, hipStream_t st) {
  constexpr int threads = (BM / WM) * (BN / WN) * WAVE, bytes = S * (BM + BN) * KB + threads / WAVE * (WN == 64 && Tag::bytes == 2 ? 2048 : 0), per_cu = 160 * 1024 / bytes;
  const int64_t tm = (p.M + BM - 1) / BM;
  p.wide = ring_wide(tm, p.N, BN);
  const int64_t tn = (p.N + p.wide - 1) / p.wide;
  if (tm * tn > 0x7ffffff0LL || p.a_stride * BM > 0xffffffffLL || p.b_stride * BN > 0xffffffffLL) return DL_ERR_LIMIT;
  if (bytes > 64 * 1024 &&
      hipFuncSetAttribute(reinterpret_cast<const void*>(&rows_ring_kernel<Tag, BM, BN, WM, WN, S>), hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess)
    return DL_ERR_LAUNCH;
  const unsigned grid = (unsigned)std::min<int64_t>((tm * tn + 7) / 8 * 8, 256 * std::min(per_cu, 4));
  hipLaunchKernelGGL((rows_ring_kernel<Tag, BM, BN, WM, WN, S>), dim3(grid), dim3(threads), bytes, st, p, (unsigned)tm, (unsigned)tn);
  return rows_status();
}

// The tile of a call: that with the least time by a model of two numbers each, microseconds for a step of a CU -- alone, and what every
// further tile of the CU adds -- measured over 21 shapes from 64 x 1000 to 8192 x 32000 (us, in the order of the list: 8192 x 32000 x 1024 283, 336, 424,
// 631, 797; 512 x 14336 x 4096 53, 36, 58, 62, 81; 61 x 50257 x 2048 34, 28, 26, 29, 33; 128 x 8000 x 4096 46, 30, 16, 12.9, 14; 64 x 4096 x 4096 44, 31, 16, 13, 11).
struct RowsShape { int bm, bn; float alone, each; };
constexpr RowsShape ROWS_SHAPES[] = {{256, 256, 1.30f, 1.72f}, {128, 256, 0.89f, 1.19f}, {64, 128, 0.37f, 0.43f}, {64, 64, 0.31f, 0.27f}, {64, 32, 0.25f, 0.175f}};
static int rows_shape(int64_t M, int64_t N) {
  int best = 0;
  float least = 0.f;
  for (int i = 0; i < 5; ++i) {
    const RowsShape& t = ROWS_SHAPES[i];
    const int64_t tiles = ((M + t.bm - 1) / t.bm) * ((N + t.bn - 1) / t.bn);
    const float time = std::max(t.alone, (float)((tiles + 255) / 256) * t.each);
    if (i == 0 || time < least) { best = i; least = time; }
  }
  return best;
}

template <class Tag>
static int launch_rows(const RowsParams& p, hipStream_t st) {
  switch (rows_shape(p.M, p.N)) {
    case 0: return launch_row_tiles<Tag, 256, 256, 128, 64>(p, st);
    case 1: return launch_row_tiles<Tag, 128, 256, 64, 64>(p, st);
    case 2: return launch_row_ring<Tag, 64, 128, 32, 64, 3>(p, st);
    case 3: return launch_row_ring<Tag, 64, 64, 32, 32, 4>(p, st);
    default: return launch_row_ring<Tag, 64, 32, 32, 16, 4>(p, st);
  }
}

}  // namespace dl

extern "C" int dl_quantize_rows(const void* x, int dtype, int64_t row_stride, int64_t rows, int64_t cols, void* codes, int64_t code_stride,
                                float* scales, void* stream) {
  using namespace dl;
  if ((unsigned)dtype > DL_F16) return DL_ERR_DTYPE;
  const int64_t width = (cols + KB - 1) / KB * KB;
  if (rows < 0 || cols < 0 || row_stride < cols || code_stride < width) return DL_ERR_SHAPE;
  if (rows == 0) return DL_OK;
  if (!scales || (cols > 0 && (!x || !codes))) return DL_ERR_NULL;      // (rows of no columns have a scale too)
  if (reinterpret_cast<uintptr_t>(x) % (dtype == DL_F32 ? 4 : 2) || reinterpret_cast<uintptr_t>(codes) % 16 || code_stride % 16 ||
      reinterpret_cast<uintptr_t>(scales) % 4)
    return DL_ERR_ALIGN;
  const RowsQuant p{reinterpret_cast<const char*>(x), row_stride, rows, cols, width, reinterpret_cast<signed char*>(codes), code_stride, scales};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (rows > 0xffffffffLL) return DL_ERR_LIMIT;
#define DL_QUANTIZE_ROWS(TAG, NT, NCH) launch_quantize<TAG, NT, NCH>(p, st)
#define DL_QUANTIZE_TAG(TAG)                                  \
  if (width <= 1024) DL_QUANTIZE_ROWS(TAG, 128, 1);           \
  else if (width <= 2048) DL_QUANTIZE_ROWS(TAG, 256, 1);      \
  else if (width <= 4096) DL_QUANTIZE_ROWS(TAG, 256, 2);      \
  else if (width <= 8192) DL_QUANTIZE_ROWS(TAG, 512, 2);      \
  else if (width <= 16384) DL_QUANTIZE_ROWS(TAG, 512, 4);     \
  else DL_QUANTIZE_ROWS(TAG, 512, 0);
  if (dtype == DL_F32) { DL_QUANTIZE_TAG(TagF32) } else if (dtype == DL_BF16) { DL_QUANTIZE_TAG(TagBF16) } else { DL_QUANTIZE_TAG(TagF16) }
#undef DL_QUANTIZE_TAG
#undef DL_QUANTIZE_ROWS
  return rows_status();
}

extern "C" int dl_matmul_rows(const void* a, int64_t a_stride, const float* a_scale, int64_t M, const void* b, int64_t b_stride, const float* b_scale,
                              int64_t N, int64_t K, void* out, int out_dtype, int64_t out_stride, void* stream) {
  using namespace dl;
  if ((unsigned)out_dtype > DL_F16) return DL_ERR_DTYPE;
  const int64_t blocks = (K + KB - 1) / KB;
  if (M < 0 || N < 0 || K <= 0 || a_stride < blocks * KB || b_stride < blocks * KB || out_stride < N) return DL_ERR_SHAPE;
  if (M == 0 || N == 0) return DL_OK;
  if (!a || !b || !a_scale || !b_scale || !out) return DL_ERR_NULL;
  if ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) % 16 || a_stride % 16 || b_stride % 16 ||
      (reinterpret_cast<uintptr_t>(a_scale) | reinterpret_cast<uintptr_t>(b_scale)) % 4 || reinterpret_cast<uintptr_t>(out) % (out_dtype == DL_F32 ? 4 : 2))
    return DL_ERR_ALIGN;
  if (K > K_MOST) return DL_ERR_LIMIT;
  const RowsParams p{reinterpret_cast<const unsigned char*>(a), a_stride, a_scale, M, reinterpret_cast<const unsigned char*>(b), b_stride, b_scale, N,
                     (int)blocks, reinterpret_cast<char*>(out), out_stride};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (out_dtype == DL_F32) return launch_rows<TagF32>(p, st);
  if (out_dtype == DL_BF16) return launch_rows<TagBF16>(p, st);
  return launch_rows<TagF16>(p, st);
}
