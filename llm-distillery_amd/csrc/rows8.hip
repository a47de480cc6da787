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
// A workgroup a row, twice: for its largest magnitude, and for the codes.
struct RowsQuant {
  const char* x; int64_t row_stride, rows, cols, width;        // width: whole blocks
  signed char* codes; int64_t code_stride;
  float* scales;
};
__device__ __forceinline__ bool not_finite(float f) { return (__float_as_uint(f) & 0x7f800000u) == 0x7f800000u; }
template <class Tag, int NT>
__global__ __launch_bounds__(NT) void quantize_whole_rows_kernel(const RowsQuant p) {
  __shared__ float red[NT / WAVE];
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const char* x = p.x + row * p.row_stride * Tag::bytes;
    float m = 0.f;
    for (int64_t col = threadIdx.x * 8; col < p.cols; col += NT * 8) {
      float f[8];
      load_eight<Tag>(x, col, p.cols, f);
#pragma unroll
      for (int e = 0; e < 8; ++e) m = not_finite(f[e]) ? __builtin_inff() : fmaxf(m, fabsf(f[e]));
    }
    m = block_max<NT>(m, red);
    const bool odd = not_finite(m);
    const float scale = fmaxf(m * ISCALE, ISCALE_MIN);
    if (threadIdx.x == 0) p.scales[row] = odd ? __builtin_nanf("") : scale;
    for (int64_t col = threadIdx.x * 8; col < p.width; col += NT * 8) {
      float f[8];
      load_eight<Tag>(x, col, p.cols, f);
      u32x2 c = {0u, 0u};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int q = odd ? 0 : (int)fminf(fmaxf(rintf(f[e] / scale), -127.f), 127.f);
        c[e / 4] |= (unsigned)(q & 255) << (e % 4 * 8);
      }
      *reinterpret_cast<u32x2*>(p.codes + row * p.code_stride + col) = c;
    }
  }
}

// ---- product ----------------------------------------------------------------------------------------
struct RowsParams {
  const unsigned char* a; int64_t a_stride; const float* sa; int64_t M;
  const unsigned char* b; int64_t b_stride; const float* sb; int64_t N;
  int blocks;
  char* out; int64_t out_stride;
};

// Tiles of BM x BN, a wave WM x WN of it, a block of 128 columns (two matrix instructions deep) per step.  A step's operands are fetched into LDS by
// loads that bypass the registers, two steps ahead of their use; a row of a tile is 128 bytes of LDS, its eight 16-byte pieces permuted
// by piece ^ (row / 2 % 8): the 16 rows x 16 bytes that a quarter of a wave reads then lie on all banks once.  (The loads write LDS in lane
// order, so it is their source addresses that are permuted.)
// Within a step a wave goes through its WM / 16 rows of tiles: the operand of the next row is read while the matrix unit works on this one.  A
// step's last barrier sits ahead of the last row, whose operands are in registers by then, so that the matrix unit is busy across it; another one at
// half the step frees b's place and half of a's.  Workgroups stay: each walks its tiles as one sequence of steps.
struct Piece { i32x4 lo, hi; };                                // a lane's 32 bytes of a row: 16 columns of either half of the block
__device__ __forceinline__ Piece row_piece(const unsigned char* lds, unsigned lo, unsigned hi, int rows) {
  return Piece{*reinterpret_cast<const i32x4*>(lds + lo + rows * KB), *reinterpret_cast<const i32x4*>(lds + hi + rows * KB)};
}

template <class Tag, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__((BM / WM) * (BN / WN) * WAVE, 2) void rows_kernel(const RowsParams p, unsigned tiles_m, unsigned tiles_n) {
  constexpr int WAVES = (BM / WM) * (BN / WN), TM = WM / 16, TN = WN / 16, NA = BM / 8 / WAVES, NB = BN / 8 / WAVES;
  static_assert(TM >= 2 && BM % (8 * WAVES) == 0 && BN % (8 * WAVES) == 0, "whole fetches");
  extern __shared__ __align__(1024) unsigned char lds[];      // two of (a: BM rows, b: BN rows of 128 bytes)
  constexpr int STEP = (BM + BN) * KB;
  const int lane = threadIdx.x & (WAVE - 1), w = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), i16 = lane % 16;      // (w: known to be the wave's)
  const int wm = (w / (BN / WN)) * WM, wn = (w % (BN / WN)) * WN;
  const TileWalk walk(tiles_m, tiles_n);
  if (walk.first >= walk.end) return;
  const unsigned steps = ((walk.end - walk.first + walk.step - 1) / walk.step) * (unsigned)p.blocks;

  // the fetching side: its tile, its block, this thread's places in them
  unsigned f_tile = walk.first;
  int f_kb = 0;
  const unsigned char *f_a, *f_b;
  unsigned f_ao[NA], f_bo[NB];
  const auto f_begin = [&]() {
    int64_t m, n;
    walk.origin(f_tile, m, n);
    m *= BM;
    n *= BN;
    f_a = p.a + m * p.a_stride;
    f_b = p.b + n * p.b_stride;
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
  // In two parts, by when their places become free: `early` after half a step (b, whose operands are in registers from a step's
  // beginning on, and of a the rows that the waves go through first), `late` at its end.
  constexpr bool HALVES = WM / 2 == WAVES * 8;                 // every other fetch of a: those rows
  constexpr int EARLY = NB + (HALVES ? NA / 2 : 0);
  const auto fetch_a = [&](unsigned char* to, int i) {
    __builtin_amdgcn_global_load_lds((global_words)(f_a + f_ao[i]), (lds_words)(to + (i * WAVES + w) * 1024), 16, 0, 0);
  };
  const auto fetch_early = [&](unsigned step) {
    unsigned char* to = lds + (step & 1u) * STEP;
#pragma unroll
    for (int i = 0; i < NB; ++i)
      __builtin_amdgcn_global_load_lds((global_words)(f_b + f_bo[i]), (lds_words)(to + BM * KB + (i * WAVES + w) * 1024), 16, 0, 0);
    if (HALVES)
#pragma unroll
      for (int i = 0; i < NA; i += 2) fetch_a(to, i);
  };
  const auto fetch_late = [&](unsigned step) {
    unsigned char* to = lds + (step & 1u) * STEP;
#pragma unroll
    for (int i = HALVES ? 1 : 0; i < NA; i += HALVES ? 2 : 1) fetch_a(to, i);
    f_a += KB;
    f_b += KB;
    if (++f_kb == p.blocks) {
      f_kb = 0;
      f_tile += walk.step;
      if (f_tile < walk.end) f_begin();
    }
  };
  const auto meet = [&]() {                                    // everyone's reads so far are done
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  // This wave's fetches are there but for the last `early` part (loads come back in order; the stores of a tile only add to the count).
  const auto landed = [&](bool early_under_way) {
    if (early_under_way) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(EARLY) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  };

  f_begin();
  fetch_early(0);
  fetch_late(0);
  landed(false);
  meet();
  if (steps > 1) {
    fetch_early(1);
    fetch_late(1);
  }
  // (the permutation of a row depends on its place among 16: the same for all operands of a lane)
  const unsigned lo = i16 * KB + ((lane / 16) ^ (i16 >> 1)) * 16, hi = lo ^ 64u;
  unsigned a_lo = wm * KB + lo, a_hi = wm * KB + hi, b_lo = (BM + wn) * KB + lo, b_hi = (BM + wn) * KB + hi;
  unsigned flip = STEP;                                        // from a place in this step's buffer to the other's
  Piece bf[TN], af[2];
#pragma unroll
  for (int j = 0; j < TN; ++j) bf[j] = row_piece(lds, b_lo, b_hi, j * 16);
  af[0] = row_piece(lds, a_lo, a_hi, 0);
  unsigned step = 0;
  for (unsigned tile = walk.first; tile < walk.end; tile += walk.step) {
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
        if (i == TM / 2 - 1 && step + 2 < steps) {
          meet();
          fetch_early(step);                                   // (into this step's buffer)
        }
      }
      landed(step + 2 < steps);
      meet();
      if (step + 2 < steps) fetch_late(step);
      a_lo += flip;
      a_hi += flip;
      b_lo += flip;
      b_hi += flip;
      flip = 0u - flip;
      constexpr int L = TM - 1;
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        acc[L][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(bf[j].lo, af[L & 1].lo, acc[L][j], 0, 0, 0);
        acc[L][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(bf[j].hi, af[L & 1].hi, acc[L][j], 0, 0, 0);
        bf[j] = row_piece(lds, b_lo, b_hi, j * 16);            // (behind the last step: what lies there, unused)
      }
      af[0] = row_piece(lds, a_lo, a_hi, 0);
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    }
    // The tile's values.  Two-byte results go through 2 KiB of LDS of the wave's own, 16 rows at a time, so that a store writes whole
    // 128-byte stretches of 8 rows instead of 32 bytes of 16; a row's 16-byte units are permuted by unit ^ (row % 8).
    int here = lane;
    asm volatile("" : "+v"(here));                             // (keeps the stores' addresses out of the steps' registers)
    const int row = here % 16, quad = here / 16;
    f32x4 sb[TN];
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) sb[j][e] = p.sb[min(n0 + wn + j * 16 + quad * 4 + e, p.N - 1)];
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const float sa = p.sa[min(m0 + wm + i * 16 + row, p.M - 1)];
      f32x4 v[TN];
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[j][e] = (float)acc[i][j][e] * (sa * sb[j][e]);
      if constexpr (Tag::bytes == 2 && WN == 64) {
        unsigned char* stage = lds + 2 * STEP + w * 2048;
        const int r8 = here / 8, unit = here % 8;
        const int64_t n = n0 + wn + unit * 8;
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          const float f[8] = {v[j][0], v[j][1], v[j][2], v[j][3], 0.f, 0.f, 0.f, 0.f};
          const u32x4 c = Chunk<Tag>::pack(f);
          *reinterpret_cast<u32x2*>(stage + row * 128 + ((j * 2 + quad / 2) ^ (row & 7)) * 16 + (quad & 1) * 8) = u32x2{c[0], c[1]};
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int64_t m = m0 + wm + i * 16 + k * 8 + r8;
          const u32x4 c = *reinterpret_cast<const u32x4*>(stage + (k * 8 + r8) * 128 + (unit ^ r8) * 16);
          char* to = p.out + (m * p.out_stride + n) * 2;
          if (m < p.M && n + 8 <= p.N) store16_stream_any(to, c);
          else if (m < p.M && n < p.N) store_chunk_elementwise<Tag>(to, 0, (int)(p.N - n), c);
        }
      } else {
        const int64_t m = m0 + wm + i * 16 + row;
        char* to = p.out + m * p.out_stride * Tag::bytes;
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          const int64_t n = n0 + wn + j * 16 + quad * 4;
          if (m < p.M && n < p.N) store_four<Tag>(to, n, p.N, v[j]);
        }
      }
    }
  }
}

static int rows_status() { return hipGetLastError() == hipSuccess ? DL_OK : DL_ERR_LAUNCH; }

template <class Tag, int BM, int BN, int WM, int WN>
static int launch_row_tiles(const RowsParams& p, hipStream_t st) {
  constexpr int threads = (BM / WM) * (BN / WN) * WAVE, bytes = 2 * (BM + BN) * KB + threads / WAVE * (WN == 64 && Tag::bytes == 2 ? 2048 : 0), per_cu = 160 * 1024 / bytes;
  const int64_t tm = (p.M + BM - 1) / BM, tn = (p.N + BN - 1) / BN;
  if (tm * tn > 0x7ffffff0LL || p.a_stride * BM > 0xffffffffLL || p.b_stride * BN > 0xffffffffLL) return DL_ERR_LIMIT;
  if (bytes > 64 * 1024 &&
      hipFuncSetAttribute(reinterpret_cast<const void*>(&rows_kernel<Tag, BM, BN, WM, WN>), hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess)
    return DL_ERR_LAUNCH;
  const unsigned grid = (unsigned)std::min<int64_t>((tm * tn + 7) / 8 * 8, 256 * std::min(per_cu, 4));
  hipLaunchKernelGGL((rows_kernel<Tag, BM, BN, WM, WN>), dim3(grid), dim3(threads), bytes, st, p, (unsigned)tm, (unsigned)tn);
  return rows_status();
}

// The tile of a call: that with the least time by a model of two numbers each, microseconds for a step of a CU -- alone, and what every
// further tile of the CU adds.
struct RowsShape { int bm, bn; float alone, each; };
constexpr RowsShape ROWS_SHAPES[] = {{256, 256, 1.55f, 1.55f}, {128, 256, 1.05f, 1.25f}, {64, 128, 0.62f, 0.43f}, {64, 64, 0.50f, 0.26f}};
static int rows_shape(int64_t M, int64_t N) {
  int best = 0;
  float least = 0.f;
  for (int i = 0; i < 4; ++i) {
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
    case 2: return launch_row_tiles<Tag, 64, 128, 32, 64>(p, st);
    default: return launch_row_tiles<Tag, 64, 64, 32, 32>(p, st);
  }
}

}  // namespace dl

extern "C" int dl_quantize_rows(const void* x, int dtype, int64_t row_stride, int64_t rows, int64_t cols, void* codes, int64_t code_stride,
                                float* scales, void* stream) {
  using namespace dl;
  if ((unsigned)dtype > DL_F16) return DL_ERR_DTYPE;
  const int64_t width = (cols + KB - 1) / KB * KB;
  if (rows < 0 || cols < 0 || row_stride < cols || code_stride < width) return DL_ERR_SHAPE;
  if (rows == 0 || cols == 0) return DL_OK;
  if (!x || !codes || !scales) return DL_ERR_NULL;
  if (reinterpret_cast<uintptr_t>(x) % (dtype == DL_F32 ? 4 : 2) || reinterpret_cast<uintptr_t>(codes) % 16 || code_stride % 16 ||
      reinterpret_cast<uintptr_t>(scales) % 4)
    return DL_ERR_ALIGN;
  const RowsQuant p{reinterpret_cast<const char*>(x), row_stride, rows, cols, width, reinterpret_cast<signed char*>(codes), code_stride, scales};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)std::min<int64_t>(rows, 65535));
  if (dtype == DL_F32) hipLaunchKernelGGL((quantize_whole_rows_kernel<TagF32, 256>), grid, dim3(256), 0, st, p);
  else if (dtype == DL_BF16) hipLaunchKernelGGL((quantize_whole_rows_kernel<TagBF16, 256>), grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL((quantize_whole_rows_kernel<TagF16, 256>), grid, dim3(256), 0, st, p);
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
