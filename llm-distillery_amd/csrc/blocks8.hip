// Matrix product in 8-bit floating point (e4m3) with a scale for every block of 128, and what makes its operands.
//
//   out[m, n] = sum over blocks kb of  sa[m, kb] * sb[n / 128, kb] * sum over the 128 columns k of kb of a[m, k] * b[n, k]
//
// a: one scale for every 128 values of a row (activations, quantised on the way); b: one for every 128 x 128 weights.
// One matrix instruction sums a whole block: v_mfma_f32_16x16x128_f8f6f4 takes 16 x 128 by 128 x 16 values, so a block's sum
// leaves the matrix unit once and is scaled and added in fp32 on the vector unit, four multiply-adds per lane beside 32
// cycles of the matrix unit.  The operands are passed with b first: a lane then holds four neighbouring columns n of one
// row m, one scale product serves all four, and the result is stored in pieces of four.
// Any order of the 128 values will do as long as both operands have the same one: a lane's 32 bytes are two 16-byte
// pieces, 64 bytes apart, so that every load instruction covers 64 contiguous bytes of a row.
#include "distill_common.hpp"
#include "distill_hip.h"
#include "product_schedule.hpp"

#include <algorithm>

namespace dl {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int QB = 128;                       // values that share a scale; bytes of a block of a row
constexpr float QSCALE = 1.f / 448.f, QSCALE_MIN = 0x1p-100f;

// ---- quantise ---------------------------------------------------------------------------------------
// scale = max(largest magnitude * (1 / 448 in fp32), 2^-100), code = x / scale (an IEEE division) rounded to e4m3, ties to even.
// Columns behind the last one are zeros, up to the end of the block.  NaN stays NaN; a block with an infinity has an infinite
// scale and NaN in the infinity's place.
template <class Tag>
__device__ __forceinline__ void load_eight(const char* row, int64_t col, int64_t cols, float* f) {
  if (col + 8 <= cols) {
    if constexpr (Tag::bytes == 2) {
      Chunk<Tag>::unpack(load16_unaligned(row + col * 2), f);
    } else {
      Chunk<Tag>::unpack(load16_unaligned(row + col * 4), f);
      Chunk<Tag>::unpack(load16_unaligned(row + col * 4 + 16), f + 4);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = col + e < cols ? load_as_float(row, Tag::id, col + e) : 0.f;
  }
}
__device__ __forceinline__ float largest_of_eight(const float* f) {
  float m = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(f[e]));
  return m;
}
__device__ __forceinline__ u32x2 code_eight(const float* f, float scale) {
  float q[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) q[e] = f[e] / scale;
  u32x2 c;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * i], q[4 * i + 1], 0, false);
    v = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * i + 2], q[4 * i + 3], v, true);
    c[i] = (unsigned)v;
  }
  return c;
}
struct QuantParams {
  const char* x; int64_t row_stride, rows, cols, blocks;
  unsigned char* codes; int64_t code_stride;
  float* scales; int64_t scale_row, scale_block;
};
// One scale per row and block: 16 threads a block, one workgroup sixteen blocks of a row.
template <class Tag>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const QuantParams p) {
  const int64_t r = blockIdx.y, kb = (int64_t)blockIdx.x * 16 + threadIdx.x / 16;
  const int t = threadIdx.x % 16;
  if (kb >= p.blocks) return;
  const int64_t col = kb * QB + t * 8;
  for (int64_t row = r; row < p.rows; row += gridDim.y) {
    float f[8];
    load_eight<Tag>(p.x + row * p.row_stride * Tag::bytes, col, p.cols, f);
    float m = largest_of_eight(f);
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, WAVE));
    const float scale = fmaxf(m * QSCALE, QSCALE_MIN);
    *reinterpret_cast<u32x2*>(p.codes + row * p.code_stride + col) = code_eight(f, scale);
    if (t == 0) p.scales[row * p.scale_row + kb * p.scale_block] = scale;
  }
}
// One scale per 128 x 128: a workgroup a block, the values in its registers between the maximum and the codes.
template <class Tag>
__global__ __launch_bounds__(256) void quantize_squares_kernel(const QuantParams p) {
  __shared__ float red[4];
  const int64_t kb = blockIdx.x, row0 = (int64_t)blockIdx.y * QB, col = kb * QB + (threadIdx.x % 16) * 8;
  float f[8][8], m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = row0 + i * 16 + threadIdx.x / 16;
    if (row < p.rows) load_eight<Tag>(p.x + row * p.row_stride * Tag::bytes, col, p.cols, f[i]);
    else
#pragma unroll
      for (int e = 0; e < 8; ++e) f[i][e] = 0.f;
    m = fmaxf(m, largest_of_eight(f[i]));
  }
  m = block_max<256>(m, red);
  const float scale = fmaxf(m * QSCALE, QSCALE_MIN);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = row0 + i * 16 + threadIdx.x / 16;
    if (row < p.rows) *reinterpret_cast<u32x2*>(p.codes + row * p.code_stride + col) = code_eight(f[i], scale);
  }
  if (threadIdx.x == 0) p.scales[blockIdx.y * p.scale_row + kb * p.scale_block] = scale;
}

// ---- product ----------------------------------------------------------------------------------------
struct BlocksParams {
  const unsigned char* a; int64_t a_stride; const float* sa; int64_t sa_row, sa_block; int64_t M;
  const unsigned char* b; int64_t b_stride; const float* sb; int64_t sb_row, sb_block; int64_t N;
  int blocks;
  char* out; int64_t out_stride;
};
__device__ __forceinline__ f32x4 block_product(const i32x8& b, const i32x8& a) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);      // e4m3 both, unscaled
}
__device__ __forceinline__ i32x8 join_pieces(const u32x4& lo, const u32x4& hi) {
  return i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
}
// Four neighbouring columns of a row, as far as it reaches.
template <class Tag>
__device__ __forceinline__ void store_four(char* row, int64_t n, int64_t N, const f32x4& v) {
  if (n + 4 <= N) {
    if constexpr (Tag::bytes == 4) {
      store16_unaligned(row + n * 4, u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])});
    } else {
      const float f[8] = {v[0], v[1], v[2], v[3], 0.f, 0.f, 0.f, 0.f};
      const u32x4 c = Chunk<Tag>::pack(f);
      const u32x2 two = {c[0], c[1]};
      __builtin_memcpy(row + n * 2, &two, 8);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < N) store_from_float(row, Tag::id, n + i, v[i]);
  }
}

// Tiles of BM x BN, a wave WM x WN of it, one block of 128 columns per step.  A step's operands are fetched into LDS by loads
// that bypass the registers, two steps ahead of their use; a row of a tile is 128 bytes of LDS, its eight 16-byte pieces permuted by
// piece ^ (row / 2 % 8): the 16 rows x 16 bytes that a quarter of a wave reads then lie on all banks once.  (The loads write LDS in
// lane order, so it is their source addresses that are permuted.)
// Within a step a wave goes through its WM / 16 rows of tiles: the operand of the next row is read while the matrix unit works on
// this one, and the products of the row before are scaled and added meanwhile.  A step's last barrier sits ahead of the last row: by
// then all operands of the step are in registers, so what follows it -- the last row's products, the first operands of the next step,
// the fetch into what has just become free -- keeps the matrix unit busy across it.  Another one at half the step frees b's place and
// half of a's, so that three quarters of the bytes have a step and a half to arrive (what the latency of memory asks for: with
// one step, waits were a third of the time).
// Workgroups stay: each walks its tiles as one sequence of steps, so that the next tile's operands arrive while the last one is stored.
// Measured: 8192 x 128256 x 4096 (bf16 out) 3.69-3.94 ms, 2190-2330 Tflop/s; the matrix units' time alone, at the 1.97 GHz that the card
// holds under this load, is 2.1 ms, the scaling's multiply-adds share the issue slots with them.  (A library product of the same operands
// with one scale for all: 3.17 ms.)  Few rows are bound by the weights' bytes: 1 x 128256 x 4096 99-117 us (4.5-5.3 TB/s),
// 61 x 50257 x 2048 25 us (4.1 TB/s), 19 where MALL still has the weights.  (Few rows in a kernel that streams the weights straight into
// the operands: 107 us for one row of 128256 x 4096, 115 for 4, 147 for 16, but 28 to 40 where these tiles take 17.5 on 50257 x 2048.)
typedef const unsigned __attribute__((address_space(1))) * global_words;
typedef unsigned __attribute__((address_space(3))) * lds_words;

// The operand that begins `lo` / `hi` bytes into LDS for this lane (its two pieces), `rows` (a constant) rows on.
__device__ __forceinline__ i32x8 tile_operand(const unsigned char* lds, unsigned lo, unsigned hi, int rows) {
  return join_pieces(*reinterpret_cast<const u32x4*>(lds + lo + rows * QB), *reinterpret_cast<const u32x4*>(lds + hi + rows * QB));
}

// The tiles of a launch: consecutive workgroups go round the 8 XCDs; each XCD has a contiguous eighth of the tiles, in bands of 8
// rows of tiles, so that the tiles it works on at a time share their operands in its L2.
struct TileWalk {
  unsigned tiles_m, tiles_n, first, step, end;
  __device__ TileWalk(unsigned tm, unsigned tn) : tiles_m(tm), tiles_n(tn) {
    const unsigned total = tm * tn, each = (total + 7) / 8, xcd = blockIdx.x & 7u;
    first = xcd * each + (blockIdx.x >> 3);
    end = min(total, (xcd + 1) * each);
    step = gridDim.x >> 3;
  }
  __device__ void origin(unsigned t, int64_t& m, int64_t& n) const {      // in tiles
    const unsigned band = t / (8u * tiles_n), high = min(8u, tiles_m - band * 8u), in = t - band * 8u * tiles_n;
    m = band * 8u + in % high;
    n = in / high;
  }
};

template <class Tag, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__((BM / WM) * (BN / WN) * WAVE, 2) void tile_kernel(const BlocksParams p, unsigned tiles_m, unsigned tiles_n) {
  constexpr int WAVES = (BM / WM) * (BN / WN), TM = WM / 16, TN = WN / 16, NA = BM / 8 / WAVES, NB = BN / 8 / WAVES;
  static_assert(WN <= QB && QB % WN == 0, "a wave's columns share their scales");
  static_assert(TM >= 2 && BM % WAVE == 0 && BN % WAVE == 0 && BM / WAVE < WAVES, "the first waves fetch a's scales, the next one b's");
  extern __shared__ __align__(1024) unsigned char lds[];      // two of (a: BM rows, b: BN rows of 128 bytes, a's BM scales, b's for every BN / 64 columns)
  constexpr int STEP = (BM + BN) * QB + BM * 4 + WAVE * 4;
  const int lane = threadIdx.x & (WAVE - 1), w = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), i16 = lane % 16;      // (w: known to be the wave's)
  const int wm = (w / (BN / WN)) * WM, wn = (w % (BN / WN)) * WN;
  const TileWalk walk(tiles_m, tiles_n);
  if (walk.first >= walk.end) return;
  const unsigned steps = ((walk.end - walk.first + walk.step - 1) / walk.step) * (unsigned)p.blocks;

  // the fetching side: its tile, its block, this thread's places in them
  unsigned f_tile = walk.first;
  int f_kb = 0;
  const unsigned char *f_a, *f_b;
  const float* f_s;
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
    f_s = w < BM / WAVE ? p.sa + min(m + w * WAVE + lane, p.M - 1) * p.sa_row : p.sb + min(n + lane * (BN / WAVE), p.N - 1) / QB * p.sb_row;
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
      __builtin_amdgcn_global_load_lds((global_words)(f_b + f_bo[i]), (lds_words)(to + BM * QB + (i * WAVES + w) * 1024), 16, 0, 0);
    if (HALVES)
#pragma unroll
      for (int i = 0; i < NA; i += 2) fetch_a(to, i);
  };
  const auto fetch_late = [&](unsigned step) {
    unsigned char* to = lds + (step & 1u) * STEP;
#pragma unroll
    for (int i = HALVES ? 1 : 0; i < NA; i += HALVES ? 2 : 1) fetch_a(to, i);
    if (w <= BM / WAVE) __builtin_amdgcn_global_load_lds((global_words)f_s, (lds_words)(to + (BM + BN) * QB + w * WAVE * 4), 4, 0, 0);
    f_a += QB;
    f_b += QB;
    f_s += w < BM / WAVE ? p.sa_block : p.sb_block;
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
  // Products are scaled and added a few behind the one that the matrix unit starts: their results are there by then.
  constexpr int Q = TM * TN;
  using Order = ProductSchedule<Q>;
  static_assert(Order::sound(), "every product is added once");
  // (the permutation of a row depends on its place among 16: the same for all operands of a lane)
  const unsigned lo = i16 * QB + ((lane / 16) ^ (i16 >> 1)) * 16, hi = lo ^ 64u;
  unsigned a_lo = wm * QB + lo, a_hi = wm * QB + hi, b_lo = (BM + wn) * QB + lo, b_hi = (BM + wn) * QB + hi, s_at = (BM + BN) * QB + (wm + i16) * 4, sb_at = (BM + BN) * QB + BM * 4 + wn * WAVE / BN * 4;
  unsigned flip = STEP;                                        // from a place in this step's buffer to the other's
  i32x8 bf[TN], af[2];
#pragma unroll
  for (int j = 0; j < TN; ++j) bf[j] = tile_operand(lds, b_lo, b_hi, j * 16);
  af[0] = tile_operand(lds, a_lo, a_hi, 0);
  unsigned step = 0;
  for (unsigned tile = walk.first; tile < walk.end; tile += walk.step) {
  int64_t m0, n0;
  walk.origin(tile, m0, n0);
  m0 *= BM;
  n0 *= BN;
  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
  for (int kb = 0; kb < p.blocks; ++kb, ++step) {
    float s[TM];
    f32x4 v[Order::PLACES];
    const auto add = [&](int q) {
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[q / TN][q % TN][e] = fmaf(v[Order::place(q)][e], s[q / TN], acc[q / TN][q % TN][e]);
      asm volatile("" : "+v"(acc[q / TN][q % TN]));            // (here, and not collected behind the barrier)
    };
    const auto add_in_slot = [&](int slot) {
      if (Order::added_in(slot) != Order::NONE) add(Order::added_in(slot));
    };
#pragma unroll
    for (int i = 0; i < TM; ++i) s[i] = *reinterpret_cast<const float*>(lds + s_at + i * 64);
    const float sb = *reinterpret_cast<const float*>(lds + sb_at);
#pragma unroll
    for (int i = 0; i < TM - 1; ++i) {
      af[(i + 1) & 1] = tile_operand(lds, a_lo, a_hi, (i + 1) * 16);
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int q = i * TN + j;
        v[Order::place(q)] = block_product(bf[j], af[i & 1]);
        if (q == 1) {
#pragma unroll
          for (int k = 0; k < TM; ++k) s[k] *= sb;
        }
        add_in_slot(q);
      }
      // a product and the four multiply-adds of an earlier one in turns, the next operand's reads behind the first
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        if (j == 0) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
      if (i == TM / 2 - 1 && step + 2 < steps) {
        meet();
        fetch_early(step);                                     // (into this step's buffer)
      }
    }
    landed(step + 2 < steps);
    meet();
    if (step + 2 < steps) fetch_late(step);
    a_lo += flip;
    a_hi += flip;
    b_lo += flip;
    b_hi += flip;
    s_at += flip;
    sb_at += flip;
    flip = 0u - flip;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int q = (TM - 1) * TN + j;
      v[Order::place(q)] = block_product(bf[j], af[(TM - 1) & 1]);
      bf[j] = tile_operand(lds, b_lo, b_hi, j * 16);           // (behind the last step: what lies there, unused)
      add_in_slot(q);
    }
    af[0] = tile_operand(lds, a_lo, a_hi, 0);
#pragma unroll
    for (int q = Order::LEFT; q < Q; ++q) add(q);
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    __builtin_amdgcn_sched_group_barrier(0x002, 4 * Order::BEHIND, 0);
  }
  // The tile's values.  Two-byte results go through 2 KiB of LDS of the wave's own, 16 rows at a time, so that a store writes whole
  // 128-byte stretches of 8 rows instead of 32 bytes of 16; a row's 16-byte units are permuted by unit ^ (row % 8).
  int here = lane;
  asm volatile("" : "+v"(here));                               // (keeps the stores' addresses out of the steps' registers)
  if constexpr (Tag::bytes == 2 && WN == 64) {
    unsigned char* stage = lds + 2 * STEP + w * 2048;
    const int row = here % 16, quad = here / 16, r8 = here / 8, unit = here % 8;
    const int64_t n = n0 + wn + unit * 8;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const float f[8] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3], 0.f, 0.f, 0.f, 0.f};
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
    }
  } else {
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int64_t m = m0 + wm + i * 16 + here % 16;
      char* row = p.out + m * p.out_stride * Tag::bytes;
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int64_t n = n0 + wn + j * 16 + here / 16 * 4;
        if (m < p.M && n < p.N) store_four<Tag>(row, n, p.N, acc[i][j]);
      }
    }
  }
  }
}

static int blocks_status() { return hipGetLastError() == hipSuccess ? DL_OK : DL_ERR_LAUNCH; }

template <class Tag, int BM, int BN, int WM, int WN>
static int launch_tiles(const BlocksParams& p, hipStream_t st) {
  constexpr int threads = (BM / WM) * (BN / WN) * WAVE, bytes = 2 * ((BM + BN) * QB + BM * 4 + WAVE * 4) + threads / WAVE * (WN == 64 && Tag::bytes == 2 ? 2048 : 0), per_cu = 160 * 1024 / bytes;
  const int64_t tm = (p.M + BM - 1) / BM, tn = (p.N + BN - 1) / BN;
  if (tm * tn > 0x7ffffff0LL || p.a_stride * BM > 0xffffffffLL || p.b_stride * BN > 0xffffffffLL) return DL_ERR_LIMIT;
  if (bytes > 64 * 1024 &&
      hipFuncSetAttribute(reinterpret_cast<const void*>(&tile_kernel<Tag, BM, BN, WM, WN>), hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess)
    return DL_ERR_LAUNCH;
  const unsigned grid = (unsigned)std::min<int64_t>((tm * tn + 7) / 8 * 8, 256 * std::min(per_cu, 4));
  hipLaunchKernelGGL((tile_kernel<Tag, BM, BN, WM, WN>), dim3(grid), dim3(threads), bytes, st, p, (unsigned)tm, (unsigned)tn);
  return blocks_status();
}

// The tile of a call: that with the least time by a model of two numbers each, microseconds for a step of a CU -- alone, and what every
// further tile of the CU adds -- measured over 15 shapes from 64 x 4096 to 4096 x 8000 (64 x 50257 x 2048: 34, 23, 21, 24 us in
// the order of the list; 128 x 128256 x 4096: 137, 118, 148, 175; 512 x 128256 x 4096: 271, 335, 428, 519; 128 x 8000 x 4096: 51, 34, 21, 17-18).
struct TileShape { int bm, bn; float alone, each; };
constexpr TileShape TILE_SHAPES[] = {{256, 256, 1.55f, 1.55f}, {128, 256, 1.05f, 1.25f}, {64, 128, 0.62f, 0.43f}, {64, 64, 0.50f, 0.26f}};
static int tile_shape(int64_t M, int64_t N) {
  int best = 0;
  float least = 0.f;
  for (int i = 0; i < 4; ++i) {
    const TileShape& t = TILE_SHAPES[i];
    const int64_t tiles = ((M + t.bm - 1) / t.bm) * ((N + t.bn - 1) / t.bn);
    const float time = std::max(t.alone, (float)((tiles + 255) / 256) * t.each);
    if (i == 0 || time < least) { best = i; least = time; }
  }
  return best;
}

template <class Tag>
static int launch_blocks(const BlocksParams& p, hipStream_t st) {
  switch (tile_shape(p.M, p.N)) {
    case 0: return launch_tiles<Tag, 256, 256, 128, 64>(p, st);
    case 1: return launch_tiles<Tag, 128, 256, 64, 64>(p, st);
    case 2: return launch_tiles<Tag, 64, 128, 32, 64>(p, st);
    default: return launch_tiles<Tag, 64, 64, 32, 32>(p, st);
  }
}

}  // namespace dl

extern "C" int dl_quantize_blocks(const void* x, int dtype, int64_t row_stride, int64_t rows, int64_t cols, int block_rows, void* codes,
                                  int64_t code_stride, float* scales, int64_t scale_row_stride, int64_t scale_block_stride, void* stream) {
  using namespace dl;
  if ((unsigned)dtype > DL_F16) return DL_ERR_DTYPE;
  const int64_t blocks = (cols + QB - 1) / QB;
  if (rows < 0 || cols < 0 || row_stride < cols || code_stride < blocks * QB || (block_rows != 1 && block_rows != QB) || scale_row_stride < 0 ||
      scale_block_stride < 0)
    return DL_ERR_SHAPE;
  if (rows == 0 || cols == 0) return DL_OK;
  if (!x || !codes || !scales) return DL_ERR_NULL;
  if (reinterpret_cast<uintptr_t>(x) % (dtype == DL_F32 ? 4 : 2) || reinterpret_cast<uintptr_t>(codes) % 16 || code_stride % 16 ||
      reinterpret_cast<uintptr_t>(scales) % 4)
    return DL_ERR_ALIGN;
  if (blocks > LAUNCH_THREADS / 256 || (block_rows == QB && (rows + QB - 1) / QB > 65535)) return DL_ERR_LIMIT;
  const QuantParams p{reinterpret_cast<const char*>(x), row_stride, rows, cols, blocks, reinterpret_cast<unsigned char*>(codes), code_stride,
                      scales, scale_row_stride, scale_block_stride};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const dim3 rows_grid((unsigned)((blocks + 15) / 16), (unsigned)std::min<int64_t>(rows, 65535)), squares_grid((unsigned)blocks, (unsigned)((rows + QB - 1) / QB));
#define DL_QUANTIZE(TAG)                                                                              \
  if (block_rows == 1) hipLaunchKernelGGL(quantize_rows_kernel<TAG>, rows_grid, dim3(256), 0, st, p); \
  else hipLaunchKernelGGL(quantize_squares_kernel<TAG>, squares_grid, dim3(256), 0, st, p);
  if (dtype == DL_F32) { DL_QUANTIZE(TagF32) } else if (dtype == DL_BF16) { DL_QUANTIZE(TagBF16) } else { DL_QUANTIZE(TagF16) }
#undef DL_QUANTIZE
  return blocks_status();
}

extern "C" int dl_matmul_blocks(const void* a, int64_t a_stride, const float* a_scale, int64_t a_scale_row, int64_t a_scale_block, int64_t M,
                                const void* b, int64_t b_stride, const float* b_scale, int64_t b_scale_row, int64_t b_scale_block, int64_t N,
                                int64_t K, void* out, int out_dtype, int64_t out_stride, void* stream) {
  using namespace dl;
  if ((unsigned)out_dtype > DL_F16) return DL_ERR_DTYPE;
  const int64_t blocks = (K + QB - 1) / QB;
  if (M < 0 || N < 0 || K <= 0 || a_stride < blocks * QB || b_stride < blocks * QB || out_stride < N || a_scale_row < 0 || a_scale_block < 0 ||
      b_scale_row < 0 || b_scale_block < 0)
    return DL_ERR_SHAPE;
  if (M == 0 || N == 0) return DL_OK;
  if (!a || !b || !a_scale || !b_scale || !out) return DL_ERR_NULL;
  if ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) % 16 || a_stride % 16 || b_stride % 16 ||
      (reinterpret_cast<uintptr_t>(a_scale) | reinterpret_cast<uintptr_t>(b_scale)) % 4 || reinterpret_cast<uintptr_t>(out) % (out_dtype == DL_F32 ? 4 : 2))
    return DL_ERR_ALIGN;
  if (blocks > 0xffffff || (N + 31) / 32 > 0x7fffffffLL) return DL_ERR_LIMIT;
  const BlocksParams p{reinterpret_cast<const unsigned char*>(a), a_stride, a_scale, a_scale_row, a_scale_block, M,
                       reinterpret_cast<const unsigned char*>(b), b_stride, b_scale, b_scale_row, b_scale_block, N, (int)blocks,
                       reinterpret_cast<char*>(out), out_stride};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (out_dtype == DL_F32) return launch_blocks<TagF32>(p, st);
  if (out_dtype == DL_BF16) return launch_blocks<TagBF16>(p, st);
  return launch_blocks<TagF16>(p, st);
}
