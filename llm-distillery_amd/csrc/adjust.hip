// Logits made ready for the sampler, and the gradient of that.
//
//   y = x > 0 ? x / repetition : x * repetition          for the tokens of the row's text
//   y -= frequency * count + presence                    for those behind the text's prompt, `count` times there
//   y += bias;   y = -inf where the row's mask has no bit
//
// A workgroup has a row, or a part of its columns.  A text's tokens are few among these and the row's bytes are what has to move, so nothing is
// done for a column that the text does not have: the tokens set a bit for their column in LDS, and count themselves (whole numbers: the order of the
// additions does not show); the columns go from registers to memory in 16-byte pieces, by way of LDS where a piece has a bit: the thread puts its
// pieces there, works on the elements whose bits are set, one after the other, and takes the pieces back.  Masked ones are taken out by a few bit
// selects.  Nothing is unpacked unless there is a bias.  Texts are asked for first and the row behind them, so that its loads are under way while
// tokens are counted; what a mask takes out throughout is not read.
// The gradient (by x: g over or times the repetition at the text's tokens; by a bias that the rows share: the sum of g over the rows; both 0
// where the mask has no bit) goes the same way; of x it reads the pieces with a bit alone.
//
// Bound by HBM where there are rows enough: 4096 x 50257 fp32, 512-token texts, a shared bias, 303 us (1.65 GB: 5.4 TB/s); 256 x 128256 bf16, texts of
// 4096, masks that allow 30 %, 29 us (134 MB: 4.6 TB/s, the first tokens and the last pieces with nothing beside them); 8192 x 128256 bf16 with a bias's
// gradient 950 us (4.2 GB, 0.2 of logits at the texts' tokens, 0.13 of sums: 4.8 TB/s).  One row of 32000 takes 4.6 us, the depth of its loads.  Tried at
// the second of these: the penalty computed in all columns and selected 54 us, a list of the text's columns that were claimed, gathered and scattered 70 (texts of
// 16384: 1036 against 290), new values picked into registers by comparisons 34, 512 or 1024 threads with one or two pieces each level to 35.  Several rows
// a workgroup for texts that rows share, so that a row adds only its own tokens' bits, is slower (the third 874 to 992 traced, without
// 846, both with totals in 32 bits): a workgroup that goes on to another row waits for the stores of the row before.
#include "distill_common.hpp"
#include "distill_hip.h"

#include <algorithm>

namespace dl {

struct AdjustParams {
  const char* x; int64_t x_stride;
  const char* g; int64_t g_stride;                             // the gradient's kernels
  char* out; int64_t out_stride;
  int64_t n_rows, V;
  const char* tokens; int itype; int64_t token_stride, n_texts, length;
  const int32_t *token_rows, *lengths, *prompt; int prompt_all;
  const float *repetition, *frequency, *presence; float repetition_all, frequency_all, presence_all;
  const char* bias; int bias_dtype; int64_t bias_stride;
  const unsigned* allowed; int64_t allowed_stride, n_masks; const int32_t* allowed_rows;
  unsigned parts, part_columns;
  int64_t first_row, first_run, runs;                          // of a launch; every `runs`-th pair of rows is a workgroup's (SUMS)
};

// What a row has besides its logits.  A lane fetches one of its settings each, so that they take one trip to memory; the same in all waves.
struct AdjustRow {
  const char* text;
  int length, prompt;                                          // entries that count, and how many of them are the prompt's
  float repetition, inverse, frequency, presence;
  const unsigned char* bits;                                   // its mask, or nothing
  __device__ __forceinline__ AdjustRow(const AdjustParams& p, int64_t r) {
    const void* const settings[7] = {p.repetition, p.frequency, p.presence, p.token_rows, p.lengths, p.prompt, p.allowed_rows};
    const int lane = threadIdx.x & (WAVE - 1);
    const void* mine = nullptr;
#pragma unroll
    for (int k = 0; k < 7; ++k) mine = lane == k ? settings[k] : mine;
    int got = 0;
    if (mine) got = reinterpret_cast<const int*>(mine)[r];
    const auto number = [&](int k) { return __builtin_amdgcn_readlane(got, k); };
    repetition = p.repetition ? __int_as_float(number(0)) : p.repetition_all;
    frequency = p.frequency ? __int_as_float(number(1)) : p.frequency_all;
    presence = p.presence ? __int_as_float(number(2)) : p.presence_all;
    int64_t t = p.token_rows ? (int64_t)number(3) : p.n_texts == 1 ? 0 : r;
    length = p.lengths ? min(number(4), (int)p.length) : (int)p.length;
    prompt = p.prompt ? number(5) : p.prompt_all;
    if (t < 0 || t >= p.n_texts || length < 0 || (repetition == 1.f && frequency == 0.f && presence == 0.f)) t = length = 0;
    text = p.tokens + t * p.token_stride * (p.itype == I64 ? 8 : 4);
    const int64_t m = p.allowed_rows ? (int64_t)number(6) : p.n_masks == 1 ? 0 : r;
    bits = m >= 0 && m < p.n_masks ? reinterpret_cast<const unsigned char*>(p.allowed + m * p.allowed_stride) : nullptr;
    inverse = 1.f / repetition;
  }
  // f / repetition, rounded once: a product with the rounded reciprocal, and what it is off by taken off (the remainder is exact).  Where the product is no
  // number or infinite, it is the quotient; so far from 1 that the reciprocal loses bits, a division.
  __device__ __forceinline__ float quotient(float f) const {
    if (!(repetition >= 0x1p-64f && repetition <= 0x1p64f)) return f / repetition;
    const float q = f * inverse, better = fmaf(fmaf(-q, repetition, f), inverse, q);
    return fabsf(q) <= 3.402823466e38f ? better : q;
  }
};

// `yes` where the element's bit is set, else `no`.
template <class Tag>
__device__ __forceinline__ u32x4 select_bits(unsigned bits, const u32x4& yes, const u32x4& no) {
  u32x4 v;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    unsigned m;
    if constexpr (Tag::bytes == 4) m = (unsigned)__builtin_amdgcn_sbfe((int)bits, k, 1);
    else m = ((unsigned)__builtin_amdgcn_sbfe((int)bits, 2 * k, 1) & 0xffffu) | ((unsigned)__builtin_amdgcn_sbfe((int)bits, 2 * k + 1, 1) & 0xffff0000u);
    v[k] = (yes[k] & m) | (no[k] & ~m);
  }
  return v;
}
// The bits of a 16-byte piece's elements, its first at column `col` (a multiple of as many).
template <class Tag>
__device__ __forceinline__ unsigned piece_bits(const unsigned char* bits, unsigned col) {
  return Tag::bytes == 2 ? bits[col >> 3] : (bits[col >> 3] >> (col & 4)) & 15u;
}

// Four neighbouring tokens of a text, as they lie there.
template <class Index>
struct FourTokens {
  u32x4 v[sizeof(Index) / 4];
  __device__ __forceinline__ void load(const char* text, int first) {
#pragma unroll
    for (int k = 0; k < (int)sizeof(Index) / 4; ++k) v[k] = load16_unaligned(text + (int64_t)first * (int)sizeof(Index) + k * 16);
  }
  // No id of 32 bits: 2^32 - 1.
  __device__ __forceinline__ unsigned get(int e) const {
    if constexpr (sizeof(Index) == 4) return v[0][e];
    else return v[e / 2][e % 2 * 2 + 1] ? ~0u : v[e / 2][e % 2 * 2];
  }
};
// A text's places are 32-bit numbers, and a workgroup's last step passes its end by less than STEP_MOST, the most tokens of a step: beyond LENGTH_MOST
// tokens that would pass 2^31 - 1.
constexpr int STEP_MOST = 8192;
constexpr int64_t LENGTH_MOST = (1LL << 31) - STEP_MOST;
__device__ const unsigned NOTHING[4] = {0u, 0u, 0u, 0u};       // in the place of a row too short for a piece
typedef double f64x2 __attribute__((ext_vector_type(2)));
typedef const char __attribute__((address_space(1))) * global_bytes;      // (said to be global, so that a choice of two is no load of any kind of memory)

// A part of the columns of a row, or (SUMS, the gradient's) of a run of rows, one after the other: what these have in common, the gradient by a shared bias,
// is added up on the way, one row of `sums` for every run, in fp64: what shows is the result's rounding, and a sum on the way may be larger than fp32 holds.
// A run is every so many-th pair of rows: the texts of neighbouring rows are of a length, those of runs of neighbours would not be (4096 x 50257 fp32,
// texts of 2048, 400 us, so 429); a pair shares the line in which one row ends and the next begins (8192 x 50257 bf16 472 us, single rows 552).
// Count: what a column's counter is held in, 16 bits where no text has more tokens than these count.
// 16 KiB of a row a workgroup, four 16-byte pieces a thread; LDS and registers leave room for four such workgroups on a CU (asked for six or eight, values
// spill; two-byte logits to be adjusted by 64-bit tokens hold 12 or 16 bytes a thread in scratch as it is).  The totals of two-byte rows, 64 registers, do
// not fit beside the rest: those of a thread's last piece are in LDS.
template <class Tag, class Index, int NT, int NCH, class Count, bool GRAD, bool SUMS>
__global__ __launch_bounds__(NT, 4) void adjust_kernel(const AdjustParams p, double* sums) {
  constexpr int N = Chunk<Tag>::N, B = Tag::bytes, NTOK = SUMS ? 1 : 2;      // (tokens of a thread at a time: four times NTOK)
  static_assert(NT * NTOK * 4 <= STEP_MOST, "places of 32 bits");
  constexpr int KEPT = SUMS && B == 2 ? NCH - 1 : NCH;         // pieces whose totals are in registers
  constexpr bool SIGNS = KEPT < NCH;                           // (which leaves no room for the logits in LDS: a bit of a register each)
  extern __shared__ __align__(16) unsigned all_lds[];          // the other totals; for each column a bit, its new value, and a counter or (GRAD) the logit
  f64x2* const last_totals = reinterpret_cast<f64x2*>(all_lds) + threadIdx.x;      // this thread's, NT apart
  unsigned* const lds = all_lds + (KEPT < NCH ? NT * N * 2 : 0);
  const unsigned group = blockIdx.x / (8u * p.parts), in = blockIdx.x % (8u * p.parts);      // the parts of a run on one XCD
  const int64_t k = (int64_t)group * 8 + (in & 7u), first = p.first_row + (SUMS ? 2 * k : k), last = SUMS ? p.n_rows : min(first + 1, p.n_rows);
  const int64_t c0 = (int64_t)(in >> 3) * p.part_columns;
  if (k >= p.runs || c0 >= p.V) return;                        // (parts are whole blocks of 128 columns: the last may be none)
  // a wave's pieces are neighbours, NCH KiB of them: all of a thread's lie within the offset of an instruction
  const unsigned tid = threadIdx.x, place = tid / WAVE * (WAVE * NCH) + tid % WAVE;
  const unsigned columns = (unsigned)min((int64_t)p.part_columns, p.V - c0), pieces = columns / N, tail = columns % N;
  const unsigned char* said = reinterpret_cast<const unsigned char*>(lds);
  char* values = reinterpret_cast<char*>(lds + p.part_columns / 32);
  char* beside = values + p.part_columns * B;
  unsigned* counts = reinterpret_cast<unsigned*>(beside);
  const u32x4 masked = GRAD ? u32x4{0u, 0u, 0u, 0u} : Chunk<Tag>::neg_inf();
  double total[SUMS ? KEPT : 1][N] = {}, total_tail = 0.0;
  if (KEPT < NCH)
#pragma unroll
    for (int e = 0; e < N; e += 2) last_totals[e / 2 * NT] = f64x2{0.0, 0.0};
#pragma unroll 1
  for (int64_t r = first; r < last; r += (SUMS && (r & 1)) ? 2 * p.runs - 1 : 1) {
    unsigned mine = place;
    if (SUMS) asm("" : "+v"(mine) : "s"((int)r));              // (said to change: offsets made from it would take registers from row to row, and spill)
    const AdjustRow row(p, r);
    const char* from = (GRAD ? p.g + (r * p.g_stride + c0) * B : p.x + (r * p.x_stride + c0) * B);
    const char* x = p.x + (r * p.x_stride + c0) * B;
    char* to = p.out + (r * p.out_stride + c0) * B;
    const char* bias = GRAD || !p.bias ? nullptr : p.bias + (r * p.bias_stride + c0) * (p.bias_dtype == F32 ? 4 : 2);
    const unsigned char* bits = row.bits ? row.bits + (c0 >> 3) : nullptr;      // (a part begins at a whole word)
    const int length = row.length, prompt = row.prompt;
    const bool counted = !GRAD && (row.frequency != 0.f || row.presence != 0.f);
    // (All loads are made, those that nobody needs from the part's or the text's beginning: a load that is branched around is waited for before
    // the next one.)
    FourTokens<Index> t[NTOK];
    u32x4 v[NCH];
    unsigned m[NCH];
    const auto fetch = [&](int at) {                           // a thread's tokens from `at` on; the text's last four where there are less
#pragma unroll
      for (int i = 0; i < NTOK; ++i) t[i].load(row.text, min(at + (i * NT + (int)tid) * 4, length - 4));
    };
    if (length >= 4) fetch(0);
#pragma unroll
    for (int i = 0; i < NCH; ++i) m[i] = 255u;
    if (bits && pieces) {
#pragma unroll
      for (int i = 0; i < NCH; ++i) m[i] = piece_bits<Tag>(bits, (mine + i * WAVE < pieces ? mine + i * WAVE : 0u) * N);
    }
    const global_bytes whole = pieces ? (global_bytes)from : (global_bytes) reinterpret_cast<const char*>(NOTHING);
#pragma unroll
    for (int i = 0; i < NCH; ++i) v[i] = __builtin_nontemporal_load((const u32x4_on_2 __attribute__((address_space(1)))*)(whole + (mine + i * WAVE < pieces && m[i] ? mine + i * WAVE : 0u) * 16u));
    if (length > 0) {
      for (unsigned i = tid; i < p.part_columns / 128; i += NT) reinterpret_cast<u32x4*>(lds)[i] = u32x4{0u, 0u, 0u, 0u};
      if (counted)
        for (unsigned i = tid; i < p.part_columns * (unsigned)sizeof(Count) / 16; i += NT) reinterpret_cast<u32x4*>(counts)[i] = u32x4{0u, 0u, 0u, 0u};
      __syncthreads();
      const auto take = [&](unsigned token, int i) {
        const unsigned c = token - (unsigned)c0;               // (no id: beyond any part)
        if (c >= columns) return;
        atomicOr(&lds[c >> 5], 1u << (c & 31u));
        if (counted && i >= prompt) atomicAdd(&counts[c * sizeof(Count) / 4], 1u << (sizeof(Count) == 4 ? 0u : (c & 1u) * 16u));
      };
      if (length < 4 && (int)tid < length) {
        const Index token = reinterpret_cast<const Index*>(row.text)[tid];
        if (token >= 0 && token <= 0x7fffffff) take((unsigned)token, (int)tid);
      }
#pragma unroll 1
      for (int at = 0; length >= 4;) {
#pragma unroll
        for (int i = 0; i < NTOK; ++i) {
          const int own = at + (i * NT + (int)tid) * 4, first_token = min(own, length - 4);      // (what is ahead of its own is another thread's)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (first_token + e >= own) take(t[i].get(e), first_token + e);
        }
        at += NTOK * NT * 4;
        if (at >= length) break;
        fetch(at);
      }
      __syncthreads();
    }
    if (GRAD)
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        if (bits) v[i] = select_bits<Tag>(m[i], v[i], masked);
        if (SUMS) {
          float f[N];
          Chunk<Tag>::unpack(v[i], f);
#pragma unroll
          for (int e = 0; e < N; e += 2) {
            const f64x2 more = {(double)f[e], (double)f[e + 1]};
            if (i < KEPT) {
              total[i < KEPT ? i : 0][e] += more[0];
              total[i < KEPT ? i : 0][e + 1] += more[1];
            } else {
              last_totals[e / 2 * NT] += more;
            }
          }
        }
      }
    const auto penalised = [&](float f, float sign, unsigned col) {
      f = sign > 0.f ? row.quotient(f) : f * row.repetition;
      if (counted) {
        const unsigned n = reinterpret_cast<const Count*>(counts)[col];
        if (n) f -= row.frequency * (float)n + row.presence;
      }
      return f;
    };
    constexpr bool OVER = B == 2;                              // (two-byte values with a bias: the sum is rounded, not the penalised value)
    unsigned c[NCH], left = 0u, positive = 0u;                 // (bits of the text's elements; SIGNS: of these the ones with a logit above 0)
    if (length > 0 && (!SUMS || p.out)) {
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        c[i] = mine + i * WAVE < pieces ? piece_bits<Tag>(said, (mine + i * WAVE) * N) & m[i] : 0u;      // (no work on masked ones)
        left |= c[i] << (i * N);
      }
      if (GRAD && pieces) {
        u32x4 xs[NCH];
#pragma unroll
        for (int i = 0; i < NCH; ++i) xs[i] = load16_unaligned(x + (c[i] ? mine + i * WAVE : 0u) * 16u);
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
          if (!c[i]) continue;
          if (!SIGNS) {
            *reinterpret_cast<u32x4*>(beside + (mine + i * WAVE) * 16u) = xs[i];
            continue;
          }
          float f[N];
          Chunk<Tag>::unpack(xs[i], f);
#pragma unroll
          for (int e = 0; e < N; ++e) positive |= (f[e] > 0.f ? 1u : 0u) << (i * N + e);
        }
      }
#pragma unroll
      for (int i = 0; i < NCH; ++i)
        if (c[i]) *reinterpret_cast<u32x4*>(values + (mine + i * WAVE) * 16u) = v[i];
#pragma unroll 1
      for (; left; left &= left - 1u) {
        const unsigned e = (unsigned)__builtin_ctz(left), col = (mine + e / N * WAVE) * N + e % N;
        const float f = load_as_float(values, Tag::id, col);
        float y = penalised(f, SIGNS ? (float)(positive >> e & 1u) : GRAD ? load_as_float(beside, Tag::id, col) : f, col);
        if (!GRAD && OVER && bias) y += load_as_float(bias, p.bias_dtype, col);
        store_from_float(values, Tag::id, col, y);
      }
#pragma unroll
      for (int i = 0; i < NCH; ++i)
        if (c[i] && !(OVER && bias)) v[i] = *reinterpret_cast<const u32x4*>(values + (mine + i * WAVE) * 16u);
    }
    if (!GRAD && bias && pieces) {
      const auto add = [&](int i, const float* a) {
        float f[N];
        Chunk<Tag>::unpack(v[i], f);
#pragma unroll
        for (int e = 0; e < N; ++e) f[e] += a[e];
        v[i] = Chunk<Tag>::pack(f);
        if (OVER && length > 0 && c[i]) v[i] = select_bits<Tag>(c[i], *reinterpret_cast<const u32x4*>(values + (mine + i * WAVE) * 16u), v[i]);
      };
      const auto place = [&](int i) { return (mine + i * WAVE < pieces ? mine + i * WAVE : 0u) * 16u; };
      if (OVER && p.bias_dtype == F32) {
        u32x4 a[NCH][2];
#pragma unroll
        for (int i = 0; i < NCH; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h) a[i][h] = load16_unaligned(bias + place(i) * 2u + h * 16);
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
          float f[8];
          Chunk<TagF32>::unpack(a[i][0], f);
          Chunk<TagF32>::unpack(a[i][1], f + 4);
          add(i, f);
        }
      } else {
        u32x4 a[NCH];
#pragma unroll
        for (int i = 0; i < NCH; ++i) a[i] = load16_unaligned(bias + place(i));
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
          float f[N];
          Chunk<Tag>::unpack(a[i], f);
          add(i, f);
        }
      }
    }
    if (!GRAD && bits) {
#pragma unroll
      for (int i = 0; i < NCH; ++i) v[i] = select_bits<Tag>(m[i], v[i], masked);
    }
    if (!SUMS || p.out) {
#pragma unroll
      for (int i = 0; i < NCH; ++i)
        if (mine + i * WAVE < pieces) store16_stream_any(to + (mine + i * WAVE) * 16u, v[i]);
    }
    if (tid < tail) {                                          // the columns behind the last whole piece
      const unsigned at = pieces * N + tid;
      const bool open = !bits || (bits[at >> 3] >> (at & 7u) & 1u);
      float f = open ? load_as_float(from, Tag::id, at) : 0.f;
      if (SUMS) total_tail += (double)f;
      if (!SUMS || p.out) {
        if (length > 0 && open && (said[at >> 3] >> (at & 7u) & 1u)) f = penalised(f, GRAD ? load_as_float(x, Tag::id, at) : f, at);
        if (!GRAD && bias) f += load_as_float(bias, p.bias_dtype, at);
        store_from_float(to, Tag::id, at, GRAD || open ? f : -__builtin_inff());
      }
    }
    if (SUMS && length > 0) __syncthreads();                   // the bits are the next row's
  }
  if (SUMS) {
    double* at = sums + (p.first_run + k) * p.V + c0;
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (place + i * WAVE < pieces) at[(place + i * WAVE) * N + e] = i < KEPT ? total[i < KEPT ? i : 0][e] : last_totals[e / 2 * NT][e % 2];
    if (tid < tail) at[pieces * N + tid] = total_tail;
  }
}

// The runs' sums, added up in fp64: 32 columns a workgroup, from `first` on, eight threads to a column, each every eighth run.
__global__ __launch_bounds__(256) void bias_join_kernel(const double* sums, int64_t runs, int64_t first, int64_t V, void* out, int dtype) {
  __shared__ double part[8][32];
  const int lane = threadIdx.x % 32, slice = threadIdx.x / 32;
  const int64_t col = first + (int64_t)blockIdx.x * 32 + lane;
  double total = 0.0;
  if (col < V)
    for (int64_t k = slice; k < runs; k += 8) total += sums[k * V + col];
  part[slice][lane] = total;
  __syncthreads();
  if (slice == 0 && col < V) {
#pragma unroll
    for (int s = 1; s < 8; ++s) total += part[s][lane];
    store_from_float(out, dtype, col, (float)total);
  }
}

static int adjust_status() { return hipGetLastError() == hipSuccess ? DL_OK : DL_ERR_LAUNCH; }

constexpr int ADJUST_NT = 256, ADJUST_NCH = 4;
constexpr int SUMS_NT = 1024;

// What a call that adds up rows is cut into: whether its workgroups are the large ones, and the rows whose sum goes to the workspace in one piece.
// Rows enough whose columns fill the parts of 1024 threads take these, which go through a text less often (8192 x 128256 bf16, texts of 8192, 1113 us, with
// 256 threads 1291; 4096 x 128256 fp32 793, 813), not few rows (512 x 128256 bf16 86, 83) or parts three quarters full (8192 x 50257 bf16 542, 479).  Runs are as long as
// leaves every CU its workgroups, all at once: 8192 x 128256 bf16 943 us, in two rounds of workgroups 965, in four 1025, of their bytes more and more sums.
struct SumsCut {
  bool wide;
  int64_t run;
  SumsCut(int64_t n_rows, int64_t V, int bytes) {
    const int64_t most = (int64_t)SUMS_NT * ADJUST_NCH * 16 / bytes;
    wide = n_rows >= 2048 && V * 10 >= (V + most - 1) / most * most * 9;
    const int64_t columns = wide ? most : most / SUMS_NT * ADJUST_NT, parts = (V + columns - 1) / columns;
    const int64_t runs = 8 * std::max<int64_t>(1, 32 * (wide ? 1 : 4) / parts);      // (an XCD has all parts of a run, and 32 CUs)
    run = std::max<int64_t>(4, (n_rows + 2 * runs - 1) / (2 * runs) * 2);
  }
  int64_t runs(int64_t n_rows) const { return (n_rows + run - 1) / run; }
};

template <class Tag, class Index, int NT, class Count, bool GRAD, bool SUMS>
static void launch_adjust(AdjustParams p, double* sums, hipStream_t st) {
  constexpr int64_t most = (int64_t)NT * ADJUST_NCH * Chunk<Tag>::N;
  p.parts = (unsigned)((p.V + most - 1) / most);
  p.part_columns = (unsigned)std::min<int64_t>(most, ((p.V + p.parts - 1) / p.parts + 127) / 128 * 128);      // (whole words of the masks, whole pieces of the bits)
  const int64_t run = SUMS ? SumsCut(p.n_rows, p.V, Tag::bytes).run : 1;
  constexpr bool SIGNS = SUMS && Tag::bytes == 2;
  constexpr size_t beside = SIGNS ? 0 : GRAD ? (size_t)Tag::bytes : sizeof(Count);
  const size_t lds = (SIGNS ? NT * 64 : 0) + (p.length > 0 ? p.part_columns / 8 + p.part_columns * (Tag::bytes + beside) : 0);
  if (NT * ADJUST_NCH * 16 > 32768 && lds > 65536 &&
      hipFuncSetAttribute(reinterpret_cast<const void*>(&adjust_kernel<Tag, Index, NT, ADJUST_NCH, Count, GRAD, SUMS>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess)
    return;                                                    // (the error is the launch's)
  const int64_t slice = LAUNCH_THREADS / NT / p.parts / 8 * 8 * run, all = p.n_rows;      // rows of a launch
  for (p.first_row = 0; p.first_row < all; p.first_row += slice) {
    p.n_rows = std::min(all, p.first_row + slice);
    p.first_run = p.first_row / run;
    p.runs = (p.n_rows - p.first_row + run - 1) / run;
    hipLaunchKernelGGL((adjust_kernel<Tag, Index, NT, ADJUST_NCH, Count, GRAD, SUMS>), dim3((unsigned)((p.runs + 7) / 8 * 8) * p.parts), dim3(NT), lds, st, p, sums);
  }
}
template <class Tag, class Index, bool GRAD, bool SUMS>
static void adjust_texts(const AdjustParams& p, double* sums, hipStream_t st) {
  if constexpr (SUMS)
    if (SumsCut(p.n_rows, p.V, Tag::bytes).wide) return launch_adjust<Tag, Index, SUMS_NT, unsigned short, GRAD, SUMS>(p, sums, st);
  if constexpr (!GRAD)
    if (p.length > 65535) return launch_adjust<Tag, Index, ADJUST_NT, unsigned, GRAD, SUMS>(p, sums, st);
  launch_adjust<Tag, Index, ADJUST_NT, unsigned short, GRAD, SUMS>(p, sums, st);
}
template <class Tag, bool GRAD, bool SUMS>
static void adjust_rows(const AdjustParams& p, double* sums, hipStream_t st) {
  if (p.itype == I64) adjust_texts<Tag, int64_t, GRAD, SUMS>(p, sums, st);
  else adjust_texts<Tag, int32_t, GRAD, SUMS>(p, sums, st);
}
template <bool GRAD, bool SUMS>
static void adjust_rows(const AdjustParams& p, int dtype, double* sums, hipStream_t st) {
  if (dtype == DL_F32) adjust_rows<TagF32, GRAD, SUMS>(p, sums, st);
  else if (dtype == DL_BF16) adjust_rows<TagBF16, GRAD, SUMS>(p, sums, st);
  else adjust_rows<TagF16, GRAD, SUMS>(p, sums, st);
}

// What both entry points ask of their common arguments.
static int adjust_check(const AdjustParams& p, int dtype) {
  if (p.n_rows < 0 || p.V < 0 || p.x_stride < p.V || p.out_stride < p.V || p.n_texts < 0 || p.length < 0 || p.n_masks < 0) return DL_ERR_SHAPE;
  if (p.n_texts > 0 && (p.token_stride < 0 || (p.n_texts > 1 && !p.token_rows && p.n_texts < p.n_rows))) return DL_ERR_SHAPE;
  if (p.n_masks > 0 && (p.allowed_stride < (p.V + 31) / 32 || (p.n_masks > 1 && !p.allowed_rows && p.n_masks < p.n_rows))) return DL_ERR_SHAPE;
  if (p.bias && p.bias_stride != 0 && p.bias_stride < p.V) return DL_ERR_SHAPE;
  if (p.V > 0x7fffffffLL || p.length > LENGTH_MOST) return DL_ERR_LIMIT;
  const uintptr_t eb = dtype == DL_F32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.out)) % eb || reinterpret_cast<uintptr_t>(p.tokens) % (p.itype == I64 ? 8 : 4) ||
      reinterpret_cast<uintptr_t>(p.allowed) % 4 || reinterpret_cast<uintptr_t>(p.bias) % (p.bias_dtype == F32 ? 4 : 2))
    return DL_ERR_ALIGN;
  return DL_OK;
}

}  // namespace dl

extern "C" int dl_adjust_rows(const void* logits, int dtype, int64_t row_stride, int64_t n_rows, int64_t V, const void* tokens, int itype,
                              int64_t token_stride, int64_t n_texts, int64_t length, const int32_t* token_rows, const int32_t* lengths,
                              const int32_t* prompt, int64_t prompt_all, const float* repetition, const float* frequency, const float* presence,
                              float repetition_all, float frequency_all, float presence_all, const void* bias, int bias_dtype, int64_t bias_stride,
                              const int32_t* allowed, int64_t allowed_stride, int64_t n_masks, const int32_t* allowed_rows, void* out,
                              int64_t out_stride, void* stream) {
  using namespace dl;
  if ((unsigned)dtype > DL_F16 || (unsigned)itype > DL_I64 || (bias && bias_dtype != DL_F32 && bias_dtype != dtype)) return DL_ERR_DTYPE;
  if (!tokens) n_texts = length = 0;
  if (!allowed) n_masks = 0;
  AdjustParams p{reinterpret_cast<const char*>(logits), row_stride, nullptr, 0, reinterpret_cast<char*>(out), out_stride, n_rows, V,
                 reinterpret_cast<const char*>(tokens), itype, token_stride, n_texts, n_texts ? length : 0, token_rows, lengths, prompt, (int)std::max<int64_t>(0, std::min<int64_t>(prompt_all, 0x7fffffff)),
                 repetition, frequency, presence, repetition_all, frequency_all, presence_all,
                 reinterpret_cast<const char*>(bias), bias_dtype, bias_stride,
                 reinterpret_cast<const unsigned*>(allowed), allowed_stride, n_masks, allowed_rows, 0, 0, 0, 0, 0};
  if (const int bad = adjust_check(p, dtype)) return bad;
  if (n_rows == 0 || V == 0) return DL_OK;
  if (!logits || !out) return DL_ERR_NULL;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  adjust_rows<false, false>(p, dtype, nullptr, st);
  return adjust_status();
}

extern "C" int64_t dl_adjust_grad_workspace_bytes(int64_t n_rows, int64_t V) {
  if (n_rows <= 0 || V <= 0) return 0;
  return std::max(dl::SumsCut(n_rows, V, 2).runs(n_rows), dl::SumsCut(n_rows, V, 4).runs(n_rows)) * V * 8;      // (of either width)
}

extern "C" int dl_adjust_grad(const void* grad, int dtype, int64_t grad_stride, const void* logits, int64_t row_stride, int64_t n_rows, int64_t V,
                              const void* tokens, int itype, int64_t token_stride, int64_t n_texts, int64_t length, const int32_t* token_rows,
                              const int32_t* lengths, const float* repetition, float repetition_all, const int32_t* allowed,
                              int64_t allowed_stride, int64_t n_masks, const int32_t* allowed_rows, void* out, int64_t out_stride,
                              void* bias_grad, int bias_dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace dl;
  if ((unsigned)dtype > DL_F16 || (unsigned)itype > DL_I64 || (bias_grad && bias_dtype != DL_F32 && bias_dtype != dtype)) return DL_ERR_DTYPE;
  if (!tokens) n_texts = length = 0;
  if (!allowed) n_masks = 0;
  if (!logits) row_stride = V;
  if (!out) out_stride = V;
  AdjustParams p{reinterpret_cast<const char*>(logits), row_stride, reinterpret_cast<const char*>(grad), grad_stride, reinterpret_cast<char*>(out), out_stride, n_rows, V,
                 reinterpret_cast<const char*>(tokens), itype, token_stride, n_texts, n_texts ? length : 0, token_rows, lengths, nullptr, 0,
                 repetition, nullptr, nullptr, repetition_all, 0.f, 0.f, nullptr, F32, 0,
                 reinterpret_cast<const unsigned*>(allowed), allowed_stride, n_masks, allowed_rows, 0, 0, 0, 0, 0};
  if (grad_stride < V) return DL_ERR_SHAPE;
  if (const int bad = adjust_check(p, dtype)) return bad;
  if (V == 0 || (n_rows == 0 && !bias_grad)) return DL_OK;
  if ((n_rows > 0 && !grad) || (out && p.length > 0 && !logits)) return DL_ERR_NULL;
  const uintptr_t eb = dtype == DL_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(grad) % eb || reinterpret_cast<uintptr_t>(bias_grad) % (bias_dtype == DL_F32 ? 4 : 2) || reinterpret_cast<uintptr_t>(workspace) % 16)
    return DL_ERR_ALIGN;
  if (bias_grad && n_rows > 0 && (!workspace || workspace_bytes < dl_adjust_grad_workspace_bytes(n_rows, V))) return DL_ERR_WORKSPACE;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (!bias_grad) {
    if (out) adjust_rows<true, false>(p, dtype, nullptr, st);
    return adjust_status();
  }
  double* sums = reinterpret_cast<double*>(workspace);
  int64_t runs = 0;
  if (n_rows > 0) {
    if (!out) p.length = 0;                                    // the bias does not feel the texts
    adjust_rows<true, true>(p, dtype, sums, st);
    runs = SumsCut(n_rows, V, dtype == DL_F32 ? 4 : 2).runs(n_rows);
  }
  constexpr int64_t MOST = LAUNCH_THREADS / 256 * 32;          // columns of a launch
  for (int64_t col = 0; col < V; col += MOST)
    hipLaunchKernelGGL(bias_join_kernel, dim3((unsigned)((std::min(MOST, V - col) + 31) / 32)), dim3(256), 0, st, sums, runs, col, V, bias_grad, bias_dtype);
  return adjust_status();
}
