// Embedding: rows of a table by token id, scaled, and the gradient of that table.
//
//   out[n, :]  = round(scale * table[token n, :])
//   grad[v, :] = round(scale * sum over {n : token n = v} of g[n, :]  (+ grad[v, :]))
//
// Both move bytes and do next to nothing else.  The lookup reads one table row per token and writes one row.  The
// gradient reads every row of g once and writes every row of the table's gradient once: tokens are sorted (stable, so
// that the rows of a token are summed in ascending order, whatever the launch), the sorted list is cut into tiles of
// equal length, and a tile's workgroup walks its entries with the running sum in registers; a token that crosses tiles
// leaves one fp32 partial sum per tile, which a last launch adds up in tile order.  No float atomics: the same bits
// every time.  A frequent token is spread over as many workgroups as it has tiles.  The rows of the gradient that no
// token names are zeroed by workgroups that ride along in the sorting launches, which would leave the card idle
// otherwise: the sort is a chain of short launches, the zeroes are most of the bytes.
#include "distill_common.hpp"
#include "distill_hip.h"

#include <algorithm>

namespace dl {

// Token n as a row of the table, or -1: outside [0, vocab) (padding).
__device__ __forceinline__ int64_t token_row(const void* tokens, int itype, int64_t n, int64_t vocab) {
  const int64_t t = load_index(tokens, itype, n);
  return t >= 0 && t < vocab ? t : -1;
}

// ---- lookup -----------------------------------------------------------------------------------------
// TPR threads share a row: a wave where there are rows enough to fill the card with waves, else a workgroup.  Table
// rows are read with ordinary loads (frequent tokens then come from L2), the result is streamed out.  Rows may start
// on any element; the columns behind the last whole 16 bytes go one by one.
template <class Tag, int TPR>
__global__ __launch_bounds__(256) void embed_rows_kernel(const char* __restrict__ table, int64_t table_stride, int64_t vocab, int64_t width,
                                                         const void* __restrict__ tokens, int itype, int64_t n_tokens, float scale,
                                                         char* __restrict__ out, int64_t out_stride) {
  using C = Chunk<Tag>;
  const int64_t n = (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
  if (n >= n_tokens) return;
  const int t = threadIdx.x % TPR;
  const int64_t v = token_row(tokens, itype, n, vocab);
  char* o = out + n * out_stride * Tag::bytes;
  const char* s = table + (v < 0 ? 0 : v) * table_stride * Tag::bytes;
  const int64_t whole = width / C::N;
  constexpr int UN = 4;
  for (int64_t c0 = t; c0 < whole; c0 += TPR * UN) {
    u32x4 x[UN];
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      const int64_t c = c0 + i * TPR;
      x[i] = u32x4{0u, 0u, 0u, 0u};
      if (v >= 0 && c < whole) x[i] = load16_unaligned(s + c * 16);
    }
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      const int64_t c = c0 + i * TPR;
      if (c >= whole) break;
      float f[C::N];
      C::unpack(x[i], f);
#pragma unroll
      for (int e = 0; e < C::N; ++e) f[e] = v < 0 ? 0.f : f[e] * scale;      // (0 * an infinite or NaN scale is not 0)
      store16_stream_any(o + c * 16, C::pack(f));
    }
  }
  for (int64_t col = whole * C::N + t; col < width; col += TPR)
    store_from_float(o, Tag::id, col, v < 0 ? 0.f : load_as_float(s, Tag::id, col) * scale);
}

// ---- zeroes that ride along ---------------------------------------------------------------------------
// Bytes [from, to) of a [vocab, width] gradient are zeroed by `blocks` workgroups of a launch.
struct ZeroShare {
  char* base; int64_t pitch_bytes, row_bytes, row0, row1; unsigned blocks;
};
// Workgroup b of z.blocks: whole rows, dealt in turn; 16 bytes per store from the row's first 16-byte boundary on.
__device__ __forceinline__ void zero_rows(const ZeroShare& z, unsigned b) {
  const int tid = threadIdx.x, nt = blockDim.x;
  for (int64_t r = z.row0 + b; r < z.row1; r += z.blocks) {
    char* row = z.base + r * z.pitch_bytes;
    const int64_t head = min((int64_t)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15), z.row_bytes), whole = (z.row_bytes - head) / 16;
    for (int64_t c = tid; c < whole; c += nt) store16_stream(row + head + c * 16, u32x4{0u, 0u, 0u, 0u});
    const int64_t beside = z.row_bytes - whole * 16;          // bytes on either side: whole elements of 2 or 4 bytes
    for (int64_t i = tid * 2; i < beside; i += nt * 2) *reinterpret_cast<unsigned short*>(row + (i < head ? i : whole * 16 + i)) = 0;
  }
}

// ---- sort ---------------------------------------------------------------------------------------------
// A token and its place as one word, token << 32 | n; tokens outside the vocabulary count as id `vocab` and end up
// behind all others.
__device__ __forceinline__ unsigned long long token_word(const void* tokens, int itype, int64_t n, int64_t vocab) {
  const int64_t t = token_row(tokens, itype, n, vocab);
  return ((unsigned long long)(t < 0 ? vocab : t) << 32) | (unsigned)n;
}

constexpr int SORT_SMALL = 1024;      // tokens one workgroup sorts in registers
__global__ __launch_bounds__(1024) void embed_sort_small_kernel(const void* __restrict__ tokens, int itype, int n, int64_t vocab,
                                                                unsigned long long* __restrict__ sorted, ZeroShare z) {
  if (blockIdx.x > 0) return zero_rows(z, blockIdx.x - 1);
  __shared__ unsigned long long xch[SORT_SMALL];
  unsigned long long w[1] = {~0ull};
  if ((int)threadIdx.x < n) w[0] = token_word(tokens, itype, threadIdx.x, vocab);
  block_sort<unsigned long long, 1024, 1>(w, xch);
  if ((int)threadIdx.x < n) sorted[threadIdx.x] = w[0];
}

// Longer lists: a stable sort by digits of `bits` bits, lowest first (two of them up to a million ids).  A pass counts
// each workgroup's digits in one launch and deals its words out in the next, where every workgroup adds up the counts
// ahead of it itself: at most SORT_BLOCKS of them.
constexpr int SORT_NT = 256, SORT_WAVES = SORT_NT / WAVE, SORT_BINS = 1024, SORT_BLOCKS = 64;
struct SortPass {
  const void* tokens; int itype; int64_t vocab;      // the first pass makes its words from the tokens
  const unsigned long long* in;                      // the later ones read them (NULL: the first)
  unsigned long long* out; unsigned* counts;         // counts: [blocks][1 << bits]
  int64_t n, per_block; int shift, bits; unsigned blocks;
};
__device__ __forceinline__ unsigned long long sort_word(const SortPass& s, int64_t i) {
  return s.in ? s.in[i] : token_word(s.tokens, s.itype, i, s.vocab);
}
__device__ __forceinline__ unsigned sort_digit(const SortPass& s, unsigned long long w) {
  return ((unsigned)(w >> 32) >> s.shift) & ((1u << s.bits) - 1u);
}

__global__ __launch_bounds__(SORT_NT) void embed_sort_count_kernel(const SortPass s, const ZeroShare z) {
  if (blockIdx.x >= s.blocks) return zero_rows(z, blockIdx.x - s.blocks);
  __shared__ unsigned h[SORT_BINS];
  const int bins = 1 << s.bits;
  for (int d = threadIdx.x; d < bins; d += SORT_NT) h[d] = 0u;
  __syncthreads();
  const int64_t lo = (int64_t)blockIdx.x * s.per_block, hi = min(s.n, lo + s.per_block);
  for (int64_t i = lo + threadIdx.x; i < hi; i += SORT_NT) atomicAdd(&h[sort_digit(s, sort_word(s, i))], 1u);
  __syncthreads();
  for (int d = threadIdx.x; d < bins; d += SORT_NT) s.counts[(int64_t)blockIdx.x * bins + d] = h[d];
}

__global__ __launch_bounds__(SORT_NT) void embed_sort_deal_kernel(const SortPass s, const ZeroShare z) {
  if (blockIdx.x >= s.blocks) return zero_rows(z, blockIdx.x - s.blocks);
  __shared__ unsigned place[SORT_WAVES][SORT_BINS];      // counts, then the next free place, of a wave's words with a digit
  __shared__ unsigned wave_total[SORT_WAVES];
  const int bins = 1 << s.bits, tid = threadIdx.x, lane = tid & (WAVE - 1), w = tid / WAVE;
  constexpr int EACH = SORT_BINS / SORT_NT;
  // this thread's digits tid * EACH ..: words of all workgroups, words of the workgroups ahead
  unsigned all[EACH], ahead[EACH], mine = 0u;
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    all[j] = ahead[j] = 0u;
    const int d = tid * EACH + j;
    if (d < bins)
      for (unsigned b = 0; b < s.blocks; ++b) {
        const unsigned c = s.counts[(int64_t)b * bins + d];
        all[j] += c;
        if (b < blockIdx.x) ahead[j] += c;
      }
    mine += all[j];
#pragma unroll
    for (int k = 0; k < SORT_WAVES; ++k)
      if (d < SORT_BINS) place[k][d] = 0u;
  }
  unsigned before = mine;                                // exclusive sum over the threads
#pragma unroll
  for (int o = 1; o < WAVE; o <<= 1) {
    const unsigned y = (unsigned)__shfl_up((int)before, o, WAVE);
    if (lane >= o) before += y;
  }
  if (lane == WAVE - 1) wave_total[w] = before;
  before -= mine;
  __syncthreads();
  for (int k = 0; k < w; ++k) before += wave_total[k];
  // every wave owns a contiguous piece of the workgroup's words
  const int64_t lo = (int64_t)blockIdx.x * s.per_block, hi = min(s.n, lo + s.per_block);
  const int64_t piece = (s.per_block + SORT_WAVES - 1) / SORT_WAVES, wlo = min(hi, lo + w * piece), whi = min(hi, wlo + piece);
  for (int64_t i = wlo + lane; i < whi; i += WAVE) atomicAdd(&place[w][sort_digit(s, sort_word(s, i))], 1u);
  __syncthreads();
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    const int d = tid * EACH + j;
    unsigned at = before + ahead[j];
    before += all[j];
#pragma unroll
    for (int k = 0; k < SORT_WAVES; ++k) {
      const unsigned c = place[k][d];
      place[k][d] = at;
      at += c;
    }
  }
  __syncthreads();
  for (int64_t i0 = wlo; i0 < whi; i0 += WAVE) {         // in order: 64 words at a time, equal digits by lane
    const bool live = i0 + lane < whi;
    const unsigned long long word = live ? sort_word(s, i0 + lane) : 0ull;
    const unsigned d = sort_digit(s, word);
    unsigned long long same = __ballot(live);
    for (int b = 0; b < s.bits; ++b) {
      const unsigned long long has = __ballot((d >> b) & 1u);
      same &= ((d >> b) & 1u) ? has : ~has;
    }
    const int rank = __popcll(same & ((1ull << lane) - 1ull));
    const int first = live ? __ffsll((unsigned long long)same) - 1 : lane;
    unsigned at = 0u;
    if (live && rank == 0) at = atomicAdd(&place[w][d], (unsigned)__popcll(same));
    at = (unsigned)__shfl((int)at, first, WAVE);
    if (live) s.out[at + rank] = word;
  }
}

// ---- sums ---------------------------------------------------------------------------------------------
constexpr int SUM_NT = 256, SUM_TILE = 32, SUM_AHEAD = 8;
struct SumParams {
  const unsigned long long* sorted; int64_t n, vocab, width;
  const char* g; int64_t g_stride;
  char* grad; int64_t grad_stride;
  float* partial;                  // [tiles][2][width]: the sum of a tile's first token (if it began earlier), of its last (if it goes on)
  float scale; unsigned slices;
};
__device__ __forceinline__ unsigned word_token(unsigned long long w) { return (unsigned)(w >> 32); }

template <class Tag>
__device__ __forceinline__ void load_columns(const char* row, int64_t col, int n, float* f) {      // n of Chunk<Tag>::N columns, zeros behind
  if (n == Chunk<Tag>::N) {
    Chunk<Tag>::unpack(load16_unaligned(row + col * Tag::bytes), f);
  } else {
#pragma unroll
    for (int e = 0; e < Chunk<Tag>::N; ++e) f[e] = e < n ? load_as_float(row, Tag::id, col + e) : 0.f;
  }
}
// The N sums of columns [col, col + n) to the gradient's row, `scale` times, onto what it holds where ADD.
template <class TagO, int N, bool ADD>
__device__ __forceinline__ void store_sum(char* row, int64_t col, int n, float scale, const float* sum) {
  using C = Chunk<TagO>;
#pragma unroll
  for (int k = 0; k < N / C::N; ++k) {
    const int have = min(max(n - k * C::N, 0), C::N);
    float old[C::N], f[C::N];
    if (ADD) load_columns<TagO>(row, col + k * C::N, have, old);
#pragma unroll
    for (int e = 0; e < C::N; ++e) f[e] = ADD ? fmaf(scale, sum[k * C::N + e], old[e]) : scale * sum[k * C::N + e];
    if (have == C::N) {
      store16_stream_any(row + (col + k * C::N) * TagO::bytes, C::pack(f));
    } else {
#pragma unroll
      for (int e = 0; e < C::N; ++e)
        if (e < have) store_from_float(row, TagO::id, col + k * C::N + e, f[e]);
    }
  }
}

template <class Tag, class TagO, bool ADD>
__global__ __launch_bounds__(SUM_NT) void embed_sum_kernel(const SumParams p) {
  using C = Chunk<Tag>;
  const int64_t tile = blockIdx.x / p.slices, t0 = tile * SUM_TILE;
  const int64_t col = ((int64_t)(blockIdx.x % p.slices) * SUM_NT + threadIdx.x) * C::N;
  const int cols = (int)min((int64_t)C::N, p.width - col);
  __shared__ unsigned long long word[SUM_TILE + 2];      // the tile's, and one on either side (~0: none)
  if (threadIdx.x < SUM_TILE + 2) {
    const int64_t i = t0 - 1 + threadIdx.x;
    word[threadIdx.x] = i >= 0 && i < p.n ? p.sorted[i] : ~0ull;
  }
  __syncthreads();
  if (cols <= 0) return;
  const int count = (int)min((int64_t)SUM_TILE, p.n - t0);
  float sum[C::N];
#pragma unroll
  for (int e = 0; e < C::N; ++e) sum[e] = 0.f;
  bool open = word_token(word[0]) == word_token(word[1]);      // the running token began in an earlier tile
  for (int i0 = 0; i0 < count; i0 += SUM_AHEAD) {
    float f[SUM_AHEAD][C::N];
#pragma unroll
    for (int j = 0; j < SUM_AHEAD; ++j)
      if (i0 + j < count && word_token(word[1 + i0 + j]) < p.vocab)
        load_columns<Tag>(p.g + (int64_t)(unsigned)word[1 + i0 + j] * p.g_stride * Tag::bytes, col, cols, f[j]);
#pragma unroll
    for (int j = 0; j < SUM_AHEAD; ++j) {
      const int i = i0 + j;
      if (i >= count) break;
      const unsigned v = word_token(word[1 + i]);
      if (v >= p.vocab) return;                                // padding: behind all tokens
#pragma unroll
      for (int e = 0; e < C::N; ++e) sum[e] += f[j][e];
      const bool same = word_token(word[2 + i]) == v;
      if (same && i + 1 < count) continue;
      if (!open && !same) {
        store_sum<TagO, C::N, ADD>(p.grad + (int64_t)v * p.grad_stride * TagO::bytes, col, cols, p.scale, sum);
      } else {
        float* part = p.partial + (tile * 2 + (open ? 0 : 1)) * p.width + col;
#pragma unroll
        for (int e = 0; e < C::N; ++e)
          if (e < cols) part[e] = sum[e];
      }
      open = false;
#pragma unroll
      for (int e = 0; e < C::N; ++e) sum[e] = 0.f;
    }
  }
}

// The tokens that cross tiles: the tile in which one begins adds up its partial sums in order.
template <class TagO, bool ADD>
__global__ __launch_bounds__(SUM_NT) void embed_join_kernel(const SumParams p) {
  const int64_t tile = blockIdx.x / p.slices, t0 = tile * SUM_TILE, t1 = t0 + SUM_TILE;
  if (t1 >= p.n) return;
  const unsigned v = word_token(p.sorted[t1 - 1]);
  if (v >= p.vocab || word_token(p.sorted[t1]) != v) return;                                     // ends with the tile
  if (word_token(p.sorted[t0]) == v && t0 > 0 && word_token(p.sorted[t0 - 1]) == v) return;      // began in an earlier one
  // how many further tiles it reaches: the first place behind it, by bisection
  int64_t lo = t1, hi = p.n;                             // sorted[lo] is the token, sorted[hi] is not
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) / 2;
    (word_token(p.sorted[mid]) == v ? lo : hi) = mid;
  }
  const int64_t last = lo / SUM_TILE;
  constexpr int N = 4;
  const int64_t per = (int64_t)p.slices * SUM_NT * N;
  for (int64_t col = ((int64_t)(blockIdx.x % p.slices) * SUM_NT + threadIdx.x) * N; col < p.width; col += per) {
    const int cols = (int)min((int64_t)N, p.width - col);
    float sum[N];
#pragma unroll
    for (int e = 0; e < N; ++e) sum[e] = e < cols ? p.partial[(tile * 2 + 1) * p.width + col + e] : 0.f;
#pragma unroll 4
    for (int64_t t = tile + 1; t <= last; ++t)
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (e < cols) sum[e] += p.partial[t * 2 * p.width + col + e];
    char* row = p.grad + (int64_t)v * p.grad_stride * TagO::bytes;
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (e < cols) store_from_float(row, TagO::id, col + e, ADD ? fmaf(p.scale, sum[e], load_as_float(row, TagO::id, col + e)) : p.scale * sum[e]);
  }
}

static int embed_status() { return hipGetLastError() == hipSuccess ? DL_OK : DL_ERR_LAUNCH; }

template <class Tag, class TagO>
static int launch_sums(const SumParams& s, bool add, hipStream_t st) {
  SumParams p = s;
  const int64_t tiles = (p.n + SUM_TILE - 1) / SUM_TILE;
  p.slices = (unsigned)((p.width + SUM_NT * Chunk<Tag>::N - 1) / (SUM_NT * Chunk<Tag>::N));
  const dim3 grid((unsigned)(tiles * p.slices)), nt(SUM_NT);
  if (add) {
    hipLaunchKernelGGL((embed_sum_kernel<Tag, TagO, true>), grid, nt, 0, st, p);
    if (tiles > 1) hipLaunchKernelGGL((embed_join_kernel<TagO, true>), grid, nt, 0, st, p);
  } else {
    hipLaunchKernelGGL((embed_sum_kernel<Tag, TagO, false>), grid, nt, 0, st, p);
    if (tiles > 1) hipLaunchKernelGGL((embed_join_kernel<TagO, false>), grid, nt, 0, st, p);
  }
  return embed_status();
}

// Places of the workspace, each on a 256-byte boundary: two lists of words, the digit counts, the partial sums.
struct EmbedSpace {
  int64_t words, counts, partial, total;
  EmbedSpace(int64_t n, int64_t width) {
    const auto up = [](int64_t b) { return (b + 255) / 256 * 256; };
    words = up(n * 8);
    counts = n > SORT_SMALL ? up((int64_t)SORT_BLOCKS * SORT_BINS * 4) : 0;
    partial = up((n + SUM_TILE - 1) / SUM_TILE * 2 * width * 4);
    total = 2 * words + counts + partial;
  }
};

}  // namespace dl

extern "C" int dl_embed_rows(const void* table, int dtype, int64_t table_stride, int64_t vocab, int64_t width, const void* tokens, int itype,
                             int64_t n_tokens, float scale, void* out, int64_t out_stride, void* stream) {
  using namespace dl;
  if ((unsigned)dtype > DL_F16 || (unsigned)itype > DL_I64) return DL_ERR_DTYPE;
  if (n_tokens < 0 || vocab < 0 || width < 0 || table_stride < width || out_stride < width) return DL_ERR_SHAPE;
  if (n_tokens == 0 || width == 0) return DL_OK;
  if (!tokens || !out || (vocab > 0 && !table)) return DL_ERR_NULL;
  const uintptr_t eb = dtype == DL_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(table) % eb || reinterpret_cast<uintptr_t>(out) % eb || reinterpret_cast<uintptr_t>(tokens) % (itype == DL_I64 ? 8 : 4))
    return DL_ERR_ALIGN;
  if (n_tokens > 0x7fffffffLL) return DL_ERR_LIMIT;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const char* t = reinterpret_cast<const char*>(table);
  char* o = reinterpret_cast<char*>(out);
  const bool few = n_tokens <= 2048;      // fewer rows than waves: a workgroup each
#define DL_EMBED(TAG)                                                                                                                        \
  if (few) hipLaunchKernelGGL((embed_rows_kernel<TAG, 256>), dim3((unsigned)n_tokens), dim3(256), 0, st, t, table_stride, vocab, width,     \
                              tokens, itype, n_tokens, scale, o, out_stride);                                                                \
  else hipLaunchKernelGGL((embed_rows_kernel<TAG, 64>), dim3((unsigned)((n_tokens + 3) / 4)), dim3(256), 0, st, t, table_stride, vocab,      \
                          width, tokens, itype, n_tokens, scale, o, out_stride);
  if (dtype == DL_F32) { DL_EMBED(TagF32) } else if (dtype == DL_BF16) { DL_EMBED(TagBF16) } else { DL_EMBED(TagF16) }
#undef DL_EMBED
  return embed_status();
}

extern "C" int64_t dl_embed_grad_workspace_bytes(int64_t n_tokens, int64_t width) {
  if (n_tokens <= 0 || width <= 0) return 0;
  return dl::EmbedSpace(n_tokens, width).total;
}

extern "C" int dl_embed_grad(const void* g, int dtype, int64_t g_stride, int64_t n_tokens, int64_t width, const void* tokens, int itype,
                             float scale, int accumulate, void* grad, int grad_dtype, int64_t grad_stride, int64_t vocab, void* workspace,
                             int64_t workspace_bytes, void* stream) {
  using namespace dl;
  if ((unsigned)dtype > DL_F16 || (unsigned)itype > DL_I64 || (grad_dtype != dtype && grad_dtype != DL_F32)) return DL_ERR_DTYPE;
  if (n_tokens < 0 || vocab < 0 || width < 0 || g_stride < width || grad_stride < width) return DL_ERR_SHAPE;
  if (vocab == 0 || width == 0 || (n_tokens == 0 && accumulate)) return DL_OK;
  if (!grad || (n_tokens > 0 && (!g || !tokens))) return DL_ERR_NULL;
  const uintptr_t eb = dtype == DL_F32 ? 4 : 2, ob = grad_dtype == DL_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(g) % eb || reinterpret_cast<uintptr_t>(grad) % ob || reinterpret_cast<uintptr_t>(tokens) % (itype == DL_I64 ? 8 : 4) ||
      reinterpret_cast<uintptr_t>(workspace) % 256)
    return DL_ERR_ALIGN;
  const int64_t slices = (width + SUM_NT * 4 - 1) / (SUM_NT * 4);
  if (n_tokens > 0x7fffffffLL || vocab > 0x7ffffffeLL || (n_tokens / SUM_TILE + 1) * slices > 0x7fffffffLL) return DL_ERR_LIMIT;
  const EmbedSpace sp(n_tokens, width);
  if (n_tokens > 0 && (!workspace || workspace_bytes < sp.total)) return DL_ERR_WORKSPACE;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  char* ws = reinterpret_cast<char*>(workspace);
  unsigned long long* words[2] = {reinterpret_cast<unsigned long long*>(ws), reinterpret_cast<unsigned long long*>(ws + sp.words)};

  // the rows to be zeroed, dealt over the sorting launches
  int digits = 0;
  while ((vocab >> digits) != 0) ++digits;                        // bits of the ids 0 .. vocab
  const int passes = n_tokens <= SORT_SMALL ? 0 : (digits + 9) / 10, launches = passes ? 2 * passes : 1;
  int64_t row = 0;
  int launch = 0;
  const auto share = [&]() {
    ZeroShare z{};
    z.base = reinterpret_cast<char*>(grad);
    z.pitch_bytes = grad_stride * (int64_t)ob;
    z.row_bytes = width * (int64_t)ob;
    z.row0 = row;
    ++launch;
    z.row1 = row = accumulate ? 0 : vocab * launch / launches;
    z.blocks = (unsigned)std::min<int64_t>(z.row1 - z.row0, 2048);
    return z;
  };
  const unsigned long long* sorted = words[0];
  if (passes == 0) {
    const ZeroShare z = share();
    hipLaunchKernelGGL(embed_sort_small_kernel, dim3(1 + z.blocks), dim3(1024), 0, st, tokens, itype, (int)n_tokens, vocab, words[0], z);
  } else {
    const int64_t per = std::max<int64_t>(2048, ((n_tokens + SORT_BLOCKS - 1) / SORT_BLOCKS + SORT_NT - 1) / SORT_NT * SORT_NT);
    SortPass s{tokens, itype, vocab, nullptr, words[0], reinterpret_cast<unsigned*>(ws + 2 * sp.words), n_tokens, per, 0, (digits + passes - 1) / passes,
               (unsigned)((n_tokens + per - 1) / per)};
    for (int k = 0; k < passes; ++k) {
      const ZeroShare a = share();
      hipLaunchKernelGGL(embed_sort_count_kernel, dim3(s.blocks + a.blocks), dim3(SORT_NT), 0, st, s, a);
      const ZeroShare b = share();
      hipLaunchKernelGGL(embed_sort_deal_kernel, dim3(s.blocks + b.blocks), dim3(SORT_NT), 0, st, s, b);
      sorted = s.out;
      s.in = s.out;
      s.out = words[(k + 1) & 1];
      s.shift += s.bits;
    }
  }
  if (n_tokens == 0) return embed_status();
  SumParams p{sorted, n_tokens, vocab, width, reinterpret_cast<const char*>(g), g_stride, reinterpret_cast<char*>(grad), grad_stride,
              reinterpret_cast<float*>(ws + 2 * sp.words + sp.counts), scale, 0};
  if (dtype == DL_F32) return launch_sums<TagF32, TagF32>(p, accumulate != 0, st);
  if (dtype == DL_BF16) return grad_dtype == DL_F32 ? launch_sums<TagBF16, TagF32>(p, accumulate != 0, st) : launch_sums<TagBF16, TagBF16>(p, accumulate != 0, st);
  return grad_dtype == DL_F32 ? launch_sums<TagF16, TagF32>(p, accumulate != 0, st) : launch_sums<TagF16, TagF16>(p, accumulate != 0, st);
}
