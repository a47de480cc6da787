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
// otherwise: the sort is a chain of short launches, the zeroes are most of the bytes.  32768 tokens x 2048 bf16 into 128256 rows, 525 MB of
// gradient and 121 MB of g: a call takes 156 us (4.1 TB/s), 134 where g is still in MALL (the sorting launches 92, the sums 33, the
// join 9).  131 x 1024 fp32 added to a gradient: a call 19 us, its three launches in a graph 13.5.
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
// TPR threads share a row: a wave where there are rows enough to fill the card with waves, else a workgroup (bf16, us for 64 / 256
// threads: 1 x 4096 3.1 / 2.6, 512 x 4096 3.8 / 3.2, 2048 x 4096 4.7 / 4.8, 8192 x 4096 20.4 / 20.4, 8192 x 1024 4.9 / 6.0).  Table
// rows are read with ordinary loads (frequent tokens then come from L2), the result is streamed out.  Rows may start
// on any element; the columns behind the last whole 16 bytes go one by one.  Bound by HBM: 32768 x 4096 bf16 70-79 us
// (419 MB; the faster, the more of the rows MALL still has).
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
// `rows` stretches of `row_bytes` at a pitch (the last one of `last`), zeroed by `blocks` workgroups of a launch.  A dense gradient is cut
// into stretches of ZERO_PIECE bytes from its first 16-byte boundary on, `head` bytes ahead of that: whole lines whatever the
// width.  Streaming stores from many short-lived workgroups: 131 MB in 22 us (from 2048 workgroups: 26; ordinary stores: 34).
constexpr int64_t ZERO_PIECE = 4096, ZERO_BLOCKS = 16384;
struct ZeroShare {
  char* base; int64_t pitch, row_bytes, last, rows; int head; unsigned blocks;
};
__device__ __forceinline__ void zero_elements(char* at, int bytes) {      // elements of 2 or 4 bytes, fewer than 16 bytes
  if ((int)threadIdx.x * 2 < bytes) reinterpret_cast<unsigned short*>(at)[threadIdx.x] = 0;
}
__device__ __forceinline__ void zero_rows(const ZeroShare& z, unsigned b) {
  const int tid = threadIdx.x, nt = blockDim.x;
  if (b == 0) zero_elements(z.base - z.head, z.head);
  for (int64_t r = b; r < z.rows; r += z.blocks) {
    char* row = z.base + r * z.pitch;
    const int64_t bytes = r + 1 < z.rows ? z.row_bytes : z.last;
    const int64_t head = min((int64_t)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15), bytes), whole = (bytes - head) / 16;
    for (int64_t c = tid; c < whole; c += nt) store16_stream(row + head + c * 16, u32x4{0u, 0u, 0u, 0u});
    zero_elements(row, (int)head);
    zero_elements(row + head + whole * 16, (int)(bytes - head - whole * 16));
  }
}
// Rows [r0, r1) of a gradient with `width` bytes of a row's `pitch`.
static ZeroShare zero_share(char* grad, int64_t pitch, int64_t width, int64_t r0, int64_t r1) {
  ZeroShare z{grad + r0 * pitch, pitch, width, width, std::max<int64_t>(r1 - r0, 0), 0, 0};
  if (pitch == width && z.rows > 0) {
    int64_t bytes = z.rows * pitch;
    z.head = (int)std::min<int64_t>((16 - (reinterpret_cast<uintptr_t>(z.base) & 15)) & 15, bytes);
    z.base += z.head;
    bytes -= z.head;
    z.pitch = z.row_bytes = ZERO_PIECE;
    z.rows = (bytes + ZERO_PIECE - 1) / ZERO_PIECE;
    z.last = bytes - (z.rows - 1) * ZERO_PIECE;
  }
  z.blocks = (unsigned)std::min<int64_t>(std::max<int64_t>(z.rows, z.head > 0), ZERO_BLOCKS);
  return z;
}

// ---- sort ---------------------------------------------------------------------------------------------
// A token and its place as one word, token << 32 | n; tokens outside the vocabulary count as id `vocab` and end up
// behind all others.
__device__ __forceinline__ unsigned long long token_word(const void* tokens, int itype, int64_t n, int64_t vocab) {
  const int64_t t = token_row(tokens, itype, n, vocab);
  return ((unsigned long long)(t < 0 ? vocab : t) << 32) | (unsigned)n;
}

constexpr int SORT_SMALL = 1024;      // tokens one workgroup sorts in registers
template <int NT>
__global__ __launch_bounds__(NT) void embed_sort_small_kernel(const void* __restrict__ tokens, int itype, int n, int64_t vocab,
                                                              unsigned long long* __restrict__ sorted, ZeroShare z) {
  if (blockIdx.x > 0) return zero_rows(z, blockIdx.x - 1);
  __shared__ unsigned long long xch[NT];
  unsigned long long w[1] = {~0ull};
  if ((int)threadIdx.x < n) w[0] = token_word(tokens, itype, threadIdx.x, vocab);
  block_sort<unsigned long long, NT, 1>(w, xch);
  if ((int)threadIdx.x < n) sorted[threadIdx.x] = w[0];
}

// Longer lists: a stable sort by digits of `bits` bits, lowest first (two of them up to a million ids).  A pass counts
// each workgroup's digits in one launch and deals its words out in the next, where every workgroup adds up the counts
// ahead of it itself: at most SORT_BLOCKS of them.
constexpr int SORT_NT = 256, SORT_WAVES = SORT_NT / WAVE, SORT_BINS = 1024, SORT_BLOCKS = 64, SORT_LEAST = 512;      // words a workgroup has at least
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
  constexpr int EACH = SORT_BINS / SORT_NT;              // (4: a pass has at least that many bins)
  static_assert(EACH == 4, "one 16-byte load per workgroup's counts");
  // this thread's digits tid * EACH ..: words of all workgroups, words of the workgroups ahead
  unsigned all[EACH], ahead[EACH], mine = 0u;
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    all[j] = ahead[j] = 0u;
#pragma unroll
    for (int k = 0; k < SORT_WAVES; ++k) place[k][tid * EACH + j] = 0u;
  }
  if (tid * EACH < bins) {
#pragma unroll 8
    for (unsigned b = 0; b < s.blocks; ++b) {
      const u32x4 c = *reinterpret_cast<const u32x4*>(s.counts + (int64_t)b * bins + tid * EACH);
#pragma unroll
      for (int j = 0; j < EACH; ++j) {
        all[j] += c[j];
        ahead[j] += b < blockIdx.x ? c[j] : 0u;
      }
    }
  }
#pragma unroll
  for (int j = 0; j < EACH; ++j) mine += all[j];
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
// Sorted words are cut into tiles of 32, or as few as 4 where that would leave most of the card idle (the depth of a tile is a chain
// of dependent memory round trips: 131 tokens x 1024 columns take 5 us with tiles of 4, 17 with 32).
constexpr int SUM_NT = 128, SUM_TILE_MOST = 32, SUM_TILE_LEAST = 4, SUM_AHEAD = 8;
static int sum_tile(int64_t n, int64_t width) {
  int tile = SUM_TILE_MOST;
  while (tile > SUM_TILE_LEAST && n * width < (int64_t)tile << 20) tile /= 2;
  return tile;
}
struct SumParams {
  const unsigned long long* sorted; int64_t n, vocab, width;
  const char* g; int64_t g_stride;
  char* grad; int64_t grad_stride;
  float* partial;                  // [tiles][2][width]: the sum of a tile's first token (if it began earlier), of its last (if it goes on)
  float scale; unsigned slices; int tile;
  int64_t tile0;                   // the launch's first tile
};
__device__ __forceinline__ unsigned word_token(unsigned long long w) { return (unsigned)(w >> 32); }

// n of the Chunk<Tag>::N columns from `col` on, zeros behind.
template <class Tag>
__device__ __forceinline__ u32x4 load_columns(const char* row, int64_t col, int n) {
  const char* at = row + col * Tag::bytes;
  if (n == Chunk<Tag>::N) return load16_unaligned(at);
  u32x4 v{0u, 0u, 0u, 0u};
#pragma unroll
  for (int e = 0; e < Chunk<Tag>::N; ++e)
    if (e < n) {
      if constexpr (Tag::bytes == 4) v[e] = reinterpret_cast<const unsigned*>(at)[e];
      else v[e / 2] |= (unsigned)reinterpret_cast<const unsigned short*>(at)[e] << (16 * (e & 1));
    }
  return v;
}
template <class Tag>
__device__ __forceinline__ void store_columns(char* row, int64_t col, int n, const float* f) {
  if (n == Chunk<Tag>::N) {
    store16_stream_any(row + col * Tag::bytes, Chunk<Tag>::pack(f));
  } else {
#pragma unroll
    for (int e = 0; e < Chunk<Tag>::N; ++e)
      if (e < n) store_from_float(row, Tag::id, col + e, f[e]);
  }
}

template <class Tag, class TagO, bool ADD>
__global__ __launch_bounds__(SUM_NT) void embed_sum_kernel(const SumParams p) {
  using C = Chunk<Tag>;
  using O = Chunk<TagO>;
  constexpr int PIECES = C::N / O::N;                          // 16-byte pieces of the gradient beside one of g
  const int64_t tile = p.tile0 + blockIdx.x / p.slices, t0 = tile * p.tile;
  const int64_t col = ((int64_t)(blockIdx.x % p.slices) * SUM_NT + threadIdx.x) * C::N;
  const int cols = (int)min((int64_t)C::N, p.width - col);
  __shared__ unsigned long long word[SUM_TILE_MOST + 2];      // the tile's, and one on either side (~0: none)
  if ((int)threadIdx.x < p.tile + 2) {
    const int64_t i = t0 - 1 + threadIdx.x;
    word[threadIdx.x] = i >= 0 && i < p.n ? p.sorted[i] : ~0ull;
  }
  __syncthreads();
  if (cols <= 0) return;
  const int count = (int)min((int64_t)p.tile, p.n - t0);
  const auto grad_row = [&](unsigned v) { return p.grad + (int64_t)v * p.grad_stride * TagO::bytes; };
  float sum[C::N];
#pragma unroll
  for (int e = 0; e < C::N; ++e) sum[e] = 0.f;
  bool open = word_token(word[0]) == word_token(word[1]);      // the running token began in an earlier tile
  for (int i0 = 0; i0 < count; i0 += SUM_AHEAD) {
    u32x4 x[SUM_AHEAD], old[ADD ? SUM_AHEAD : 1][PIECES];
#pragma unroll
    for (int j = 0; j < SUM_AHEAD; ++j) {
      const unsigned v = i0 + j < count ? word_token(word[1 + i0 + j]) : (unsigned)p.vocab;
      if (v >= p.vocab) continue;
      x[j] = load_columns<Tag>(p.g + (int64_t)(unsigned)word[1 + i0 + j] * p.g_stride * Tag::bytes, col, cols);
      if (ADD && word_token(word[2 + i0 + j]) != v)
#pragma unroll
        for (int k = 0; k < PIECES; ++k) old[ADD ? j : 0][k] = load_columns<TagO>(grad_row(v), col + k * O::N, min(max(cols - k * O::N, 0), O::N));
    }
#pragma unroll
    for (int j = 0; j < SUM_AHEAD; ++j) {
      const int i = i0 + j;
      if (i >= count) break;
      const unsigned v = word_token(word[1 + i]);
      if (v >= p.vocab) return;                                // padding: behind all tokens
      float f[C::N];
      C::unpack(x[j], f);
#pragma unroll
      for (int e = 0; e < C::N; ++e) sum[e] += f[e];
      const bool same = word_token(word[2 + i]) == v;
      if (same && i + 1 < count) continue;
      if (!open && !same) {
#pragma unroll
        for (int k = 0; k < PIECES; ++k) {
          float to[O::N];
          if (ADD) O::unpack(old[ADD ? j : 0][k], to);
#pragma unroll
          for (int e = 0; e < O::N; ++e) to[e] = ADD ? fmaf(p.scale, sum[k * O::N + e], to[e]) : p.scale * sum[k * O::N + e];
          store_columns<TagO>(grad_row(v), col + k * O::N, min(max(cols - k * O::N, 0), O::N), to);
        }
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

// The tokens that cross tiles: the tile in which one begins adds up its partial sums in order, 8 loads in flight per thread; a
// token that crosses more than 64 tiles is dealt to the workgroup's waves, a contiguous stretch of tiles each, whose sums then meet
// in LDS in order.
constexpr int JOIN_NT = 256, JOIN_COLS = 4, JOIN_AHEAD = 8, JOIN_DEALT = 64;
__device__ __forceinline__ void add_partials(const SumParams& p, int64_t from, int64_t to, int64_t col, int cols, float* sum) {      // tiles [from, to)
  if (cols == JOIN_COLS) {
    for (int64_t t = from; t < to; t += JOIN_AHEAD) {
      u32x4 x[JOIN_AHEAD];
#pragma unroll
      for (int j = 0; j < JOIN_AHEAD; ++j)
        if (t + j < to) x[j] = load16_unaligned(p.partial + (t + j) * 2 * p.width + col);
#pragma unroll
      for (int j = 0; j < JOIN_AHEAD; ++j)
        if (t + j < to)
#pragma unroll
          for (int e = 0; e < JOIN_COLS; ++e) sum[e] += __uint_as_float(x[j][e]);
    }
  } else {
    for (int64_t t = from; t < to; ++t)
#pragma unroll
      for (int e = 0; e < JOIN_COLS; ++e)
        if (e < cols) sum[e] += p.partial[t * 2 * p.width + col + e];
  }
}
template <class TagO, bool ADD>
__global__ __launch_bounds__(JOIN_NT) void embed_join_kernel(const SumParams p) {
  __shared__ float met[JOIN_NT / WAVE][WAVE * JOIN_COLS];
  const int64_t tile = p.tile0 + blockIdx.x / p.slices, t0 = tile * p.tile, t1 = t0 + p.tile;
  if (t1 >= p.n) return;
  const unsigned v = word_token(p.sorted[t1 - 1]);
  if (v >= p.vocab || word_token(p.sorted[t1]) != v) return;                                     // ends with the tile
  if (word_token(p.sorted[t0]) == v && t0 > 0 && word_token(p.sorted[t0 - 1]) == v) return;      // began in an earlier one
  int64_t lo = t1, hi = p.n;                             // where it ends, by bisection: sorted[lo] is the token, sorted[hi] is not
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) / 2;
    (word_token(p.sorted[mid]) == v ? lo : hi) = mid;
  }
  const int64_t end = lo / p.tile + 1, span = end - tile - 1;
  char* row = p.grad + (int64_t)v * p.grad_stride * TagO::bytes;
  const int lane = threadIdx.x & (WAVE - 1), w = threadIdx.x / WAVE;
  constexpr int NW = JOIN_NT / WAVE;
  const auto finish = [&](const float* sum, int64_t col, int cols) {
#pragma unroll
    for (int e = 0; e < JOIN_COLS; ++e)
      if (e < cols) store_from_float(row, TagO::id, col + e, ADD ? fmaf(p.scale, sum[e], load_as_float(row, TagO::id, col + e)) : p.scale * sum[e]);
  };
  const int64_t slice0 = (int64_t)(blockIdx.x % p.slices) * JOIN_NT * JOIN_COLS;
  if (span <= JOIN_DEALT) {
    const int64_t col = slice0 + threadIdx.x * JOIN_COLS;
    const int cols = (int)min((int64_t)JOIN_COLS, p.width - col);
    if (cols <= 0) return;
    float sum[JOIN_COLS];
#pragma unroll
    for (int e = 0; e < JOIN_COLS; ++e) sum[e] = e < cols ? p.partial[(tile * 2 + 1) * p.width + col + e] : 0.f;
    add_partials(p, tile + 1, end, col, cols, sum);
    finish(sum, col, cols);
    return;
  }
  const int64_t each = (span + NW - 1) / NW, from = min(end, tile + 1 + w * each), to = min(end, from + each);
  for (int q = 0; q < NW; ++q) {
    const int64_t col = slice0 + (q * WAVE + lane) * JOIN_COLS;
    const int cols = (int)min((int64_t)JOIN_COLS, p.width - col);
    float sum[JOIN_COLS] = {0.f, 0.f, 0.f, 0.f};
    if (cols > 0) {
      if (w == 0)
#pragma unroll
        for (int e = 0; e < JOIN_COLS; ++e)
          if (e < cols) sum[e] = p.partial[(tile * 2 + 1) * p.width + col + e];
      add_partials(p, from, to, col, cols, sum);
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < JOIN_COLS; ++e) met[w][lane * JOIN_COLS + e] = sum[e];
    __syncthreads();
    if (w == q && cols > 0) {
#pragma unroll
      for (int e = 0; e < JOIN_COLS; ++e) {
        sum[e] = met[0][lane * JOIN_COLS + e];
        for (int k = 1; k < NW; ++k) sum[e] += met[k][lane * JOIN_COLS + e];
      }
      finish(sum, col, cols);
    }
  }
}

static int embed_status() { return hipGetLastError() == hipSuccess ? DL_OK : DL_ERR_LAUNCH; }

template <class Tag, class TagO>
static int launch_sums(const SumParams& s, bool add, hipStream_t st) {
  SumParams p = s, j = s;
  const int64_t tiles = (p.n + p.tile - 1) / p.tile;
  p.slices = (unsigned)((p.width + SUM_NT * Chunk<Tag>::N - 1) / (SUM_NT * Chunk<Tag>::N));
  j.slices = (unsigned)((p.width + JOIN_NT * JOIN_COLS - 1) / (JOIN_NT * JOIN_COLS));
  const auto launch = [&](SumParams& q, int64_t end, int threads, auto kernel) {      // tiles [0, end)
    for (const int64_t most = LAUNCH_THREADS / threads / q.slices; q.tile0 < end; q.tile0 += most)
      hipLaunchKernelGGL(kernel, dim3((unsigned)(std::min(most, end - q.tile0) * q.slices)), dim3(threads), 0, st, q);
  };
  // (the last tile is no joined token's first)
  if (add) {
    launch(p, tiles, SUM_NT, embed_sum_kernel<Tag, TagO, true>);
    launch(j, tiles - 1, JOIN_NT, embed_join_kernel<TagO, true>);
  } else {
    launch(p, tiles, SUM_NT, embed_sum_kernel<Tag, TagO, false>);
    launch(j, tiles - 1, JOIN_NT, embed_join_kernel<TagO, false>);
  }
  return embed_status();
}

// Places of the workspace, each on a 256-byte boundary: two lists of words, the digit counts, the partial sums.
struct EmbedSpace {
  int64_t words, counts, partial, total;
  int tile;
  EmbedSpace(int64_t n, int64_t width) {
    const auto up = [](int64_t b) { return (b + 255) / 256 * 256; };
    words = up(n * 8);
    counts = n > SORT_SMALL ? up((int64_t)SORT_BLOCKS * SORT_BINS * 4) : 0;
    tile = sum_tile(n, width);
    partial = up((n + tile - 1) / tile * 2 * width * 4);
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
  constexpr int64_t MOST = LAUNCH_THREADS / 256 * 4;      // tokens of a launch
#define DL_EMBED(TAG)                                                                                                                     \
  if (few) hipLaunchKernelGGL((embed_rows_kernel<TAG, 256>), dim3((unsigned)n), dim3(256), 0, st, t, table_stride, vocab, width, ids,    \
                              itype, n, scale, to, out_stride);                                                                           \
  else hipLaunchKernelGGL((embed_rows_kernel<TAG, 64>), dim3((unsigned)((n + 3) / 4)), dim3(256), 0, st, t, table_stride, vocab, width,   \
                          ids, itype, n, scale, to, out_stride);
  for (int64_t n0 = 0; n0 < n_tokens; n0 += MOST) {
    const int64_t n = std::min(MOST, n_tokens - n0);
    const void* ids = reinterpret_cast<const char*>(tokens) + n0 * (itype == DL_I64 ? 8 : 4);
    char* to = o + n0 * out_stride * (int64_t)eb;
    if (dtype == DL_F32) { DL_EMBED(TagF32) } else if (dtype == DL_BF16) { DL_EMBED(TagBF16) } else { DL_EMBED(TagF16) }
  }
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
  if (n_tokens > 0x7fffffffLL || vocab > 0x7ffffffeLL || slices > LAUNCH_THREADS / JOIN_NT) return DL_ERR_LIMIT;
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
    ++launch;
    const int64_t first = row;
    row = accumulate ? 0 : vocab * launch / launches;
    return zero_share(reinterpret_cast<char*>(grad), grad_stride * (int64_t)ob, width * (int64_t)ob, first, row);
  };
  const unsigned long long* sorted = words[0];
  if (passes == 0) {
    const ZeroShare z = share();
    if (n_tokens <= 256) hipLaunchKernelGGL(embed_sort_small_kernel<256>, dim3(1 + z.blocks), dim3(256), 0, st, tokens, itype, (int)n_tokens, vocab, words[0], z);
    else hipLaunchKernelGGL(embed_sort_small_kernel<1024>, dim3(1 + z.blocks), dim3(1024), 0, st, tokens, itype, (int)n_tokens, vocab, words[0], z);
  } else {
    const int64_t per = std::max<int64_t>(SORT_LEAST, ((n_tokens + SORT_BLOCKS - 1) / SORT_BLOCKS + SORT_NT - 1) / SORT_NT * SORT_NT);
    SortPass s{tokens, itype, vocab, nullptr, words[0], reinterpret_cast<unsigned*>(ws + 2 * sp.words), n_tokens, per, 0, std::max(2, (digits + passes - 1) / passes),
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
              reinterpret_cast<float*>(ws + 2 * sp.words + sp.counts), scale, 0, sp.tile, 0};
  if (dtype == DL_F32) return launch_sums<TagF32, TagF32>(p, accumulate != 0, st);
  if (dtype == DL_BF16) return grad_dtype == DL_F32 ? launch_sums<TagBF16, TagF32>(p, accumulate != 0, st) : launch_sums<TagBF16, TagBF16>(p, accumulate != 0, st);
  return grad_dtype == DL_F32 ? launch_sums<TagF16, TagF32>(p, accumulate != 0, st) : launch_sums<TagF16, TagF16>(p, accumulate != 0, st);
}
