// Sampling: one token per row of logits, from a given random number, with temperature, top-k, top-p and min-p.
//
// The tokens of a row go in descending order of their logits, equal logits by their index.  Their weights are whole numbers,
//   W_i = floor(2^31 2^t_i),   t_i = (x_i - max x) log2(e) / T   (fp32, every operation rounded by itself),
// the power from a polynomial whose products and sums are rounded one by one.  Sums of whole numbers are exact, so the
// choice depends neither on the order of any additions nor on how a row is dealt to threads and workgroups: the same
// logits and the same random number give the same token on any launch, and on any machine with IEEE arithmetic.  (What is
// lost of a row's mass: below 2^-31 of the largest weight per token; the random number itself has 24 bits.)
//   top-k  the first k tokens;  top-p  tokens with less than floor(p * mass of those) ahead of them;  min-p  up to the
//   first token whose weight is below min_p * 2^31.  All three cut the ordered list behind some token, so what is kept is
//   a prefix, and the token is the one in whose stretch of the prefix's mass floor(u * mass) falls.
// So a row needs three look-ups in its ordered weights, not a sort: a histogram of (mass, count) over 1024 bins, a 32nd of a
// power of two wide, says in which bin each answer lies, and only the bins up to there (usually a few dozen tokens), or
// just that bin, are collected and sorted in LDS.  A bin that holds more than the list (equal logits, flat rows) is
// narrowed by eight bits of the logits' order at a time; what remains after 32 bits are equal logits, whose weights are
// equal too.
// Most rows need no histogram: while the maximum is looked for, every thread keeps the largest logit that it meets, and the q-th largest
// of those has at least q tokens at or above it, not many more.  They are listed in the sweep that adds up the row, and where the answers
// lie among them (top-k always) two sweeps are all.
#include "distill_common.hpp"
#include "distill_hip.h"

#include <algorithm>

namespace dl {

typedef unsigned long long u64;

constexpr int SAMPLE_BINS = 1024, SAMPLE_CAP = 2048;
constexpr int64_t SAMPLE_MAX_V = 1 << 22;      // a row's mass stays below 2^53

struct SampleParams {
  const void* logits; int64_t row_stride, n_rows, V;
  const float* u;
  const float* T; const int32_t* k; const float* p; const float* m;      // one per row, or NULL: the ones below for all rows
  float T0, p0, m0; int k0;
  int64_t* token; float* logp; int32_t* kept;
  // n rows from row r on
  SampleParams rows(int64_t r, int64_t n, int bytes) const {
    SampleParams q = *this;
    q.logits = reinterpret_cast<const char*>(logits) + r * row_stride * bytes;
    q.n_rows = n;
    q.u += r;
    q.token += r;
    if (T) q.T += r;
    if (k) q.k += r;
    if (this->p) q.p += r;
    if (m) q.m += r;
    if (logp) q.logp += r;
    if (kept) q.kept += r;
    return q;
  }
};

// What the weights of a row are relative to.
struct RowScale { float top, rate; };

// Rows in which only the maximum has a weight: T <= 0 (or NaN), T so small that 1 / T is infinite, an infinite maximum.
__device__ __forceinline__ bool only_the_maximum(float top, float T) { return !(T > 0.f) || LOG2E / T == INFINITY || top == INFINITY; }
// t of a logit, at least -64 (NaN as well)
__device__ __forceinline__ float sample_t(const RowScale& s, float x) {
#pragma clang fp contract(off)
  const float d = x - s.top;
  return fmaxf(d * s.rate, -64.f);
}
// 2^(t + 31), every operation rounded by itself.  t plus 1.5 * 2^23 is rint(t) in the lowest bits; the coefficients carry the 2^31 (a
// power of two changes no rounding), and 2^rint(t) is added to the exponent.  The polynomial is the one of degree 5 with p(0) = 1 whose
// largest relative error over [-1/2, 1/2] is least (a linear program over a grid), its coefficients rounded to fp32: off by 1.1e-7 of 2^f at
// most, 1.9e-7 as evaluated here.
__device__ __forceinline__ float sample_power(float t) {
#pragma clang fp contract(off)
  const float r = t + 0x1.8p23f, f = t - (r - 0x1.8p23f);
  float p = 0x1.5bba14p21f;
  p = p * f + 0x1.3cea88p24f;
  p = p * f + 0x1.c6b752p26f;
  p = p * f + 0x1.ebf9bcp28f;
  p = p * f + 0x1.62e42ap30f;
  p = p * f + 0x1p31f;
  return __uint_as_float(__float_as_uint(p) + (__float_as_uint(r) << 23));
}
__device__ __forceinline__ unsigned sample_weight(float t) { return (unsigned)sample_power(t); }
__device__ __forceinline__ int sample_bin(float t) { return min((int)(t * -32.f), SAMPLE_BINS - 1); }      // rounded towards 0
// Ascending with the logit; -0 counts as 0.
__device__ __forceinline__ unsigned order_of(float x) {
  const unsigned b = __float_as_uint(x + 0.f);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float logit_of(unsigned order) { return __uint_as_float(order ^ ((order >> 31) ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ u64 sample_word(float x, int column) { return ((u64)~order_of(x) << 32) | (unsigned)column; }
__device__ __forceinline__ float word_logit(u64 w) { return logit_of(~(unsigned)(w >> 32)); }
// floor(mass * part / 2^24)
__device__ __forceinline__ u64 share_of(u64 mass, unsigned part) { return (mass >> 24) * part + (((mass & 0xffffffu) * part) >> 24); }

// f(logits, n, column) for a row's columns in pieces of n <= 8 (4-byte logits: 4) neighbours, on any element boundary; the pieces of a
// thread that are whole come eight loads ahead.  Places behind n hold -inf.
template <class Tag, int NT, bool UNROLLED = true, class F>
__device__ __forceinline__ void each_piece(const char* row, int64_t V, F f) {
  using C = Chunk<Tag>;
  const int n = (int)V, whole = n / C::N;
  constexpr int UN = 4;
  u32x4 v[UN], ahead[UN];
  const auto fetch = [&](int c0, u32x4* to) {
#pragma unroll
    for (int i = 0; i < UN; ++i)
      if (c0 + i * NT < whole) to[i] = load16_unaligned(row + (int64_t)(c0 + i * NT) * 16);
  };
  float x[C::N];
  fetch(threadIdx.x, v);
  for (int c0 = threadIdx.x; c0 < whole; c0 += NT * UN) {
    fetch(c0 + NT * UN, ahead);                  // the next four are on their way while these are worked on
    if constexpr (UNROLLED) {
#pragma unroll
      for (int i = 0; i < UN; ++i) {
        if (c0 + i * NT >= whole) break;
        C::unpack(v[i], x);
        f(x, C::N, (c0 + i * NT) * C::N);
      }
    } else {
#pragma unroll 1
      for (int i = 0; i < UN; ++i) {
        if (c0 + i * NT >= whole) break;
        C::unpack(v[0], x);
        f(x, C::N, (c0 + i * NT) * C::N);
#pragma unroll
        for (int j = 1; j < UN; ++j) v[j - 1] = v[j];
      }
    }
#pragma unroll
    for (int i = 0; i < UN; ++i) v[i] = ahead[i];
  }
  const int col = whole * C::N + (int)threadIdx.x;
  if (col < n) {
#pragma unroll
    for (int e = 1; e < C::N; ++e) x[e] = -INFINITY;
    x[0] = load_as_float(row, Tag::id, col);
    f(x, 1, col);
  }
}
// f(logit, column) for every column.
template <class Tag, int NT, bool UNROLLED = true, class F>
__device__ __forceinline__ void each_logit(const char* row, int64_t V, F f) {
  each_piece<Tag, NT, UNROLLED>(row, V, [&](const float* x, int n, int col) {
#pragma unroll
    for (int e = 0; e < Chunk<Tag>::N; ++e)
      if (e < n) f(x[e], col + e);
  });
}

// A bin behind which every token has less weight than `least`: the threshold's, and two more for what rounding does to it.
__device__ __forceinline__ int bin_behind(unsigned least) { return min((int)((31.f - log2f((float)least)) * 32.f) + 2, SAMPLE_BINS - 1); }

// A list of tokens in order with their masses: those of some bins, or some of one bin's.
struct SampleLds {
  u64 mass[SAMPLE_BINS + 1];                 // of a bin; then of all bins ahead of it
  u64 word[SAMPLE_CAP], upto[SAMPLE_CAP];    // the list; the mass up to and with each of its tokens
  u64 wave_mass[32], hit_mass;
  unsigned count[SAMPLE_BINS + 1], wave_count[32];
  unsigned n, hit;
  float red[16];
};
// (the same for a row, whose address a called function gets without that knowledge)
__device__ __forceinline__ const char* global_row(const char* row) { return (const char*)(const __attribute__((address_space(1))) char*)row; }
__device__ __forceinline__ SampleLds& sample_lds() {      // (known as LDS also in functions that are called)
  __shared__ SampleLds s;
  return s;
}

// (Every function of it is inlined: the list's bounds stay in registers and what they index is known to be LDS.  Called, they go through
// scratch memory and generic addresses: 512 x 128256 bf16, T = 1.5, top-p 0.98: 351 us, inlined 184.  ROLLED: the sweeps' code once and not
// four times, for the function that holds every path; 3 % slower in the others.)
template <int NT, bool ROLLED = false>
struct Sampler {
  static constexpr int NW = NT / WAVE;
  SampleLds& s = sample_lds();
  const char* row;
  int64_t V;
  RowScale sc;
  // the list in LDS: bins [lo_bin, hi_bin] whole (hi_bin < 0: none), tokens and mass ahead of it
  int lo_bin = 0, hi_bin = -1, n = 0;
  unsigned ahead = 0;
  u64 ahead_mass = 0;
  bool overflow = false;                     // more tokens than the list holds

  __device__ __forceinline__ Sampler(const char* r, int64_t v, const RowScale& scale) : row(r), V(v), sc(scale) {}

  // Sums over the workgroup of a pair; the result in every thread.
  __device__ __forceinline__ void sum(u64& mass, unsigned& count) {
    const int lane = threadIdx.x & (WAVE - 1), w = threadIdx.x / WAVE;
#pragma unroll
    for (int o = WAVE / 2; o > 0; o >>= 1) {
      mass += __shfl_xor(mass, o, WAVE);
      count += __shfl_xor(count, o, WAVE);
    }
    __syncthreads();
    if (lane == 0) { s.wave_mass[w] = mass; s.wave_count[w] = count; }
    __syncthreads();
    mass = 0;
    count = 0;
    for (int i = 0; i < NW; ++i) { mass += s.wave_mass[i]; count += s.wave_count[i]; }
  }
  // Exclusive sums over the workgroup's threads, in order.
  __device__ __forceinline__ void scan(u64& mass, unsigned& count) {
    const int lane = threadIdx.x & (WAVE - 1), w = threadIdx.x / WAVE;
    const u64 m0 = mass;
    const unsigned c0 = count;
#pragma unroll
    for (int o = 1; o < WAVE; o <<= 1) {
      const u64 a = __shfl_up(mass, o, WAVE);
      const unsigned b = __shfl_up(count, o, WAVE);
      if (lane >= o) { mass += a; count += b; }
    }
    __syncthreads();
    if (lane == WAVE - 1) { s.wave_mass[w] = mass; s.wave_count[w] = count; }
    __syncthreads();
    mass -= m0;
    count -= c0;
    for (int i = 0; i < w; ++i) { mass += s.wave_mass[i]; count += s.wave_count[i]; }
  }
  // Masses and counts of bins -> of all bins ahead; entry `bins` gets the totals.
  template <int BINS>
  __device__ __forceinline__ void scan_bins(u64* mass, unsigned* count) {
    constexpr int EACH = (BINS + NT - 1) / NT;
    u64 m[EACH], mm = 0;
    unsigned c[EACH], cc = 0;
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      const int b = threadIdx.x * EACH + j;
      m[j] = b < BINS ? mass[b] : 0;
      c[j] = b < BINS ? count[b] : 0;
      mm += m[j];
      cc += c[j];
    }
    scan(mm, cc);
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      const int b = threadIdx.x * EACH + j;
      if (b < BINS) { mass[b] = mm; count[b] = cc; }
      mm += m[j];
      cc += c[j];
      if (b == BINS - 1) { mass[BINS] = mm; count[BINS] = cc; }
    }
    __syncthreads();
  }
  // The one index b < bins for which test(b) holds, in every thread.
  template <class Test>
  __device__ __forceinline__ int find(int bins, Test test) {
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += NT)
      if (test(b)) s.hit = (unsigned)b;
    __syncthreads();
    return (int)s.hit;
  }
  __device__ __forceinline__ int bin_of_count(unsigned q) { return find(SAMPLE_BINS, [&](int b) { return s.count[b] < q && s.count[b + 1] >= q; }); }
  __device__ __forceinline__ int bin_reaching(u64 m) { return find(SAMPLE_BINS, [&](int b) { return s.mass[b] < m && s.mass[b + 1] >= m; }); }
  __device__ __forceinline__ int bin_passing(u64 m) { return find(SAMPLE_BINS, [&](int b) { return s.mass[b] <= m && s.mass[b + 1] > m; }); }

  // Tokens for which in(t, x) holds (and that have a weight; only below < t <= above is asked) into the list, in order, with their masses
  // behind `mass`.  Most of a row is far below: one comparison for several logits themselves, with room for what rounding
  // does to t, is all that it costs.
  template <class Tag, class In>
  __device__ __forceinline__ void collect(unsigned before, u64 mass, float above, float below, In in) {
    collect<Tag>(before, mass, above, below, in, [](float) {});
  }
  // (`also` is called with every logit of the row)
  template <class Tag, class In, class Also>
  __device__ __forceinline__ void collect(unsigned before, u64 mass, float above, float below, In in, Also also) {
    const float far = sc.top + fmaxf(below, -33.f) / sc.rate;
    const float least = far - 1e-5f * (fabsf(far) + fabsf(sc.top));
    __syncthreads();
    if (threadIdx.x == 0) s.n = 0;
    __syncthreads();
    each_piece<Tag, NT, !ROLLED>(row, V, [&](const float* x, int count, int col) {
      float most = x[0];
#pragma unroll
      for (int e = 0; e < Chunk<Tag>::N; ++e) {
        if (e < count) also(x[e]);
        most = fmaxf(most, x[e]);
      }
      if (!(most >= least)) return;
#pragma unroll
      for (int e = 0; e < Chunk<Tag>::N; ++e) {
        if (!(x[e] >= least)) continue;
        const float t = sample_t(sc, x[e]);
        if (in(t, x[e]) && sample_weight(t) > 0) {
          const unsigned at = atomicAdd(&s.n, 1u);
          if (at < SAMPLE_CAP) s.word[at] = sample_word(x[e], col + e);
        }
      }
    });
    __syncthreads();
    overflow = s.n > SAMPLE_CAP;
    n = min((int)s.n, SAMPLE_CAP);
    ahead = before;
    ahead_mass = mass;
    if (overflow) return;
    sort(above, below);
    constexpr int EACH = SAMPLE_CAP / NT;
    unsigned w[EACH], none = 0;
    u64 sum_w = 0;
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      const int i = threadIdx.x * EACH + j;
      w[j] = i < n ? sample_weight(sample_t(sc, word_logit(s.word[i]))) : 0u;
      sum_w += w[j];
    }
    scan(sum_w, none);
    sum_w += mass;
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      const int i = threadIdx.x * EACH + j;
      sum_w += w[j];
      if (i < n) s.upto[i] = sum_w;
    }
    __syncthreads();
  }
  // The list's words, of tokens above t = `below` and at most t = `above`, ascending.  Up to 256: every word's place is the number of words
  // below it (all are different).
  __device__ __forceinline__ void sort(float above, float below) {
    const int tid = threadIdx.x;
    if (n <= 256) {
      u64 mine = 0;
      int place = 0;
      if (tid < n) {
        mine = s.word[tid];
        for (int j = 0; j < n; ++j) place += s.word[j] < mine;
      }
      __syncthreads();
      if (tid < n) s.word[place] = mine;
    } else if (sort_by_bins(above, below)) {
    } else if (n <= NT) {
      sort_in_registers<1>();
    } else {
      sort_in_registers<SAMPLE_CAP / NT>();
    }
    __syncthreads();
  }
  // More: dealt to 1024 bins of t, then every word counts those below it in its bin.  (top_k = 400 of 2048 x 50257
  // rows: 254 us with a bitonic sort through registers, 169 so.  Where a bin holds too many words, equal logits mostly, that sort is
  // what is left: false.)
  __device__ __forceinline__ bool sort_by_bins(float above, float below) {
    constexpr int BINS = 1024, MOST = 192, EACH = SAMPLE_CAP / NT, PER = BINS / NT;
    unsigned* start = reinterpret_cast<unsigned*>(s.upto);       // free until the masses go there
    const float scale = (float)BINS / (above - fmaxf(below, -32.f));
    for (int b = threadIdx.x; b <= BINS; b += NT) start[b] = 0;
    if (threadIdx.x == 0) s.hit = 0;
    __syncthreads();
    u64 w[EACH];
    unsigned slot[EACH];
    int bin[EACH];
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      const int i = j * NT + (int)threadIdx.x;
      if (i >= n) continue;
      w[j] = s.word[i];
      bin[j] = min(max((int)((above - sample_t(sc, word_logit(w[j]))) * scale), 0), BINS - 1);
      slot[j] = atomicAdd(&start[bin[j]], 1u);
    }
    __syncthreads();
    unsigned c[PER], all = 0;
    bool many = false;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      c[j] = start[threadIdx.x * PER + j];
      all += c[j];
      many = many || c[j] > MOST;
    }
    if (many) s.hit = 1;
    u64 none = 0;
    scan(none, all);                                             // (its barriers: the counts are read)
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      start[threadIdx.x * PER + j] = all;
      all += c[j];
    }
    if (threadIdx.x == 0) start[BINS] = (unsigned)n;
    __syncthreads();
    if (s.hit) return false;
#pragma unroll
    for (int j = 0; j < EACH; ++j)
      if (j * NT + (int)threadIdx.x < n) s.word[start[bin[j]] + slot[j]] = w[j];
    __syncthreads();
    unsigned place[EACH];
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      if (j * NT + (int)threadIdx.x >= n) continue;
      const unsigned first = start[bin[j]], last = start[bin[j] + 1];
      place[j] = first;
      for (unsigned i = first; i < last; ++i) place[j] += s.word[i] < w[j];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < EACH; ++j)
      if (j * NT + (int)threadIdx.x < n) s.word[place[j]] = w[j];
    return true;
  }
  template <int EACH>
  __device__ __forceinline__ void sort_in_registers() {
    u64 w[EACH];
#pragma unroll
    for (int j = 0; j < EACH; ++j) w[j] = (int)threadIdx.x * EACH + j < n ? s.word[threadIdx.x * EACH + j] : ~0ull;
    __syncthreads();
    block_sort<u64, NT, EACH>(w, s.word);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < EACH; ++j) s.word[threadIdx.x * EACH + j] = w[j];
  }
  // (The tokens ahead are counted on the way: the counts of the bins may be estimates.)
  template <class Tag>
  __device__ __forceinline__ void collect_bins(int lo, int hi) {
    const float above = -(float)lo * 0.03125f, below = hi == SAMPLE_BINS - 1 ? -65.f : -(float)(hi + 1) * 0.03125f;      // bin lo .. hi: below < t <= above
    unsigned before = 0;
    collect<Tag>(0, s.mass[lo], above, below, [&](float t, float) {
      before += t > above;
      return t <= above && t > below;
    });
    u64 none = 0;
    if (lo > 0) sum(none, before);
    ahead = before;
    lo_bin = lo;
    hi_bin = hi;
  }
  // Bins [lo, hi] and, further down, `end`, in one sweep: the list has the tokens of both, their masses those of the row.  (in_list_reaching
  // is for masses that `end` reaches then, in_list_token for those that [lo, hi] or `end` passes.)
  template <class Tag>
  __device__ __forceinline__ void collect_two(int lo, int hi, int end) {
    const float above = -(float)lo * 0.03125f, below = -(float)(hi + 1) * 0.03125f, above_end = -(float)end * 0.03125f, below_end = end == SAMPLE_BINS - 1 ? -65.f : -(float)(end + 1) * 0.03125f;
    const u64 gap = s.mass[end] - s.mass[hi + 1];
    unsigned before = 0, first = 0;
    collect<Tag>(0, s.mass[lo], above, below_end, [&](float t, float) {
      before += t > above_end;
      const bool one = t <= above && t > below, two = t <= above_end && t > below_end;
      first += one;
      return one || two;
    });
    if (overflow) return;
    for (int i = threadIdx.x; i < n; i += NT)
      if (sample_t(sc, word_logit(s.word[i])) <= above_end) s.upto[i] += gap;
    u64 both = ((u64)first << 32) | before;
    unsigned none = 0;
    sum(both, none);
    ahead = (unsigned)both - (unsigned)(both >> 32);             // of the row's place and the list's, from `end` on
    lo_bin = lo;
    hi_bin = hi;
  }
  // The likeliest tokens without a histogram of the row: every thread has met some logits while the row's maximum was looked for,
  // and the q-th largest of the threads' own maxima (`met`) has at least q tokens at or above it, not many more: the last of
  // the bins that hold them (count: zeros before).  The list then gets those bins, in a sweep in which `also` sees the row.
  __device__ __forceinline__ int likeliest_bins(float met, unsigned q) {
    const float t = sample_t(sc, met);
    if (t >= -31.f) atomicAdd(&s.count[sample_bin(t)], 1u);      // (a token has a weight from t = -31 on)
    __syncthreads();
    scan_bins<SAMPLE_BINS>(s.mass, s.count);
    return s.count[SAMPLE_BINS] < q ? SAMPLE_BINS - 1 : bin_of_count(q);
  }
  template <class Tag, class Also>
  __device__ __forceinline__ void collect_likeliest(int hi, Also also) {
    const float below = hi == SAMPLE_BINS - 1 ? -65.f : -(float)(hi + 1) * 0.03125f;
    collect<Tag>(0, 0, 0.f, below, [&](float t, float) { return t > below; }, also);
    lo_bin = 0;
    hi_bin = hi;
  }
  // Look-ups in the list as it is.
  __device__ __forceinline__ void in_list_reaching(u64 m, unsigned& tokens, u64& mass) {
    const int i = find(n, [&](int j) { return s.upto[j] >= m && (j == 0 ? ahead_mass : s.upto[j - 1]) < m; });
    tokens = ahead + (unsigned)i + 1;
    mass = s.upto[i];
  }
  __device__ __forceinline__ int in_list_token(u64 m, float& t) {
    const int i = find(n, [&](int k) { return s.upto[k] > m && (k == 0 ? ahead_mass : s.upto[k - 1]) <= m; });
    t = sample_t(sc, word_logit(s.word[i]));
    return (int)(unsigned)s.word[i];
  }
  // (a list from the first token on, and all tokens behind it below `least` or `tokens` within it)
  __device__ __forceinline__ void in_list_below(unsigned least, unsigned& tokens, u64& mass) {
    __syncthreads();
    if (threadIdx.x == 0) s.hit = min(tokens, (unsigned)n);
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += NT)
      if (s.upto[i] - (i == 0 ? 0 : s.upto[i - 1]) < least) atomicMin(&s.hit, (unsigned)i);
    __syncthreads();
    const unsigned q = s.hit;
    if (q < tokens) {
      tokens = q;
      mass = s.upto[q - 1];
    }
  }

  // Equal logits too many for the list, after narrow(): the order of their logit, tokens and mass ahead of them.
  bool ties = false;
  unsigned tie_order = 0, tie_weight = 0;

  // Makes the list hold the part of `bin` in which tokens-ahead-of-it <= target < ... (by_count), or the mass does, or sets `ties`.
  template <class Tag>
  __device__ __forceinline__ void narrow(int bin, bool by_count, u64 target) {
    u64* mass = s.word;                                       // 257 of each, in the list's place
    unsigned* count = reinterpret_cast<unsigned*>(s.upto);
    unsigned prefix = 0, before = s.count[bin];
    u64 before_mass = s.mass[bin];
    for (int shift = 24; shift >= 0; shift -= 8) {
      __syncthreads();
      for (int i = threadIdx.x; i <= 256; i += NT) { mass[i] = 0; count[i] = 0; }
      __syncthreads();
      each_logit<Tag, NT, !ROLLED>(row, V, [&](float x, int) {
        const float t = sample_t(sc, x);
        if (sample_bin(t) != bin) return;
        const unsigned o = order_of(x), w = sample_weight(t);
        if (w == 0 || (shift < 24 && (o >> (shift + 8)) != prefix)) return;
        const int slot = 255 - (int)((o >> shift) & 255u);
        atomicAdd(&mass[slot], (u64)w);
        atomicAdd(&count[slot], 1u);
      });
      __syncthreads();
      scan_bins<256>(mass, count);
      const u64 m0 = before_mass;
      const unsigned c0 = before;
      const int slot = find(256, [&](int b) {
        return by_count ? c0 + count[b] <= target && target < c0 + count[b + 1] : m0 + mass[b] <= target && target < m0 + mass[b + 1];
      });
      const unsigned inside = count[slot + 1] - count[slot];
      const u64 inside_mass = mass[slot + 1] - mass[slot];
      before = c0 + count[slot];
      before_mass = m0 + mass[slot];
      prefix = (prefix << 8) | (unsigned)(255 - slot);
      if (inside <= SAMPLE_CAP) {
        const unsigned want = prefix;
        const int sh = shift;
        collect<Tag>(before, before_mass, 0.f, -65.f, [&](float t, float x) { return sample_bin(t) == bin && (order_of(x) >> sh) == want; });
        lo_bin = 0;
        hi_bin = -1;                                          // part of a bin: of no use to other look-ups
        return;
      }
      if (shift == 0) {
        ties = true;
        tie_order = prefix;
        tie_weight = (unsigned)(inside_mass / inside);
        ahead = before;
        ahead_mass = before_mass;
        lo_bin = 0;
        hi_bin = -1;
      }
    }
  }
  // The list (or `ties`) so that it holds the target of bin `bin`.
  template <class Tag>
  __device__ __forceinline__ void reach(int bin, bool by_count, u64 target) {
    ties = false;
    if (bin >= lo_bin && bin <= hi_bin) return;
    if (s.count[bin + 1] - s.count[bin] <= SAMPLE_CAP) collect_bins<Tag>(bin, bin);
    else narrow<Tag>(bin, by_count, target);
  }
  // Mass of the first q tokens.
  template <class Tag>
  __device__ __forceinline__ u64 mass_of_first(unsigned q, int bin) {
    reach<Tag>(bin, true, q - 1);
    if (ties) return ahead_mass + (u64)(q - ahead) * tie_weight;
    return s.upto[q - ahead - 1];
  }
  // The number of tokens, and their mass, up to the first one at which the mass reaches m.
  template <class Tag>
  __device__ __forceinline__ void first_reaching(u64 m, int bin, unsigned& tokens, u64& mass) {
    reach<Tag>(bin, false, m - 1);
    if (ties) {
      const u64 q = (m - ahead_mass + tie_weight - 1) / tie_weight;
      tokens = ahead + (unsigned)q;
      mass = ahead_mass + q * tie_weight;
      return;
    }
    in_list_reaching(m, tokens, mass);
  }
  // The token in whose stretch m falls, and its t.
  template <class Tag>
  __device__ __forceinline__ int token_at(u64 m, int bin, float& t) {
    reach<Tag>(bin, false, m);
    if (ties) {
      const unsigned j = (unsigned)((m - ahead_mass) / tie_weight);
      t = sample_t(sc, logit_of(tie_order));
      return equal_logit<Tag>(j);
    }
    return in_list_token(m, t);
  }
  // The column of the j-th logit of order `tie_order`: every wave counts those of a stretch of columns, then the one that
  // holds the j-th walks its stretch again.
  template <class Tag>
  __device__ __forceinline__ int equal_logit(unsigned j) {
    const int lane = threadIdx.x & (WAVE - 1), w = threadIdx.x / WAVE;
    const int64_t each = (V + NW - 1) / NW, lo = min(V, w * each), hi = min(V, lo + each);
    unsigned mine = 0;
    for (int64_t c = lo + lane; c < hi; c += WAVE) mine += order_of(load_as_float(row, Tag::id, c)) == tie_order;
#pragma unroll
    for (int o = WAVE / 2; o > 0; o >>= 1) mine += __shfl_xor(mine, o, WAVE);
    __syncthreads();
    if (lane == 0) s.wave_count[w] = mine;
    __syncthreads();
    unsigned before = 0;
    for (int i = 0; i < w; ++i) before += s.wave_count[i];
    if (j >= before && j < before + mine) {
      for (int64_t c0 = lo; c0 < hi; c0 += WAVE) {
        const bool is = c0 + lane < hi && order_of(load_as_float(row, Tag::id, c0 + lane)) == tie_order;
        const u64 all = __ballot(is);
        if (is && before + __popcll(all & ((1ull << lane) - 1ull)) == j) s.hit = (unsigned)(c0 + lane);
        before += __popcll(all);
        if (before > j) break;
      }
    }
    __syncthreads();
    return (int)s.hit;
  }
  // The number of tokens ahead of the first whose weight is below `least`, and their mass, if that comes before `tokens`.
  template <class Tag>
  __device__ __forceinline__ void cut_below(unsigned least, unsigned& tokens, u64& mass) {
    const int behind = bin_behind(least);
    if (hi_bin < 0 || lo_bin > 0) {
      if (s.count[behind + 1] <= SAMPLE_CAP) collect_bins<Tag>(0, behind);
    }
    if (hi_bin >= 0 && lo_bin == 0 && (hi_bin >= behind || tokens <= (unsigned)n)) {
      in_list_below(least, tokens, mass);
      return;
    }
    // Too many for the list: the largest logit with too small a weight, then what lies above it.
    unsigned worst = 0;
    each_logit<Tag, NT, !ROLLED>(row, V, [&](float x, int) {
      const unsigned w = sample_weight(sample_t(sc, x));
      if (w > 0 && w < least) worst = max(worst, order_of(x));
    });
    worst = wave_max(worst);
    __syncthreads();
    if ((threadIdx.x & (WAVE - 1)) == 0) s.wave_count[threadIdx.x / WAVE] = worst;
    __syncthreads();
    for (int i = 0; i < NW; ++i) worst = max(worst, s.wave_count[i]);
    u64 m = 0;
    unsigned c = 0;
    each_logit<Tag, NT, !ROLLED>(row, V, [&](float x, int) {
      const unsigned w = sample_weight(sample_t(sc, x));
      if (w > 0 && order_of(x) > worst) { m += w; ++c; }
    });
    sum(m, c);
    if (c < tokens) {
      tokens = c;
      mass = m;
    }
  }
};

// The row's settings as whole numbers.
struct RowCuts { int k; unsigned part, least, u; bool top_p; };      // part, u: of 2^24
__device__ __forceinline__ RowCuts row_cuts(const SampleParams& p, int64_t r, float T) {
  const float top_p = p.p ? p.p[r] : p.p0, min_p = p.m ? p.m[r] : p.m0;
  RowCuts c;
  c.k = T > 0.f ? (p.k ? p.k[r] : p.k0) : 1;
  c.top_p = top_p < 1.f;
  c.part = (unsigned)(fminf(fmaxf(top_p, 0.f), 1.f) * 0x1p24f);
  c.least = min_p > 0.f ? (unsigned)(fminf(min_p, 1.f) * 0x1p31f) : 0u;
  c.u = (unsigned)fminf(fmaxf(p.u[r], 0.f) * 0x1p24f, 0x1p24f - 1.f);
  return c;
}
__device__ __forceinline__ u64 mass_wanted(u64 mass, unsigned part) {
  const u64 m = share_of(mass, part);
  return m > 0 ? m : 1;
}
struct RowResult { int token; unsigned kept; float t; };

// Rows whose maxima share the mass: equal weights, in the order of their columns.
template <class Tag, int NT>
__device__ __attribute__((noinline)) RowResult sample_maximum(const char* row, int64_t V, float top, const RowCuts cuts, unsigned& ties) {
  row = global_row(row);
  SampleLds& s = sample_lds();
  Sampler<NT> a(row, V, RowScale{top, 0.f});
  u64 none = 0;
  ties = 0;
  unsigned first = 0xffffffffu;
  each_logit<Tag, NT>(row, V, [&](float x, int col) {
    if (x == top) {
      ++ties;
      first = min(first, (unsigned)col);
    }
  });
  a.sum(none, ties);
  first = wave_min(first);
  __syncthreads();
  if ((threadIdx.x & (WAVE - 1)) == 0) s.wave_count[threadIdx.x / WAVE] = first;
  __syncthreads();
  for (int i = 0; i < Sampler<NT>::NW; ++i) first = min(first, s.wave_count[i]);
  unsigned n = cuts.k > 0 ? min(ties, (unsigned)cuts.k) : ties;
  if (cuts.top_p) n = (unsigned)((mass_wanted((u64)n << 31, cuts.part) + 0x7fffffffull) >> 31);
  const unsigned j = (unsigned)(share_of((u64)n << 31, cuts.u) >> 31);
  a.tie_order = order_of(top);
  return RowResult{j == 0 ? (int)first : a.template equal_logit<Tag>(j), n, 0.f};
}

__device__ __forceinline__ void clear_bins(SampleLds& s, int threads) {
  __syncthreads();
  for (int b = threadIdx.x; b <= SAMPLE_BINS; b += threads) { s.mass[b] = 0; s.count[b] = 0; }
  __syncthreads();
}

// Any row: a histogram of masses and counts, every look-up by the bins.
template <class Tag, int NT>
__device__ __attribute__((noinline)) RowResult sample_any(const char* row, int64_t V, const RowScale sc, const RowCuts cuts) {
  row = global_row(row);
  SampleLds& s = sample_lds();
  Sampler<NT, true> a(row, V, sc);
  clear_bins(s, NT);
  each_logit<Tag, NT, false>(row, V, [&](float x, int) {
    const float t = sample_t(sc, x);
    const unsigned w = sample_weight(t);
    if (w > 0) {
      const int b = sample_bin(t);
      atomicAdd(&s.mass[b], (u64)w);
      atomicAdd(&s.count[b], 1u);
    }
  });
  __syncthreads();
  a.template scan_bins<SAMPLE_BINS>(s.mass, s.count);
  unsigned tokens = s.count[SAMPLE_BINS];
  u64 mass = s.mass[SAMPLE_BINS];
  if (cuts.k > 0 && (unsigned)cuts.k < tokens) {
    const int bin = a.bin_of_count(cuts.k);
    if (s.count[bin + 1] <= SAMPLE_CAP) a.template collect_bins<Tag>(0, bin);      // holds whatever is asked below
    mass = a.template mass_of_first<Tag>(cuts.k, bin);
    tokens = cuts.k;
  }
  if (cuts.top_p) {
    const u64 want = mass_wanted(mass, cuts.part);
    const int bin = a.bin_reaching(want);
    if (a.hi_bin < 0 && s.count[bin + 1] <= SAMPLE_CAP) a.template collect_bins<Tag>(0, bin);
    a.template first_reaching<Tag>(want, bin, tokens, mass);
  }
  if (cuts.least > 0) a.template cut_below<Tag>(cuts.least, tokens, mass);
  const u64 want = share_of(mass, cuts.u);
  RowResult res;
  res.token = a.template token_at<Tag>(want, a.bin_passing(want), res.t);
  res.kept = tokens;
  return res;
}

// The usual rows: all that is asked lies among the likeliest tokens.  Two sweeps over the row, this is the second.  False: not
// decided here.  `powers`: the sum of 2^(t + 31).
template <class Tag, int NT>
__device__ __forceinline__ bool sample_likeliest(const char* row, int64_t V, const RowScale& sc, const RowCuts& cuts, float met, float& powers, RowResult& res) {
  SampleLds& s = sample_lds();
  Sampler<NT> a(row, V, sc);
  unsigned tokens = 0, live = 0;
  u64 mass = 0;
  if (cuts.k > 0) {
    a.template collect_likeliest<Tag>(a.likeliest_bins(met, cuts.k), [&](float x) { powers += fast_exp2(sample_t(sc, x)); });
    powers = block_sum<NT>(powers, s.red) * 0x1p31f;
    if (a.overflow || (a.n < cuts.k && a.hi_bin < SAMPLE_BINS - 1)) return false;
    tokens = min(a.n, cuts.k);
    mass = s.upto[tokens - 1];
  } else {
    const int hi = a.likeliest_bins(met, 128);      // (a list of somewhat more: up to 256 are sorted by counting)
    // what lies behind them could outweigh the maximum several times: the histogram at once
    if (hi < SAMPLE_BINS - 1 && (float)V * fast_exp2(-(float)(hi + 1) * 0.03125f) > 8.f) return false;
    a.template collect_likeliest<Tag>(hi, [&](float x) {
      const float e = sample_power(sample_t(sc, x));
      powers += e;
      const unsigned w = (unsigned)e;
      mass += w;
      live += __popcll(__ballot(w > 0));      // (of the wave: the scalar unit counts)
    });
    tokens = (threadIdx.x & (WAVE - 1)) == 0 ? live : 0u;
    powers = block_sum<NT>(powers, s.red);
    a.sum(mass, tokens);
    if (a.overflow) return false;
  }
  const u64 listed = s.upto[a.n - 1];
  if (cuts.top_p) {
    const u64 want = mass_wanted(mass, cuts.part);
    if (want > listed) {
      if (cuts.least == 0 || bin_behind(cuts.least) > a.hi_bin) return false;      // (else min-p cuts ahead of that)
    } else {
      a.in_list_reaching(want, tokens, mass);
    }
  }
  if (cuts.least > 0) {
    if (tokens > (unsigned)a.n && bin_behind(cuts.least) > a.hi_bin) return false;
    a.in_list_below(cuts.least, tokens, mass);
  }
  const u64 want = share_of(mass, cuts.u);
  if (want >= listed) return false;
  res.token = a.in_list_token(want, res.t);
  res.kept = tokens;
  return true;
}

// Rows with top-k whose first k tokens fit the list: counts of tokens per bin, first of those within 2^-16 of the most likely one
// (few, and with them few additions in LDS), of all if that is not enough.  Bins are counted whole or not at all -- t > -16 is bins 0 to
// 511, and behind t = -31 no token has a weight -- so a bin holds no more tokens for the list than were counted.  False: not decided here.
template <class Tag, int NT>
__device__ __forceinline__ bool sample_top_k(const char* row, int64_t V, const RowScale& sc, RowCuts cuts, RowResult& res) {
  SampleLds& s = sample_lds();
  Sampler<NT> a(row, V, sc);
  constexpr float ALL = -0x1.f00002p4f;      // the number before -31
  float below = -16.f;
  for (;;) {
    clear_bins(s, NT);
    each_logit<Tag, NT>(row, V, [&](float x, int) {
      const float t = sample_t(sc, x);
      if (t > below) atomicAdd(&s.count[sample_bin(t)], 1u);
    });
    __syncthreads();
    a.template scan_bins<SAMPLE_BINS>(s.mass, s.count);
    if (s.count[SAMPLE_BINS] >= (unsigned)cuts.k || below == ALL) break;
    below = ALL;
  }
  cuts.k = min(cuts.k, (int)s.count[SAMPLE_BINS]);
  const int bin = a.bin_of_count(cuts.k);
  if (s.count[bin + 1] > SAMPLE_CAP) return false;
  a.template collect_bins<Tag>(0, bin);
  unsigned tokens = cuts.k;
  u64 mass = s.upto[tokens - 1];
  if (cuts.top_p) a.in_list_reaching(mass_wanted(mass, cuts.part), tokens, mass);
  if (cuts.least > 0) a.in_list_below(cuts.least, tokens, mass);
  res.token = a.in_list_token(share_of(mass, cuts.u), res.t);
  res.kept = tokens;
  return true;
}

// Rows without top-k: a histogram of masses.  Counts of tokens are only needed to choose between lists; a bin's mass over its
// middle weight gives them to 1 %, and whether a list held all is known when it is made.
template <class Tag, int NT>
__device__ __forceinline__ bool sample_by_mass(const char* row, int64_t V, const RowScale& sc, const RowCuts& cuts, float& powers, RowResult& res) {
  SampleLds& s = sample_lds();
  Sampler<NT> a(row, V, sc);
  unsigned tokens = 0;
  powers = 0.f;
  clear_bins(s, NT);
  each_logit<Tag, NT>(row, V, [&](float x, int) {
    const float t = sample_t(sc, x), e = sample_power(t);
    powers += e;
    const unsigned w = (unsigned)e;
    if (w > 0) {
      ++tokens;
      atomicAdd(&s.mass[sample_bin(t)], (u64)w);
    }
  });
  powers = block_sum<NT>(powers, s.red);
  for (int b = threadIdx.x; b < SAMPLE_BINS; b += NT)
    if (s.mass[b] > 0) s.count[b] = (unsigned)((float)s.mass[b] * fast_exp2((float)b * 0.03125f + (0.015625f - 31.f))) + 1u;
  __syncthreads();
  a.template scan_bins<SAMPLE_BINS>(s.mass, s.count);
  u64 mass = s.mass[SAMPLE_BINS], none = 0;
  constexpr unsigned FITS = SAMPLE_CAP - SAMPLE_CAP / 16;
  a.sum(none, tokens);
  if (cuts.top_p || cuts.least > 0) {
    const u64 want = cuts.top_p ? mass_wanted(mass, cuts.part) : mass;
    const int end_p = cuts.top_p ? a.bin_reaching(want) : SAMPLE_BINS - 1, behind = cuts.least > 0 ? bin_behind(cuts.least) : SAMPLE_BINS - 1;
    const int end = min(end_p, behind);
    if (s.count[end + 1] <= FITS) a.template collect_bins<Tag>(0, end);
    else if (cuts.least == 0 && s.count[end + 1] - s.count[end] <= FITS) {
      // the token's bin as well: what is kept has a mass between those ahead of and with `end`
      const int from = a.bin_passing(share_of(s.mass[end], cuts.u)), to = a.bin_passing(share_of(s.mass[end + 1], cuts.u));
      if (s.count[end + 1] - s.count[min(from, end)] <= FITS) a.template collect_bins<Tag>(min(from, end), end);
      else if (to < end && s.count[to + 1] - s.count[from] + s.count[end + 1] - s.count[end] <= FITS) a.template collect_two<Tag>(from, to, end);
      else a.template collect_bins<Tag>(end, end);
    } else return false;
    if (a.overflow) return false;
    if (cuts.top_p && end_p <= behind) a.in_list_reaching(want, tokens, mass);
    if (cuts.least > 0) a.in_list_below(cuts.least, tokens, mass);
  }
  const u64 want = share_of(mass, cuts.u);
  const int bin = a.bin_passing(want);
  if (bin < a.lo_bin || bin > a.hi_bin) {
    if (s.count[bin + 1] - s.count[bin] > FITS) return false;
    a.template collect_bins<Tag>(bin, bin);
    if (a.overflow) return false;
  }
  res.token = a.in_list_token(want, res.t);
  res.kept = tokens;
  return true;
}

template <class Tag, int NT>
__global__ __launch_bounds__(NT) __attribute__((amdgpu_waves_per_eu(4, 8))) void sample_row_kernel(const SampleParams p) {
  SampleLds& s = sample_lds();
  const int64_t r = blockIdx.x;
  const char* row = reinterpret_cast<const char*>(p.logits) + r * p.row_stride * Tag::bytes;
  for (int b = threadIdx.x; b <= SAMPLE_BINS; b += NT) { s.mass[b] = 0; s.count[b] = 0; }
  float met = -INFINITY;                     // the largest logit that this thread has met
  each_logit<Tag, NT>(row, p.V, [&](float x, int) { met = fmaxf(met, x); });
  const float top = block_max<NT>(met, s.red);
  if (top == -INFINITY) {                    // nothing to draw from
    if (threadIdx.x == 0) {
      p.token[r] = -1;
      if (p.logp) p.logp[r] = -INFINITY;
      if (p.kept) p.kept[r] = 0;
    }
    return;
  }
  const float T = p.T ? p.T[r] : p.T0;
  const RowCuts cuts = row_cuts(p, r, T);
  RowResult res;
  float logp;
  if (only_the_maximum(top, T)) {
    unsigned ties;
    res = sample_maximum<Tag, NT>(row, p.V, top, cuts, ties);
    logp = -logf((float)ties);
  } else {
    const RowScale sc{top, LOG2E / T};
    float powers = 0.f;
    if (!sample_likeliest<Tag, NT>(row, p.V, sc, cuts, met, powers, res)) {
      const bool done = cuts.k > 0 ? sample_top_k<Tag, NT>(row, p.V, sc, cuts, res) : sample_by_mass<Tag, NT>(row, p.V, sc, cuts, powers, res);
      if (!done) res = sample_any<Tag, NT>(row, p.V, sc, cuts);
    }
    logp = (res.t - log2f(powers * 0x1p-31f)) * LN2;
  }
  if (threadIdx.x == 0) {
    p.token[r] = res.token;
    if (p.logp) p.logp[r] = logp;
    if (p.kept) p.kept[r] = (int)res.kept;
  }
}

// A workgroup per row: 1024 threads where every row has a CU to itself, 512 beyond, so that rows share one.  bf16, us for 512 / 1024
// threads, top-k 50 and top-p 0.95 (T = 1.5 and top-p 0.98): 256 x 128256 35.4 / 34.6 (153 / 102), 300 x 128256 41.7 / 54.7 (166 / 164),
// 512 x 32000 20.8 / 30.6 (53 / 70), 1024 x 50257 53 / 78 (140 / 193); 2048 x 50257 fp32 139 / 179 (276 / 375).
// Bound by vector work and additions in LDS where a row is flat (four sweeps over it, the first from HBM, the others from L2 and MALL), by
// the two sweeps' latency and the barriers between them for single rows: 1 x 32000 14.6 us; 256 x 128256 bf16 with mixed settings 75-96 us
// (0.7-0.9 TB/s, by how flat the flattest row is); 2048 x 50257 fp32 without top-k 209-218 us (1.9 TB/s).
template <class Tag>
static int launch_sample(const SampleParams& p, hipStream_t st) {
  if (p.n_rows <= 256) hipLaunchKernelGGL((sample_row_kernel<Tag, 1024>), dim3((unsigned)p.n_rows), dim3(1024), 0, st, p);
  else
    for (int64_t r = 0, most = LAUNCH_THREADS / 512; r < p.n_rows; r += most) {      // (one launch up to 8388607 rows)
      const SampleParams q = p.rows(r, std::min(most, p.n_rows - r), Tag::bytes);
      hipLaunchKernelGGL((sample_row_kernel<Tag, 512>), dim3((unsigned)q.n_rows), dim3(512), 0, st, q);
    }
  return hipGetLastError() == hipSuccess ? DL_OK : DL_ERR_LAUNCH;
}

}  // namespace dl

extern "C" int dl_sample_rows(const void* logits, int dtype, int64_t row_stride, int64_t n_rows, int64_t V, const float* u,
                              const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                              float temperature_all, int top_k_all, float top_p_all, float min_p_all, int64_t* token, float* logp,
                              int32_t* kept, void* stream) {
  using namespace dl;
  if ((unsigned)dtype > DL_F16) return DL_ERR_DTYPE;
  if (n_rows < 0 || V <= 0 || row_stride < V) return DL_ERR_SHAPE;
  if (n_rows == 0) return DL_OK;
  if (!logits || !u || !token) return DL_ERR_NULL;
  if (reinterpret_cast<uintptr_t>(logits) % (dtype == DL_F32 ? 4 : 2) || reinterpret_cast<uintptr_t>(token) % 8 ||
      (reinterpret_cast<uintptr_t>(u) | reinterpret_cast<uintptr_t>(temperature) | reinterpret_cast<uintptr_t>(top_k) |
       reinterpret_cast<uintptr_t>(top_p) | reinterpret_cast<uintptr_t>(min_p) | reinterpret_cast<uintptr_t>(logp) |
       reinterpret_cast<uintptr_t>(kept)) % 4)
    return DL_ERR_ALIGN;
  if (V > SAMPLE_MAX_V || n_rows > 0x7fffffffLL) return DL_ERR_LIMIT;
  SampleParams p{logits, row_stride, n_rows, V, u, temperature, top_k, top_p, min_p, temperature_all, top_p_all, min_p_all, top_k_all,
                 token, logp, kept};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (dtype == DL_F32) return launch_sample<TagF32>(p, st);
  if (dtype == DL_BF16) return launch_sample<TagBF16>(p, st);
  return launch_sample<TagF16>(p, st);
}
