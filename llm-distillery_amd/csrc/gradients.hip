// The norm of many tensors together, and the tensors scaled and clipped by it.
//
//   norm = scale * sqrt(sum of the squares of all elements);   element *= scale * min(1, max_norm / norm)
//
// The tensors' addresses and sizes travel with the launches, TABLE of them at a time.  They are cut into pieces of PIECE 16-byte chunks, from each
// tensor's first 16-byte boundary on (what lies ahead of it goes with the first piece, what lies behind the last whole chunk with the last).
// Squares are added up in fp64 (no sum overflows, none of a billion elements loses anything that fp32 shows) by workgroups that stay and take every
// so many-th piece, one sum per workgroup goes to the workspace, and these are added up in their order: no atomics, the same bits on every call.
// The second pass has a workgroup for every piece, the last piece first: what was read last may still be in MALL.
// Bound by HBM: 1.2 billion bf16 elements (2.4 GB) 1176 us, of it the squares 353 (6.8 TB/s), their sum 5, the product 818 (5.8 TB/s read and written: a
// copy of the size by the library reaches 4.9); 203 million fp32 elements of odd sizes, only read, 128 us, the squares 119 to 124.  Few small tensors
// (1 million elements in 11): 5 and 8 us on the card, less than the host needs for two launches.  Tried at the first of these: every workgroup
// a contiguous share of all 1261 us, long-lived workgroups that take every so many-th piece in the second pass 1245, its stores kept in the caches 1322, half
// as many chunks a thread 1361.
#include "distill_common.hpp"
#include "distill_hip.h"

#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

namespace dl {

constexpr int TABLE = 240, GRAD_NT = 256, GRAD_NCH = 16, PIECE = GRAD_NT * GRAD_NCH;
constexpr unsigned GRAD_GRID = 2048;
constexpr int ADDRESS_BITS = 56;                               // of a pointer; the dtype sits above them

struct GradTable {
  int n;
  unsigned pieces;                                             // of all tensors in the table
  unsigned long long at[TABLE];
  unsigned end[TABLE];                                         // pieces of the entries up to this one
  unsigned edges[TABLE];                                       // chunks of the last piece, elements behind them, elements ahead of the first: 13, 3 and 3 bits
};
static_assert(sizeof(GradTable) + 64 <= 4096, "a launch's arguments");

// A tensor's elements ahead of its first 16-byte boundary, the chunks from there on, the pieces that these make.
struct GradCut {
  int64_t head, chunks, tail, pieces;
  GradCut(const void* at, int64_t size, int dtype) {
    const int bytes = dtype == F32 ? 4 : 2;
    head = std::min<int64_t>(size, (int64_t)((16u - (unsigned)(reinterpret_cast<uintptr_t>(at) & 15u)) & 15u) / bytes);
    chunks = (size - head) * bytes / 16;
    tail = size - head - chunks * (16 / bytes);
    pieces = std::max<int64_t>(1, (chunks + PIECE - 1) / PIECE);
  }
  unsigned edges() const { return (unsigned)(chunks - (pieces - 1) * PIECE) | (unsigned)tail << 13 | (unsigned)head << 16; }
};

// A piece: `chunks` from `body` on; `n_ahead` and `n_behind` elements that belong to it besides.
struct GradPiece {
  char *body, *ahead, *behind;
  int dtype, chunks, n_ahead, n_behind;
};
// Piece q of the table.  A thread looks at an entry; the one whose entry has the piece says so to the others.
struct GradFind { unsigned long long at; unsigned begin, end, edges; };
__device__ __forceinline__ void find_entry(const GradTable& t, unsigned q, GradFind& found) {
  static_assert(TABLE <= GRAD_NT, "a thread an entry");
  const int tid = threadIdx.x;
  if (tid < t.n) {
    const unsigned end = t.end[tid], begin = tid ? t.end[tid - 1] : 0u;
    if (begin <= q && q < end) found = GradFind{t.at[tid], begin, end, t.edges[tid]};
  }
  __syncthreads();
}
__device__ __forceinline__ GradPiece piece_of(const GradFind& f, unsigned q) {
  const int dtype = (int)(f.at >> ADDRESS_BITS), head = (int)(f.edges >> 16);
  const bool last = q + 1 == f.end;
  char* const base = reinterpret_cast<char*>(f.at & ((1ull << ADDRESS_BITS) - 1));
  char* const body = base + head * (dtype == F32 ? 4 : 2) + (int64_t)(q - f.begin) * (PIECE * 16);
  const int chunks = last ? (int)(f.edges & 0x1fffu) : PIECE;
  return GradPiece{body, base, body + chunks * 16, dtype, chunks, q == f.begin ? head : 0, last ? (int)(f.edges >> 13 & 7u) : 0};
}
__device__ __forceinline__ int grad_chunk(int i) { return (int)(threadIdx.x / WAVE) * (WAVE * GRAD_NCH) + i * WAVE + (int)(threadIdx.x % WAVE); }

__device__ __forceinline__ double block_total(double v, double* scratch) {
  v = wave_sum(v);
  if ((threadIdx.x & (WAVE - 1)) == 0) scratch[threadIdx.x / WAVE] = v;
  __syncthreads();
  double total = 0.0;
#pragma unroll
  for (int w = 0; w < GRAD_NT / WAVE; ++w) total += scratch[w];
  return total;
}

template <class Tag>
__device__ __forceinline__ double piece_squares(const GradPiece& p) {
  constexpr int N = Chunk<Tag>::N;
  constexpr int HALF = GRAD_NCH / 2;                           // (all at a time: registers that spill)
  double sum = 0.0;
#pragma unroll 1
  for (int h = 0; h < GRAD_NCH; h += HALF) {
    u32x4 v[HALF];
#pragma unroll
    for (int i = 0; i < HALF; ++i) {
      v[i] = u32x4{0u, 0u, 0u, 0u};
      if (grad_chunk(h + i) < p.chunks) v[i] = load16_stream(p.body + grad_chunk(h + i) * 16);
    }
#pragma unroll
    for (int i = 0; i < HALF; ++i) {
      float f[N];
      Chunk<Tag>::unpack(v[i], f);
#pragma unroll
      for (int e = 0; e < N; ++e) sum = fma((double)f[e], (double)f[e], sum);
    }
  }
  for (int side = 0; side < 2; ++side)
    if ((int)threadIdx.x < (side ? p.n_behind : p.n_ahead)) {
      const double f = (double)load_as_float(side ? p.behind : p.ahead, Tag::id, threadIdx.x);
      sum = fma(f, f, sum);
    }
  return sum;
}

__global__ __launch_bounds__(GRAD_NT, 4) void squares_kernel(const GradTable t, double* sums) {
  __shared__ GradFind found;
  __shared__ double scratch[GRAD_NT / WAVE];
  double sum = 0.0;
#pragma unroll 1
  for (unsigned q = blockIdx.x; q < t.pieces; q += gridDim.x) {
    if (q == blockIdx.x || q >= found.end) {                   // (the same in all threads)
      __syncthreads();
      find_entry(t, q, found);
    }
    const GradPiece p = piece_of(found, q);
    sum += p.dtype == F32 ? piece_squares<TagF32>(p) : p.dtype == BF16 ? piece_squares<TagBF16>(p) : piece_squares<TagF16>(p);
  }
  const double total = block_total(sum, scratch);
  if (threadIdx.x == 0) sums[blockIdx.x] = total;
}

// scale * sqrt of the sums' sum: the same in every workgroup.
__device__ __forceinline__ double norm_of(const double* sums, unsigned n, float scale, double* scratch) {
  double v = 0.0;
  unsigned i = threadIdx.x;
  for (; i + 7 * GRAD_NT < n; i += 8 * GRAD_NT) {              // eight at a time on their way
    double w[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) w[k] = sums[i + k * GRAD_NT];
#pragma unroll
    for (int k = 0; k < 8; ++k) v += w[k];
  }
  for (; i < n; i += GRAD_NT) v += sums[i];
  return sqrt(block_total(v, scratch)) * (double)scale;
}
// `keep`: where the norm goes as it is, over the sums.
__global__ __launch_bounds__(GRAD_NT) void norm_kernel(double* sums, unsigned n, float scale, float* norm, bool keep) {
  __shared__ double scratch[GRAD_NT / WAVE];
  const double v = norm_of(sums, n, scale, scratch);           // (all have read theirs)
  if (threadIdx.x == 0) {
    norm[0] = (float)v;
    if (keep) sums[0] = v;
  }
}

// f times a factor of 64 bits, which may be smaller than fp32 holds: a product in 64 bits, so that the one rounding that shows is the result's.
__device__ __forceinline__ float scaled(float f, double by) { return (float)((double)f * by); }
template <class Tag>
__device__ __forceinline__ void scale_piece(const GradPiece& p, double by) {
  constexpr int N = Chunk<Tag>::N;
  u32x4 v[GRAD_NCH];
#pragma unroll
  for (int i = 0; i < GRAD_NCH; ++i) {
    v[i] = u32x4{0u, 0u, 0u, 0u};
    if (grad_chunk(i) < p.chunks) v[i] = load16_stream(p.body + grad_chunk(i) * 16);
  }
#pragma unroll
  for (int i = 0; i < GRAD_NCH; ++i) {
    float f[N];
    Chunk<Tag>::unpack(v[i], f);
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = scaled(f[e], by);
    if (grad_chunk(i) < p.chunks) store16_stream(p.body + grad_chunk(i) * 16, Chunk<Tag>::pack(f));
  }
  for (int side = 0; side < 2; ++side)
    if ((int)threadIdx.x < (side ? p.n_behind : p.n_ahead)) {
      char* at = side ? p.behind : p.ahead;
      store_from_float(at, Tag::id, threadIdx.x, scaled(load_as_float(at, Tag::id, threadIdx.x), by));
    }
}
// The norm: of `n_sums` sums, and is written; or (none) the first of them; or (no `sums`) given.
__global__ __launch_bounds__(GRAD_NT, 4) void scale_kernel(const GradTable t, const double* sums, unsigned n_sums, float scale, float max_norm, float* norm) {
  __shared__ GradFind found;
  __shared__ double scratch[GRAD_NT / WAVE];
  const double all = !sums ? (double)norm[0] : n_sums ? norm_of(sums, n_sums, scale, scratch) : sums[0];
  if (n_sums && blockIdx.x == 0 && threadIdx.x == 0) norm[0] = (float)all;
  const double by = all > (double)max_norm ? (double)max_norm / all * (double)scale : (double)scale;
  if (!((float)all <= 3.402823466e38f)) return;                // NaN or, as fp32 shows it, infinite: left as they are
  if (fabs(by - 1.0) <= 0x1p-25) return;                       // less than half a step of any element: they would stay what they are
  const unsigned q = t.pieces - 1u - blockIdx.x;
  find_entry(t, q, found);
  const GradPiece p = piece_of(found, q);
  if (p.dtype == F32) scale_piece<TagF32>(p, by);
  else if (p.dtype == BF16) scale_piece<TagBF16>(p, by);
  else scale_piece<TagF16>(p, by);
}

static int gradients_status() { return hipGetLastError() == hipSuccess ? DL_OK : DL_ERR_LAUNCH; }

constexpr int64_t PIECES = LAUNCH_THREADS / GRAD_NT;          // of a table

// Table by table: `each(table, the workgroups that add up squares of the tables before)`.
template <class Each>
static unsigned for_tables(const void* const* tensors, const int64_t* sizes, const int32_t* dtypes, int64_t n, Each each) {
  unsigned before = 0;
  GradTable t;
  t.n = 0;
  int64_t pieces = 0;
  for (int64_t i = 0; i <= n; ++i) {
    if (i < n && sizes[i] == 0) continue;
    const GradCut cut(i < n ? tensors[i] : nullptr, i < n ? sizes[i] : 0, i < n ? dtypes[i] : DL_F32);
    if (t.n > 0 && (i == n || t.n == TABLE || pieces + cut.pieces > PIECES)) {
      t.pieces = (unsigned)pieces;
      each(t, before);
      before += std::min(t.pieces, GRAD_GRID);
      t.n = 0;
      pieces = 0;
    }
    if (i == n) break;
    pieces += cut.pieces;
    t.at[t.n] = reinterpret_cast<unsigned long long>(tensors[i]) | (unsigned long long)dtypes[i] << ADDRESS_BITS;
    t.edges[t.n] = cut.edges();
    t.end[t.n++] = (unsigned)pieces;
  }
  return before;
}
static unsigned launch_squares(const void* const* tensors, const int64_t* sizes, const int32_t* dtypes, int64_t n, double* sums, hipStream_t st) {
  return for_tables(tensors, sizes, dtypes, n, [&](const GradTable& t, unsigned before) {
    hipLaunchKernelGGL(squares_kernel, dim3(std::min(t.pieces, GRAD_GRID)), dim3(GRAD_NT), 0, st, t, sums + before);
  });
}
constexpr unsigned FEW_SUMS = 512;                             // so many every workgroup adds up for itself (a launch less: 4 us)

static int gradients_check(const void* const* tensors, const int64_t* sizes, const int32_t* dtypes, int64_t n, float scale, bool apart) {
  if (n < 0 || !(scale > 0.f) || !(scale <= 3.4e38f)) return DL_ERR_SHAPE;
  if (n > 0 && (!tensors || !sizes || !dtypes)) return DL_ERR_NULL;
  for (int64_t i = 0; i < n; ++i) {
    if ((unsigned)dtypes[i] > DL_F16) return DL_ERR_DTYPE;
    if (sizes[i] < 0) return DL_ERR_SHAPE;
    if (sizes[i] > 0 && !tensors[i]) return DL_ERR_NULL;
    if (reinterpret_cast<uintptr_t>(tensors[i]) % (dtypes[i] == DL_F32 ? 4 : 2)) return DL_ERR_ALIGN;
    if (reinterpret_cast<uintptr_t>(tensors[i]) >> ADDRESS_BITS || sizes[i] > (int64_t)PIECE * 4 * (PIECES - 1)) return DL_ERR_LIMIT;
  }
  if (!apart) return DL_OK;
  try {
    std::vector<std::pair<uintptr_t, uintptr_t>> spans;
    spans.reserve((size_t)n);
    for (int64_t i = 0; i < n; ++i)
      if (sizes[i] > 0) spans.emplace_back(reinterpret_cast<uintptr_t>(tensors[i]), reinterpret_cast<uintptr_t>(tensors[i]) + (uintptr_t)sizes[i] * (dtypes[i] == DL_F32 ? 4 : 2));
    std::sort(spans.begin(), spans.end());
    for (size_t i = 1; i < spans.size(); ++i)
      if (spans[i].first < spans[i - 1].second) return DL_ERR_OVERLAP;
  } catch (const std::bad_alloc&) {
    return DL_ERR_LIMIT;
  }
  return DL_OK;
}

}  // namespace dl

extern "C" int64_t dl_grad_norm_workspace_bytes(const int64_t* sizes, int64_t n_tensors) {
  if (!sizes || n_tensors <= 0) return 0;
  int64_t tables = 1, in = 0, pieces = 0;
  for (int64_t i = 0; i < n_tensors; ++i) {
    if (sizes[i] <= 0) continue;
    const int64_t more = sizes[i] / (4 * (int64_t)dl::PIECE) + 1;      // (of the widest dtype: at least as many as there are)
    if (in == dl::TABLE || pieces + more > dl::PIECES) { ++tables; in = pieces = 0; }
    ++in;
    pieces += more;
  }
  return tables * dl::GRAD_GRID * 8;
}

extern "C" int dl_grad_norm(const void* const* tensors, const int64_t* sizes, const int32_t* dtypes, int64_t n_tensors, float scale, float* norm,
                            void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace dl;
  if (const int bad = gradients_check(tensors, sizes, dtypes, n_tensors, scale, false)) return bad;
  if (!norm) return DL_ERR_NULL;
  if (reinterpret_cast<uintptr_t>(workspace) % 8 || reinterpret_cast<uintptr_t>(norm) % 4) return DL_ERR_ALIGN;
  if (n_tensors > 0 && (!workspace || workspace_bytes < dl_grad_norm_workspace_bytes(sizes, n_tensors))) return DL_ERR_WORKSPACE;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  double* sums = reinterpret_cast<double*>(workspace);
  const unsigned n = launch_squares(tensors, sizes, dtypes, n_tensors, sums, st);
  hipLaunchKernelGGL(norm_kernel, dim3(1), dim3(GRAD_NT), 0, st, sums, n, scale, norm, false);
  return gradients_status();
}

extern "C" int dl_clip_grads(void* const* tensors, const int64_t* sizes, const int32_t* dtypes, int64_t n_tensors, float scale, float max_norm,
                             float* norm, int norm_given, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace dl;
  if (const int bad = gradients_check(tensors, sizes, dtypes, n_tensors, scale, true)) return bad;
  if (!(max_norm >= 0.f)) return DL_ERR_SHAPE;
  if (!norm) return DL_ERR_NULL;
  if (reinterpret_cast<uintptr_t>(workspace) % 8 || reinterpret_cast<uintptr_t>(norm) % 4) return DL_ERR_ALIGN;
  if (!norm_given && n_tensors > 0 && (!workspace || workspace_bytes < dl_grad_norm_workspace_bytes(sizes, n_tensors))) return DL_ERR_WORKSPACE;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  double* sums = norm_given ? nullptr : reinterpret_cast<double*>(workspace);
  unsigned n = 0;
  if (!norm_given) {
    n = launch_squares(tensors, sizes, dtypes, n_tensors, sums, st);
    if (n == 0 || n > FEW_SUMS) {
      hipLaunchKernelGGL(norm_kernel, dim3(1), dim3(GRAD_NT), 0, st, sums, n, scale, norm, n > 0);
      n = 0;
    }
  }
  for_tables(tensors, sizes, dtypes, n_tensors, [&](const GradTable& t, unsigned) {
    hipLaunchKernelGGL(scale_kernel, dim3(t.pieces), dim3(GRAD_NT), 0, st, t, sums, n, scale, max_norm, norm);
  });
  return gradients_status();
}
