// The norm of many tensors together, and the tensors scaled and clipped by it.
//
//   norm = scale * sqrt(sum of the squares of all elements);   element *= scale * min(1, max_norm / norm)
//
// The tensors' addresses and sizes travel with the launches, TABLE of them at a time.  They are cut into pieces of PIECE elements and the
// pieces dealt evenly to the workgroups.  Squares are added up in fp64 (no sum overflows, none of a billion elements loses anything that
// fp32 shows), one sum per workgroup goes to the workspace, and whoever needs the norm adds these up in their order: no atomics, the same
// bits on every call, two launches for up to TABLE tensors.
#include "distill_common.hpp"
#include "distill_hip.h"

#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

namespace dl {

constexpr int TABLE = 240, GRAD_NT = 256, PIECE = 8192;
constexpr unsigned GRAD_GRID = 2048;
constexpr int ADDRESS_BITS = 56;                               // of a pointer; the dtype sits above them

struct GradTable {
  int n;
  unsigned pieces;                                             // of all tensors in the table
  unsigned long long at[TABLE];
  int64_t size[TABLE];
};

// The pieces of a workgroup, one after the other: `each(address, dtype, elements)`.
template <class Each>
__device__ __forceinline__ void for_pieces(const GradTable& t, unsigned long long* at, int64_t* size, unsigned* first, Each each) {
  const int tid = threadIdx.x;
  static_assert(TABLE <= GRAD_NT, "a thread an entry");
  unsigned mine = 0;
  if (tid < t.n) {
    at[tid] = t.at[tid];
    size[tid] = t.size[tid];
    mine = (unsigned)((t.size[tid] + PIECE - 1) / PIECE);
  }
  first[tid] = mine;
  __syncthreads();
  for (int o = 1; o < GRAD_NT; o <<= 1) {                      // sums up to each entry
    const unsigned v = tid >= o ? first[tid - o] : 0u;
    __syncthreads();
    first[tid] += v;
    __syncthreads();
  }
  const unsigned begin = (unsigned)((uint64_t)t.pieces * blockIdx.x / gridDim.x), end = (unsigned)((uint64_t)t.pieces * (blockIdx.x + 1) / gridDim.x);
  int lo = 0, hi = t.n - 1;                                    // the first entry whose pieces end behind `begin`
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (first[mid] > begin) hi = mid;
    else lo = mid + 1;
  }
  for (unsigned q = begin; q < end; ++q) {
    while (first[lo] <= q) ++lo;
    const int64_t from = (int64_t)(q - (lo ? first[lo - 1] : 0u)) * PIECE;
    const int dtype = (int)(at[lo] >> ADDRESS_BITS);
    each(reinterpret_cast<char*>(at[lo] & ((1ull << ADDRESS_BITS) - 1)) + from * (dtype == F32 ? 4 : 2), dtype, (int)min(size[lo] - from, (int64_t)PIECE));
  }
}

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
__device__ __forceinline__ double piece_squares(const char* at, int n) {
  constexpr int N = Chunk<Tag>::N;
  double sum = 0.0;
  for (int c = threadIdx.x * N; c < n; c += GRAD_NT * N) {
    if (c + N <= n) {
      float f[N];
      Chunk<Tag>::unpack(load16_stream_any(at + c * Tag::bytes), f);
#pragma unroll
      for (int e = 0; e < N; ++e) sum = fma((double)f[e], (double)f[e], sum);
    } else {
      for (int e = c; e < n; ++e) {
        const double f = (double)load_as_float(at, Tag::id, e);
        sum = fma(f, f, sum);
      }
    }
  }
  return sum;
}

__global__ __launch_bounds__(GRAD_NT) void squares_kernel(const GradTable t, double* sums) {
  __shared__ unsigned long long at[TABLE];
  __shared__ int64_t size[TABLE];
  __shared__ unsigned first[GRAD_NT];
  __shared__ double scratch[GRAD_NT / WAVE];
  double sum = 0.0;
  for_pieces(t, at, size, first, [&](const char* p, int dtype, int n) {
    sum += dtype == F32 ? piece_squares<TagF32>(p, n) : dtype == BF16 ? piece_squares<TagBF16>(p, n) : piece_squares<TagF16>(p, n);
  });
  const double total = block_total(sum, scratch);
  if (threadIdx.x == 0) sums[blockIdx.x] = total;
}

// scale * sqrt of the sums' sum: the same in every workgroup.
__device__ __forceinline__ double norm_of(const double* sums, unsigned n, float scale, double* scratch) {
  double v = 0.0;
  for (unsigned i = threadIdx.x; i < n; i += GRAD_NT) v += sums[i];
  return sqrt(block_total(v, scratch)) * (double)scale;
}
__global__ __launch_bounds__(GRAD_NT) void norm_kernel(const double* sums, unsigned n, float scale, float* norm) {
  __shared__ double scratch[GRAD_NT / WAVE];
  const double v = norm_of(sums, n, scale, scratch);
  if (threadIdx.x == 0) norm[0] = (float)v;
}

template <class Tag>
__device__ __forceinline__ void scale_piece(char* at, int n, float by) {
  constexpr int N = Chunk<Tag>::N;
  for (int c = threadIdx.x * N; c < n; c += GRAD_NT * N) {
    if (c + N <= n) {
      float f[N];
      Chunk<Tag>::unpack(load16_stream_any(at + c * Tag::bytes), f);
#pragma unroll
      for (int e = 0; e < N; ++e) f[e] *= by;
      store16_stream_any(at + c * Tag::bytes, Chunk<Tag>::pack(f));
    } else {
      for (int e = c; e < n; ++e) store_from_float(at, Tag::id, e, load_as_float(at, Tag::id, e) * by);
    }
  }
}
// `sums`: the norm is theirs, and is written; else it is there.
__global__ __launch_bounds__(GRAD_NT) void scale_kernel(const GradTable t, const double* sums, unsigned n_sums, float scale, float max_norm, float* norm) {
  __shared__ unsigned long long at[TABLE];
  __shared__ int64_t size[TABLE];
  __shared__ unsigned first[GRAD_NT];
  __shared__ double scratch[GRAD_NT / WAVE];
  const double all = sums ? norm_of(sums, n_sums, scale, scratch) : (double)norm[0];
  if (sums && blockIdx.x == 0 && threadIdx.x == 0) norm[0] = (float)all;
  const float by = (float)(all > (double)max_norm ? (double)max_norm / all * (double)scale : (double)scale);
  if (!(all <= 1.7976931348623157e308) || by == 1.f) return;   // NaN or infinite: left as they are
  for_pieces(t, at, size, first, [&](char* p, int dtype, int n) {
    if (dtype == F32) scale_piece<TagF32>(p, n, by);
    else if (dtype == BF16) scale_piece<TagBF16>(p, n, by);
    else scale_piece<TagF16>(p, n, by);
  });
}

static int gradients_status() { return hipGetLastError() == hipSuccess ? DL_OK : DL_ERR_LAUNCH; }

// Table by table: `each(table, grid, the grids of the tables before)`.
template <class Each>
static unsigned for_tables(const void* const* tensors, const int64_t* sizes, const int32_t* dtypes, int64_t n, Each each) {
  unsigned before = 0;
  GradTable t;
  t.n = 0;
  int64_t pieces = 0;
  for (int64_t i = 0; i <= n; ++i) {
    if (i < n && sizes[i] == 0) continue;
    const int64_t more = i < n ? (sizes[i] + PIECE - 1) / PIECE : 0;
    if (t.n > 0 && (i == n || t.n == TABLE || pieces + more > 0x7fffffffLL)) {
      t.pieces = (unsigned)pieces;
      const unsigned grid = (unsigned)std::min<int64_t>(pieces, GRAD_GRID);
      each(t, grid, before);
      before += grid;
      t.n = 0;
      pieces = 0;
    }
    if (i == n) break;
    t.at[t.n] = reinterpret_cast<unsigned long long>(tensors[i]) | (unsigned long long)dtypes[i] << ADDRESS_BITS;
    t.size[t.n++] = sizes[i];
    pieces += more;
  }
  return before;
}

static int gradients_check(const void* const* tensors, const int64_t* sizes, const int32_t* dtypes, int64_t n, float scale, bool apart) {
  if (n < 0 || !(scale > 0.f) || !(scale <= 3.4e38f)) return DL_ERR_SHAPE;
  if (n > 0 && (!tensors || !sizes || !dtypes)) return DL_ERR_NULL;
  for (int64_t i = 0; i < n; ++i) {
    if ((unsigned)dtypes[i] > DL_F16) return DL_ERR_DTYPE;
    if (sizes[i] < 0) return DL_ERR_SHAPE;
    if (sizes[i] > 0 && !tensors[i]) return DL_ERR_NULL;
    if (reinterpret_cast<uintptr_t>(tensors[i]) % (dtypes[i] == DL_F32 ? 4 : 2)) return DL_ERR_ALIGN;
    if (reinterpret_cast<uintptr_t>(tensors[i]) >> ADDRESS_BITS || sizes[i] > (int64_t)PIECE * 0x7fffffffLL) return DL_ERR_LIMIT;
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
    const int64_t more = (sizes[i] + dl::PIECE - 1) / dl::PIECE;
    if (in == dl::TABLE || pieces + more > 0x7fffffffLL) { ++tables; in = pieces = 0; }
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
  const unsigned n = for_tables(tensors, sizes, dtypes, n_tensors, [&](const GradTable& t, unsigned grid, unsigned before) {
    hipLaunchKernelGGL(squares_kernel, dim3(grid), dim3(GRAD_NT), 0, st, t, sums + before);
  });
  hipLaunchKernelGGL(norm_kernel, dim3(1), dim3(GRAD_NT), 0, st, sums, n, scale, norm);
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
    n = for_tables(tensors, sizes, dtypes, n_tensors, [&](const GradTable& t, unsigned grid, unsigned before) {
      hipLaunchKernelGGL(squares_kernel, dim3(grid), dim3(GRAD_NT), 0, st, t, sums + before);
    });
    if (n == 0) hipLaunchKernelGGL(norm_kernel, dim3(1), dim3(GRAD_NT), 0, st, sums, n, scale, norm);
  }
  for_tables(tensors, sizes, dtypes, n_tensors, [&](const GradTable& t, unsigned grid, unsigned) {
    hipLaunchKernelGGL(scale_kernel, dim3(grid), dim3(GRAD_NT), 0, st, t, sums, n, scale, max_norm, norm);
  });
  return gradients_status();
}
