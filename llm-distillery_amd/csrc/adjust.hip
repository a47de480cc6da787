// Logits made ready for the sampler, and the gradient of that.
//
//   y = x > 0 ? x / repetition : x * repetition          for the tokens of the row's text
//   y -= frequency * count + presence                    for those behind the text's prompt, `count` times there
//   y += bias;   y = -inf where the row's mask has no bit
//
// A workgroup has a row, or a part of its columns.  It counts the text's tokens that fall into its columns in LDS -- whole numbers, so
// the order of the additions does not show -- and then goes through the columns once.  The gradient (by x: g, times what the penalty
// multiplied with; by a bias that the rows share: the sum of g over the rows, both 0 where the mask has no bit) needs of x only the sign
// at the text's tokens.
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
  const int32_t *token_rows, *lengths, *prompt; int64_t prompt_all;
  const float *repetition, *frequency, *presence; float repetition_all, frequency_all, presence_all;
  const char* bias; int bias_dtype; int64_t bias_stride;
  const unsigned* allowed; int64_t allowed_stride, n_masks; const int32_t* allowed_rows;
  unsigned parts, part_columns;
  int64_t first_row;
};

// What a row has besides its logits.
struct AdjustRow {
  const char* text;
  int64_t length, prompt;                                      // entries that count, and how many of them are the prompt's
  float repetition, frequency, presence;
  const unsigned char* bits;                                   // its mask, or nothing
  __device__ __forceinline__ AdjustRow(const AdjustParams& p, int64_t r) {
    repetition = p.repetition ? p.repetition[r] : p.repetition_all;
    frequency = p.frequency ? p.frequency[r] : p.frequency_all;
    presence = p.presence ? p.presence[r] : p.presence_all;
    int64_t t = p.token_rows ? (int64_t)p.token_rows[r] : p.n_texts == 1 ? 0 : r;
    length = p.lengths ? min((int64_t)p.lengths[r], p.length) : p.length;
    if (t < 0 || t >= p.n_texts || length < 0 || (repetition == 1.f && frequency == 0.f && presence == 0.f)) t = length = 0;
    prompt = p.prompt ? (int64_t)p.prompt[r] : p.prompt_all;
    text = p.tokens + t * p.token_stride * (p.itype == I64 ? 8 : 4);
    const int64_t m = p.allowed_rows ? (int64_t)p.allowed_rows[r] : p.n_masks == 1 ? 0 : r;
    bits = m >= 0 && m < p.n_masks ? reinterpret_cast<const unsigned char*>(p.allowed + m * p.allowed_stride) : nullptr;
  }
};

// The counters of a part's columns: one 32-bit word a column (WIDE), or half a word, whose top bit says that the prompt has the token and
// whose other bits count up to 32767 tokens behind it.
template <bool WIDE>
struct Counters {
  static constexpr unsigned PROMPT = WIDE ? 0x80000000u : 0x8000u;
  static constexpr int64_t MOST = WIDE ? 0x7fffffff : 0x7fff;
  __device__ static __forceinline__ void add(unsigned* words, unsigned column, bool prompt) {
    unsigned* w = words + (WIDE ? column : column >> 1);
    const unsigned at = WIDE ? 0u : (column & 1u) * 16u;
    if (prompt) atomicOr(w, PROMPT << at);
    else atomicAdd(w, 1u << at);
  }
  // The counters of N neighbouring columns; whether there is any.
  template <int N>
  __device__ static __forceinline__ bool load(const unsigned* words, unsigned column, unsigned (&c)[N]) {
    constexpr int W = WIDE ? N : N / 2;
    unsigned w[W], any = 0u;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      w[i] = words[(WIDE ? column : column >> 1) + i];
      any |= w[i];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) c[i] = WIDE ? w[i % W] : (w[i / 2] >> (i % 2 * 16)) & 0xffffu;
    return any != 0u;
  }
};

// N values from column `col` on of a row of V (those that are there), as floats.
template <class Tag>
__device__ __forceinline__ u32x4 load_columns(const char* row, int64_t col, int64_t V) {
  if (col + Chunk<Tag>::N <= V) return load16_stream_any(row + col * Tag::bytes);
  return load_chunk_elementwise<Tag>(row + col * Tag::bytes, 0, (int)(V - col));
}
template <class Tag>
__device__ __forceinline__ void store_columns(char* row, int64_t col, int64_t V, const u32x4& v) {
  if (col + Chunk<Tag>::N <= V) store16_stream_any(row + col * Tag::bytes, v);
  else store_chunk_elementwise<Tag>(row + col * Tag::bytes, 0, (int)(V - col), v);
}
template <int N>
__device__ __forceinline__ unsigned mask_bits(const unsigned char* bits, int64_t col) {
  return N == 8 ? bits[col >> 3] : (bits[col >> 3] >> (col & 4)) & 15u;
}

template <class Tag, int NT, int NCH, bool WIDE, bool GRAD>
__global__ __launch_bounds__(NT) void adjust_kernel(const AdjustParams p) {
  constexpr int N = Chunk<Tag>::N;
  extern __shared__ __align__(16) unsigned counts[];
  const unsigned group = blockIdx.x / (8u * p.parts), in = blockIdx.x % (8u * p.parts);      // the parts of a row on one XCD
  const int64_t r = p.first_row + (int64_t)group * 8 + (in & 7u);
  if (r >= p.n_rows) return;
  const int64_t c0 = (int64_t)(in >> 3) * p.part_columns, columns = min((int64_t)p.part_columns, p.V - c0);
  const AdjustRow row(p, r);
  const char* from = (GRAD ? p.g + r * p.g_stride * Tag::bytes : p.x + r * p.x_stride * Tag::bytes) + c0 * Tag::bytes;
  char* to = p.out + r * p.out_stride * Tag::bytes + c0 * Tag::bytes;
  u32x4 v[NCH];
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int64_t col = (int64_t)(i * NT + (int)threadIdx.x) * N;
    if (col < columns) v[i] = load_columns<Tag>(from, col, columns);
  }
  if (row.length > 0) {
    for (unsigned i = threadIdx.x; i < p.part_columns / (WIDE ? 4u : 8u); i += NT) reinterpret_cast<u32x4*>(counts)[i] = u32x4{0u, 0u, 0u, 0u};
    __syncthreads();
    for (int64_t i = threadIdx.x; i < row.length; i += NT) {
      const int64_t c = load_index(row.text, p.itype, i) - c0;
      if (c >= 0 && c < columns) Counters<WIDE>::add(counts, (unsigned)c, GRAD || i < row.prompt);
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int64_t col = (int64_t)(i * NT + (int)threadIdx.x) * N;
    if (col >= columns) break;
    float f[N];
    Chunk<Tag>::unpack(v[i], f);
    unsigned c[N];
    if (row.length > 0 && Counters<WIDE>::template load<N>(counts, (unsigned)col, c)) {
      float x[N];
      if (GRAD) Chunk<Tag>::unpack(load_columns<Tag>(p.x + (r * p.x_stride + c0) * Tag::bytes, col, columns), x);
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (c[e]) {
          f[e] = (GRAD ? x[e] : f[e]) > 0.f ? f[e] / row.repetition : f[e] * row.repetition;
          const unsigned count = c[e] & (Counters<WIDE>::PROMPT - 1u);
          if (!GRAD && count) f[e] -= row.frequency * (float)count + row.presence;
        }
    }
    if (!GRAD && p.bias) {
      const char* b = p.bias + (r * p.bias_stride + c0) * (p.bias_dtype == F32 ? 4 : 2);
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (col + e < columns) f[e] += load_as_float(b, p.bias_dtype, col + e);
    }
    if (row.bits) {
      const unsigned m = mask_bits<N>(row.bits, c0 + col);
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (!(m >> e & 1u)) f[e] = GRAD ? 0.f : -__builtin_inff();
    }
    store_columns<Tag>(to, col, columns, Chunk<Tag>::pack(f));
  }
}

// The gradient of a bias that the rows share: sums over `rows` rows at a time in fp32, the sums' in fp64.
template <class Tag, int NT>
__global__ __launch_bounds__(NT) void bias_sums_kernel(const AdjustParams p, float* sums, int64_t rows) {
  constexpr int N = Chunk<Tag>::N;
  const int64_t col = ((int64_t)blockIdx.x * NT + threadIdx.x) * N, first = (int64_t)blockIdx.y * rows;
  if (col >= p.V) return;
  float total[N] = {};
  for (int64_t r = first; r < min(first + rows, p.n_rows); ++r) {
    const AdjustRow row(p, r);
    const unsigned m = row.bits ? mask_bits<N>(row.bits, col) : 255u;
    float f[N];
    Chunk<Tag>::unpack(load_columns<Tag>(p.g + r * p.g_stride * Tag::bytes, col, p.V), f);
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (m >> e & 1u) total[e] += f[e];
  }
#pragma unroll
  for (int e = 0; e < N; ++e)
    if (col + e < p.V) sums[(int64_t)blockIdx.y * p.V + col + e] = total[e];
}
template <int NT>
__global__ __launch_bounds__(NT) void bias_join_kernel(const float* sums, int64_t groups, int64_t V, void* out, int dtype) {
  const int64_t col = (int64_t)blockIdx.x * NT + threadIdx.x;
  if (col >= V) return;
  double total = 0.0;
  for (int64_t k = 0; k < groups; ++k) total += (double)sums[k * V + col];
  store_from_float(out, dtype, col, (float)total);
}

static int adjust_status() { return hipGetLastError() == hipSuccess ? DL_OK : DL_ERR_LAUNCH; }

template <class Tag, int NT, int NCH, bool WIDE, bool GRAD>
static void launch_adjust(AdjustParams p, hipStream_t st) {
  const int64_t most = (int64_t)NT * NCH * Chunk<Tag>::N;
  p.parts = (unsigned)((p.V + most - 1) / most);
  p.part_columns = (unsigned)((p.V + p.parts - 1) / p.parts + 31) / 32 * 32;
  const size_t lds = p.length > 0 ? p.part_columns * (WIDE ? 4 : 2) : 0;
  const int64_t slice = LAUNCH_THREADS / NT / p.parts / 8 * 8;      // rows of a launch
  for (p.first_row = 0; p.first_row < p.n_rows; p.first_row += slice) {
    AdjustParams q = p;
    q.n_rows = std::min(p.n_rows, p.first_row + slice);
    hipLaunchKernelGGL((adjust_kernel<Tag, NT, NCH, WIDE, GRAD>), dim3((unsigned)((q.n_rows - q.first_row + 7) / 8 * 8) * p.parts), dim3(NT), lds, st, q);
  }
}
template <class Tag, bool GRAD>
static void adjust_rows(const AdjustParams& p, hipStream_t st) {
  if (p.length > Counters<false>::MOST) launch_adjust<Tag, 256, 4, true, GRAD>(p, st);
  else launch_adjust<Tag, 256, 4, false, GRAD>(p, st);
}

// Rows that one thread adds up: 64, or as many as leave no more runs than a launch has blocks in y.
static int64_t bias_rows(int64_t n_rows) { return std::max<int64_t>(64, (n_rows + 65534) / 65535); }

// What both entry points ask of their common arguments.
static int adjust_check(const AdjustParams& p, int dtype) {
  if (p.n_rows < 0 || p.V < 0 || p.x_stride < p.V || p.out_stride < p.V || p.n_texts < 0 || p.length < 0 || p.n_masks < 0) return DL_ERR_SHAPE;
  if (p.n_texts > 0 && (p.token_stride < 0 || (p.n_texts > 1 && !p.token_rows && p.n_texts < p.n_rows))) return DL_ERR_SHAPE;
  if (p.n_masks > 0 && (p.allowed_stride < (p.V + 31) / 32 || (p.n_masks > 1 && !p.allowed_rows && p.n_masks < p.n_rows))) return DL_ERR_SHAPE;
  if (p.bias && p.bias_stride != 0 && p.bias_stride < p.V) return DL_ERR_SHAPE;
  if (p.V > 0x7fffffffLL || p.length > 0x7fffffffLL) return DL_ERR_LIMIT;
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
                 reinterpret_cast<const char*>(tokens), itype, token_stride, n_texts, n_texts ? length : 0, token_rows, lengths, prompt, prompt_all,
                 repetition, frequency, presence, repetition_all, frequency_all, presence_all,
                 reinterpret_cast<const char*>(bias), bias_dtype, bias_stride,
                 reinterpret_cast<const unsigned*>(allowed), allowed_stride, n_masks, allowed_rows, 0, 0, 0};
  if (const int bad = adjust_check(p, dtype)) return bad;
  if (n_rows == 0 || V == 0) return DL_OK;
  if (!logits || !out) return DL_ERR_NULL;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (dtype == DL_F32) adjust_rows<TagF32, false>(p, st);
  else if (dtype == DL_BF16) adjust_rows<TagBF16, false>(p, st);
  else adjust_rows<TagF16, false>(p, st);
  return adjust_status();
}

extern "C" int64_t dl_adjust_grad_workspace_bytes(int64_t n_rows, int64_t V) {
  if (n_rows <= 0 || V <= 0) return 0;
  const int64_t rows = dl::bias_rows(n_rows);
  return (n_rows + rows - 1) / rows * V * 4;
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
                 reinterpret_cast<const unsigned*>(allowed), allowed_stride, n_masks, allowed_rows, 0, 0, 0};
  if (grad_stride < V) return DL_ERR_SHAPE;
  if (const int bad = adjust_check(p, dtype)) return bad;
  if (V == 0 || (n_rows == 0 && !bias_grad)) return DL_OK;
  if ((n_rows > 0 && !grad) || (out && p.length > 0 && !logits)) return DL_ERR_NULL;
  const uintptr_t eb = dtype == DL_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(grad) % eb || reinterpret_cast<uintptr_t>(bias_grad) % (bias_dtype == DL_F32 ? 4 : 2) || reinterpret_cast<uintptr_t>(workspace) % 16)
    return DL_ERR_ALIGN;
  const int64_t run = bias_rows(n_rows), groups = (n_rows + run - 1) / run;
  if (bias_grad && groups > 0 && (!workspace || workspace_bytes < dl_adjust_grad_workspace_bytes(n_rows, V))) return DL_ERR_WORKSPACE;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (bias_grad) {
    float* sums = reinterpret_cast<float*>(workspace);
    const dim3 grid((unsigned)((V + 256 * 16 / eb - 1) / (256 * 16 / eb)), (unsigned)groups);
    if (groups > 0) {
      if (dtype == DL_F32) hipLaunchKernelGGL((bias_sums_kernel<TagF32, 256>), grid, dim3(256), 0, st, p, sums, run);
      else if (dtype == DL_BF16) hipLaunchKernelGGL((bias_sums_kernel<TagBF16, 256>), grid, dim3(256), 0, st, p, sums, run);
      else hipLaunchKernelGGL((bias_sums_kernel<TagF16, 256>), grid, dim3(256), 0, st, p, sums, run);
    }
    hipLaunchKernelGGL((bias_join_kernel<256>), dim3((unsigned)((V + 255) / 256)), dim3(256), 0, st, sums, groups, V, bias_grad, bias_dtype);
  }
  if (out && n_rows > 0) {
    if (dtype == DL_F32) adjust_rows<TagF32, true>(p, st);
    else if (dtype == DL_BF16) adjust_rows<TagBF16, true>(p, st);
    else adjust_rows<TagF16, true>(p, st);
  }
  return adjust_status();
}
