// Matrix product in 8-bit integers with a scale for every row of either operand, and what makes its operands.
//
//   out[m, n] = (sum over k of a[m, k] * b[n, k]) * (sa[m] * sb[n])
//
// a: states, quantised on the way; b: weights, a row for every output channel.  Sums are exact: v_mfma_i32_16x16x64_i8 adds 64 products at a
// time in 32-bit integers, and K_MOST of the largest stay below 2^31.  The operands are passed with b first: a lane then holds four
// neighbouring columns n of one row m, and the result is stored in pieces of four.
#include "distill_common.hpp"
#include "distill_hip.h"

#include <algorithm>

namespace dl {

typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int KB = 128;                                        // columns are stored in whole blocks of these
constexpr int64_t K_MOST = 130944;                             // 1023 blocks: 128 * 128 as often stays below 2^31
constexpr float ISCALE = 1.f / 127.f, ISCALE_MIN = 0x1p-100f;

// ---- quantise ---------------------------------------------------------------------------------------
// A workgroup a row, twice: for its largest magnitude, and for the codes.
template <class Tag>
__device__ __forceinline__ void load_some(const char* row, int64_t col, int64_t cols, float* f) {      // eight
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
      load_some<Tag>(x, col, p.cols, f);
#pragma unroll
      for (int e = 0; e < 8; ++e) m = not_finite(f[e]) ? __builtin_inff() : fmaxf(m, fabsf(f[e]));
    }
    m = block_max<NT>(m, red);
    const bool odd = not_finite(m);
    const float scale = fmaxf(m * ISCALE, ISCALE_MIN);
    if (threadIdx.x == 0) p.scales[row] = odd ? __builtin_nanf("") : scale;
    for (int64_t col = threadIdx.x * 8; col < p.width; col += NT * 8) {
      float f[8];
      load_some<Tag>(x, col, p.cols, f);
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
template <class Tag>
__device__ __forceinline__ void store_four_columns(char* row, int64_t n, int64_t N, const float* v) {
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

// Tiles of BM x BN, a wave WM x WN of it, a block of 128 columns at a time through LDS.  A row of a tile is 128 bytes, its eight 16-byte
// pieces permuted by piece ^ (row % 8).
template <class Tag, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__((BM / WM) * (BN / WN) * WAVE) void rows_kernel(const RowsParams p) {
  constexpr int NT = (BM / WM) * (BN / WN) * WAVE, TM = WM / 16, TN = WN / 16;
  __shared__ __align__(16) unsigned char lds[(BM + BN) * KB];
  const int lane = threadIdx.x & (WAVE - 1), w = threadIdx.x / WAVE, i16 = lane % 16, quad = lane / 16;
  const int wm = (w / (BN / WN)) * WM, wn = (w % (BN / WN)) * WN;
  const int64_t m0 = (int64_t)blockIdx.x * BM, n0 = (int64_t)blockIdx.y * BN;
  i32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
  for (int kb = 0; kb < p.blocks; ++kb) {
    for (int c = threadIdx.x; c < (BM + BN) * 8; c += NT) {
      const int row = c / 8, piece = c % 8;
      const unsigned char* from = row < BM ? p.a + min(m0 + row, p.M - 1) * p.a_stride : p.b + min(n0 + row - BM, p.N - 1) * p.b_stride;
      *reinterpret_cast<u32x4*>(lds + row * KB + (piece ^ (row & 7)) * 16) = *reinterpret_cast<const u32x4*>(from + (int64_t)kb * KB + piece * 16);
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      i32x4 af[TM], bf[TN];
#pragma unroll
      for (int i = 0; i < TM; ++i) af[i] = *reinterpret_cast<const i32x4*>(lds + (wm + i * 16 + i16) * KB + ((h * 4 + quad) ^ (i16 & 7)) * 16);
#pragma unroll
      for (int j = 0; j < TN; ++j) bf[j] = *reinterpret_cast<const i32x4*>(lds + (BM + wn + j * 16 + i16) * KB + ((h * 4 + quad) ^ (i16 & 7)) * 16);
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(bf[j], af[i], acc[i][j], 0, 0, 0);
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int64_t m = m0 + wm + i * 16 + i16;
    if (m >= p.M) continue;
    const float sa = p.sa[m];
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int64_t n = n0 + wn + j * 16 + quad * 4;
      if (n >= p.N) continue;
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = (float)acc[i][j][e] * (sa * p.sb[min(n + e, p.N - 1)]);
      store_four_columns<Tag>(p.out + m * p.out_stride * Tag::bytes, n, p.N, v);
    }
  }
}

static int rows_status() { return hipGetLastError() == hipSuccess ? DL_OK : DL_ERR_LAUNCH; }

template <class Tag>
static int launch_rows(const RowsParams& p, hipStream_t st) {
  constexpr int B = 128;
  const int64_t tm = (p.M + B - 1) / B, tn = (p.N + B - 1) / B;
  if (tm * tn * 256 > LAUNCH_THREADS || tn > 65535) return DL_ERR_LIMIT;
  hipLaunchKernelGGL((rows_kernel<Tag, B, B, 64, 64>), dim3((unsigned)tm, (unsigned)tn), dim3(256), 0, st, p);
  return rows_status();
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
