// What the products over 8-bit operands share: whole rows in, tiles of rows through LDS, rows out.
#pragma once
#include "distill_common.hpp"

namespace dl {

typedef float f32x4 __attribute__((ext_vector_type(4)));

// Eight neighbouring values of a row, zeros behind its last column.
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

typedef const unsigned __attribute__((address_space(1))) * global_words;
typedef unsigned __attribute__((address_space(3))) * lds_words;

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

}  // namespace dl
