// Generalised Jensen-Shannon divergence against a top-K teacher with the rest of the vocabulary as one more outcome.
//
// Outcomes: the K listed ids and "the rest", every column that is not listed.
//   P  the teacher: exp(t_val) on the listed ids; the rest has what they leave of 1, at least rest_min; divided by their sum
//   Q  the student: softmax(x / T), the rest's columns added up
//   beta = 0: KL(P|Q);  beta = 1: KL(Q|P);  between: beta KL(P|M) + (1 - beta) KL(Q|M) with M = beta P + (1 - beta) Q
// Gradient: with s_j = q_j dL/dq_j (beta = 0: -p_j; 1: q_j log(q_j / p_j); between: (1 - beta) q_j log(q_j / m_j)) and S their sum,
//   dL/dz_k = s_k - q_k S on a listed id, and softmax over the rest's columns times (s_rest - q_rest S) on those:
// the rest's columns need one number per row, so the row is read once, written once and costs one exponential per column (two-byte
// logits: their powers stay in registers as fp16; four-byte ones: as fp32).  Bound by HBM traffic, 2 V bytes x the element size per row:
// 8192 x 128256 bf16, K = 200: 799-856 us (4.9-5.3 TB/s); 4093 x 50257, K = 100: 182-204 us (a tenth of the rows masked; 50304 columns,
// whose rows begin on 16 bytes: 15 % less); 2048 x 128256 fp32 in parts 432 us (4.9 TB/s); 131 x 32000 fp32, K = 400: 17 us, the latency
// of its phases.
//
// Layout as in the forward-KL kernels: a row, or one column part of it, sits in its workgroup's registers; parts exchange
// (max, sum) of the rest's columns through records in a workspace, with a bounded wait and a second launch for parts
// that gave up.  Listed columns are taken out of the registers (-inf in their place, by a bit per column in LDS) before the
// row's statistics, so that the rest's mass is a sum of what it consists of and not 1 minus the listed mass: a confident
// student leaves it 1e-8, which that difference would lose.  Every thread keeps a few entries in registers: their ids are asked
// for ahead of the row, their logits (all K of a row, in every part: the lines are on their way to some workgroup of the XCD
// anyway) behind it, and their maxima and sums travel in the barriers that the row's own need.
#include "topk_div.hpp"
#include "distill_hip.h"

namespace dl {

struct RestParams {
  const void* logits; int64_t row_stride, n_rows, V;
  const int32_t* row_map;
  const void* t_val; int t_val_dtype; const void* t_idx; int t_idx_itype; int K;
  int64_t n_trows; const int32_t* t_cnt;
  float beta, inv_T, rest_min, grad_scale;
  float* row_loss; void* grad; int64_t grad_stride;
  void* workspace; int parts; int spin_limit;
  // n rows from row r on
  RestParams rows(int64_t r, int64_t n, int bytes) const {
    RestParams q = *this;
    q.logits = reinterpret_cast<const char*>(logits) + r * row_stride * bytes;
    q.n_rows = n;
    if (row_loss) q.row_loss += r;
    if (grad) q.grad = reinterpret_cast<char*>(grad) + r * grad_stride * bytes;
    if (row_map) {
      q.row_map += r;
    } else {                             // row r's teacher is row r
      q.t_val = reinterpret_cast<const char*>(t_val) + r * K * (t_val_dtype == F32 ? 4 : 2);
      q.t_idx = reinterpret_cast<const char*>(t_idx) + r * K * (t_idx_itype == I64 ? 8 : 4);
      q.n_trows = n_trows > r ? n_trows - r : 0;
      if (t_cnt) q.t_cnt += r;
    }
    return q;
  }
};

// Lists of the row's entries by the 16-byte chunk of their column (chunks that share a head share a list), and a byte per
// chunk of the part: which of its columns are listed.
struct RestLds {
  int *idx, *next, *head;
  float *lp, *red, *xm, *xs;
  int* xok;
  unsigned *own, *mask;
  __device__ RestLds(unsigned char* base, int K, int threads) {
    const int Kp = (K + 3) & ~3;
    idx = reinterpret_cast<int*>(base);
    next = idx + Kp;
    lp = reinterpret_cast<float*>(next + Kp);
    red = lp + Kp;
    xm = red + 64;
    xs = xm + MAX_PARTS;
    xok = reinterpret_cast<int*>(xs + MAX_PARTS);
    head = xok + MAX_PARTS;
    own = reinterpret_cast<unsigned*>(head + CORRECTION_HEADS);
    mask = own + threads;
  }
  static size_t bytes(int K, int threads, int chunks) {
    return (size_t)(3 * ((K + 3) & ~3) + 64 + 3 * MAX_PARTS + CORRECTION_HEADS + threads + (threads * chunks + 3) / 4) * 4;
  }
};

// One outcome's part of the loss, and s = q dL/dq.  The logarithm of the mixture goes through log1p / expm1 on the side
// where the exponential is at most 1, so that it neither overflows nor loses a student close to the teacher.
__device__ __forceinline__ void rest_outcome(float lp, float lq, float beta, float& loss, float& slope) {
  const float p = expf(lp), q = expf(lq), r = lp - lq;
  if (beta == 0.f) {
    loss += p == 0.f ? 0.f : p * r;      // (an entry without mass adds nothing, where the student has none either: r is infinite)
    slope = -p;
  } else if (beta == 1.f) {
    slope = q == 0.f ? 0.f : -q * r;
    loss += slope;
  } else {
    float over_p, over_q;                // log(m / p), log(m / q)
    if (r > 0.f) {
      over_p = log1pf((1.f - beta) * expm1f(-r));
      over_q = r + over_p;
    } else {
      over_q = log1pf(beta * expm1f(r));
      over_p = over_q - r;
    }
    slope = q == 0.f ? 0.f : -(1.f - beta) * q * over_q;
    loss += slope - beta * p * over_p;
  }
}

// The listed columns of a chunk (`bits`) become -inf.
template <class Tag>
__device__ __forceinline__ void take_out(u32x4& c, unsigned bits) {
  if constexpr (Tag::bytes == 4) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c[j] = (bits >> j) & 1u ? 0xff800000u : c[j];
  } else {
    constexpr unsigned inf = Tag::id == BF16 ? 0xff80u : 0xfc00u;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      c[j] = (bits >> (2 * j)) & 1u ? (c[j] & 0xffff0000u) | inf : c[j];
      c[j] = (bits >> (2 * j + 1)) & 1u ? (c[j] & 0xffffu) | (inf << 16) : c[j];
    }
  }
}

// Makes the compiler work `v` out here: a sum that is only needed behind a branch is put off to there otherwise, and all that goes into
// it stays in registers.
__device__ __forceinline__ void keep(float& v) { asm volatile("" : "+v"(v)); }

// J entries per thread (K <= J * NT).  `RETRY`: the part is finished by the second launch; every record of the row is there.
template <class Tag, int NT, int NCH, int J, bool SPLIT, bool RETRY>
__device__ __forceinline__ void rest_part(const RestParams& p, const RestLds& s, int64_t r, int h) {
  using C = Chunk<Tag>;
  using M = ChunkMap<NT, NCH>;
  const int tid = threadIdx.x, P = SPLIT ? p.parts : 1;
  const int64_t lo = (int64_t)h * NT * NCH * C::N;
  const int n_cols = (int)min(p.V - lo, (int64_t)NT * NCH * C::N), nch = n_cols / C::N, tail = n_cols - nch * C::N;
  char* gpart = p.grad ? reinterpret_cast<char*>(p.grad) + (r * p.grad_stride + lo) * Tag::bytes : nullptr;
  const auto leave = [&]() {             // a row that counts for nothing
    if (gpart) zero_row_any<Tag, NT>(gpart, n_cols);
    if (tid == 0 && h == 0 && p.row_loss) p.row_loss[r] = 0.f;
  };
  const int64_t trow = teacher_row(p.row_map, r, p.n_trows);
  if (trow < 0) return leave();
  const char* row = reinterpret_cast<const char*>(p.logits) + r * p.row_stride * Tag::bytes;
  const char* rpart = row + lo * Tag::bytes;

  int64_t id[J];
  float lp[J], z[J];
  const int cnt = p.t_cnt ? min(p.K, max(p.t_cnt[trow], 0)) : p.K;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int k = j * NT + tid;
    id[j] = k < cnt ? load_index(p.t_idx, p.t_idx_itype, trow * p.K + k) : -1;
    lp[j] = k < cnt ? load_as_float(p.t_val, p.t_val_dtype, trow * p.K + k) : -INFINITY;
  }
  u32x4 reg[NCH];
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int c = M::chunk(i, tid);
    reg[i] = C::neg_inf();
    if (c < nch) reg[i] = load16_unaligned(rpart + (int64_t)c * 16);
    else if (c == nch && tail) reg[i] = load_chunk_elementwise<Tag>(rpart, c, n_cols);
  }
  correction_clear<NT>(s.head, s.own);
#pragma unroll
  for (int i = 0; i < (NCH + 3) / 4; ++i)
    if (i * NT + tid < (NT * NCH + 3) / 4) s.mask[i * NT + tid] = 0u;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int k = j * NT + tid;
    z[j] = -INFINITY;
    if (!(id[j] >= 0 && id[j] < p.V && lp[j] != -INFINITY)) lp[j] = -INFINITY;      // does not count
    if (k < p.K) {
      s.idx[k] = lp[j] != -INFINITY ? (int)id[j] : -1;
      s.lp[k] = lp[j];
    }
    if (lp[j] != -INFINITY) {
      s.next[k] = atomicExch(&s.head[(int)(id[j] / C::N) & (CORRECTION_HEADS - 1)], k);
      if (id[j] >= lo && id[j] < lo + n_cols) {
        const int at = (int)(id[j] - lo), c = at / C::N;
        atomicOr(&s.own[M::owner(c)], 1u << M::reg(c));
        atomicOr(&s.mask[c / 4], 1u << (8 * (c % 4) + at % C::N));
      }
      z[j] = load_as_float(row, Tag::id, id[j]);
    }
  }
  __syncthreads();
  // An id that is listed again has its masses added up, in the order of its entries, in the first of them; the others no longer count.
#pragma unroll
  for (int j = 0; j < J; ++j) {
    if (lp[j] == -INFINITY) continue;
    const int k = j * NT + tid, first = s.head[(int)(id[j] / C::N) & (CORRECTION_HEADS - 1)];
    bool again = false, later = false;
    for (int q = first; q >= 0; q = s.next[q])
      if (q != k && s.idx[q] == (int)id[j]) { again = true; later = later || q < k; }
    if (later) {
      lp[j] = -INFINITY;
    } else if (again) {
      float sum = expf(lp[j]);
      for (int at = k;;) {
        int next = p.K;
        for (int q = first; q >= 0; q = s.next[q])
          if (q > at && q < next && s.idx[q] == (int)id[j]) next = q;
        if (next == p.K) break;
        sum += expf(s.lp[next]);
        at = next;
      }
      lp[j] = logf(sum);
    }
  }
  const unsigned mine = s.own[tid];
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    forget(reg[i]);                      // (chunk by chunk: no pile-up of masks and halves)
    if (mine & (1u << i)) take_out<Tag>(reg[i], reinterpret_cast<const unsigned char*>(s.mask)[M::chunk(i, tid)]);
    forget(reg[i]);
  }

  // maxima of the rest's columns and of the listed ones; then the sums of the powers over them, and the teacher's mass.  The rest's
  // powers 2^(x a - mb), mb the largest one's x a rounded, stay in the registers for the gradient.  Logits are scaled inside fused
  // multiply-adds and only ever less a maximum: what a power or a log-probability is off by goes with its logit's distance from that
  // maximum, not with the logit (fp32 logits near 32768 in the middle of a row: losses off by 1e-3 with a product of their own).
  const float a = p.inv_T * LOG2E;
  float mx = -INFINITY, zmax = -INFINITY;
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    float f[C::N];
    forget(reg[i]);
    C::unpack(reg[i], f);
#pragma unroll
    for (int e = 0; e < C::N; ++e) mx = fmaxf(mx, f[e]);
    keep(mx);
  }
#pragma unroll
  for (int j = 0; j < J; ++j)
    if (lp[j] != -INFINITY) zmax = fmaxf(zmax, z[j]);
  block_max2<NT>(mx, zmax, s.red);
  constexpr float BIAS = C::stash_bias;
  float mb_own = mx * a - BIAS, zb = zmax * a;
  keep(mb_own);                          // (rounded here: what follows has one value for each)
  keep(zb);
  float mb = mb_own + BIAS;
  // A rest of nothing but masked columns counts as none, whatever they are masked with (distill_common.hpp: MASKED_BELOW; two-byte
  // logits are thousands apart at -2^20 already), and so does a row.
  constexpr float LOW = Tag::bytes == 2 ? -0x1p20f : MASKED_BELOW;
  const bool masked = mb < LOW;
  if (masked) { mb_own = -BIAS; mb = -INFINITY; }
  float sm = 0.f, zs = 0.f, ps = 0.f;
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    float f[C::N];
    forget(reg[i]);
    C::unpack(reg[i], f);
#pragma unroll
    for (int e = 0; e < C::N; ++e) {
      f[e] = fast_exp2(fmaf(f[e], a, -mb_own));
      sm += f[e];
    }
    keep(sm);
    reg[i] = C::stash(f);
    forget(reg[i]);
  }
  sm *= __builtin_exp2f(-BIAS);
#pragma unroll
  for (int j = 0; j < J; ++j)
    if (lp[j] != -INFINITY) {
      ps += expf(lp[j]);
      zs += zb == -INFINITY ? (z[j] == z[j] ? 0.f : z[j]) : fast_exp2(fmaf(z[j], a, -zb));
    }
  block_sum3<NT>(sm, zs, ps, s.red);

  if (SPLIT) {
    PartStats* ws = reinterpret_cast<PartStats*>(p.workspace) + r * P;
    if (tid == 0 && !RETRY) part_publish(ws + h, mb, sm, 0.f);
    if (tid < P) {
      float om = mb, os = sm, ob;
      s.xok[tid] = (tid == h) || part_collect(ws + tid, RETRY ? 0x7fffffff : p.spin_limit, om, os, ob);
      s.xm[tid] = om; s.xs[tid] = os;
    }
    __syncthreads();
    bool all_ok = true;
    for (int j = 0; j < P; ++j) all_ok = all_ok && (s.xok[j] != 0);
    if (!all_ok) {                       // nothing is written yet; the part's own record is out
      if (tid == 0) {
        RetryList list(p.workspace, p.n_rows, P);
        list.entries[atomicAdd(list.count, 1u)] = (unsigned)(r * P + h);
      }
      return;
    }
    float top = s.xm[0];
    for (int j = 1; j < P; ++j) top = fmaxf(top, s.xm[j]);
    float S = 0.f;
    if (top == -INFINITY) {
      for (int j = 0; j < P; ++j) S += s.xs[j];                       // 0, or NaN
    } else {
      for (int j = 0; j < P; ++j) S += s.xs[j] * fast_exp2(s.xm[j] - top);
    }
    mb = top;
    sm = S;
  }

  // the K outcomes and the rest (none where no column outside the list has an unmasked logit: a sum of 0)
  const bool rest = !(sm == 0.f);
  if (!rest && zb < LOW && zs == zs) return leave();                  // no unmasked logit (nor NaN)
  if (!rest && ps == 0.f) return leave();                             // nothing to compare
  const float top = rest ? fmaxf(zb, mb) : zb, lr = fast_log2(sm);    // (lr: log2 of the rest's sum, from mb on)
  const float lse = fast_log2((zb == -INFINITY ? zs : zs * fast_exp2(zb - top)) + (rest ? sm * fast_exp2(mb - top) : 0.f));      // from top on
  const float p0 = rest ? fmaxf(1.f - ps, p.rest_min) : 0.f, lz = logf(ps + p0);
  float loss = 0.f, slopes = 0.f, slope[J];
#pragma unroll
  for (int j = 0; j < J; ++j)
    if (lp[j] != -INFINITY) {
      rest_outcome(lp[j] - lz, (fmaf(z[j], a, -top) - lse) * LN2, p.beta, loss, slope[j]);
      slopes += slope[j];
    }
  block_sum2<NT>(loss, slopes, s.red);
  float slope0 = 0.f, q0 = 0.f;
  if (rest) {
    const float lq0 = (mb - top + (lr - lse)) * LN2;
    rest_outcome(logf(p0) - lz, lq0, p.beta, loss, slope0);
    slopes += slope0;
    q0 = expf(lq0);
  }
  if (tid == 0 && h == 0 && p.row_loss) p.row_loss[r] = loss;
  if (!gpart) return;
  const float c = p.inv_T * p.grad_scale;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int k = j * NT + tid;
    if (lp[j] != -INFINITY) s.lp[k] = (slope[j] - fast_exp2(fmaf(z[j], a, -top) - lse) * slopes) * c;
    else if (k < p.K) s.idx[k] = -1;
  }
  const float kc = !rest || masked ? 0.f : fast_exp2(mb_own - mb - lr) * (slope0 - q0 * slopes) * c;      // stashed power -> gradient
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int ch = M::chunk(i, tid);
    if (ch < nch || (ch == nch && tail)) {
      float f[C::N];
      forget(reg[i]);
      C::unstash(reg[i], f);
#pragma unroll
      for (int e = 0; e < C::N; ++e) f[e] *= kc;
      if (mine & (1u << i)) {
        const int gc = (int)(lo / C::N) + ch;
        for (int k = s.head[gc & (CORRECTION_HEADS - 1)]; k >= 0; k = s.next[k]) {
          const int e = s.idx[k] - gc * C::N;
          if (e < 0 || e >= C::N) continue;                           // (entries that do not count: -1)
          const float v = s.lp[k];
#pragma unroll
          for (int j = 0; j < C::N; ++j) f[j] = j == e ? v : f[j];
        }
      }
      if (ch < nch) store16_stream_any(gpart + (int64_t)ch * 16, C::pack(f));
      else store_chunk_elementwise<Tag>(gpart, ch, n_cols, C::pack(f));
    }
  }
}

template <class Tag, int NT, int NCH, int J, bool SPLIT>
__global__ __launch_bounds__(NT) __attribute__((amdgpu_waves_per_eu(4, 8))) void rest_kernel(const RestParams p) {
  extern __shared__ __align__(16) unsigned char smem[];
  const RestLds s(smem, p.K, NT);
  const int P = SPLIT ? p.parts : 1;
  const unsigned grp = SPLIT ? blockIdx.x / (8u * P) : 0u, t_in = SPLIT ? blockIdx.x % (8u * P) : 0u;
  const int64_t r = SPLIT ? (int64_t)grp * 8 + (t_in & 7u) : xcd_banded_row(blockIdx.x);
  if (r >= p.n_rows) return;
  rest_part<Tag, NT, NCH, J, SPLIT, false>(p, s, r, SPLIT ? (int)(t_in >> 3) : 0);
}

template <class Tag, int NT, int NCH, int J>
__device__ __attribute__((noinline)) void rest_part_again(const RestParams& p, const RestLds& s, unsigned at) {
  rest_part<Tag, NT, NCH, J, true, true>(p, s, (int64_t)(at / (unsigned)p.parts), (int)(at % (unsigned)p.parts));
}
template <class Tag, int NT, int NCH, int J>
__global__ __launch_bounds__(NT) __attribute__((amdgpu_waves_per_eu(4, 8))) void rest_retry_kernel(const RestParams p) {
  extern __shared__ __align__(16) unsigned char smem[];
  const RestLds s(smem, p.K, NT);
  const RetryList list(p.workspace, p.n_rows, p.parts);
  const unsigned n = *list.count;
#pragma unroll 1
  for (unsigned e = blockIdx.x; e < n; e += gridDim.x) {
    rest_part_again<Tag, NT, NCH, J>(p, s, list.entries[e]);
    __syncthreads();
  }
}

// Threads and chunks per thread of a workgroup, parts per row, for rows of `nch` chunks (parts == 0: too wide).  Rows stay whole as far as
// 512 threads' registers go (us, whole / in parts, K = 200 bf16: 64 x 50304 16.9 / 23.6, 4096 x 50304 174 / 188, 4096 x 50257 201 / 212,
// 1024 x 65536 59.9 / 67.3).
struct RestShape { int NT, NCH, parts; };
static RestShape rest_shape(int64_t nch) {
  if (nch <= 256 * 4) return {256, 4, 1};
  if (nch <= 256 * 8) return {256, 8, 1};
  if (nch <= 512 * 8) return {512, 8, 1};
  if (nch <= 512 * 13) return {512, 13, 1};
  if (nch <= 512 * 16) return {512, 16, 1};
  const int64_t parts = (nch + 256 * 16 - 1) / (256 * 16);
  if (parts > MAX_PARTS) return {0, 0, 0};
  const int64_t per_thread = (nch + parts * 256 - 1) / (parts * 256);
  return {256, per_thread <= 13 ? 13 : per_thread <= 14 ? 14 : 16, (int)parts};
}

// Entries per thread: two, or as many as the most entries ask for (us at K = 200 for 2 / as many: 4096 x 50304 174 / 223,
// 4096 x 128256 417 / 439).
template <class Tag, int NT, int NCH, int J>
static void launch_rest_row_j(const RestParams& p, hipStream_t st) {
  hipLaunchKernelGGL((rest_kernel<Tag, NT, NCH, J, false>), dim3(xcd_banded_grid(p.n_rows)), dim3(NT), RestLds::bytes(p.K, NT, NCH), st, p);
}
template <class Tag, int NT, int NCH>
static void launch_rest_row(const RestParams& p, hipStream_t st) {
  if (p.K <= 2 * NT) launch_rest_row_j<Tag, NT, NCH, 2>(p, st);
  else launch_rest_row_j<Tag, NT, NCH, DL_MAX_TOPK / NT>(p, st);
}
template <class Tag, int NT, int NCH, int J>
static void launch_rest_parts_j(const RestParams& p, hipStream_t st) {
  const size_t lds = RestLds::bytes(p.K, NT, NCH);
  hipLaunchKernelGGL((rest_kernel<Tag, NT, NCH, J, true>), dim3((unsigned)((p.n_rows + 7) / 8 * 8 * p.parts)), dim3(NT), lds, st, p);
  hipLaunchKernelGGL((rest_retry_kernel<Tag, NT, NCH, J>), dim3((unsigned)std::min<int64_t>(p.n_rows * p.parts, 256)), dim3(NT), lds, st, p);
}
template <class Tag, int NT, int NCH>
static void launch_rest_parts(const RestParams& p, hipStream_t st) {
  const int64_t n16 = split_clear_words(p.n_rows, p.parts);
  hipLaunchKernelGGL(clear_workspace_kernel<256>, dim3((unsigned)((n16 + 255) / 256)), dim3(256), 0, st, reinterpret_cast<u32x4*>(p.workspace), n16);
  if (p.K <= 2 * NT) launch_rest_parts_j<Tag, NT, NCH, 2>(p, st);
  else launch_rest_parts_j<Tag, NT, NCH, DL_MAX_TOPK / NT>(p, st);
}

template <class Tag>
static int launch_rest(const RestParams& all, const RestShape& sh, hipStream_t st) {
  // rows of a launch (one launch up to 8388544 rows that stay whole); launches follow each other on the same workspace
  const int64_t most = LAUNCH_THREADS / (sh.NT * sh.parts) / 64 * 64;
  for (int64_t r = 0; r < all.n_rows; r += most) {
    const RestParams p = all.rows(r, std::min(most, all.n_rows - r), Tag::bytes);
    if (sh.parts == 1) {
      if (sh.NT == 256) sh.NCH == 4 ? launch_rest_row<Tag, 256, 4>(p, st) : launch_rest_row<Tag, 256, 8>(p, st);
      else if (sh.NCH == 8) launch_rest_row<Tag, 512, 8>(p, st);
      else if (sh.NCH == 13) launch_rest_row<Tag, 512, 13>(p, st);
      else launch_rest_row<Tag, 512, 16>(p, st);
    } else {
      if (sh.NCH == 13) launch_rest_parts<Tag, 256, 13>(p, st);
      else if (sh.NCH == 14) launch_rest_parts<Tag, 256, 14>(p, st);
      else launch_rest_parts<Tag, 256, 16>(p, st);
    }
  }
  return launch_status();
}

static int64_t rest_chunks(int dtype, int64_t V) { return dtype == DL_F32 ? (V + 3) / 4 : (V + 7) / 8; }

}  // namespace dl

extern "C" int64_t dl_div_topk_rest_workspace_bytes(int dtype, int64_t n_rows, int64_t V) {
  using namespace dl;
  if ((unsigned)dtype > DL_F16 || n_rows <= 0 || V <= 0) return 0;
  const RestShape sh = rest_shape(rest_chunks(dtype, V));
  return sh.parts > 1 ? RetryList::bytes(n_rows, sh.parts) : 0;
}

extern "C" int dl_div_topk_rest(float beta, const void* logits, int logits_dtype, int64_t row_stride, int64_t n_rows, int64_t V,
                                const int32_t* row_map, const void* t_val, int t_val_dtype, const void* t_idx, int t_idx_itype, int K,
                                int64_t n_teacher_rows, const int32_t* t_cnt, float inv_T, float rest_min, float grad_scale,
                                float* row_loss, void* grad, int64_t grad_stride, void* workspace, int64_t workspace_bytes, int flags,
                                void* stream) {
  using namespace dl;
  if ((unsigned)logits_dtype > DL_F16 || (unsigned)t_val_dtype > DL_F16 || (unsigned)t_idx_itype > DL_I64) return DL_ERR_DTYPE;
  if (n_rows < 0 || V <= 0 || K < 0 || n_teacher_rows < 0 || row_stride < V || (grad && grad_stride < V)) return DL_ERR_SHAPE;
  if (!(beta >= 0.f && beta <= 1.f) || !(rest_min > 0.f && rest_min < 1.f) || !(inv_T > 0.f)) return DL_ERR_SHAPE;
  if (n_rows == 0) return DL_OK;
  if (!logits || (n_teacher_rows > 0 && K > 0 && (!t_val || !t_idx)) || (!row_loss && !grad)) return DL_ERR_NULL;
  if (K > DL_MAX_TOPK) return DL_ERR_LIMIT;
  const uintptr_t eb = logits_dtype == DL_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(logits) % eb || reinterpret_cast<uintptr_t>(grad) % eb || reinterpret_cast<uintptr_t>(workspace) % 16 ||
      reinterpret_cast<uintptr_t>(t_val) % (t_val_dtype == DL_F32 ? 4 : 2) || reinterpret_cast<uintptr_t>(t_idx) % (t_idx_itype == DL_I64 ? 8 : 4))
    return DL_ERR_ALIGN;
  const RestShape sh = rest_shape(rest_chunks(logits_dtype, V));
  if (sh.parts == 0 || (n_rows + 64) * sh.parts > 0x7fffffffLL) return DL_ERR_LIMIT;
  if (sh.parts > 1 && (!workspace || workspace_bytes < RetryList::bytes(n_rows, sh.parts))) return DL_ERR_WORKSPACE;
  RestParams p{logits, row_stride, n_rows, V, row_map, t_val, t_val_dtype, t_idx, t_idx_itype, K, n_teacher_rows, t_cnt, beta, inv_T, rest_min,
               grad_scale, row_loss, grad, grad_stride, workspace, sh.parts, (flags & DL_TOPK_NO_WAIT) ? 0 : SPIN_LIMIT};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (logits_dtype == DL_F32) return launch_rest<TagF32>(p, sh, st);
  if (logits_dtype == DL_BF16) return launch_rest<TagBF16>(p, sh, st);
  return launch_rest<TagF16>(p, sh, st);
}
