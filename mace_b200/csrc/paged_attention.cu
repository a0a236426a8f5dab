// Attention of one new token per sequence over a paged key-value cache.
//
//   s_j = scale q . k_j,   out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),   lse = m + log sum_j e^(s_j - m)
//
// One pass over the cache with a running maximum m; exponentials are powers of two, so that scale log2(e) is one factor.  A block
// has one run of slots of one kv head and up to ROWS of the query heads that share it, so that a slot is read once for all of them;
// the runs are as many as fill the SMs, and the block that arrives last of a head's runs joins them.
// Slots behind the length, outside the window or in a page that the pool lacks are -inf before the maximum, and their values
// zeros: 0 times the NaN that an unused row may hold would be NaN.
#include <cmath>

#include "elements.cuh"
#include "kv_cache.h"
#include "sm100_ptx.cuh"

namespace {

constexpr int THREADS = 128;
constexpr int WARPS = THREADS / 32;
constexpr int MAX_SPLITS = 128;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

struct AttentionParams {
  const void *q, *k, *v;
  const int32_t *table, *lengths;
  void *out;
  float *lse;
  float *logits;        // [batch][heads][logits_stride], in powers of two; null: no weights asked for
  float *lse2;          // [batch][heads], beside them
  float *partial;       // of (unit, run): row maxima, row sums, rows of dim
  unsigned *arrived;    // of a unit
  const float *weights_in;
  float *weights_out;
  int64_t q_stride, out_stride, num_pages, logits_stride, weights_stride, window;
  int heads, kv_heads, group, blocks, dim, page_size, max_pages, longest, splits, split_len;
  uint32_t page_mul, page_shift;
  float scale2;         // scale log2(e)
  int *status;
};

// Which part of the problem a block has.
struct Place {
  int unit, batch, kv_head, head0, heads, split, active, begin, end;
  __device__ __forceinline__ Place(const AttentionParams &p, int rows) {
    // (blocks of heads that share a run follow one another, so that the run comes from memory once)
    int x = blockIdx.x;
    const int block = x % p.blocks;
    x /= p.blocks;
    split = x % p.splits;
    x /= p.splits;
    kv_head = x % p.kv_heads;
    batch = x / p.kv_heads;
    unit = x * p.blocks + block;
    head0 = kv_head * p.group + block * rows;
    heads = min(rows, p.group - block * rows);
    bool bad;
    const int length = kv::usable_length(mb_load(p.lengths + batch), p.longest, &bad);
    if (bad && threadIdx.x == 0) mb_report_bad_index(p.status);
    const int first = kv::window_begin(length, p.window);
    active = max(1, (length - first + p.split_len - 1) / p.split_len);
    begin = first + split * p.split_len;
    end = min(begin + p.split_len, length);
  }
};

// The row of slot `slot` in the pools, in elements; -1: there is none.
__device__ __forceinline__ int64_t slot_offset(const AttentionParams &p, const int32_t *table, int kv_head, int slot) {
  const int page = static_cast<int>(fast_div(slot, p.page_mul, p.page_shift));
  const int64_t at = kv::row_offset(mb_load(table + page), p.num_pages, p.kv_heads, kv_head, p.page_size, slot - page * p.page_size, p.dim);
  if (at < 0) mb_report_bad_index(p.status);
  return at;
}

// What `W` warps of the block hold of their slots -- per row a maximum, a sum and `dim` values `pitch` apart -- joined, and
// written as the result or as a run's part of it.  All in shared memory; coef: W x R floats of room, total: 2 R.
template <typename T, int R>
__device__ void finish(const AttentionParams &p, const Place &at, int W, int pitch, const float *top, const float *sum, const float *acc,
                       float *coef, float *total) {
  __shared__ int last;
  const int t = threadIdx.x;
  if (t < at.heads) {
    float m = -INFINITY, l = 0.f;
    for (int w = 0; w < W; ++w) m = fmaxf(m, top[w * R + t]);
    for (int w = 0; w < W; ++w) {
      const float c = top[w * R + t] == -INFINITY ? 0.f : exp2f(top[w * R + t] - m);
      coef[w * R + t] = c;
      l += sum[w * R + t] * c;
    }
    total[t] = m;
    total[R + t] = l;
  }
  __syncthreads();
  const bool whole = at.active == 1;
  float *part = whole ? nullptr : p.partial + (static_cast<int64_t>(at.unit) * p.splits + at.split) * R * (p.dim + 2);
  for (int i = t; i < at.heads * p.dim; i += THREADS) {
    const int h = i / p.dim, d = i - h * p.dim;
    float o = 0.f;
    for (int w = 0; w < W; ++w) o += acc[(w * R + h) * pitch + d] * coef[w * R + h];
    if (whole) {
      const float l = total[R + h];
      static_cast<T *>(p.out)[at.batch * p.out_stride + static_cast<int64_t>(at.head0 + h) * p.dim + d] =
          elem::narrow<T>(l == 0.f ? 0.f : o / l);
    } else {
      part[2 * R + h * p.dim + d] = o;
    }
  }
  if (!whole) {
    if (t < at.heads) {
      part[t] = total[t];
      part[R + t] = total[R + t];
    }
    __threadfence();
    __syncthreads();
    if (t == 0) last = atomicAdd(p.arrived + at.unit, 1u) == static_cast<unsigned>(at.active - 1);
    __syncthreads();
    if (!last) return;
    __threadfence();
    if (t == 0) p.arrived[at.unit] = 0;
    const float *parts = p.partial + static_cast<int64_t>(at.unit) * p.splits * R * (p.dim + 2);
    const int64_t step = R * (p.dim + 2);
    if (t < at.heads) {
      float m = -INFINITY, l = 0.f;
      for (int s = 0; s < at.active; ++s) m = fmaxf(m, __ldcg(parts + s * step + t));
      for (int s = 0; s < at.active; ++s) {
        const float ms = __ldcg(parts + s * step + t);
        l += __ldcg(parts + s * step + R + t) * (ms == -INFINITY ? 0.f : exp2f(ms - m));
      }
      total[t] = m;
      total[R + t] = l;
    }
    __syncthreads();
    for (int i = t; i < at.heads * p.dim; i += THREADS) {
      const int h = i / p.dim, d = i - h * p.dim;
      const float m = total[h], l = total[R + h];
      float o = 0.f;
      for (int s = 0; s < at.active; ++s) {
        const float ms = __ldcg(parts + s * step + h);
        o += __ldcg(parts + s * step + 2 * R + i) * (ms == -INFINITY ? 0.f : exp2f(ms - m));
      }
      static_cast<T *>(p.out)[at.batch * p.out_stride + static_cast<int64_t>(at.head0 + h) * p.dim + d] =
          elem::narrow<T>(l == 0.f ? 0.f : o / l);
    }
  }
  if (t < at.heads) {
    const float m = total[t], l = total[R + t];
    const int64_t to = static_cast<int64_t>(at.batch) * p.heads + at.head0 + t;
    const float lse2 = l == 0.f ? -INFINITY : m + log2f(l);
    if (p.lse != nullptr) p.lse[to] = lse2 * LN2;
    if (p.logits != nullptr) p.lse2[to] = lse2;
  }
}

// ---- on CUDA cores: every type, size and alignment -----------------------------------------------------------------------
//
// A warp takes 16 slots at a time; LANES of its lanes share a slot's row, N words of four values each (row: q and the accumulators
// of R query heads are in registers).  The R dot products of a slot are summed over its lanes by halving: each exchange
// leaves half the lanes with half of the heads.

template <typename T, bool VEC>
__device__ __forceinline__ void load_four(const T *p, int valid, float *v) {
  if (VEC) {
    elem::Vec<T, 4> w;
    if (valid > 0) w.load(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = valid > 0 ? elem::widen(w.v[i]) : 0.f;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < valid ? elem::widen(mb_load(p + i)) : 0.f;
  }
}

template <typename T, int R, int LANES, int N, bool VEC>
__global__ void __launch_bounds__(THREADS) paged_attention_kernel(const AttentionParams p) {
  constexpr int SLOTS = 16;             // a warp's at a time
  constexpr int AT_ONCE = 32 / LANES;   // of these, in one pass of its lanes
  constexpr int DIM = LANES * 4 * N;
  __shared__ float scores[WARPS][SLOTS * R], fix[WARPS][R];
  __shared__ int64_t rows[WARPS][SLOTS];
  __shared__ float top_s[WARPS * R], sum_s[WARPS * R], coef[WARPS * R], total[2 * R];
  __shared__ float acc_s[WARPS * R * DIM];
  mb_grid_dep_launch();
  mb_grid_dep_wait();
  const Place at(p, R);
  if (at.split >= at.active) return;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int mine = lane / LANES, word = lane % LANES;   // which slot of a pass, which words of its row
  const T *q = static_cast<const T *>(p.q), *k = static_cast<const T *>(p.k), *v = static_cast<const T *>(p.v);
  const int32_t *table = p.table + static_cast<int64_t>(at.batch) * p.max_pages;

  float qr[R][4 * N], acc[R][4 * N];
#pragma unroll
  for (int h = 0; h < R; ++h)
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int d = (n * LANES + word) * 4;
      load_four<T, VEC>(q + at.batch * p.q_stride + static_cast<int64_t>(at.head0 + h) * p.dim + d, h < at.heads ? p.dim - d : 0, qr[h] + 4 * n);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[h][4 * n + i] = 0.f;
    }
  // lane l keeps maximum and sum of heads l / 16, l / 16 + 2, ..
  constexpr int KEPT = (R + 1) / 2;
  float top[KEPT], sum[KEPT];
#pragma unroll
  for (int i = 0; i < KEPT; ++i) top[i] = -INFINITY, sum[i] = 0.f;

  for (int base = at.begin + warp * SLOTS; base < at.end; base += WARPS * SLOTS) {
    __syncwarp();
    if (lane < SLOTS) rows[warp][lane] = base + lane < at.end ? slot_offset(p, table, at.kv_head, base + lane) : -1;
    __syncwarp();
#pragma unroll 4
    for (int pass = 0; pass < SLOTS / AT_ONCE; ++pass) {
      const int slot = pass * AT_ONCE + mine;
      const int64_t row = rows[warp][slot];
      float kr[4 * N], dot[R];
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int d = (n * LANES + word) * 4;
        load_four<T, VEC>(k + row + d, row >= 0 ? p.dim - d : 0, kr + 4 * n);
      }
#pragma unroll
      for (int h = 0; h < R; ++h) {
        dot[h] = 0.f;
#pragma unroll
        for (int i = 0; i < 4 * N; ++i) dot[h] += qr[h][i] * kr[i];
      }
      // halving: lanes whose bit is set keep the upper half of the heads that are left
      int head = 0;
#pragma unroll
      for (int bit = LANES / 2, left = R; bit > 0; bit /= 2) {
        if (left > 1) {
          left /= 2;
          const bool upper = (word & bit) != 0;
          head += upper ? left : 0;
#pragma unroll
          for (int i = 0; i < R / 2; ++i)
            if (i < left) {
              const float give = upper ? dot[i] : dot[i + left], keep = upper ? dot[i + left] : dot[i];
              dot[i] = keep + __shfl_xor_sync(0xffffffffu, give, bit);
            }
        } else {
          dot[0] += __shfl_xor_sync(0xffffffffu, dot[0], bit);
        }
      }
      // (lanes whose low bits are set have the same sum once more)
      if (word % (LANES / R) == 0) scores[warp][head * SLOTS + slot] = row >= 0 ? dot[0] * p.scale2 : -INFINITY;
    }
    __syncwarp();
    bool grew = false;
#pragma unroll
    for (int i = 0; i < KEPT; ++i) {
      const int h = 2 * i + lane / SLOTS, slot = lane % SLOTS;
      const bool used = R > 1 || lane < SLOTS;
      const float s = used ? scores[warp][h * SLOTS + slot] : -INFINITY;
      if (p.logits != nullptr && used && h < at.heads && base + slot < at.end)
        p.logits[(static_cast<int64_t>(at.batch) * p.heads + at.head0 + h) * p.logits_stride + base + slot] = s;
      float m = s;
#pragma unroll
      for (int o = 8; o > 0; o /= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      m = fmaxf(m, top[i]);
      const float safe = m == -INFINITY ? 0.f : m;
      const float e = exp2f(s - safe), back = exp2f(top[i] - safe);
      float l = e;
#pragma unroll
      for (int o = 8; o > 0; o /= 2) l += __shfl_xor_sync(0xffffffffu, l, o);
      sum[i] = sum[i] * back + l;
      grew = grew || m != top[i];
      top[i] = m;
      if (used) {
        scores[warp][h * SLOTS + slot] = e;
        if (slot == 0) fix[warp][h] = back;
      }
    }
    __syncwarp();
    if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
      for (int h = 0; h < R; ++h) {
        const float back = fix[warp][h];
#pragma unroll
        for (int i = 0; i < 4 * N; ++i) acc[h][i] *= back;
      }
    }
#pragma unroll 4
    for (int pass = 0; pass < SLOTS / AT_ONCE; ++pass) {
      const int slot = pass * AT_ONCE + mine;
      const int64_t row = rows[warp][slot];
      float vr[4 * N];
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int d = (n * LANES + word) * 4;
        load_four<T, VEC>(v + row + d, row >= 0 ? p.dim - d : 0, vr + 4 * n);
      }
#pragma unroll
      for (int h = 0; h < R; ++h) {
        const float e = scores[warp][h * SLOTS + slot];
#pragma unroll
        for (int i = 0; i < 4 * N; ++i) acc[h][i] += e * vr[i];
      }
    }
  }
  // a row's accumulators over the passes' slots, then to shared memory for the other warps
#pragma unroll
  for (int h = 0; h < R; ++h)
#pragma unroll
    for (int i = 0; i < 4 * N; ++i) {
#pragma unroll
      for (int o = LANES; o < 32; o *= 2) acc[h][i] += __shfl_xor_sync(0xffffffffu, acc[h][i], o);
      if (mine == 0) acc_s[(warp * R + h) * DIM + (i / 4 * LANES + word) * 4 + i % 4] = acc[h][i];
    }
#pragma unroll
  for (int i = 0; i < KEPT; ++i) {
    const int h = 2 * i + lane / SLOTS;
    if (lane % SLOTS == 0 && h < R) {
      top_s[warp * R + h] = top[i];
      sum_s[warp * R + h] = sum[i];
    }
  }
  __syncthreads();
  finish<T, R>(p, at, WARPS, DIM, top_s, sum_s, acc_s, coef, total);
}

// ---- on the tensor cores: 16-bit types, rows of whole 16-byte words -----------------------------------------------------------
//
// Up to 16 query heads are the rows of mma.sync m16n8k16 (a decode step has no 128 rows for tcgen05 to multiply, and the cache's bytes
// bound it by far: 16 rows cost 16 operations a byte where 250 would be needed).  Every warp has a ring of its own in shared
// memory that its cp.asyncs fill with CHUNK slots' keys and values at a time, two stages ahead, so that no barrier joins warps
// before the end.  Rows are swizzled in 16-byte words for ldmatrix.  Probabilities are multiplied as two 16-bit values, hi + lo:
// their sum is the fp32 one to 2^-16 (bf16) or 2^-22, and the second product costs nothing that the memory does not hide.

template <typename T> struct Mma;
template <> struct Mma<__half> {
  static __device__ __forceinline__ void run(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ void split(float x, float y, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = *reinterpret_cast<const uint32_t *>(&l);
  }
};
template <> struct Mma<__nv_bfloat16> {
  static __device__ __forceinline__ void run(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ void split(float x, float y, uint32_t &hi, uint32_t &lo) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    const float2 f = __bfloat1622float2(h);
    const __nv_bfloat162 l = __floats2bfloat162_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = *reinterpret_cast<const uint32_t *>(&l);
  }
};

template <bool TRANS>
__device__ __forceinline__ void load_matrices(uint32_t addr, uint32_t (&r)[4]) {
  if (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

template <int DIM>
struct Ring {
  static constexpr int CHUNK = DIM == 64 ? 32 : 16;         // slots
  static constexpr int ROW = DIM * 2, WORDS = DIM / 8;      // bytes of a row, its 16-byte words
  static constexpr int PART = CHUNK * ROW, STAGE = 2 * PART;  // keys, then values
  static constexpr int STAGES = 3;
  static constexpr int BYTES = WARPS * STAGES * STAGE;
  static constexpr int PITCH = DIM + 4;                     // floats between rows of the accumulators at the end
  static_assert(WARPS * 16 * PITCH * 4 <= BYTES, "accumulators reuse the ring");
};

template <typename T, int DIM>
__global__ void __launch_bounds__(THREADS) paged_attention_mma_kernel(const AttentionParams p) {
  using G = Ring<DIM>;
  constexpr int R = 16, CHUNK = G::CHUNK, KEY_TILES = CHUNK / 8, DIM_STEPS = DIM / 16, STAGES = G::STAGES;
  extern __shared__ __align__(1024) uint8_t ring[];
  __shared__ unsigned valid[WARPS][STAGES];
  __shared__ float top_s[WARPS * R], sum_s[WARPS * R], coef[WARPS * R], total[2 * R];
  mb_grid_dep_launch();
  mb_grid_dep_wait();
  const Place at(p, R);
  if (at.split >= at.active) return;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, row = lane / 4, pair = lane % 4;
  const T *k = static_cast<const T *>(p.k), *v = static_cast<const T *>(p.v);
  const int32_t *table = p.table + static_cast<int64_t>(at.batch) * p.max_pages;
  const uint32_t mine = sm100::smem_u32(ring) + warp * STAGES * G::STAGE;

  // the queries of rows `row` and `row` + 8
  uint32_t q[DIM_STEPS][4];
#pragma unroll
  for (int s = 0; s < DIM_STEPS; ++s)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int h = row + i % 2 * 8, d = s * 16 + i / 2 * 8 + pair * 2;
      elem::Vec<T, 2> two;
      two.word = 0;
      if (h < at.heads && d < p.dim) {
        const T *src = static_cast<const T *>(p.q) + at.batch * p.q_stride + static_cast<int64_t>(at.head0 + h) * p.dim + d;
        two.v[0] = mb_load(src);
        two.v[1] = mb_load(src + 1);
      }
      q[s][i] = two.word;
    }
  float acc[2 * DIM_STEPS][4], top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 2 * DIM_STEPS; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;

  const int chunks = (at.end - at.begin + CHUNK - 1) / CHUNK;   // of all warps; this one has warp, warp + WARPS, ..
  const auto offset_of = [&](int chunk) -> int64_t {
    const int slot = at.begin + chunk * CHUNK + lane;
    return lane < CHUNK && chunk < chunks && slot < at.end ? slot_offset(p, table, at.kv_head, slot) : -1;
  };
  // `where`: lane l's offset of the chunk's slot l
  const auto fetch = [&](int chunk, int stage, int64_t where) {
    if (chunk < chunks) {
      const unsigned ok = __ballot_sync(0xffffffffu, where >= 0);
      if (lane == 0) valid[warp][stage] = ok;
      const int word = lane % G::WORDS;
#pragma unroll
      for (int i = 0; i < CHUNK * G::WORDS / 32; ++i) {
        const int r = i * (32 / G::WORDS) + lane / G::WORDS;
        const int64_t from = __shfl_sync(0xffffffffu, where, r);
        const bool there = from >= 0 && word * 8 < p.dim;
        const int64_t src = there ? from + word * 8 : 0;
        const uint32_t dst = mine + stage * G::STAGE + r * G::ROW + ((word ^ (r & 7)) << 4);
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(k + src), "r"(there ? 16 : 0) : "memory");
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + G::PART), "l"(v + src), "r"(there ? 16 : 0) : "memory");
      }
    }
    sm100::cp_async_commit();
  };
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) fetch(warp + s * WARPS, s, offset_of(warp + s * WARPS));
  int64_t ahead = offset_of(warp + (STAGES - 1) * WARPS);

  int stage = 0;
  for (int chunk = warp; chunk < chunks; chunk += WARPS) {
    sm100::cp_async_wait<STAGES - 2>();
    __syncwarp();
    fetch(chunk + (STAGES - 1) * WARPS, stage == 0 ? STAGES - 1 : stage - 1, ahead);
    ahead = offset_of(chunk + STAGES * WARPS);
    const uint32_t keys = mine + stage * G::STAGE, values = keys + G::PART;
    const unsigned ok = valid[warp][stage];
    float s[KEY_TILES][4];
#pragma unroll
    for (int t = 0; t < KEY_TILES; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[t][j] = 0.f;
#pragma unroll
    for (int d = 0; d < DIM_STEPS; ++d)
#pragma unroll
      for (int t = 0; t < KEY_TILES; t += 2) {
        uint32_t b[4];
        const int r = t * 8 + lane % 8 + lane / 16 * 8, word = 2 * d + lane / 8 % 2;
        load_matrices<false>(keys + r * G::ROW + ((word ^ (r & 7)) << 4), b);
        Mma<T>::run(s[t], q[d], b[0], b[1]);
        Mma<T>::run(s[t + 1], q[d], b[2], b[3]);
      }
    const int slot = at.begin + chunk * CHUNK + pair * 2;
    float m[2] = {top[0], top[1]};
#pragma unroll
    for (int t = 0; t < KEY_TILES; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[t][j] = (ok >> (t * 8 + pair * 2 + j % 2) & 1u) != 0 ? s[t][j] * p.scale2 : -INFINITY;
        m[j / 2] = fmaxf(m[j / 2], s[t][j]);
      }
    if (p.logits != nullptr) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (row + 8 * h < at.heads) {
          float *to = p.logits + (static_cast<int64_t>(at.batch) * p.heads + at.head0 + row + 8 * h) * p.logits_stride + slot;
#pragma unroll
          for (int t = 0; t < KEY_TILES; ++t)
#pragma unroll
            for (int j = 0; j < 2; ++j)
              if (slot + t * 8 + j < at.end) to[t * 8 + j] = s[t][2 * h + j];
        }
    }
    bool grew = false;
    float back[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      m[h] = fmaxf(m[h], __shfl_xor_sync(0xffffffffu, m[h], 1));
      m[h] = fmaxf(m[h], __shfl_xor_sync(0xffffffffu, m[h], 2));
      grew = grew || m[h] != top[h];
      const float safe = m[h] == -INFINITY ? 0.f : m[h];
      back[h] = exp2f(top[h] - safe);
      top[h] = m[h];
      m[h] = safe;
      sum[h] *= back[h];
    }
    if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
      for (int i = 0; i < 2 * DIM_STEPS; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] *= back[j / 2];
    }
#pragma unroll
    for (int t = 0; t < KEY_TILES; t += 2) {
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float x = exp2f(s[t + u][2 * h] - m[h]), y = exp2f(s[t + u][2 * h + 1] - m[h]);
          sum[h] += x + y;
          Mma<T>::split(x, y, hi[2 * u + h], lo[2 * u + h]);
        }
#pragma unroll
      for (int d = 0; d < DIM_STEPS; ++d) {
        uint32_t b[4];
        const int r = t * 8 + lane % 16, word = 2 * d + lane / 16;
        load_matrices<true>(values + r * G::ROW + ((word ^ (r & 7)) << 4), b);
        Mma<T>::run(acc[2 * d], hi, b[0], b[1]);
        Mma<T>::run(acc[2 * d + 1], hi, b[2], b[3]);
        Mma<T>::run(acc[2 * d], lo, b[0], b[1]);
        Mma<T>::run(acc[2 * d + 1], lo, b[2], b[3]);
      }
    }
    stage = stage + 1 == STAGES ? 0 : stage + 1;
  }
  sm100::cp_async_wait<0>();
  __syncthreads();
  float *acc_s = reinterpret_cast<float *>(ring);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
    sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
    if (row + 8 * h < at.heads) {
      const int r = warp * R + row + 8 * h;
      if (pair == 0) {
        top_s[r] = top[h];
        sum_s[r] = sum[h];
      }
#pragma unroll
      for (int i = 0; i < 2 * DIM_STEPS; ++i)
        *reinterpret_cast<float2 *>(acc_s + r * G::PITCH + i * 8 + pair * 2) = make_float2(acc[i][2 * h], acc[i][2 * h + 1]);
    }
  }
  __syncthreads();
  finish<T, R>(p, at, WARPS, G::PITCH, top_s, sum_s, acc_s, coef, total);
}

template <typename T, int DIM>
int launch_mma(mb_context *ctx, const AttentionParams &p, unsigned grid, int index) {
  const auto kern = paged_attention_mma_kernel<T, DIM>;
  if (!(ctx->attention_attr_mask & (1u << index))) {
    MB_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Ring<DIM>::BYTES));
    ctx->attention_attr_mask |= 1u << index;
  }
  MB_CUDA(ctx, mb_launch_chained(ctx, kern, dim3(grid), dim3(THREADS), Ring<DIM>::BYTES, p));
  return MB_SUCCESS;
}

template <typename T>
int launch_mma(mb_context *ctx, const AttentionParams &p, unsigned grid, int index) {
  if (p.dim <= 64) return launch_mma<T, 64>(ctx, p, grid, index);
  if (p.dim <= 128) return launch_mma<T, 128>(ctx, p, grid, index + 1);
  return launch_mma<T, 256>(ctx, p, grid, index + 2);
}

// What each slot has received of the query heads' probabilities, on top of what it had.
__global__ void __launch_bounds__(256) attention_weights_kernel(const AttentionParams p, int chunks) {
  mb_grid_dep_launch();
  mb_grid_dep_wait();
  const int unit = blockIdx.x / chunks, batch = unit / p.kv_heads, kv_head = unit % p.kv_heads;
  const int slot = (blockIdx.x % chunks) * 256 + threadIdx.x;
  bool bad;
  const int length = kv::usable_length(mb_load(p.lengths + batch), p.longest, &bad);
  if (slot >= length) return;
  const int64_t to = static_cast<int64_t>(unit) * p.weights_stride + slot;
  float w = 0.f;
  if (slot >= kv::window_begin(length, p.window)) {
    const int64_t head = static_cast<int64_t>(batch) * p.heads + kv_head * p.group;
    for (int g = 0; g < p.group; ++g) {
      const float lse2 = mb_load(p.lse2 + head + g);
      if (lse2 != -INFINITY) w += exp2f(mb_load(p.logits + (head + g) * p.logits_stride + slot) - lse2);
    }
  }
  p.weights_out[to] = (p.weights_in != nullptr ? mb_load(p.weights_in + to) : 0.f) + w;
}

template <typename T, int R, int LANES, int N>
cudaError_t launch_cores(mb_context *ctx, const AttentionParams &p, unsigned grid, bool vec) {
  if (vec) return mb_launch_chained(ctx, paged_attention_kernel<T, R, LANES, N, true>, dim3(grid), dim3(THREADS), 0, p);
  return mb_launch_chained(ctx, paged_attention_kernel<T, R, LANES, N, false>, dim3(grid), dim3(THREADS), 0, p);
}

template <typename T, int R>
cudaError_t launch_cores(mb_context *ctx, const AttentionParams &p, unsigned grid, bool vec) {
  if (p.dim <= 32) return launch_cores<T, R, 8, 1>(ctx, p, grid, vec);
  if (p.dim <= 64) return launch_cores<T, R, 16, 1>(ctx, p, grid, vec);
  if (p.dim <= 128) return launch_cores<T, R, 32, 1>(ctx, p, grid, vec);
  return launch_cores<T, R, 32, 2>(ctx, p, grid, vec);
}

// The runs a head's slots are cut into: about four blocks per SM where the sequences are as long as they may be, of 64 slots at least.
void cut_runs(const mb_context *ctx, AttentionParams &p, int64_t units) {
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>(4ll * ctx->num_sms / std::max<int64_t>(units, 1), MAX_SPLITS));
  const int64_t most = std::max<int64_t>(p.longest, 1);
  p.split_len = static_cast<int>(std::max<int64_t>(64, ceil_div64(ceil_div64(most, want), 64) * 64));
  p.splits = static_cast<int>(ceil_div64(most, p.split_len));
}

}  // namespace

extern "C" int mb_paged_attention(mb_context *ctx, const void *q, const void *k_cache, const void *v_cache, const int32_t *page_table,
                                  const int32_t *lengths, void *out, float *lse, const float *weights_in, float *weights_out,
                                  int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t q_stride,
                                  int64_t out_stride, int64_t num_pages, int64_t page_size, int64_t max_pages, int64_t max_length,
                                  int64_t window, int64_t weights_stride, float scale, int dtype) {
  if (ctx == nullptr) return MB_INVALID_ARGS;
  const kv::Verdict verdict = kv::check_attention(q, k_cache, v_cache, page_table, lengths, out, lse, weights_in, weights_out, batch,
                                                  heads, kv_heads, head_dim, q_stride, out_stride, num_pages, page_size, max_pages,
                                                  max_length, window, weights_stride, dtype);
  if (verdict.code != MB_SUCCESS) return mb_fail(ctx, verdict.code, "mb_paged_attention: %s", verdict.why);
  if (batch == 0) return MB_SUCCESS;
  MB_CUDA(ctx, cudaSetDevice(ctx->device));
  AttentionParams p = {};
  p.q = q; p.k = k_cache; p.v = v_cache; p.table = page_table; p.lengths = lengths; p.out = out; p.lse = lse;
  p.weights_in = weights_in; p.weights_out = weights_out;
  p.q_stride = q_stride; p.out_stride = out_stride; p.num_pages = num_pages; p.weights_stride = weights_stride; p.window = window;
  p.heads = static_cast<int>(heads); p.kv_heads = static_cast<int>(kv_heads); p.group = static_cast<int>(heads / kv_heads);
  p.dim = static_cast<int>(head_dim); p.page_size = static_cast<int>(page_size); p.max_pages = static_cast<int>(max_pages);
  p.longest = kv::longest_of(max_length, max_pages, page_size);
  fast_div_make(static_cast<uint32_t>(page_size), &p.page_mul, &p.page_shift);
  p.scale2 = scale * LOG2E;
  p.status = ctx->dev_status;

  const bool by_mma = dtype != MB_F32 && ctx->use_tensor_cores && head_dim % 8 == 0 && kv::aligned(k_cache, 16) && kv::aligned(v_cache, 16);
  const int rows = by_mma ? 16 : p.group >= 5 ? 8 : p.group >= 3 ? 4 : p.group;
  p.blocks = (p.group + rows - 1) / rows;
  const int64_t units = batch * kv_heads * p.blocks;
  cut_runs(ctx, p, units);
  if (units * p.splits > kv::MOST) return mb_fail(ctx, MB_UNSUPPORTED, "mb_paged_attention: too many sequences and heads");
  const size_t partial = p.splits > 1 ? align_up(sizeof(float) * units * p.splits * rows * (p.dim + 2), 256) : 0;
  size_t logits = 0, lse2 = 0;
  if (weights_out != nullptr && p.longest > 0) {
    p.logits_stride = align_up(p.longest, 4);
    lse2 = align_up(sizeof(float) * batch * heads, 256);
    logits = sizeof(float) * batch * heads * p.logits_stride;
  }
  char *room = nullptr;
  if (partial + lse2 + logits > 0) {
    void *ptr = nullptr;
    MB_RETURN_IF_ERROR(mb_op_scratch(ctx, partial + lse2 + logits, &ptr));
    room = static_cast<char *>(ptr);
  }
  if (partial > 0) {
    p.partial = reinterpret_cast<float *>(room);
    MB_RETURN_IF_ERROR(mb_op_counters(ctx, units, &p.arrived));
  }
  if (logits > 0) {
    p.lse2 = reinterpret_cast<float *>(room + partial);
    p.logits = reinterpret_cast<float *>(room + partial + lse2);
  }
  const unsigned grid = static_cast<unsigned>(units * p.splits);
  cudaError_t e = cudaSuccess;
  if (by_mma) {
    if (dtype == MB_F16) MB_RETURN_IF_ERROR(launch_mma<__half>(ctx, p, grid, 0));
    else MB_RETURN_IF_ERROR(launch_mma<__nv_bfloat16>(ctx, p, grid, 3));
  } else MB_FOR_ELEMENT(dtype, {
    const uintptr_t word = 4 * sizeof(T);
    const bool vec = p.dim % 4 == 0 && q_stride % 4 == 0 && kv::aligned(q, word) && kv::aligned(k_cache, word) && kv::aligned(v_cache, word);
    e = rows == 8 ? launch_cores<T, 8>(ctx, p, grid, vec) : rows == 4 ? launch_cores<T, 4>(ctx, p, grid, vec)
      : rows == 2 ? launch_cores<T, 2>(ctx, p, grid, vec) : launch_cores<T, 1>(ctx, p, grid, vec);
  });
  MB_CUDA(ctx, e);
  ctx->launches++;
  if (logits > 0) {
    const int chunks = (p.longest + 255) / 256;
    if (batch * kv_heads * chunks > kv::MOST) return mb_fail(ctx, MB_UNSUPPORTED, "mb_paged_attention: too many slots");
    MB_CUDA(ctx, mb_launch_chained(ctx, attention_weights_kernel, dim3(static_cast<unsigned>(batch * kv_heads * chunks)), dim3(256), 0, p, chunks));
    ctx->launches++;
  }
  return MB_SUCCESS;
}
