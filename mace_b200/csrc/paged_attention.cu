// Attention of one new token per sequence over a paged key-value cache.
//
//   s_j = scale q . k_j,   out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),   lse = m + log sum_j e^(s_j - m)
//
// One pass over the cache with a running maximum m; exponentials are powers of two, so that scale log2(e) is one factor.  A block
// has one run of slots of one kv head and up to ROWS of the query heads that share it, so that a slot is read once for all of them;
// the runs are as many as fill the SMs, and the block that arrives last of a head's runs joins them.
// Slots behind the length, outside the window or in a page that the pool lacks are -inf before the maximum, and their values
// zeros: 0 times the NaN that an unused row may hold would be NaN.
#include <algorithm>
#include <cmath>

#include "elements.cuh"
#include "gemm_u8_cut.cuh"
#include "kv_cache.h"
#include "sm100_ptx.cuh"

namespace {

constexpr int THREADS = 128;
constexpr int WARPS = THREADS / 32;
constexpr int MAX_SPLITS = 128;
constexpr int LEAST_RUN = kv::LEAST_RUN;
constexpr int SCANNED = 1024;    // sequences whose lengths every block reads
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// What a probability is multiplied by until the end, relative to one of the running maximum, as a power of two.  Halves reach from 2^-24
// to 2^16 only, and most probabilities are small: the largest are brought to their upper end.  The other types' values may be as large as
// an fp32 sum can be: probabilities are brought down by so much that 2^24 slots of the maximum's weight sum up to at most one (and
// what has less than 2^-102 of its weight, e^-70, loses bits, where without the factor it would be 2^-126).
template <typename T> constexpr int LIFT = -24;
template <> constexpr int LIFT<__half> = 15;
template <typename T> constexpr float RAISED = LIFT<T> < 0 ? 1.f / (1 << -LIFT<T>) : static_cast<float>(1 << (LIFT<T> < 0 ? 0 : LIFT<T>));

struct AttentionParams {
  const void *q, *k, *v;
  const int32_t *table, *lengths;
  void *out;
  float *lse;
  float *logits;        // [batch][heads][logits_stride], in powers of two; null: no weights asked for
  float *lse2;          // [batch][heads], beside them
  float *partial;       // of a run: row maxima, row sums, rows of `pitch` values
  unsigned *arrived;    // of a unit
  const float *weights_in;
  float *weights_out;
  int64_t q_stride, out_stride, num_pages, logits_stride, weights_stride, window;
  int batch, heads, kv_heads, group, blocks, dim, pitch, page_size, max_pages, longest, wanted;   // wanted: runs, about
  int cluster;                 // above 1: every head's slots over a cluster of so many blocks
  int fixed_runs, fixed_run;   // batches above SCANNED: every head has so many runs of so many slots
  uint32_t page_mul, page_shift;
  float scale2;         // scale log2(e)
  int *status;
};

// Which part of the problem a block has.  The lengths are in device memory, so the blocks cut the work themselves: all slots of all
// heads over the blocks that are resident at once give a run's length, a sequence has as many runs as it needs, and a
// prefix sum over the sequences says whose run this block's is.  No block is without work but the few behind the last run, and a
// batch of one long and many short sequences fills the SMs as well as one of equals.  (Runs cut by the longest sequence, which
// the host knows: a batch of 32 from 1 to 4096 slots took 57 us instead of 49.)
struct Place {
  int unit, batch, kv_head, head0, heads, split, active, first, begin, end;   // slots from `first` on; the run is begin .. end
  int record;                                                                 // of the unit's first run; the next ones p.blocks apart

  // Slots of a sequence that a run is made of; they begin at a multiple of `chunk`, below `first` where a window does not.
  static __device__ __forceinline__ int slots_of(const AttentionParams &p, int b, int chunk, int *first, int *from, bool *bad) {
    const int length = kv::usable_length(mb_load(p.lengths + b), p.longest, bad);
    *first = kv::window_begin(length, p.window);
    *from = *first / chunk * chunk;
    return length - *from;
  }
  // The runs of a sequence, at most *run slots each, made as long as one another.
  static __device__ __forceinline__ int runs_of(int slots, int *run) {
    const unsigned n = static_cast<unsigned>(slots), most = static_cast<unsigned>(*run);
    const unsigned runs = max(1u, (n + most - 1) / most);
    const unsigned each = max(((n + runs - 1) / runs + 63) / 64 * 64, 64u);
    *run = static_cast<int>(each);
    return static_cast<int>(max(1u, (n + each - 1) / each));
  }

  // false: there is no such run.
  __device__ __forceinline__ bool find(const AttentionParams &p, int rows, int chunk) {
    __shared__ long long sums[WARPS];
    __shared__ int tops[WARPS], counts[WARPS], found[2];
    const int t = threadIdx.x, lane = t % 32, warp = t / 32, per_run = p.kv_heads * p.blocks;
    int from;
    bool bad;
    if (p.cluster > 1) {
      split = static_cast<int>(sm100::cluster_ctarank());
      int x = blockIdx.x / p.cluster;
      unit = x;
      const int block = x % p.blocks;
      x /= p.blocks;
      kv_head = x % p.kv_heads;
      batch = x / p.kv_heads;
      const int slots = slots_of(p, batch, chunk, &first, &from, &bad);
      if (bad && t == 0) mb_report_bad_index(p.status);
      const int run = static_cast<int>((static_cast<unsigned>(slots) + p.cluster * 16 - 1) / (p.cluster * 16)) * 16;
      active = p.cluster;
      record = 0;
      place(p, rows, block, from, slots, run);
      if (begin > from + slots) begin = end = from + slots;
      return true;
    }
    if (p.fixed_runs > 0) {
      int x = blockIdx.x;
      const int block = x % p.blocks;
      x /= p.blocks;
      split = x % p.fixed_runs;
      unit = x / p.fixed_runs * p.blocks + block;
      record = x / p.fixed_runs * p.fixed_runs * p.blocks + block;
      kv_head = x / p.fixed_runs % p.kv_heads;
      batch = x / p.fixed_runs / p.kv_heads;
      const int slots = slots_of(p, batch, chunk, &first, &from, &bad);
      if (bad && t == 0) mb_report_bad_index(p.status);
      int run = p.fixed_run;
      active = runs_of(slots, &run);
      if (split >= active) return false;
      place(p, rows, block, from, slots, run);
      return true;
    }
    long long total = 0;
    int top = 0;
    for (int b = t; b < p.batch; b += THREADS) {
      const int slots = slots_of(p, b, chunk, &first, &from, &bad);
      total += slots;
      top = max(top, slots);
      if (bad && blockIdx.x == 0) mb_report_bad_index(p.status);
    }
    top = static_cast<int>(__reduce_max_sync(0xffffffffu, static_cast<unsigned>(top)));
#pragma unroll
    for (int o = 16; o > 0; o /= 2) total += __shfl_xor_sync(0xffffffffu, total, o);
    if (lane == 0) {
      sums[warp] = total;
      tops[warp] = top;
    }
    __syncthreads();
    total = 0;
    for (int w = 0; w < WARPS; ++w) {
      total += sums[w];
      top = max(top, tops[w]);
    }
    // (no sequence may have more than MAX_SPLITS runs)
    const long long share = max((total * per_run + p.wanted - 1) / p.wanted, static_cast<long long>((top + MAX_SPLITS - 1) / MAX_SPLITS));
    const int most = static_cast<int>(min(max(static_cast<long long>(LEAST_RUN), (share + 63) / 64 * 64), 0x7fffffc0ll));
    int before = 0;   // runs of the sequences in front of this round's
    for (int base = 0; base < p.batch; base += THREADS) {
      const int b = base + t;
      int slots = 0, mine = 0;
      if (b < p.batch) {
        slots = slots_of(p, b, chunk, &first, &from, &bad);
        int run = most;
        mine = runs_of(slots, &run) * per_run;
      }
      int upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o *= 2) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      if (lane == 31) counts[warp] = upto;
      __syncthreads();
      int all = 0;
      for (int w = 0; w < WARPS; ++w) {
        if (w == warp) upto += all;
        all += counts[w];
      }
      upto += before;
      const int x = blockIdx.x;
      if (x < upto && x >= upto - mine) {
        found[0] = b;
        found[1] = upto - mine;
      }
      before += all;
      __syncthreads();
      if (x < before) break;
    }
    if (static_cast<int>(blockIdx.x) >= before) return false;
    batch = found[0];
    const int slots = slots_of(p, batch, chunk, &first, &from, &bad);
    int run = most;
    active = runs_of(slots, &run);
    // (blocks of heads that share a run follow one another, so that the run comes from memory once)
    int x = blockIdx.x - found[1];
    const int block = x % p.blocks;
    x /= p.blocks;
    split = x % active;
    kv_head = x / active;
    unit = (batch * p.kv_heads + kv_head) * p.blocks + block;
    record = found[1] + kv_head * active * p.blocks + block;
    place(p, rows, block, from, slots, run);
    return true;
  }

  __device__ __forceinline__ void place(const AttentionParams &p, int rows, int block, int from, int slots, int run) {
    head0 = kv_head * p.group + block * rows;
    heads = min(rows, p.group - block * rows);
    begin = from + split * run;
    end = from + slots - begin < run ? from + slots : begin + run;
  }
};

// The row of slot `slot` in the pools, in elements; -1: there is none.
__device__ __forceinline__ int64_t slot_offset(const AttentionParams &p, const int32_t *table, int kv_head, int slot) {
  const int page = static_cast<int>(fast_div(slot, p.page_mul, p.page_shift));
  const int64_t at = kv::row_offset(mb_load(table + page), p.num_pages, p.kv_heads, kv_head, p.page_size, slot - page * p.page_size, p.dim);
  if (at < 0) mb_report_bad_index(p.status);
  return at;
}

__device__ __forceinline__ float load_remote(uint32_t addr, int rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(sm100::mapa_shared(addr, rank)) : "memory");
  return v;
}

// The log-sum-exp of the block's row h, for the caller and for the weights.  l: the sum as it was kept.
template <typename T>
__device__ __forceinline__ void tell(const AttentionParams &p, const Place &at, int h, float m, float l) {
  const int64_t to = static_cast<int64_t>(at.batch) * p.heads + at.head0 + h;
  const float lse2 = l == 0.f ? -INFINITY : m + log2f(l * (1.f / RAISED<T>));
  if (p.lse != nullptr) p.lse[to] = lse2 * LN2;
  if (p.logits != nullptr) p.lse2[to] = lse2;
}

// What the warps of the block hold of their slots -- per row a maximum, a sum and `dim` values `pitch` apart -- joined, and
// written as the result or as a run's part of it.  All in shared memory; coef: WARPS x R floats of room, total: 2 R; acc is room for
// 2 R MAX_SPLITS floats when its values have been read.
template <typename T, int R>
__device__ void finish(const AttentionParams &p, const Place &at, int pitch, const float *top, const float *sum, float *room,
                       float *coef, float *total) {
  const float *acc = room;
  __shared__ int last;
  const int t = threadIdx.x;
  if (t < at.heads) {
    float m = -INFINITY, l = 0.f;
    for (int w = 0; w < WARPS; ++w) m = fmaxf(m, top[w * R + t]);
    for (int w = 0; w < WARPS; ++w) {
      const float c = top[w * R + t] == -INFINITY ? 0.f : exp2f(top[w * R + t] - m);
      coef[w * R + t] = c;
      l += sum[w * R + t] * c;
    }
    total[t] = m;
    total[R + t] = l;
  }
  __syncthreads();
  const bool whole = at.active == 1, apart = p.cluster > 1;   // apart: the runs of a head are the blocks of a cluster
  constexpr int HEAD = R == 1 ? 4 : 2 * R;   // (the values behind them by 16 bytes)
  const int record = HEAD + R * p.pitch, words = p.pitch / 4;
  float *part = whole || apart ? nullptr : p.partial + static_cast<int64_t>(at.record + at.split * p.blocks) * record;
  const auto store = [&](int h, int d, float4 o, float l) {
    T *to = static_cast<T *>(p.out) + at.batch * p.out_stride + static_cast<int64_t>(at.head0 + h) * p.dim + d;
    const float v[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (d + j < p.dim) to[j] = elem::narrow<T>(l == 0.f ? 0.f : v[j] / l);
  };
  for (int i = t; i < at.heads * words; i += THREADS) {
    const int h = i / words, d = (i - h * words) * 4;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float4 v = *reinterpret_cast<const float4 *>(acc + (w * R + h) * pitch + d);
      const float c = coef[w * R + h];
      o.x += v.x * c;
      o.y += v.y * c;
      o.z += v.z * c;
      o.w += v.w * c;
    }
    if (whole) store(h, d, o, total[R + h]);
    else if (apart) *reinterpret_cast<float4 *>(room + h * pitch + d) = o;   // (over the first warp's, which only this thread reads)
    else *reinterpret_cast<float4 *>(part + HEAD + h * p.pitch + d) = o;
  }
  if (apart) {
    // every block joins its share of the values out of all blocks' shared memory
    sm100::cluster_sync_all();
    const uint32_t tops = sm100::smem_u32(total), values = sm100::smem_u32(room);
    for (int i = at.split * THREADS + t; i < at.heads * words; i += p.cluster * THREADS) {
      const int h = i / words, d = (i - h * words) * 4;
      float m = -INFINITY, l = 0.f;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int s = 0; s < p.cluster; ++s) {
        const float ms = load_remote(tops + h * 4, s), ls = load_remote(tops + (R + h) * 4, s);
        float4 v;
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(sm100::mapa_shared(values + (h * pitch + d) * 4, s)) : "memory");
        const float top = fmaxf(m, ms), old = m == -INFINITY ? 0.f : exp2f(m - top), c = ms == -INFINITY ? 0.f : exp2f(ms - top);
        l = l * old + ls * c;
        o.x = o.x * old + v.x * c;
        o.y = o.y * old + v.y * c;
        o.z = o.z * old + v.z * c;
        o.w = o.w * old + v.w * c;
        m = top;
      }
      store(h, d, o, l);
      if (d == 0) tell<T>(p, at, h, m, l);
    }
    sm100::cluster_sync_all();   // (no block may leave while another reads its shared memory)
    return;
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
    // all runs' maxima and sums at once, then a warp per row, then the values, four to a load and AT_ONCE runs in flight
    constexpr int AT_ONCE = 8;
    const float *parts = p.partial + static_cast<int64_t>(at.record) * record;
    const int64_t step = static_cast<int64_t>(record) * p.blocks;
    float *tops = room, *sums = room + MAX_SPLITS * R;
    for (int i = t; i < at.active * R; i += THREADS) {
      const int s = i / R, h = i % R;
      const bool used = h < at.heads;
      tops[i] = used ? __ldcg(parts + s * step + h) : -INFINITY;
      sums[i] = used ? __ldcg(parts + s * step + R + h) : 0.f;
    }
    __syncthreads();
    for (int h = t / 32; h < at.heads; h += WARPS) {
      float m = -INFINITY, l = 0.f;
      for (int s = t % 32; s < at.active; s += 32) m = fmaxf(m, tops[s * R + h]);
#pragma unroll
      for (int o = 16; o > 0; o /= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      for (int s = t % 32; s < at.active; s += 32) {
        const float ms = tops[s * R + h], c = ms == -INFINITY ? 0.f : exp2f(ms - m);
        tops[s * R + h] = c;
        l += sums[s * R + h] * c;
      }
#pragma unroll
      for (int o = 16; o > 0; o /= 2) l += __shfl_xor_sync(0xffffffffu, l, o);
      if (t % 32 == 0) {
        total[h] = m;
        total[R + h] = l;
      }
    }
    __syncthreads();
    for (int i = t; i < at.heads * words; i += THREADS) {
      const int h = i / words, d = (i - h * words) * 4;
      const float *from = parts + HEAD + h * p.pitch + d;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int s0 = 0; s0 < at.active; s0 += AT_ONCE) {
        float4 v[AT_ONCE];
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j)
          if (s0 + j < at.active) v[j] = __ldcg(reinterpret_cast<const float4 *>(from + (s0 + j) * step));
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j)
          if (s0 + j < at.active) {
            const float c = tops[(s0 + j) * R + h];
            o.x += v[j].x * c;
            o.y += v[j].y * c;
            o.z += v[j].z * c;
            o.w += v[j].w * c;
          }
      }
      store(h, d, o, total[R + h]);
    }
  }
  if (t < at.heads) tell<T>(p, at, t, total[t], total[R + t]);
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
  __shared__ __align__(16) float acc_s[WARPS * R * DIM < 2 * R * MAX_SPLITS ? 2 * R * MAX_SPLITS : WARPS * R * DIM];
  mb_grid_dep_launch();
  mb_grid_dep_wait();
  Place at;
  if (!at.find(p, R, 1)) return;
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
      const float e = exp2f(s - safe) * RAISED<T>, back = exp2f(top[i] - safe);
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
  finish<T, R>(p, at, DIM, top_s, sum_s, acc_s, coef, total);
}

// ---- on the tensor cores: 16-bit types, rows of whole 16-byte words -----------------------------------------------------------
//
// mma.sync m16n8k16 with slots as rows and 8 query heads as columns: S^T = K Q^T, then O^T = V^T P^T.  (A decode step has no 128 rows
// for tcgen05 to multiply, and the cache's bytes bound it by far.  With heads as the 16 rows, as a prompt's attention has
// them, a group of four or eight leaves half of every product and of every exponential unused: 787 instructions per 16 slots where this
// form takes about 200, and 210 us instead of 165 for two sequences of 120001.)  Every warp has a ring of its own in shared memory that
// its cp.asyncs fill with CHUNK slots' keys and values at a time, so that no barrier joins warps before the end.  Rows are
// swizzled in 16-byte words for ldmatrix.  Probabilities are multiplied as two 16-bit values, hi + lo: their sum is the fp32 one to
// 2^-16, and the second product costs nothing that the memory does not hide.  Two bf16 values are that at any size; two halves only
// while lo is not cut off at 2^-24, which RAISED keeps true of 24 powers of two below the maximum (16.6 nats).  A chunk with
// smaller ones among its probabilities, as every one is whose sequence has a slot that outweighs the others by more, multiplies them again,
// 2^24 times as large (a slot of hardly any weight may still be all there is: the heaviest slot's value may be zero).

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

template <> struct Mma<float> {
  // tf32, 8 of the depth
  static __device__ __forceinline__ void run(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  // x as the nearest tf32 number and what that leaves, 12 bits, of which the MMA takes 11: together x to 2^-23 (of an infinity, or of a
  // number that has none above it: NaN)
  static __device__ __forceinline__ void split(uint32_t x, uint32_t &hi, uint32_t &lo) {
    hi = (x + 0x1000u) & 0xffffe000u;
    lo = __float_as_uint(__uint_as_float(x) - __uint_as_float(hi));
  }
  // x cut off and what that leaves, 13 bits of which the MMA takes 11: together x to 3 x 2^-23, and never above it, so that the type's
  // largest values stay finite (what is infinite gives NaN)
  static __device__ __forceinline__ void cut(uint32_t x, uint32_t &hi, uint32_t &lo) {
    hi = x & 0xffffe000u;
    lo = __float_as_uint(__uint_as_float(x) - __uint_as_float(hi));
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

// An 8 x 8 matrix of 16-bit values, two of a row to a lane, transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

__device__ __forceinline__ void copy_word(uint32_t dst, const void *src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_word(uint32_t dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

template <typename T, int DIM>
struct Ring {
  static constexpr int CHUNK = 16;                                // slots
  static constexpr int ROW = DIM * sizeof(T), WORDS = ROW / 16;   // bytes of a row, its 16-byte words
  static constexpr int EACH = 16 / sizeof(T);                     // values of a word
  static constexpr int PART = CHUNK * ROW, STAGE = 2 * PART;      // keys, then values
  static constexpr int STAGES = ROW == 256 ? 2 : 3;               // (two of 256-byte rows: three blocks an SM)
  static constexpr int BYTES = WARPS * STAGES * STAGE;
  static constexpr int PITCH = DIM + 4;                       // floats between rows of the accumulators at the end
  static constexpr int MOST_HEADS = DIM * sizeof(T) <= 256 ? 24 : 16;
  static_assert(2 * MOST_HEADS * MAX_SPLITS * 4 <= BYTES, "what joins the runs reuses it too");
  static_assert(WARPS * MOST_HEADS * PITCH * 4 <= BYTES, "accumulators reuse the ring");
};

// Where the words of a row of values lie: 16-bit rows are read by ldmatrix, eight at a time; fp32 ones as single values, four rows of two
// words at a time.
template <bool F32>
__device__ __forceinline__ int value_swizzle(int r) {
  return F32 ? (r * 2 & 7) | (r >> 2 & 1) : r & 7;
}

// HEADS: tiles of 8 query heads.  WHOLE: a chunk of slots lies in one page, and rows have DIM values.
template <typename T, int DIM, int HEADS, bool WHOLE>
__global__ void __launch_bounds__(THREADS, DIM * sizeof(T) == 128 && HEADS == 2 ? 4 : 0) paged_attention_mma_kernel(const AttentionParams p) {
  using G = Ring<T, DIM>;
  constexpr bool F32 = sizeof(T) == 4, HALVES = LIFT<T> > 0;
  constexpr float LEAST = 1.f / 512.f;   // (halves: what is 2^-16 exact as a pair of them)
  constexpr int R = 8 * HEADS, CHUNK = G::CHUNK, STAGES = G::STAGES;
  constexpr int STEPS = G::WORDS / 2, DIM_STEPS = DIM / 16;   // of a product with the keys (two words of a row), with the values
  extern __shared__ __align__(1024) uint8_t ring[];
  __shared__ unsigned valid[WARPS][STAGES];
  __shared__ float top_s[WARPS * R], sum_s[WARPS * R], coef[WARPS * R], total[2 * R];
  __shared__ __align__(16) float weight_s[F32 ? WARPS : 1][CHUNK][8];   // a chunk's probabilities, to be read as the other operand
  mb_grid_dep_launch();
  mb_grid_dep_wait();
  Place at;
  if (!at.find(p, R, CHUNK)) return;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, row = lane / 4, pair = lane % 4;
  const T *k = static_cast<const T *>(p.k), *v = static_cast<const T *>(p.v);
  const int32_t *table = p.table + static_cast<int64_t>(at.batch) * p.max_pages;
  const uint32_t mine = sm100::smem_u32(ring) + warp * STAGES * G::STAGE;

  const int chunks = (at.end - at.begin + CHUNK - 1) / CHUNK;   // of all warps; this one has warp, warp + WARPS, ..
  // Where chunk's slot l lies, for lane l; with WHOLE, where its first slot does, if all of them are there, else -1.
  const auto slot_of = [&](int chunk) -> int64_t {
    const int slot = at.begin + chunk * CHUNK + lane;
    return lane < CHUNK && slot >= at.first && slot < at.end ? slot_offset(p, table, at.kv_head, slot) : -1;
  };
  const auto offset_of = [&](int chunk) -> int64_t {
    if (chunk >= chunks) return -1;
    if (!WHOLE) return slot_of(chunk);
    const int slot = at.begin + chunk * CHUNK;
    return slot >= at.first && slot + CHUNK <= at.end ? slot_offset(p, table, at.kv_head, slot) : -1;
  };
  const int word = lane % G::WORDS, line = lane / G::WORDS;
  constexpr int LINES = 32 / G::WORDS;   // rows that one instruction copies
  const auto fetch = [&](int chunk, int stage, int64_t where) {
    if (chunk < chunks) {
      const uint32_t to = mine + stage * G::STAGE + line * G::ROW;
      if (WHOLE && where >= 0) {
        const T *ks = k + where + line * DIM + word * G::EACH, *vs = v + where + line * DIM + word * G::EACH;
        if (lane == 0) valid[warp][stage] = 0xffffu;
#pragma unroll
        for (int i = 0; i < CHUNK / LINES; ++i) {
          const int r = i * LINES + line;
          copy_word(to + i * LINES * G::ROW + ((word ^ (r & 7)) << 4), ks + i * LINES * DIM);
          copy_word(to + i * LINES * G::ROW + G::PART + ((word ^ value_swizzle<F32>(r)) << 4), vs + i * LINES * DIM);
        }
      } else {
        if (WHOLE) where = slot_of(chunk);
        const unsigned ok = __ballot_sync(0xffffffffu, where >= 0);
        if (lane == 0) valid[warp][stage] = ok;
#pragma unroll
        for (int i = 0; i < CHUNK / LINES; ++i) {
          const int64_t from = __shfl_sync(0xffffffffu, where, i * LINES + line);
          const bool there = from >= 0 && word * G::EACH < p.dim;
          const int64_t src = there ? from + word * G::EACH : 0;
          const int r = i * LINES + line;
          copy_word(to + i * LINES * G::ROW + ((word ^ (r & 7)) << 4), k + src, there ? 16 : 0);
          copy_word(to + i * LINES * G::ROW + G::PART + ((word ^ value_swizzle<F32>(r)) << 4), v + src, there ? 16 : 0);
        }
      }
    }
    sm100::cp_async_commit();
  };
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) fetch(warp + s * WARPS, s, offset_of(warp + s * WARPS));
  int64_t ahead = offset_of(warp + (STAGES - 1) * WARPS);

  // the queries: head `row` of each tile; fp32 ones as they are, split where they are used
  uint32_t q[HEADS][STEPS][2];
#pragma unroll
  for (int t = 0; t < HEADS; ++t)
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        constexpr int N = 4 / sizeof(T);
        const int h = t * 8 + row, d = s * 2 * G::EACH + i * G::EACH + pair * N;
        elem::Vec<T, N> part;
        part.word = 0;
        if (h < at.heads && d < p.dim) {
          const T *src = static_cast<const T *>(p.q) + at.batch * p.q_stride + static_cast<int64_t>(at.head0 + h) * p.dim + d;
#pragma unroll
          for (int j = 0; j < N; ++j) part.v[j] = mb_load(src + j);
        }
        q[t][s][i] = part.word;
      }
  // heads 2 pair and 2 pair + 1 of each tile: values row and row + 8 of every 16, maximum, and this lane's part of the sum
  float acc[HEADS][DIM_STEPS][4], top[HEADS][2], sum[HEADS][2];
#pragma unroll
  for (int t = 0; t < HEADS; ++t) {
#pragma unroll
    for (int j = 0; j < 2; ++j) top[t][j] = -INFINITY, sum[t][j] = 0.f;
#pragma unroll
    for (int d = 0; d < DIM_STEPS; ++d)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[t][d][j] = 0.f;
  }
  // ldmatrix: keys row lane % 16, values row lane % 8 + lane / 16 * 8; their words' swizzle within 128 bytes
  const uint32_t key_row = lane % 16 * G::ROW, value_row = (lane % 8 + lane / 16 * 8) * G::ROW;
  uint32_t key_word[4], value_word[4];
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    key_word[d] = key_row + (((2 * d + lane / 16) ^ (lane & 7)) << 4);
    // fp32: value `row` (+ 8: d & 1) of every 16 and slot `pair` (+ 4: d & 2) of every 8; every other 16 four words on
    value_word[d] = F32 ? (pair + d / 2 * 4) * G::ROW + (((row / 4 + d % 2 * 2) ^ value_swizzle<F32>(pair + d / 2 * 4)) << 4) + row % 4 * 4
                        : value_row + (((2 * d + lane / 8 % 2) ^ (lane & 7)) << 4);
  }

  int stage = 0;
  for (int chunk = warp; chunk < chunks; chunk += WARPS) {
    sm100::cp_async_wait<STAGES - 2>();
    __syncwarp();
    fetch(chunk + (STAGES - 1) * WARPS, stage == 0 ? STAGES - 1 : stage - 1, ahead);
    ahead = offset_of(chunk + STAGES * WARPS);
    const uint32_t keys = mine + stage * G::STAGE, values = keys + G::PART;
    const unsigned ok = valid[warp][stage];
    // slots row and row + 8: s[t][0, 1] and s[t][2, 3] are heads 2 pair and 2 pair + 1
    float s[HEADS][4];
#pragma unroll
    for (int t = 0; t < HEADS; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[t][j] = 0.f;
    // (fp32: an MMA cuts its sum off, always towards zero; so large products gather in fours, small ones by themselves)
    float large[4] = {0.f, 0.f, 0.f, 0.f}, small[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int d = 0; d < STEPS; ++d) {
      uint32_t a[4];
      load_matrices<false>(keys + key_word[d % 4] + d / 4 * 128, a);
      if constexpr (F32) {
        uint32_t hi[4], lo[4], qh[2], ql[2];
#pragma unroll
        for (int i = 0; i < 4; ++i) Mma<T>::split(a[i], hi[i], lo[i]);
#pragma unroll
        for (int i = 0; i < 2; ++i) Mma<T>::split(q[0][d][i], qh[i], ql[i]);
        Mma<T>::run(small, hi, ql[0], ql[1]);
        Mma<T>::run(small, lo, qh[0], qh[1]);
        Mma<T>::run(large, hi, qh[0], qh[1]);
        if (d % 4 == 3) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            s[0][j] += d == STEPS - 1 ? large[j] + small[j] : large[j];
            large[j] = 0.f;
          }
        }
      } else {
#pragma unroll
        for (int t = 0; t < HEADS; ++t) Mma<T>::run(s[t], a, q[t][d][0], q[t][d][1]);
      }
    }
    if constexpr (F32) {
      // NaN: an infinite key or query, which a pair of tf32 numbers does not hold, or one that is NaN.  Once more, by the definition.
      if (__any_sync(0xffffffffu, s[0][0] != s[0][0] || s[0][1] != s[0][1] || s[0][2] != s[0][2] || s[0][3] != s[0][3])) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int h = pair * 2 + j % 2, r = row + j / 2 * 8;
          const T *src = static_cast<const T *>(p.q) + at.batch * p.q_stride + static_cast<int64_t>(at.head0 + h) * p.dim;
          float dot = 0.f;
          for (int d = 0; d < p.dim && h < at.heads; ++d) {
            float x;
            asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(keys + r * G::ROW + ((d / 4 ^ (r & 7)) << 4) + d % 4 * 4) : "memory");
            dot += x * elem::widen(mb_load(src + d));
          }
          s[0][j] = dot;
        }
        __syncwarp();
      }
    }
#pragma unroll
    for (int t = 0; t < HEADS; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[t][j] *= p.scale2;
    if (ok != 0xffffu) {
#pragma unroll
      for (int t = 0; t < HEADS; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if ((ok >> (row + j / 2 * 8) & 1u) == 0) s[t][j] = -INFINITY;
    }
    if (p.logits != nullptr) {
      const int slot = at.begin + chunk * CHUNK + row;
#pragma unroll
      for (int t = 0; t < HEADS; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int h = t * 8 + pair * 2 + j % 2, n = slot + j / 2 * 8;
          if (h < at.heads && n < at.end)
            p.logits[(static_cast<int64_t>(at.batch) * p.heads + at.head0 + h) * p.logits_stride + n] = s[t][j];
        }
    }
    float m[HEADS][2];
    bool grew = false;
#pragma unroll
    for (int t = 0; t < HEADS; ++t)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        m[t][j] = fmaxf(s[t][j], s[t][j + 2]);
        grew = grew || m[t][j] > top[t][j];
      }
    // (a maximum that no lane exceeds stays: neither the exchange nor the factors are needed)
    if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
      for (int t = 0; t < HEADS; ++t)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
          for (int o = 4; o < 32; o *= 2) m[t][j] = fmaxf(m[t][j], __shfl_xor_sync(0xffffffffu, m[t][j], o));
          m[t][j] = fmaxf(m[t][j], top[t][j]);
          const float back = m[t][j] == -INFINITY ? 1.f : exp2f(top[t][j] - m[t][j]);
          top[t][j] = m[t][j];
          sum[t][j] *= back;
#pragma unroll
          for (int d = 0; d < DIM_STEPS; ++d) {
            acc[t][d][j] *= back;
            acc[t][d][j + 2] *= back;
          }
        }
    }
    if constexpr (F32) {
      // probabilities to the other operand's place, by way of shared memory
      const float m0 = top[0][0] == -INFINITY ? 0.f : top[0][0], m1 = top[0][1] == -INFINITY ? 0.f : top[0][1];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float x = exp2f(s[0][2 * i] - m0) * RAISED<T>, y = exp2f(s[0][2 * i + 1] - m1) * RAISED<T>;
        sum[0][0] += x;
        sum[0][1] += y;
        *reinterpret_cast<float2 *>(&weight_s[warp][row + 8 * i][2 * pair]) = make_float2(x, y);
      }
      __syncwarp();
      uint32_t ph[4], pl[4];   // slots pair, pair + 4 of the first eight, of the others
#pragma unroll
      for (int i = 0; i < 4; ++i) Mma<T>::split(__float_as_uint(weight_s[warp][i * 4 + pair][row]), ph[i], pl[i]);
#pragma unroll
      for (int d = 0; d < DIM_STEPS; ++d) {
        uint32_t hi[2][4], lo[2][4];
        float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            // (the swizzle's low three bits: every other 16 values are four words on)
            const uint32_t addr = values + half * 8 * G::ROW + ((value_word[i] ^ (d % 2 << 6)) + d / 2 * 128);
            uint32_t x;
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(x) : "r"(addr) : "memory");
            Mma<T>::cut(x, hi[half][i], lo[half][i]);
          }
        // small products first; what the chunk gives is added to the sum by rounding
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          Mma<T>::run(part, hi[half], pl[2 * half], pl[2 * half + 1]);
          Mma<T>::run(part, lo[half], ph[2 * half], ph[2 * half + 1]);
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) Mma<T>::run(part, hi[half], ph[2 * half], ph[2 * half + 1]);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[0][d][j] += part[j];
      }
      __syncwarp();
    } else {
      uint32_t least = 0xffffffffu;   // the smallest probability's bits less one: zeros come last
#pragma unroll
      for (int t = 0; t < HEADS; ++t) {
        const float m0 = top[t][0] == -INFINITY ? 0.f : top[t][0], m1 = top[t][1] == -INFINITY ? 0.f : top[t][1];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          s[t][2 * i] = exp2f(s[t][2 * i] - m0) * RAISED<T>;
          s[t][2 * i + 1] = exp2f(s[t][2 * i + 1] - m1) * RAISED<T>;
          sum[t][0] += s[t][2 * i];
          sum[t][1] += s[t][2 * i + 1];
          if (HALVES) least = min(least, min(__float_as_uint(s[t][2 * i]) - 1u, __float_as_uint(s[t][2 * i + 1]) - 1u));
        }
      }
      if constexpr (HALVES) {
        if (__any_sync(0xffffffffu, least < __float_as_uint(LEAST) - 1u)) {
          // those below LEAST by themselves, STEP times as large each time (an fp32 probability is above 2^-149: six times)
          constexpr float STEP = RAISED<T> / LEAST;
          float x[HEADS][4], down = 1.f;
#pragma unroll
          for (int t = 0; t < HEADS; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              x[t][j] = s[t][j] < LEAST ? s[t][j] : 0.f;
              s[t][j] = s[t][j] < LEAST ? 0.f : s[t][j];
            }
          bool more = true;
          while (__any_sync(0xffffffffu, more)) {
            more = false;
            down *= 1.f / STEP;
            uint32_t hi[HEADS][2], lo[HEADS][2];
#pragma unroll
            for (int t = 0; t < HEADS; ++t)
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                float now[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                  float &v = x[t][2 * i + j];
                  v *= STEP;
                  now[j] = v < LEAST ? 0.f : v;
                  v = v < LEAST ? v : 0.f;
                  more = more || v > 0.f;
                }
                Mma<T>::split(now[0], now[1], hi[t][i], lo[t][i]);
                hi[t][i] = transposed(hi[t][i]);
                lo[t][i] = transposed(lo[t][i]);
              }
#pragma unroll
            for (int d = 0; d < DIM_STEPS; ++d) {
              uint32_t a[4];
              load_matrices<true>(values + value_word[d % 4] + d / 4 * 128, a);
#pragma unroll
              for (int t = 0; t < HEADS; ++t) {
                float part[4] = {0.f, 0.f, 0.f, 0.f};
                Mma<T>::run(part, a, lo[t][0], lo[t][1]);
                Mma<T>::run(part, a, hi[t][0], hi[t][1]);
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[t][d][j] += part[j] * down;
              }
            }
          }
        }
      }
      uint32_t hi[HEADS][2], lo[HEADS][2];
#pragma unroll
      for (int t = 0; t < HEADS; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          Mma<T>::split(s[t][2 * i], s[t][2 * i + 1], hi[t][i], lo[t][i]);
          hi[t][i] = transposed(hi[t][i]);
          lo[t][i] = transposed(lo[t][i]);
        }
#pragma unroll
      for (int d = 0; d < DIM_STEPS; ++d) {
        uint32_t a[4];
        load_matrices<true>(values + value_word[d % 4] + d / 4 * 128, a);
#pragma unroll
        for (int t = 0; t < HEADS; ++t) {
          Mma<T>::run(acc[t][d], a, hi[t][0], hi[t][1]);
          Mma<T>::run(acc[t][d], a, lo[t][0], lo[t][1]);
        }
      }
    }
    stage = stage + 1 == STAGES ? 0 : stage + 1;
  }
  sm100::cp_async_wait<0>();
  __syncthreads();
  float *acc_s = reinterpret_cast<float *>(ring);
#pragma unroll
  for (int t = 0; t < HEADS; ++t)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int o = 4; o < 32; o *= 2) sum[t][j] += __shfl_xor_sync(0xffffffffu, sum[t][j], o);
      const int h = t * 8 + pair * 2 + j;
      if (h < at.heads) {
        const int r = warp * R + h;
        if (row == 0) {
          top_s[r] = top[t][j];
          sum_s[r] = sum[t][j];
        }
#pragma unroll
        for (int d = 0; d < DIM_STEPS; ++d) {
          acc_s[r * G::PITCH + d * 16 + row] = acc[t][d][j];
          acc_s[r * G::PITCH + d * 16 + row + 8] = acc[t][d][j + 2];
        }
      }
    }
  __syncthreads();
  finish<T, R>(p, at, G::PITCH, top_s, sum_s, acc_s, coef, total);
}

template <typename T, int DIM, int HEADS, bool WHOLE>
int launch_mma(mb_context *ctx, const AttentionParams &p, unsigned grid, int index) {
  const auto kern = paged_attention_mma_kernel<T, DIM, HEADS, WHOLE>;
  index += (HEADS - 1) * 2 + WHOLE;
  if (!(ctx->attention_attr_mask & (1ull << index))) {
    MB_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Ring<T, DIM>::BYTES));
    MB_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));   // clusters of 16
    ctx->attention_attr_mask |= 1ull << index;
  }
  MB_CUDA(ctx, mb_launch_clusters(ctx, kern, grid, THREADS, Ring<T, DIM>::BYTES, p.cluster, p));
  return MB_SUCCESS;
}

template <typename T, int DIM>
int launch_mma(mb_context *ctx, const AttentionParams &p, unsigned grid, int rows, int index) {
  const bool whole = p.dim == DIM && p.page_size % Ring<T, DIM>::CHUNK == 0;
  if constexpr (sizeof(T) == 2 && DIM <= 128) {
    if (rows > 16) return whole ? launch_mma<T, DIM, 3, true>(ctx, p, grid, index) : launch_mma<T, DIM, 3, false>(ctx, p, grid, index);
  }
  if constexpr (sizeof(T) == 2) {
    if (rows > 8) return whole ? launch_mma<T, DIM, 2, true>(ctx, p, grid, index) : launch_mma<T, DIM, 2, false>(ctx, p, grid, index);
  }
  return whole ? launch_mma<T, DIM, 1, true>(ctx, p, grid, index) : launch_mma<T, DIM, 1, false>(ctx, p, grid, index);
}

template <typename T>
int launch_mma(mb_context *ctx, const AttentionParams &p, unsigned grid, int rows, int index) {
  if (p.dim <= 64) return launch_mma<T, 64>(ctx, p, grid, rows, index);
  if (sizeof(T) == 4 || p.dim <= 128) return launch_mma<T, 128>(ctx, p, grid, rows, index + 6);
  if constexpr (sizeof(T) == 2) return launch_mma<T, 256>(ctx, p, grid, rows, index + 12);
  return MB_SUCCESS;
}

// What each slot has received of the query heads' probabilities, on top of what it had.  Four slots a thread (kv::WEIGHT_SLOTS a block): a
// word of every head's logits, all in flight together.
__global__ void __launch_bounds__(256) attention_weights_kernel(const AttentionParams p, int chunks) {
  mb_grid_dep_launch();
  mb_grid_dep_wait();
  const int unit = blockIdx.x / chunks, batch = unit / p.kv_heads, kv_head = unit % p.kv_heads;
  const int slot = (blockIdx.x % chunks) * kv::WEIGHT_SLOTS + threadIdx.x * 4;
  bool bad;
  const int length = kv::usable_length(mb_load(p.lengths + batch), p.longest, &bad);
  if (slot >= length) return;
  const int first = kv::window_begin(length, p.window);
  const int64_t to = static_cast<int64_t>(unit) * p.weights_stride + slot;
  float w[4] = {0.f, 0.f, 0.f, 0.f}, had[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) had[j] = p.weights_in != nullptr && slot + j < length ? mb_load(p.weights_in + to + j) : 0.f;
  if (slot + 3 >= first) {
    // (rows of logits are whole words; what is outside first .. length is not used)
    const int64_t head = static_cast<int64_t>(batch) * p.heads + kv_head * p.group;
#pragma unroll 4
    for (int g = 0; g < p.group; ++g) {
      const float lse2 = mb_load(p.lse2 + head + g);
      const float4 s = mb_load(reinterpret_cast<const float4 *>(p.logits + (head + g) * p.logits_stride + slot));
      if (lse2 != -INFINITY) {
        w[0] += exp2f(s.x - lse2);
        w[1] += exp2f(s.y - lse2);
        w[2] += exp2f(s.z - lse2);
        w[3] += exp2f(s.w - lse2);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (slot + j < length) p.weights_out[to + j] = had[j] + (slot + j >= first ? w[j] : 0.f);
}

template <typename T, int R, int LANES, int N>
cudaError_t launch_cores(mb_context *ctx, const AttentionParams &p, unsigned grid, bool vec) {
  if (vec) return mb_launch_clusters(ctx, paged_attention_kernel<T, R, LANES, N, true>, grid, THREADS, 0, p.cluster, p);
  return mb_launch_clusters(ctx, paged_attention_kernel<T, R, LANES, N, false>, grid, THREADS, 0, p.cluster, p);
}

template <typename T, int R>
cudaError_t launch_cores(mb_context *ctx, const AttentionParams &p, unsigned grid, bool vec) {
  if (p.dim <= 32) return launch_cores<T, R, 8, 1>(ctx, p, grid, vec);
  if (p.dim <= 64) return launch_cores<T, R, 16, 1>(ctx, p, grid, vec);
  if (p.dim <= 128) return launch_cores<T, R, 32, 1>(ctx, p, grid, vec);
  return launch_cores<T, R, 32, 2>(ctx, p, grid, vec);
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

  const bool f32 = dtype == MB_F32;
  // (a pool without pages has no address that a copy of no bytes could name)
  const bool by_mma = ctx->use_tensor_cores && num_pages > 0 && head_dim % (f32 ? 4 : 8) == 0 && (!f32 || head_dim <= 128) && kv::aligned(k_cache, 16) &&
                      kv::aligned(v_cache, 16);
  // Rows of a block: as many of a group's heads as registers hold, since every block of heads reads the run again (20 heads of 128 in one
  // block of 24 142 us, in two of 16 171).
  const bool three = by_mma && !f32 && head_dim <= 128 && (p.group + 23) / 24 < (p.group + 15) / 16;
  const int rows = three ? 24 : by_mma ? (p.group > 8 && !f32 ? 16 : 8) : p.group >= 5 ? 8 : p.group >= 3 ? 4 : p.group;
  p.blocks = (p.group + rows - 1) / rows;
  p.batch = static_cast<int>(batch);
  p.pitch = static_cast<int>(align_up(p.dim, 4));
  const int64_t units = batch * kv_heads * p.blocks;
  const int per_sm = three ? 2 : !by_mma ? (rows * p.dim >= 1024 ? 3 : 5) : p.dim * kv::type_bytes(dtype) > 256 ? 1 : p.dim * kv::type_bytes(dtype) > 128 ? 3 : 4;
  // Small work: each head's slots over a cluster, which joins without memory.  What a block of one can be given: 1024 slots of 16-bit
  // types on the tensor cores, 512 of fp32 ones up to 64, 256 up to 128, and 128 on CUDA cores, whose clusters are of 8 (one head of 128, bf16, on clusters
  // and as runs: 1000 slots 7.0 and 9.4 us, 16000 21.2 and 25.3, 32000 34.1 and 27.1; fp32 4000 15.7 and 15.4, 8000 23.7 and 19.6; fp32 of 256,
  // CUDA cores, 1000 26.4 and 28.3, 2000 70.7 and 43.2).  All of a launch's are resident at once: where a block fills an SM, as many as
  // the device's clusters of one CTA an SM (8 heads of 256, 2000 slots, on 128 CTAs in clusters of 16, of which 112 are resident: 20.8 us,
  // as runs 16.2).
  int64_t room_for[5];
  for (int i = 0; i < 5; ++i) room_for[i] = per_sm > 1 ? 2 * ctx->num_sms : mb_resident_cluster_ctas(ctx, 1 << i);
  const int share = !by_mma ? 128 : !f32 ? 1024 : head_dim <= 64 ? 512 : 256;
  p.cluster = kv::cluster_of(units, p.longest, 2 * head_dim * kv::type_bytes(dtype), by_mma ? 16 : 8, share, room_for);
  // The runs wanted of all heads together: one round of resident blocks where the heads leave room for it, less one for each head, whose
  // last run is not a whole one; else half as many again as are resident.  (256 heads of 4096 slots, 444 blocks resident: 444 wanted
  // 105 us, 666 90, 888 97; 512 ragged ones of up to 8192: 168, 164, 164.  As many as fill the last round, up to 8 of them: 94 and 173.)
  const int64_t slots = static_cast<int64_t>(per_sm) * ctx->num_sms;
  p.wanted = static_cast<int>(units * 2 <= slots ? slots - units : slots * 3 / 2);
  int64_t runs = std::min<int64_t>(units + p.wanted, units * std::max<int64_t>(1, ceil_div64(p.longest + 15, LEAST_RUN)));
  if (p.cluster > 1) {
    runs = units * p.cluster;
  } else if (batch > SCANNED) {
    // (reading thousands of lengths in every block costs more than it evens out)
    p.fixed_runs = static_cast<int>(std::min<int64_t>(16, std::max<int64_t>(1, ceil_div64(p.longest, 4096))));
    p.fixed_run = static_cast<int>(ceil_div64(ceil_div64(std::max<int64_t>(p.longest + 15, 1), p.fixed_runs), 64) * 64);
    runs = units * p.fixed_runs;
  }
  if (runs > kv::MOST) return mb_fail(ctx, MB_UNSUPPORTED, "mb_paged_attention: too many sequences and heads");
  const size_t partial = runs > units && p.cluster == 1 ? align_up(sizeof(float) * runs * (rows * p.pitch + std::max(4, 2 * rows)), 256) : 0;
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
  const unsigned grid = static_cast<unsigned>(runs);
  cudaError_t e = cudaSuccess;
  if (by_mma) {
    if (f32) MB_RETURN_IF_ERROR(launch_mma<float>(ctx, p, grid, rows, 36));
    else if (dtype == MB_F16) MB_RETURN_IF_ERROR(launch_mma<__half>(ctx, p, grid, rows, 0));
    else MB_RETURN_IF_ERROR(launch_mma<__nv_bfloat16>(ctx, p, grid, rows, 18));
  } else MB_FOR_ELEMENT(dtype, {
    const uintptr_t word = 4 * sizeof(T);
    const bool vec = p.dim % 4 == 0 && q_stride % 4 == 0 && kv::aligned(q, word) && kv::aligned(k_cache, word) && kv::aligned(v_cache, word);
    e = rows == 8 ? launch_cores<T, 8>(ctx, p, grid, vec) : rows == 4 ? launch_cores<T, 4>(ctx, p, grid, vec)
      : rows == 2 ? launch_cores<T, 2>(ctx, p, grid, vec) : launch_cores<T, 1>(ctx, p, grid, vec);
  });
  MB_CUDA(ctx, e);
  ctx->launches++;
  if (logits > 0) {
    const int chunks = (p.longest + kv::WEIGHT_SLOTS - 1) / kv::WEIGHT_SLOTS;
    MB_CUDA(ctx, mb_launch_chained(ctx, attention_weights_kernel, dim3(static_cast<unsigned>(batch * kv_heads * chunks)), dim3(256), 0, p, chunks));
    ctx->launches++;
  }
  return MB_SUCCESS;
}
