// Eviction from a paged cache by accumulated attention weight: of every kv head's slots the heaviest are kept, in order.
//
// Two kernels.  The first finds, per sequence and kv head, the weight of the last slot that is kept: a radix selection from the top
// digit down, on the weights' order-preserving integers.  Above that weight everything stays, of those equal to it the lowest slots; a
// prefix sum over counts then gives every kept slot its place.  The second copies rows of keys and values.
#include <algorithm>

#include "elements.cuh"
#include "gemm_u8_cut.cuh"
#include "kv_cache.h"
#include "sm100_ptx.cuh"

namespace {

constexpr int COPY_THREADS = 256;
constexpr int COPY_EACH = 2;   // words a thread has in flight, of keys and of values each (four: 57.9 us for 54.5 at 16 x 8 heads of 2048 kept)

struct EvictParams {
  const void *k_src, *v_src;
  void *k_dst, *v_dst;
  const int32_t *src_table, *dst_table, *lengths;
  const float *weights;
  int32_t *dst_lengths, *kept;
  float *dst_weights;
  int64_t weights_stride, src_pages, dst_pages;
  int dst_weights_stride;
  int kv_heads, dim, page_size, src_max_pages, dst_max_pages, longest, budget, sinks, recent;
  uint32_t page_mul, page_shift;
  int cluster, cached;   // CTAs that select for a head; whether a run of weights fits into one's shared memory
  int words, chunks;     // of a row; blocks of a head's rows
  uint32_t word_mul, word_shift;
  int *status;
};

// Larger weights give larger numbers, -0 and 0 the same, NaN the smallest.
__device__ __forceinline__ uint32_t order_of(float w) {
  if (w != w) return 0;
  const uint32_t u = __float_as_uint(w + 0.f);
  return (u & 0x80000000u) != 0 ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ unsigned load_remote_u32(uint32_t addr, int rank) {
  unsigned v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(sm100::mapa_shared(addr, rank)) : "memory");
  return v;
}

// A cluster of CTAs per sequence and kv head, each with a run of the candidates, whose order-preserving integers it keeps in shared
// memory (where they fit: `cached`).  Digits of 11, 11 and 10 bits; every CTA counts its own, after a cluster barrier each adds up all
// CTAs' counts through distributed shared memory and comes to the same digit.  What bounds it: two passes over counts and a cluster
// barrier for each digit, about 1 us, not the weights (33333 of them, 4 heads: 39 us with one CTA a head and bytes as digits, 18 here).
constexpr int DIGIT = 2048, GROUPS = DIGIT / 32;

// The sum over the lanes up to this one.
__device__ __forceinline__ unsigned upto_lane(unsigned v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const unsigned below = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += below;
  }
  return v;
}

template <int SELECT_THREADS>
__global__ void __launch_bounds__(SELECT_THREADS, 1024 / SELECT_THREADS) evict_select_kernel(const EvictParams p) {
  constexpr int SELECT_WARPS = SELECT_THREADS / 32;
  extern __shared__ uint32_t keys[];
  __shared__ __align__(8) unsigned counts[3][DIGIT], groups[3][GROUPS];
  __shared__ unsigned above[SELECT_WARPS], equal[SELECT_WARPS], mine[2];
  __shared__ unsigned digit_s, left_s, held_s;
  mb_grid_dep_launch();
  mb_grid_dep_wait();
  const int rank = p.cluster > 1 ? static_cast<int>(sm100::cluster_ctarank()) : 0;
  const int unit = blockIdx.x / p.cluster, batch = unit / p.kv_heads;
  const int t = threadIdx.x, warp = t / 32, lane = t % 32;
  bool bad;
  const int length = kv::usable_length(mb_load(p.lengths + batch), p.longest, &bad);
  if (bad && t == 0 && rank == 0) mb_report_bad_index(p.status);
  const float *w = p.weights + unit * p.weights_stride;
  int32_t *kept = p.kept + static_cast<int64_t>(unit) * p.budget;
  const int all = p.cluster * SELECT_THREADS, me = rank * SELECT_THREADS + t;
  if (length <= p.budget) {   // (the whole cluster agrees)
    for (int64_t j = me; j < p.budget; j += all) kept[j] = j < length ? static_cast<int32_t>(j) : -1;
    return;
  }
  // candidates lie between the first and the last slots that stay in any case
  const int first = p.sinks, end = length - p.recent, places = p.budget - p.sinks - p.recent;
  const int run = (end - first + p.cluster - 1) / p.cluster;
  const int from = min(static_cast<int64_t>(first) + static_cast<int64_t>(rank) * run, static_cast<int64_t>(end));
  const int until = end - from < run ? end : from + run;
  const auto key = [&](int j) { return p.cached ? keys[j - from] : order_of(mb_load(w + j)); };
  uint32_t limit = 0xffffffffu;   // (no place: nothing is above, and none of the equal ones is taken)
  unsigned ties = 0;
  for (int i = t; i < 3 * DIGIT; i += SELECT_THREADS) (&counts[0][0])[i] = 0;
  if (p.cached) {
    for (int base = from + t; base - t < until; base += 8 * SELECT_THREADS) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = until - base > i * SELECT_THREADS ? mb_load(w + base + i * SELECT_THREADS) : 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (until - base > i * SELECT_THREADS) keys[base - from + i * SELECT_THREADS] = order_of(v[i]);
    }
  }
  for (int j = me; j < first; j += all) kept[j] = j;
  for (int j = me; j < p.recent; j += all) kept[p.budget - p.recent + j] = end + j;
  __syncthreads();
  if (places > 0) {
    uint32_t prefix = 0, mask = 0;
    unsigned left = places;
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
      const uint32_t digits = pass == 2 ? 1023u : 2047u;
      unsigned *count = counts[pass];
#pragma unroll 4
      for (int base = from; base < until; base += SELECT_THREADS) {
        const int j = base + t;
        const uint32_t u = j < until ? key(j) : 0;
        const bool counts_in = j < until && (u & mask) == prefix;
        const unsigned in = __ballot_sync(0xffffffffu, counts_in);
        if (in == 0) continue;
        const uint32_t d = (u >> shift) & digits;
        // (weights that are all alike would queue at one counter)
        int same = 0;
        if (in == 0xffffffffu) __match_all_sync(0xffffffffu, d, &same);
        if (same) {
          if (lane == 0) atomicAdd(count + d, 32u);
        } else if (counts_in) {
          atomicAdd(count + d, 1u);
        }
      }
      __syncthreads();
      // sums of 32 digits each, so that what the CTAs read of one another is 64 sums and then 32 counts
      for (int g = warp; g < GROUPS; g += SELECT_WARPS) {
        const unsigned sum = __reduce_add_sync(0xffffffffu, count[g * 32 + lane]);
        if (lane == 0) groups[pass][g] = sum;
      }
      if (p.cluster > 1) sm100::cluster_sync_all();
      else __syncthreads();
      if (warp == 0) {
        // lane l has groups 63 - 2 l and 62 - 2 l, then digit 31 - l of the group that is found: from the largest down
        const int g = GROUPS - 2 - 2 * lane;
        unsigned low = 0, high = 0;
        if (p.cluster > 1) {
          const uint32_t addr = sm100::smem_u32(&groups[pass][g]);
#pragma unroll 8
          for (int s = 0; s < p.cluster; ++s) {
            unsigned x, y;
            asm volatile("ld.shared::cluster.v2.u32 {%0, %1}, [%2];" : "=r"(x), "=r"(y) : "r"(sm100::mapa_shared(addr, s)) : "memory");
            low += x;
            high += y;
          }
        } else {
          low = groups[pass][g];
          high = groups[pass][g + 1];
        }
        unsigned before = upto_lane(low + high, lane) - low - high;
        const unsigned here = __ballot_sync(0xffffffffu, before < left && left <= before + low + high);
        const int who = __ffs(here) - 1;
        const bool upper = left <= before + high;
        const int group = __shfl_sync(0xffffffffu, upper ? g + 1 : g, who);
        const unsigned base = __shfl_sync(0xffffffffu, upper ? before : before + high, who);
        const int d = group * 32 + 31 - lane;
        unsigned n = 0;
        if (p.cluster > 1) {
          const uint32_t addr = sm100::smem_u32(count + d);
#pragma unroll 8
          for (int s = 0; s < p.cluster; ++s) n += load_remote_u32(addr, s);
        } else {
          n = count[d];
        }
        before = base + upto_lane(n, lane) - n;
        if (before < left && left <= before + n) {
          digit_s = d;
          left_s = left - before;
          held_s = n;
        }
      }
      __syncthreads();
      prefix |= digit_s << shift;
      mask |= digits << shift;
      left = left_s;
      // (all that begin with these digits stay: nothing left to tell apart)
      if (held_s == left && prefix != 0) {
        limit = prefix - 1;
        break;
      }
      if (pass == 2) {
        limit = prefix;
        ties = left;
      }
    }
  }
  // every warp has a part of the run: what it holds, then what lies before it, then where its own go
  const int part = (until - from + SELECT_THREADS - 1) / SELECT_THREADS * 32;
  const int mine_from = min(from + warp * part, until), mine_until = until - mine_from < part ? until : mine_from + part;
  unsigned a = 0, e = 0;
  for (int j = mine_from + lane; j < mine_until; j += 32) {
    const uint32_t u = key(j);
    a += u > limit;
    e += u == limit;
  }
  a = __reduce_add_sync(0xffffffffu, a);
  e = __reduce_add_sync(0xffffffffu, e);
  __syncthreads();
  if (lane == 0) {
    above[warp] = a;
    equal[warp] = e;
  }
  __syncthreads();
  a = e = 0;
  for (int i = 0; i < warp; ++i) {
    a += above[i];
    e += equal[i];
  }
  if (p.cluster > 1) {
    if (t == SELECT_THREADS - 32) {   // (the last warp's first lane has all but its own)
      mine[0] = a + above[warp];
      mine[1] = e + equal[warp];
    }
    sm100::cluster_sync_all();
    for (int s = 0; s < rank; ++s) {
      a += load_remote_u32(sm100::smem_u32(&mine[0]), s);
      e += load_remote_u32(sm100::smem_u32(&mine[1]), s);
    }
    // (no CTA may leave while another reads its counts: arrive here, wait at the end)
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  }
  for (int base = mine_from; base < mine_until; base += 32) {
    const int j = base + lane;
    const uint32_t u = j < mine_until ? key(j) : 0;
    const unsigned more = __ballot_sync(0xffffffffu, j < mine_until && u > limit), same = __ballot_sync(0xffffffffu, j < mine_until && u == limit);
    const unsigned lower = (1u << lane) - 1u;
    const unsigned rank_of = e + __popc(same & lower);
    if ((more >> lane & 1u) != 0 || ((same >> lane & 1u) != 0 && rank_of < ties)) {
      kept[first + a + __popc(more & lower) + min(rank_of, ties)] = j;
    }
    a += __popc(more);
    e += __popc(same);
  }
  if (p.cluster > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Rows of keys and values to their new slots, a word per item, their weights (zeros behind them where asked for), and the new lengths (here,
// because the other kernel reads the old ones and the two may be the same memory).
// (CLEAR apart: its loop in the other form costs 5 of 54 us.)
template <typename Word, bool CLEAR>
__global__ void __launch_bounds__(COPY_THREADS) evict_copy_kernel(const EvictParams p) {
  mb_grid_dep_launch();
  mb_grid_dep_wait();
  const int unit = blockIdx.x / p.chunks, chunk = blockIdx.x % p.chunks;
  const int batch = unit / p.kv_heads, head = unit % p.kv_heads;
  if (chunk == 0 && head == 0 && threadIdx.x == 0) {
    bool bad;
    p.dst_lengths[batch] = min(kv::usable_length(mb_load(p.lengths + batch), p.longest, &bad), p.budget);
  }
  if constexpr (CLEAR) {   // (the length may be the new one already: cut by the budget, both are the same)
    bool bad;
    const int64_t length = min(kv::usable_length(mb_load(p.lengths + batch), p.longest, &bad), p.budget);
    float *row = p.dst_weights + static_cast<int64_t>(unit) * p.dst_weights_stride;
    for (int64_t j = length + chunk * COPY_THREADS + threadIdx.x; j < p.dst_weights_stride; j += static_cast<int64_t>(p.chunks) * COPY_THREADS) row[j] = 0.f;
  }
  const int32_t *kept = p.kept + static_cast<int64_t>(unit) * p.budget;
  const int32_t *src_table = p.src_table + static_cast<int64_t>(batch) * p.src_max_pages;
  const int32_t *dst_table = p.dst_table + static_cast<int64_t>(batch) * p.dst_max_pages;
  const int rows = COPY_THREADS * COPY_EACH / p.words;   // whole rows of a block; at least one
  // three loads that wait for one another, each for all items at once: slots, pages, rows
  int slot[COPY_EACH], src_page[COPY_EACH], dst_page[COPY_EACH];
#pragma unroll
  for (int i = 0; i < COPY_EACH; ++i) {
    const int row = static_cast<int>(fast_div(i * COPY_THREADS + threadIdx.x, p.word_mul, p.word_shift));
    const int64_t j = static_cast<int64_t>(chunk) * rows + row;
    slot[i] = row < rows && j < p.budget ? mb_load(kept + j) : -1;
  }
#pragma unroll
  for (int i = 0; i < COPY_EACH; ++i) {
    const int row = static_cast<int>(fast_div(i * COPY_THREADS + threadIdx.x, p.word_mul, p.word_shift));
    const int j = chunk * rows + row;
    src_page[i] = slot[i] >= 0 ? mb_load(src_table + fast_div(slot[i], p.page_mul, p.page_shift)) : -1;
    dst_page[i] = slot[i] >= 0 ? mb_load(dst_table + fast_div(j, p.page_mul, p.page_shift)) : -1;
  }
  Word k[COPY_EACH], v[COPY_EACH];
  float weight[COPY_EACH];
  int64_t to[COPY_EACH];
#pragma unroll
  for (int i = 0; i < COPY_EACH; ++i) {
    const int item = i * COPY_THREADS + threadIdx.x;
    const int row = static_cast<int>(fast_div(item, p.word_mul, p.word_shift)), word = item - row * p.words, j = chunk * rows + row;
    const int at_slot = max(slot[i], 0);
    const int64_t from = kv::row_offset(src_page[i], p.src_pages, p.kv_heads, head, p.page_size,
                                        at_slot - static_cast<int>(fast_div(at_slot, p.page_mul, p.page_shift)) * p.page_size, p.words);
    const int64_t at = kv::row_offset(dst_page[i], p.dst_pages, p.kv_heads, head, p.page_size,
                                      j - static_cast<int>(fast_div(j, p.page_mul, p.page_shift)) * p.page_size, p.words);
    const bool there = from >= 0 && at >= 0;
    if (!there && slot[i] >= 0) mb_report_bad_index(p.status);
    to[i] = there ? at + word : -1;
    if (there) {
      k[i] = mb_load(static_cast<const Word *>(p.k_src) + from + word);
      v[i] = mb_load(static_cast<const Word *>(p.v_src) + from + word);
    }
    if (slot[i] >= 0 && word == 0) weight[i] = mb_load(p.weights + unit * p.weights_stride + slot[i]);
  }
#pragma unroll
  for (int i = 0; i < COPY_EACH; ++i) {
    const int item = i * COPY_THREADS + threadIdx.x;
    const int row = static_cast<int>(fast_div(item, p.word_mul, p.word_shift));
    if (slot[i] >= 0 && item == row * p.words) p.dst_weights[static_cast<int64_t>(unit) * (CLEAR ? p.dst_weights_stride : p.budget) + chunk * rows + row] = weight[i];
    if (to[i] >= 0) {
      static_cast<Word *>(p.k_dst)[to[i]] = k[i];
      static_cast<Word *>(p.v_dst)[to[i]] = v[i];
    }
  }
}

static_assert(COPY_THREADS * COPY_EACH == kv::COPY_WORDS, "words of a block");

template <typename Word>
int launch_copy(mb_context *ctx, EvictParams &p, int64_t units, const kv::CopyShape &copy, bool clear) {
  p.words = static_cast<int>(copy.words);
  fast_div_make(p.words, &p.word_mul, &p.word_shift);
  p.chunks = static_cast<int>(ceil_div64(std::min(p.budget, std::max(p.longest, 1)), copy.rows));
  MB_CUDA(ctx, mb_launch_chained(ctx, clear ? evict_copy_kernel<Word, true> : evict_copy_kernel<Word, false>, dim3(static_cast<unsigned>(units * p.chunks)), dim3(COPY_THREADS), 0, p));
  ctx->launches++;
  return MB_SUCCESS;
}

int evict(mb_context *ctx, const char *who, const void *k_src, const void *v_src, const int32_t *src_table, const int32_t *lengths,
          const float *weights, void *k_dst, void *v_dst, const int32_t *dst_table, int32_t *dst_lengths, float *dst_weights,
          int32_t *kept, int64_t batch, int64_t kv_heads, int64_t head_dim, int64_t page_size, int64_t src_pages,
          int64_t src_max_pages, int64_t dst_pages, int64_t dst_max_pages, int64_t max_length, int64_t weights_stride,
          int64_t dst_weights_stride, bool clear, int64_t budget, int64_t sinks, int64_t recent, int dtype) {
  if (ctx == nullptr) return MB_INVALID_ARGS;
  const kv::Verdict verdict = kv::check_evict(k_src, v_src, src_table, lengths, weights, k_dst, v_dst, dst_table, dst_lengths,
                                              dst_weights, kept, batch, kv_heads, head_dim, page_size, src_pages, src_max_pages,
                                              dst_pages, dst_max_pages, max_length, weights_stride, budget, sinks, recent, dtype,
                                              dst_weights_stride);
  if (verdict.code != MB_SUCCESS) return mb_fail(ctx, verdict.code, "%s: %s", who, verdict.why);
  if (batch == 0) return MB_SUCCESS;
  MB_CUDA(ctx, cudaSetDevice(ctx->device));
  EvictParams p = {};
  p.k_src = k_src; p.v_src = v_src; p.k_dst = k_dst; p.v_dst = v_dst;
  p.src_table = src_table; p.dst_table = dst_table; p.lengths = lengths; p.weights = weights;
  p.dst_lengths = dst_lengths; p.kept = kept; p.dst_weights = dst_weights;
  p.weights_stride = weights_stride; p.dst_weights_stride = static_cast<int>(dst_weights_stride); p.src_pages = src_pages; p.dst_pages = dst_pages;
  p.kv_heads = static_cast<int>(kv_heads); p.dim = static_cast<int>(head_dim); p.page_size = static_cast<int>(page_size);
  p.src_max_pages = static_cast<int>(src_max_pages); p.dst_max_pages = static_cast<int>(dst_max_pages);
  p.longest = kv::longest_of(max_length, src_max_pages, page_size);
  p.budget = static_cast<int>(budget); p.sinks = static_cast<int>(sinks); p.recent = static_cast<int>(recent);
  fast_div_make(static_cast<uint32_t>(page_size), &p.page_mul, &p.page_shift);
  p.status = ctx->dev_status;

  const int64_t units = batch * kv_heads, row_bytes = head_dim * kv::type_bytes(dtype);
  const kv::CopyShape copy = kv::copy_shape(kv::copy_bits(k_src, v_src, k_dst, v_dst, row_bytes), row_bytes);
  // A CTA of 1024 threads an SM, or, where there are more heads than SMs, two of 512; 4096 weights or more to each of a cluster.
  // (16 sequences of 8192, 8 heads: two CTAs of 512 a head 17.7 us, one of 1024 14.7.)
  constexpr int MOST_KEYS = 20 << 10;
  const bool large = units <= ctx->num_sms;
  p.cluster = 1;
  while (p.cluster < 16 && units * p.cluster * 2 <= ctx->num_sms && p.longest > 4096 * p.cluster) p.cluster *= 2;
  while (p.cluster < 16 && p.longest > MOST_KEYS * p.cluster) p.cluster *= 2;
  const int64_t keys = ceil_div64(p.longest, p.cluster);
  p.cached = keys <= MOST_KEYS;
  if (!ctx->evict_attr_set) {
    for (const auto kern : {evict_select_kernel<512>, evict_select_kernel<1024>}) {
      MB_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, MOST_KEYS * 4));
      MB_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));   // clusters of 16
    }
    ctx->evict_attr_set = true;
  }
  MB_CUDA(ctx, mb_launch_clusters(ctx, large ? evict_select_kernel<1024> : evict_select_kernel<512>, static_cast<unsigned>(units * p.cluster),
                                  large ? 1024 : 512, p.cached ? static_cast<size_t>(keys) * 4 : 0, p.cluster, p));
  ctx->launches++;
  if (copy.word == 16) return launch_copy<uint4>(ctx, p, units, copy, clear);
  if (copy.word == 4) return launch_copy<uint32_t>(ctx, p, units, copy, clear);
  return launch_copy<uint16_t>(ctx, p, units, copy, clear);
}

}  // namespace

extern "C" {

int mb_kv_evict(mb_context *ctx, const void *k_src, const void *v_src, const int32_t *src_table, const int32_t *lengths,
                const float *weights, void *k_dst, void *v_dst, const int32_t *dst_table, int32_t *dst_lengths, float *dst_weights,
                int32_t *kept, int64_t batch, int64_t kv_heads, int64_t head_dim, int64_t page_size, int64_t src_pages,
                int64_t src_max_pages, int64_t dst_pages, int64_t dst_max_pages, int64_t max_length, int64_t weights_stride,
                int64_t budget, int64_t sinks, int64_t recent, int dtype) {
  return evict(ctx, "mb_kv_evict", k_src, v_src, src_table, lengths, weights, k_dst, v_dst, dst_table, dst_lengths, dst_weights, kept,
               batch, kv_heads, head_dim, page_size, src_pages, src_max_pages, dst_pages, dst_max_pages, max_length, weights_stride,
               budget, false, budget, sinks, recent, dtype);
}

int mb_kv_evict_strided(mb_context *ctx, const void *k_src, const void *v_src, const int32_t *src_table, const int32_t *lengths,
                        const float *weights, void *k_dst, void *v_dst, const int32_t *dst_table, int32_t *dst_lengths,
                        float *dst_weights, int32_t *kept, int64_t batch, int64_t kv_heads, int64_t head_dim, int64_t page_size,
                        int64_t src_pages, int64_t src_max_pages, int64_t dst_pages, int64_t dst_max_pages, int64_t max_length,
                        int64_t weights_stride, int64_t dst_weights_stride, int64_t budget, int64_t sinks, int64_t recent, int dtype) {
  if (dst_weights_stride == 0) dst_weights_stride = -1;   // (the check's word for rows of budget)
  return evict(ctx, "mb_kv_evict_strided", k_src, v_src, src_table, lengths, weights, k_dst, v_dst, dst_table, dst_lengths, dst_weights,
               kept, batch, kv_heads, head_dim, page_size, src_pages, src_max_pages, dst_pages, dst_max_pages, max_length,
               weights_stride, dst_weights_stride, true, budget, sinks, recent, dtype);
}

}  // extern "C"
