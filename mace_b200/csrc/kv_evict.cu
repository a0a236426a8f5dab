// Eviction from a paged cache by accumulated attention weight: of every kv head's slots the heaviest are kept, in order.
//
// Two kernels.  The first finds, per sequence and kv head, the weight of the last slot that is kept: a radix selection from the top
// byte down, on the weights' order-preserving integers.  Above that weight everything stays, of those equal to it the lowest slots; a
// prefix sum over counts then gives every kept slot its place.  The second copies rows of keys and values.
#include "elements.cuh"
#include "kv_cache.h"

namespace {

constexpr int SELECT_THREADS = 1024;
constexpr int SELECT_WARPS = SELECT_THREADS / 32;
constexpr int COPY_THREADS = 256;
constexpr int COPY_EACH = 4;   // words a thread has in flight, of keys and of values each

struct EvictParams {
  const void *k_src, *v_src;
  void *k_dst, *v_dst;
  const int32_t *src_table, *dst_table, *lengths;
  const float *weights;
  int32_t *dst_lengths, *kept;
  float *dst_weights;
  int64_t weights_stride, src_pages, dst_pages;
  int kv_heads, dim, page_size, src_max_pages, dst_max_pages, longest, budget, sinks, recent;
  uint32_t page_mul, page_shift;
  int words, chunks;   // of a row; blocks of a head's rows
  uint32_t word_mul, word_shift;
  int *status;
};

// Larger weights give larger numbers, -0 and 0 the same, NaN the smallest.
__device__ __forceinline__ uint32_t order_of(float w) {
  if (w != w) return 0;
  const uint32_t u = __float_as_uint(w + 0.f);
  return (u & 0x80000000u) != 0 ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(SELECT_THREADS) evict_select_kernel(const EvictParams p) {
  __shared__ unsigned count[256];
  __shared__ unsigned above[SELECT_WARPS], equal[SELECT_WARPS];
  __shared__ unsigned digit_s, left_s;
  mb_grid_dep_launch();
  mb_grid_dep_wait();
  const int unit = blockIdx.x, batch = unit / p.kv_heads;
  const int t = threadIdx.x, warp = t / 32, lane = t % 32;
  bool bad;
  const int length = kv::usable_length(mb_load(p.lengths + batch), p.longest, &bad);
  if (bad && t == 0) mb_report_bad_index(p.status);
  const float *w = p.weights + unit * p.weights_stride;
  int32_t *kept = p.kept + static_cast<int64_t>(unit) * p.budget;
  float *to = p.dst_weights + static_cast<int64_t>(unit) * p.budget;
  if (length <= p.budget) {
    for (int j = t; j < p.budget; j += SELECT_THREADS) {
      kept[j] = j < length ? j : -1;
      if (j < length) to[j] = mb_load(w + j);
    }
    return;
  }
  // candidates lie between the first and the last slots that stay in any case
  const int first = p.sinks, end = length - p.recent, places = p.budget - p.sinks - p.recent;
  uint32_t limit = 0xffffffffu;   // (no place: nothing is above, and none of the equal ones is taken)
  unsigned ties = 0;
  if (places > 0) {
    uint32_t prefix = 0, mask = 0;
    unsigned left = places;
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (t < 256) count[t] = 0;
      __syncthreads();
      for (int j = first + t; j < end; j += SELECT_THREADS) {
        const uint32_t u = order_of(mb_load(w + j));
        if ((u & mask) == prefix) atomicAdd(count + ((u >> shift) & 255u), 1u);
      }
      __syncthreads();
      if (warp == 0) {
        // lane l has digits 255 - 8 l .. 248 - 8 l, so that lanes go from the largest down
        unsigned mine = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) mine += count[255 - 8 * lane - i];
        unsigned before = mine;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
          const unsigned v = __shfl_up_sync(0xffffffffu, before, o);
          if (lane >= o) before += v;
        }
        before -= mine;
        if (before < left && left <= before + mine) {
          int d = 255 - 8 * lane;
          while (before + count[d] < left) before += count[d--];
          digit_s = d;
          left_s = left - before;
        }
      }
      __syncthreads();
      prefix |= digit_s << shift;
      mask |= 255u << shift;
      left = left_s;
    }
    limit = prefix;
    ties = left;
  }
  for (int j = t; j < first; j += SELECT_THREADS) {
    kept[j] = j;
    to[j] = mb_load(w + j);
  }
  for (int j = t; j < p.recent; j += SELECT_THREADS) {
    kept[p.budget - p.recent + j] = end + j;
    to[p.budget - p.recent + j] = mb_load(w + end + j);
  }
  // every warp has a run of the candidates: what it holds, then what lies before it, then where its own go
  const int run = (end - first + SELECT_THREADS - 1) / SELECT_THREADS * 32;
  const int from = min(first + warp * run, end), until = min(from + run, end);
  unsigned a = 0, e = 0;
  for (int j = from + lane; j < until; j += 32) {
    const uint32_t u = order_of(mb_load(w + j));
    a += u > limit;
    e += u == limit;
  }
  a = __reduce_add_sync(0xffffffffu, a);
  e = __reduce_add_sync(0xffffffffu, e);
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
  for (int base = from; base < until; base += 32) {
    const int j = base + lane;
    const float value = j < until ? mb_load(w + j) : 0.f;
    const uint32_t u = order_of(value);
    const unsigned more = __ballot_sync(0xffffffffu, j < until && u > limit), same = __ballot_sync(0xffffffffu, j < until && u == limit);
    const unsigned lower = (1u << lane) - 1u;
    const unsigned rank = e + __popc(same & lower);
    const bool stays = (more >> lane & 1u) != 0 || ((same >> lane & 1u) != 0 && rank < ties);
    if (stays) {
      const int at = first + a + __popc(more & lower) + min(rank, ties);
      kept[at] = j;
      to[at] = value;
    }
    a += __popc(more);
    e += __popc(same);
  }
}

// Rows of keys and values to their new slots, a word per item, and the new lengths (here, because the other kernel reads the old ones
// and the two may be the same memory).
template <typename Word>
__global__ void __launch_bounds__(COPY_THREADS) evict_copy_kernel(const EvictParams p) {
  mb_grid_dep_launch();
  mb_grid_dep_wait();
  const int unit = blockIdx.x / p.chunks, chunk = blockIdx.x % p.chunks;
  const int batch = unit / p.kv_heads, head = unit % p.kv_heads;
  if (chunk == 0 && head == 0 && threadIdx.x == 0) {
    bool bad;
    p.dst_lengths[batch] = min(kv::usable_length(mb_load(p.lengths + batch), p.longest, &bad), p.budget);
  }
  const int32_t *kept = p.kept + static_cast<int64_t>(unit) * p.budget;
  const int32_t *src_table = p.src_table + static_cast<int64_t>(batch) * p.src_max_pages;
  const int32_t *dst_table = p.dst_table + static_cast<int64_t>(batch) * p.dst_max_pages;
  const int rows = COPY_THREADS * COPY_EACH / p.words;   // whole rows of a block; at least one
  Word k[COPY_EACH], v[COPY_EACH];
  int64_t to[COPY_EACH];
#pragma unroll
  for (int i = 0; i < COPY_EACH; ++i) {
    const int item = i * COPY_THREADS + threadIdx.x;
    const int row = static_cast<int>(fast_div(item, p.word_mul, p.word_shift)), word = item - row * p.words;
    const int64_t j = static_cast<int64_t>(chunk) * rows + row;
    to[i] = -1;
    if (row >= rows || j >= p.budget) continue;
    const int slot = mb_load(kept + j);
    if (slot < 0) continue;
    const int from_page = static_cast<int>(fast_div(slot, p.page_mul, p.page_shift));
    const int to_page = static_cast<int>(fast_div(static_cast<uint32_t>(j), p.page_mul, p.page_shift));
    const int64_t from = kv::row_offset(mb_load(src_table + from_page), p.src_pages, p.kv_heads, head, p.page_size,
                                        slot - from_page * p.page_size, p.words);
    const int64_t at = kv::row_offset(mb_load(dst_table + to_page), p.dst_pages, p.kv_heads, head, p.page_size,
                                      static_cast<int>(j) - to_page * p.page_size, p.words);
    if (from < 0 || at < 0) {
      mb_report_bad_index(p.status);
      continue;
    }
    to[i] = at + word;
    k[i] = mb_load(static_cast<const Word *>(p.k_src) + from + word);
    v[i] = mb_load(static_cast<const Word *>(p.v_src) + from + word);
  }
#pragma unroll
  for (int i = 0; i < COPY_EACH; ++i)
    if (to[i] >= 0) {
      static_cast<Word *>(p.k_dst)[to[i]] = k[i];
      static_cast<Word *>(p.v_dst)[to[i]] = v[i];
    }
}

template <typename Word>
int launch_copy(mb_context *ctx, EvictParams &p, int64_t units, int64_t row_bytes) {
  const int64_t words = row_bytes / sizeof(Word);
  if (words > COPY_THREADS * COPY_EACH) return mb_fail(ctx, MB_UNSUPPORTED, "mb_kv_evict: head_dim too large");
  p.words = static_cast<int>(words);
  fast_div_make(p.words, &p.word_mul, &p.word_shift);
  p.chunks = static_cast<int>(ceil_div64(std::min(p.budget, std::max(p.longest, 1)), COPY_THREADS * COPY_EACH / p.words));
  if (units * p.chunks > kv::MOST) return mb_fail(ctx, MB_UNSUPPORTED, "mb_kv_evict: too many slots");
  MB_CUDA(ctx, mb_launch_chained(ctx, evict_copy_kernel<Word>, dim3(static_cast<unsigned>(units * p.chunks)), dim3(COPY_THREADS), 0, p));
  ctx->launches++;
  return MB_SUCCESS;
}

}  // namespace

extern "C" int mb_kv_evict(mb_context *ctx, const void *k_src, const void *v_src, const int32_t *src_table, const int32_t *lengths,
                           const float *weights, void *k_dst, void *v_dst, const int32_t *dst_table, int32_t *dst_lengths,
                           float *dst_weights, int32_t *kept, int64_t batch, int64_t kv_heads, int64_t head_dim, int64_t page_size,
                           int64_t src_pages, int64_t src_max_pages, int64_t dst_pages, int64_t dst_max_pages, int64_t max_length,
                           int64_t weights_stride, int64_t budget, int64_t sinks, int64_t recent, int dtype) {
  if (ctx == nullptr) return MB_INVALID_ARGS;
  const kv::Verdict verdict = kv::check_evict(k_src, v_src, src_table, lengths, weights, k_dst, v_dst, dst_table, dst_lengths,
                                              dst_weights, kept, batch, kv_heads, head_dim, page_size, src_pages, src_max_pages,
                                              dst_pages, dst_max_pages, max_length, weights_stride, budget, sinks, recent, dtype);
  if (verdict.code != MB_SUCCESS) return mb_fail(ctx, verdict.code, "mb_kv_evict: %s", verdict.why);
  if (batch == 0) return MB_SUCCESS;
  MB_CUDA(ctx, cudaSetDevice(ctx->device));
  EvictParams p = {};
  p.k_src = k_src; p.v_src = v_src; p.k_dst = k_dst; p.v_dst = v_dst;
  p.src_table = src_table; p.dst_table = dst_table; p.lengths = lengths; p.weights = weights;
  p.dst_lengths = dst_lengths; p.kept = kept; p.dst_weights = dst_weights;
  p.weights_stride = weights_stride; p.src_pages = src_pages; p.dst_pages = dst_pages;
  p.kv_heads = static_cast<int>(kv_heads); p.dim = static_cast<int>(head_dim); p.page_size = static_cast<int>(page_size);
  p.src_max_pages = static_cast<int>(src_max_pages); p.dst_max_pages = static_cast<int>(dst_max_pages);
  p.longest = kv::longest_of(max_length, src_max_pages, page_size);
  p.budget = static_cast<int>(budget); p.sinks = static_cast<int>(sinks); p.recent = static_cast<int>(recent);
  fast_div_make(static_cast<uint32_t>(page_size), &p.page_mul, &p.page_shift);
  p.status = ctx->dev_status;

  // the widest word that a row and the four pools are made of
  const int64_t units = batch * kv_heads, row_bytes = head_dim * kv::type_bytes(dtype);
  const uintptr_t bits = reinterpret_cast<uintptr_t>(k_src) | reinterpret_cast<uintptr_t>(v_src) | reinterpret_cast<uintptr_t>(k_dst) |
                         reinterpret_cast<uintptr_t>(v_dst) | static_cast<uintptr_t>(row_bytes);
  if (row_bytes / (bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 2) > COPY_THREADS * COPY_EACH)
    return mb_fail(ctx, MB_UNSUPPORTED, "mb_kv_evict: head_dim too large");
  MB_CUDA(ctx, mb_launch_chained(ctx, evict_select_kernel, dim3(static_cast<unsigned>(units)), dim3(SELECT_THREADS), 0, p));
  ctx->launches++;
  if (bits % 16 == 0) return launch_copy<uint4>(ctx, p, units, row_bytes);
  if (bits % 4 == 0) return launch_copy<uint32_t>(ctx, p, units, row_bytes);
  return launch_copy<uint16_t>(ctx, p, units, row_bytes);
}
