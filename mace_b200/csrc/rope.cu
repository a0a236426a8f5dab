// Rotary positions, alone (mb_rope) and on a step's way into the paged cache (mb_rope_kv_append), and their frequencies.
//
// A pair (a, b) of a head's values is turned by t = position * freq: (a cos t - b sin t, a sin t + b cos t), times a factor.
// The angle of a far position has to be reduced before it is rounded: position 10^6 at one radian each is held to 0.06
// radians in 32 bits.  So turns = position * freq / 2 pi is formed in 64 bits, its whole part dropped there, and only the fraction
// becomes a float for sincospif.  A block works out the sines and cosines of its tokens once, into shared memory, while its loads are
// in flight; all heads share them.
#include <cmath>

#include "elements.cuh"
#include "kv_cache.h"

namespace {

constexpr int THREADS = 256;
constexpr int U = 2;          // items of a thread: with two words of 16 bytes each, 64 bytes in flight
constexpr int TABLE = 2048;   // sines and cosines a block holds at most, beyond a single token's

// One of the call's tensors: queries (or all there is), which go to rows of a tensor, keys and values, which go to slots of a pool;
// values are copied.
struct Part {
  const void *src;
  void *dst;
  int64_t src_token, src_head, dst_token, dst_head;  // strides in elements
};

struct RopeParams {
  Part part[3];
  int end[2];                        // heads up to which they are queries, keys
  const int32_t *positions, *slots;
  const double *freq;
  int64_t tokens;
  int per_token, tokens_per_block;   // items of a token; tokens of a block
  int per_head;                      // items of a head: first those that turn, then those that copy
  uint32_t token_mul, token_shift, head_mul, head_shift, page_mul, page_shift, half_mul, half_shift;
  int copy_two;                      // ... two words each
  int half, turning, dim, page_size, kv_heads;  // half: rotary_dim / 2; turning: items of a head that turn
  int64_t num_pages, page_row;       // page_row: elements between the heads of a page
  float cos_factor, sin_factor;
  int *status;
};

// What an item is: with V elements to a word, items 0 .. turning - 1 of a head turn two words (half layout: those at jV and half + jV;
// interleaved: neighbours, from 2jV on), the others copy two behind the rotated part, or one where their number is odd.
template <typename T, int V, bool INTERLEAVED>
struct Item {
  elem::Vec<T, V> a, b;
  int at, next, pair;       // a's place in the head, b's behind it; the first pair's number, -1: behind the rotated part
  int token, head, which;   // of the block; of its tensor, the tensor
  bool two;                 // there is a second word

  // Where it comes from, and the loads.  (Where it goes needs the tokens' slots: those are read in the meantime.)
  __device__ __forceinline__ void fetch(const RopeParams &p, int64_t token0, int tokens, int index) {
    token = p.tokens_per_block == 1 ? 0 : static_cast<int>(fast_div(index, p.token_mul, p.token_shift));
    const int rest = index - token * p.per_token;
    which = -1;
    if (token >= tokens || rest >= p.per_token) return;
    head = static_cast<int>(fast_div(rest, p.head_mul, p.head_shift));
    const int j = rest - head * p.per_head;
    which = (head >= p.end[0]) + (head >= p.end[1]);
    head -= which == 0 ? 0 : which == 1 ? p.end[0] : p.end[1];
    const Part &part = p.part[which];
    const T *src = static_cast<const T *>(part.src) + (token0 + token) * part.src_token + head * part.src_head;
    const bool turns = j < p.turning;
    at = turns ? (INTERLEAVED ? 2 * j * V : j * V) : 2 * p.half + (j - p.turning) * (p.copy_two ? 2 * V : V);
    pair = turns ? j * V : -1;
    two = turns || p.copy_two;
    next = !turns ? V : INTERLEAVED ? V : p.half;
    a.load(src + at);
    if (two) b.load(src + at + next);
  }

  static constexpr int PAIRS = V;   // that a turning item has

  // Where pair q of a token lies in its table: two of an item's side by side, words of neighbouring items next to each other, so that
  // lanes read 16 bytes each without meeting in a bank.
  static __device__ __forceinline__ int table_at(int q, int items) {
    if (PAIRS == 1) return q;
    const int j = q / PAIRS, i = q % PAIRS;
    return ((i / 2) * items + j) * 2 + i % 2;
  }

  __device__ __forceinline__ void finish(const RopeParams &p, int64_t token0, const float2 *table, const int64_t *rows) {
    if (which < 0) return;
    const Part &part = p.part[which];
    int64_t to;
    if (which == 0) {
      to = (token0 + token) * part.dst_token + head * part.dst_head;
    } else {
      to = rows[token];
      if (to < 0) return;
      to += head * p.page_row;
    }
    T *dst = static_cast<T *>(part.dst) + to;
    if (pair >= 0 && which != 2) {
      float2 cs[PAIRS];
      if constexpr (PAIRS == 1) {
        cs[0] = table[token * p.half + pair];
      } else {
#pragma unroll
        for (int i = 0; i < PAIRS; i += 2) {
          const float4 w = *reinterpret_cast<const float4 *>(table + token * p.half + ((i / 2) * p.turning + pair / PAIRS) * 2);
          cs[i] = make_float2(w.x, w.y);
          cs[i + 1] = make_float2(w.z, w.w);
        }
      }
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) {
        // half layout (and single values): a's i-th and b's; interleaved: two neighbours, of a, then of b
        constexpr bool APART = !INTERLEAVED || V == 1;
        elem::Vec<T, V> &first = APART || i < V / 2 ? a : b, &second = APART || i >= V / 2 ? b : a;
        T &lo = first.v[APART ? i : 2 * i % V], &hi = second.v[APART ? i : (2 * i + 1) % V];
        const float x = elem::widen(lo), y = elem::widen(hi), c = cs[i].x, s = cs[i].y;
        lo = elem::narrow<T>(x * c - y * s);
        hi = elem::narrow<T>(x * s + y * c);
      }
    }
    a.store(dst + at);
    if (two) b.store(dst + at + next);
  }
};

template <typename T, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(THREADS) rope_kernel(const RopeParams p) {
  extern __shared__ __align__(16) float2 table[];
  mb_grid_dep_launch();
  mb_grid_dep_wait();
  const int64_t token0 = static_cast<int64_t>(blockIdx.x) * p.tokens_per_block;
  const int tokens = static_cast<int>(min(static_cast<int64_t>(p.tokens_per_block), p.tokens - token0));
  Item<T, V, INTERLEAVED> item[U];
#pragma unroll
  for (int u = 0; u < U; ++u) item[u].fetch(p, token0, tokens, (blockIdx.y * U + u) * THREADS + threadIdx.x);
  int64_t *rows = reinterpret_cast<int64_t *>(table + tokens * p.half);   // where the tokens' first heads go in the pools, -1: nowhere
  if (p.slots != nullptr) {
    for (int i = THREADS - 1 - threadIdx.x; i < tokens; i += THREADS) {   // (from the last warp down: the first ones have the table)
      const int slot = mb_load(p.slots + token0 + i);
      int64_t to = -1;
      if (slot >= 0) {
        const int page = static_cast<int>(fast_div(slot, p.page_mul, p.page_shift));
        to = kv::row_offset(page, p.num_pages, p.kv_heads, 0, p.page_size, slot - page * p.page_size, p.dim);
        if (to < 0) mb_report_bad_index(p.status);
      }
      rows[i] = to;
    }
  }
  for (int i = threadIdx.x; i < tokens * p.half; i += THREADS) {
    const int token = tokens == 1 ? 0 : static_cast<int>(fast_div(i, p.half_mul, p.half_shift));
    const double turns = mb_load(p.positions + token0 + token) * (mb_load(p.freq + (i - token * p.half)) * 0.15915494309189533577);
    float s, c;
    sincospif(2.f * static_cast<float>(turns - rint(turns)), &s, &c);
    table[token * p.half + Item<T, V, INTERLEAVED>::table_at(i - token * p.half, p.turning)] = make_float2(c * p.cos_factor, s * p.sin_factor);
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < U; ++u) item[u].finish(p, token0, table, rows);
}

template <typename T, int V, bool INTERLEAVED>
int launch(mb_context *ctx, RopeParams &p, int heads) {
  const int behind = (p.dim - 2 * p.half) / V;
  p.turning = p.half / V;
  p.copy_two = behind % 2 == 0;
  p.per_head = p.turning + (p.copy_two ? behind / 2 : behind);
  if (p.per_head > INT32_MAX / heads) return mb_fail(ctx, MB_UNSUPPORTED, "mb_rope: a token has too many values");
  p.per_token = p.per_head * heads;
  int64_t tokens = std::min<int64_t>(U * THREADS / p.per_token, p.tokens);
  if (p.half > 0) tokens = std::min<int64_t>(tokens, TABLE / p.half);
  // a few tokens: a block each, as far as there are SMs
  tokens = std::min<int64_t>(tokens, ceil_div64(p.tokens, ctx->num_sms));
  p.tokens_per_block = static_cast<int>(std::max<int64_t>(tokens, 1));
  fast_div_make(p.per_token, &p.token_mul, &p.token_shift);
  fast_div_make(p.per_head, &p.head_mul, &p.head_shift);
  const int64_t blocks = ceil_div64(p.tokens, p.tokens_per_block);
  const int64_t rows = ceil_div64(static_cast<int64_t>(p.per_token) * p.tokens_per_block, U * THREADS);
  if (rows > 65535) return mb_fail(ctx, MB_UNSUPPORTED, "mb_rope: a token has too many values");
  fast_div_make(p.half, &p.half_mul, &p.half_shift);
  const size_t smem = (sizeof(float2) * p.half + (p.slots != nullptr ? sizeof(int64_t) : 0)) * p.tokens_per_block;
  if (smem > (48u << 10)) return mb_fail(ctx, MB_UNSUPPORTED, "mb_rope: rotary_dim too large for a block's table of sines");
  MB_CUDA(ctx, mb_launch_chained(ctx, rope_kernel<T, V, INTERLEAVED>, dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(rows)),
                                 dim3(THREADS), smem, p));
  ctx->launches++;
  return MB_SUCCESS;
}

// The widest word that every row and place allows: 16 bytes, two elements, or one.
template <typename T>
int dispatch(mb_context *ctx, RopeParams &p, bool interleaved, int heads) {
  const int parts = p.slots != nullptr ? 3 : 1;
  bool words[2] = {true, true};
  constexpr int wide = 16 / sizeof(T);
  const int sizes[2] = {wide, 2};
  for (int i = 0; i < 2; ++i) {
    const int v = sizes[i], behind = p.dim - 2 * p.half;
    words[i] = behind % v == 0 && p.half % v == 0;
    for (int w = 0; w < parts; ++w) {
      const Part &part = p.part[w];
      words[i] = words[i] && kv::aligned(part.src, v * sizeof(T)) && kv::aligned(part.dst, v * sizeof(T)) &&
                 part.src_token % v == 0 && part.src_head % v == 0 && part.dst_token % v == 0 && part.dst_head % v == 0 &&
                 (w == 0 || p.dim % v == 0);
    }
  }
  if (interleaved) {
    if (words[0]) return launch<T, wide, true>(ctx, p, heads);
    if (words[1]) return launch<T, 2, true>(ctx, p, heads);
    return launch<T, 1, true>(ctx, p, heads);
  }
  if (words[0]) return launch<T, wide, false>(ctx, p, heads);
  if (words[1]) return launch<T, 2, false>(ctx, p, heads);
  return launch<T, 1, false>(ctx, p, heads);
}

}  // namespace

extern "C" {

int mb_rope_frequencies(int scaling, int64_t rotary_dim, double base, double factor, double original_length, double low, double high,
                        double *host_freq, float *host_magnitude) {
  if (host_freq == nullptr || host_magnitude == nullptr || rotary_dim < 0 || rotary_dim % 2 != 0 || rotary_dim > kv::MOST_DIM ||
      !(base > 0.0) || !std::isfinite(base))
    return MB_INVALID_ARGS;
  if (scaling < MB_ROPE_PLAIN || scaling > MB_ROPE_RAMP) return MB_INVALID_ARGS;
  if (scaling != MB_ROPE_PLAIN && (!(factor >= 1.0) || !std::isfinite(factor))) return MB_INVALID_ARGS;
  if (scaling == MB_ROPE_BASE && rotary_dim < 4) return MB_INVALID_ARGS;
  const bool bands = scaling == MB_ROPE_BANDS || scaling == MB_ROPE_RAMP;
  if (bands && (!(original_length > 0.0) || !std::isfinite(original_length) || !(low > 0.0) || !(high > low) || !std::isfinite(high)))
    return MB_INVALID_ARGS;
  const double pi = 3.14159265358979323846;
  const double d = static_cast<double>(rotary_dim);
  if (scaling == MB_ROPE_BASE) base *= std::pow(factor, d / (d - 2.0));
  // the pair (not a whole one) that makes so many turns over the original length
  const auto pair_of = [&](double turns) { return d * std::log(original_length / (turns * 2.0 * pi)) / (2.0 * std::log(base)); };
  double first = 0.0, last = 0.0;
  if (scaling == MB_ROPE_RAMP) {
    if (base <= 1.0) return MB_INVALID_ARGS;
    first = std::fmax(std::floor(pair_of(high)), 0.0);
    last = std::fmin(std::ceil(pair_of(low)), d - 1.0);
    if (first == last) last += 0.001;   // (a ramp without width)
  }
  for (int64_t i = 0; i < rotary_dim / 2; ++i) {
    double f = std::pow(base, -2.0 * static_cast<double>(i) / d);
    if (scaling == MB_ROPE_LINEAR) f /= factor;
    if (bands) {
      double kept;
      if (scaling == MB_ROPE_BANDS)
        kept = (original_length * f / (2.0 * pi) - low) / (high - low);
      else if (last < first)   // (every pair turns less than `low` times, or every one more than `high` times)
        kept = last < 0.0 ? 0.0 : 1.0;
      else
        kept = 1.0 - (static_cast<double>(i) - first) / (last - first);
      kept = std::fmin(std::fmax(kept, 0.0), 1.0);
      f = f * kept + f / factor * (1.0 - kept);
    }
    host_freq[i] = f;
  }
  *host_magnitude = scaling == MB_ROPE_RAMP ? static_cast<float>(0.1 * std::log(factor) + 1.0) : 1.f;
  return MB_SUCCESS;
}

int mb_rope(mb_context *ctx, const void *x, void *y, const int32_t *positions, const double *freq, int64_t tokens, int64_t heads,
            int64_t head_dim, int64_t rotary_dim, int64_t x_token_stride, int64_t x_head_stride, int64_t y_token_stride,
            int64_t y_head_stride, int interleaved, int inverse, float magnitude, int dtype) {
  if (ctx == nullptr) return MB_INVALID_ARGS;
  const kv::Verdict v = kv::check_rope(x, y, positions, freq, tokens, heads, head_dim, rotary_dim, x_token_stride, x_head_stride,
                                       y_token_stride, y_head_stride, dtype);
  if (v.code != MB_SUCCESS) return mb_fail(ctx, v.code, "mb_rope: %s", v.why);
  if (tokens == 0) return MB_SUCCESS;
  MB_CUDA(ctx, cudaSetDevice(ctx->device));
  RopeParams p = {};
  p.part[0] = {x, y, x_token_stride, x_head_stride, y_token_stride, y_head_stride};
  p.end[0] = p.end[1] = static_cast<int>(heads);
  p.positions = positions; p.freq = freq; p.tokens = tokens;
  p.half = static_cast<int>(rotary_dim / 2); p.dim = static_cast<int>(head_dim);
  p.cos_factor = magnitude; p.sin_factor = inverse ? -magnitude : magnitude;
  p.status = ctx->dev_status;
  int st = MB_SUCCESS;
  MB_FOR_ELEMENT(dtype, st = dispatch<T>(ctx, p, interleaved != 0, static_cast<int>(heads)));
  return st;
}

int mb_rope_kv_append(mb_context *ctx, const void *q, void *q_out, const void *k, const void *v, void *k_cache, void *v_cache,
                      const int32_t *positions, const int32_t *slots, const double *freq, int64_t tokens, int64_t heads,
                      int64_t kv_heads, int64_t head_dim, int64_t rotary_dim, int64_t q_token_stride, int64_t q_out_token_stride,
                      int64_t k_token_stride, int64_t v_token_stride, int64_t num_pages, int64_t page_size, int interleaved,
                      float magnitude, int dtype) {
  if (ctx == nullptr) return MB_INVALID_ARGS;
  const kv::Verdict verdict =
      kv::check_append(q, q_out, k, v, k_cache, v_cache, positions, slots, freq, tokens, heads, kv_heads, head_dim, rotary_dim,
                       q_token_stride, q_out_token_stride, k_token_stride, v_token_stride, num_pages, page_size, dtype);
  if (verdict.code != MB_SUCCESS) return mb_fail(ctx, verdict.code, "mb_rope_kv_append: %s", verdict.why);
  if (tokens == 0) return MB_SUCCESS;
  MB_CUDA(ctx, cudaSetDevice(ctx->device));
  RopeParams p = {};
  const int h = static_cast<int>(heads), hk = static_cast<int>(kv_heads);
  p.part[0] = {q, q_out, q_token_stride, head_dim, q_out_token_stride, head_dim};
  p.part[1] = {k, k_cache, k_token_stride, head_dim, 0, 0};
  p.part[2] = {v, v_cache, v_token_stride, head_dim, 0, 0};
  p.end[0] = h; p.end[1] = h + hk;
  p.page_row = page_size * head_dim;
  p.positions = positions; p.slots = slots; p.freq = freq; p.tokens = tokens;
  p.half = static_cast<int>(rotary_dim / 2); p.dim = static_cast<int>(head_dim);
  p.num_pages = num_pages; p.page_size = static_cast<int>(page_size); p.kv_heads = hk;
  fast_div_make(static_cast<uint32_t>(page_size), &p.page_mul, &p.page_shift);
  p.cos_factor = p.sin_factor = magnitude;
  p.status = ctx->dev_status;
  int st = MB_SUCCESS;
  MB_FOR_ELEMENT(dtype, st = dispatch<T>(ctx, p, interleaved != 0, h + 2 * hk));
  return st;
}

}  // extern "C"
