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
constexpr int TABLE = 2048;   // sines and cosines a block holds at most, beyond a single token's

// One of the call's tensors: `heads` heads of every token.  The destination is rows of a tensor, or slots of a pool.
struct Part {
  const void *src;
  void *dst;
  int64_t src_token, src_head, dst_token, dst_head;  // strides in elements
  int heads;
  int turned;    // 0: copied
  int to_slots;  // the destination is the paged pool
};

struct RopeParams {
  Part part[3];
  int parts;
  const int32_t *positions, *slots;
  const double *freq;
  int64_t tokens;
  int per_token, tokens_per_block;   // items of a token; tokens of a block
  int per_head;                      // items of a head: first those that turn, then those that copy
  uint32_t token_mul, token_shift, head_mul, head_shift, page_mul, page_shift;
  int half, turning, dim, page_size, kv_heads;  // half: rotary_dim / 2; turning: items of a head that turn
  int64_t num_pages;
  float cos_factor, sin_factor;
  int *status;
};

// What an item is: with V elements to a word, items 0 .. turning - 1 of a head turn (half layout: the words at jV and half + jV;
// interleaved: the word at jV, or with V = 1 the pair at 2j), the others copy a word behind the rotated part.
template <typename T, int V, bool INTERLEAVED>
struct Item {
  elem::Vec<T, V> a, b;
  T *dst;          // of the head; null: nothing to do
  int at, pair;    // a's place in the head; the first pair's number, or -1: copied
  int token;       // of the block

  static constexpr bool TWO = !INTERLEAVED || V == 1;   // a turning item has two words

  __device__ __forceinline__ void fetch(const RopeParams &p, int64_t token0, int tokens, int index) {
    dst = nullptr;
    token = p.tokens_per_block == 1 ? 0 : static_cast<int>(fast_div(index, p.token_mul, p.token_shift));
    const int rest = index - token * p.per_token;
    if (token >= tokens || rest >= p.per_token) return;
    int head = static_cast<int>(fast_div(rest, p.head_mul, p.head_shift));
    const int j = rest - head * p.per_head;
    int which = 0;
    while (which + 1 < p.parts && head >= p.part[which].heads) head -= p.part[which++].heads;
    const Part &part = p.part[which];
    const T *src = static_cast<const T *>(part.src) + (token0 + token) * part.src_token + head * part.src_head;
    const bool turns = j < p.turning;
    if (turns) {
      at = INTERLEAVED && V == 1 ? 2 * j : j * V;
      pair = !part.turned ? -1 : INTERLEAVED && V > 1 ? j * (V / 2) : j * V;
    } else {
      at = 2 * p.half + (j - p.turning) * V;
      pair = -2;
    }
    if (part.to_slots) {
      const int slot = mb_load(p.slots + token0 + token);
      if (slot < 0) return;
      const int page = static_cast<int>(fast_div(slot, p.page_mul, p.page_shift));
      const int64_t to = kv::row_offset(page, p.num_pages, p.kv_heads, head, p.page_size, slot - page * p.page_size, p.dim);
      if (to < 0) {
        mb_report_bad_index(p.status);
        return;
      }
      dst = static_cast<T *>(part.dst) + to;
    } else {
      dst = static_cast<T *>(part.dst) + (token0 + token) * part.dst_token + head * part.dst_head;
    }
    a.load(src + at);
    if (TWO && turns) b.load(src + other(p));
  }

  static constexpr int PAIRS = TWO ? V : V / 2;         // that a turning item has

  // Where pair q of a token lies in its table: two of an item's side by side, words of neighbouring items next to each other, so that
  // lanes read 16 bytes each without meeting in a bank.
  static __device__ __forceinline__ int table_at(int q, int items) {
    if (PAIRS == 1) return q;
    const int j = q / PAIRS, i = q % PAIRS;
    return ((i / 2) * items + j) * 2 + i % 2;
  }

  __device__ __forceinline__ int other(const RopeParams &p) const { return INTERLEAVED ? at + 1 : at + p.half; }

  __device__ __forceinline__ void finish(const RopeParams &p, const float2 *table) {
    if (dst == nullptr) return;
    if (pair >= 0) {
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
        T &lo = TWO ? a.v[i] : a.v[(2 * i) % V], &hi = TWO ? b.v[i] : a.v[(2 * i + 1) % V];
        const float x = elem::widen(lo), y = elem::widen(hi), c = cs[i].x, s = cs[i].y;
        lo = elem::narrow<T>(x * c - y * s);
        hi = elem::narrow<T>(x * s + y * c);
      }
    }
    a.store(dst + at);
    if (TWO && pair != -2) b.store(dst + other(p));
  }
};

template <typename T, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(THREADS) rope_kernel(const RopeParams p) {
  // two words per item: two items a thread; else four.  64 bytes of a thread's are in flight.
  constexpr int U = Item<T, V, INTERLEAVED>::TWO ? 2 : 4;
  extern __shared__ __align__(16) float2 table[];
  mb_grid_dep_launch();
  mb_grid_dep_wait();
  const int64_t token0 = static_cast<int64_t>(blockIdx.x) * p.tokens_per_block;
  const int tokens = static_cast<int>(min(static_cast<int64_t>(p.tokens_per_block), p.tokens - token0));
  Item<T, V, INTERLEAVED> item[U];
#pragma unroll
  for (int u = 0; u < U; ++u) item[u].fetch(p, token0, tokens, (blockIdx.y * U + u) * THREADS + threadIdx.x);
  for (int i = threadIdx.x; i < tokens * p.half; i += THREADS) {
    const int token = i / p.half;
    const double turns = mb_load(p.positions + token0 + token) * (mb_load(p.freq + (i - token * p.half)) * 0.15915494309189533577);
    float s, c;
    sincospif(2.f * static_cast<float>(turns - rint(turns)), &s, &c);
    table[token * p.half + Item<T, V, INTERLEAVED>::table_at(i - token * p.half, p.turning)] = make_float2(c * p.cos_factor, s * p.sin_factor);
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < U; ++u) item[u].finish(p, table);
}

template <typename T, int V, bool INTERLEAVED>
int launch(mb_context *ctx, RopeParams &p, int heads) {
  constexpr int U = Item<T, V, INTERLEAVED>::TWO ? 2 : 4;
  p.turning = INTERLEAVED && V > 1 ? 2 * p.half / V : p.half / V;
  p.per_head = p.turning + (p.dim - 2 * p.half) / V;
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
  const size_t smem = sizeof(float2) * p.tokens_per_block * p.half;
  if (smem > (48u << 10)) return mb_fail(ctx, MB_UNSUPPORTED, "mb_rope: rotary_dim above 12288");
  MB_CUDA(ctx, mb_launch_chained(ctx, rope_kernel<T, V, INTERLEAVED>, dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(rows)),
                                 dim3(THREADS), smem, p));
  ctx->launches++;
  return MB_SUCCESS;
}

// The widest word that every row and place allows: 16 bytes, two elements, or one.
template <typename T>
int dispatch(mb_context *ctx, RopeParams &p, bool interleaved) {
  int heads = 0;
  bool words[2] = {true, true};
  constexpr int wide = 16 / sizeof(T);
  const int sizes[2] = {wide, 2};
  for (int i = 0; i < 2; ++i) {
    const int v = sizes[i], behind = p.dim - 2 * p.half;
    words[i] = behind % v == 0 && (interleaved ? 2 * p.half : p.half) % v == 0;
    for (int w = 0; w < p.parts; ++w) {
      const Part &part = p.part[w];
      words[i] = words[i] && kv::aligned(part.src, v * sizeof(T)) && kv::aligned(part.dst, v * sizeof(T)) &&
                 part.src_token % v == 0 && part.src_head % v == 0 && part.dst_token % v == 0 && part.dst_head % v == 0 &&
                 (!part.to_slots || p.dim % v == 0);
    }
  }
  for (int w = 0; w < p.parts; ++w) heads += p.part[w].heads;
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
  p.part[0] = {x, y, x_token_stride, x_head_stride, y_token_stride, y_head_stride, static_cast<int>(heads), 1, 0};
  p.parts = 1;
  p.positions = positions; p.freq = freq; p.tokens = tokens;
  p.half = static_cast<int>(rotary_dim / 2); p.dim = static_cast<int>(head_dim);
  p.cos_factor = magnitude; p.sin_factor = inverse ? -magnitude : magnitude;
  p.status = ctx->dev_status;
  int st = MB_SUCCESS;
  MB_FOR_ELEMENT(dtype, st = dispatch<T>(ctx, p, interleaved != 0));
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
  p.part[0] = {q, q_out, q_token_stride, head_dim, q_out_token_stride, head_dim, h, 1, 0};
  p.part[1] = {k, k_cache, k_token_stride, head_dim, 0, 0, hk, 1, 1};
  p.part[2] = {v, v_cache, v_token_stride, head_dim, 0, 0, hk, 0, 1};
  p.parts = 3;
  p.positions = positions; p.slots = slots; p.freq = freq; p.tokens = tokens;
  p.half = static_cast<int>(rotary_dim / 2); p.dim = static_cast<int>(head_dim);
  p.num_pages = num_pages; p.page_size = static_cast<int>(page_size); p.kv_heads = hk;
  fast_div_make(static_cast<uint32_t>(page_size), &p.page_mul, &p.page_shift);
  p.cos_factor = p.sin_factor = magnitude;
  p.status = ctx->dev_status;
  int st = MB_SUCCESS;
  MB_FOR_ELEMENT(dtype, st = dispatch<T>(ctx, p, interleaved != 0));
  return st;
}

}  // extern "C"
