// What the operators on the paged cache share and what needs no GPU: the arithmetic of pages and lengths, and the checks of
// arguments.  Plain C++, so that it is tested on the host as well (tests/kv_cache_unit.cc).
#pragma once

#include <stdint.h>

#include "../../include/mace_b200.h"

#ifdef __CUDACC__
#define MB_HD __host__ __device__ __forceinline__
#else
#define MB_HD inline
#endif

namespace kv {

// Where row `row` of a page lies in its pool, in elements; -1 for a page that the pool does not have.
MB_HD int64_t row_offset(int32_t page, int64_t num_pages, int kv_heads, int head, int page_size, int row, int dim) {
  if (page < 0 || page >= num_pages) return -1;
  return ((static_cast<int64_t>(page) * kv_heads + head) * page_size + row) * dim;
}

// The slots of a sequence that count: lengths outside [0, longest] (longest: what the call and its table allow) are cut and told.
MB_HD int usable_length(int32_t length, int longest, bool *bad) {
  *bad = length < 0 || length > longest;
  return length < 0 ? 0 : length > longest ? longest : length;
}

MB_HD int longest_of(int64_t max_length, int64_t max_pages, int64_t page_size) {
  const int64_t room = max_pages * page_size;
  return static_cast<int>(max_length < room ? max_length : room);
}

// The first slot that a window of the last `window` ones leaves (0: no window).
MB_HD int window_begin(int length, int64_t window) {
  return window > 0 && length > window ? static_cast<int>(length - window) : 0;
}

// Slots that are worth a block of attention of their own (1000 slots, 8 heads: 64 12.2 us, 128 10.8, 256 13.7).
constexpr int LEAST_RUN = 128;

// The blocks of a cluster that shares a head's slots (1: none; the slots are cut into runs that meet in memory).  Clusters are for work
// that is over before parts could meet in memory (1000 slots, 8 heads: 10.4 us as runs, 7.7 on clusters of 8), so they take up
// to 64 MiB of keys and values, and no block more than `share` slots: a head or two over a long context are a cluster or two, which leave
// most SMs idle.  room[i]: blocks in clusters of 2^i that the device holds at once.
inline int cluster_of(int64_t units, int64_t longest, int64_t slot_bytes, int most, int64_t share, const int64_t *room) {
  if (longest * slot_bytes > (64ll << 20) / units) return 1;
  int blocks = 1;
  for (int i = 1; blocks < most && units * blocks * 2 <= room[i] && longest > LEAST_RUN * blocks; ++i) blocks *= 2;
  return longest > share * blocks ? 1 : blocks;
}

// Slots of a sequence that a block of the second kernel of attention with weights has.
constexpr int WEIGHT_SLOTS = 1024;

// What a check of arguments says: code MB_SUCCESS, or the status to return and why.
struct Verdict {
  int code;
  const char *why;
};
inline Verdict fine() { return {MB_SUCCESS, nullptr}; }
inline Verdict invalid(const char *why) { return {MB_INVALID_ARGS, why}; }
inline Verdict unsupported(const char *why) { return {MB_UNSUPPORTED, why}; }

inline bool is_type(int dtype) { return dtype == MB_F32 || dtype == MB_F16 || dtype == MB_BF16; }
inline int type_bytes(int dtype) { return dtype == MB_F32 ? 4 : 2; }
inline bool aligned(const void *p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

// Extents above these are refused, so that counts fit 31 bits and byte offsets 63 (a tensor's two strides together).
constexpr int64_t MOST = INT32_MAX;
constexpr int64_t MOST_DIM = 1 << 16;   // rotary head_dim
constexpr int64_t MOST_SLOTS = MOST - (1 << 16);   // of a sequence: an index that steps past the last by a cluster's threads (16 x 1024) fits
constexpr int64_t MOST_STRIDE = 1ll << 40, MOST_OFFSET = 1ll << 59;

#define KV_REQUIRE(cond, why) \
  do {                        \
    if (!(cond)) return ::kv::invalid(why); \
  } while (0)

inline Verdict check_heads(int64_t count, int64_t heads, int64_t dim, int dtype) {
  KV_REQUIRE(is_type(dtype), "element type is not MB_F32, MB_F16 or MB_BF16");
  KV_REQUIRE(count >= 0 && heads >= 1 && dim >= 1, "negative size, or no heads");
  if (count > MOST || heads > MOST || dim > MOST_DIM || heads * dim > MOST) return unsupported("tensor too large");
  return fine();
}

inline Verdict check_rotary(int64_t dim, int64_t rotary, int64_t tokens, int64_t heads) {
  KV_REQUIRE(rotary >= 0 && rotary <= dim && rotary % 2 == 0, "rotary_dim must be even and at most head_dim");
  if (tokens * heads > (MOST << 8)) return unsupported("tensor too large");
  return fine();
}

// Whether the last of `count` rows `stride` apart has a place.
inline bool reaches(int64_t count, int64_t stride) { return count <= 1 || stride == 0 || count - 1 <= MOST_OFFSET / stride; }

inline Verdict check_stride(int64_t stride, int64_t count) {
  KV_REQUIRE(stride >= 0 && stride <= MOST_STRIDE && reaches(count, stride), "stride is negative or too large");
  return fine();
}

// outer >= (count - 1) * step + width, however large they are.
inline bool holds(int64_t outer, int64_t count, int64_t step, int64_t width) {
  return outer >= width && (count <= 1 || step == 0 || (outer - width) / step >= count - 1);
}

// Rows of `width` elements, `count` of them, in a buffer that is written: they may not overlap.
inline Verdict check_rows(int64_t count, int64_t stride, int64_t width) {
  KV_REQUIRE(stride >= 0 && stride <= MOST_STRIDE && reaches(count, stride) && (count <= 1 || stride >= width), "output rows overlap, or stride is too large");
  return fine();
}

inline Verdict check_pool(int64_t num_pages, int64_t page_size, int64_t kv_heads, int64_t dim) {
  KV_REQUIRE(num_pages >= 0 && page_size >= 1, "bad number or size of pages");
  if (page_size > MOST || num_pages > MOST / page_size || kv_heads * dim > MOST) return unsupported("more than 2^31 - 1 slots");
  if (num_pages * page_size > MOST_OFFSET / (kv_heads * dim)) return unsupported("pool too large");
  return fine();
}

// Whether two stretches of 4-byte values have none in common.
inline bool apart(const void *a, int64_t na, const void *b, int64_t nb) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y ? (y - x) / 4 >= static_cast<uintptr_t>(na) : (x - y) / 4 >= static_cast<uintptr_t>(nb);
}

#define KV_PASS(expr)                              \
  do {                                             \
    const Verdict kv_v = (expr);                   \
    if (kv_v.code != MB_SUCCESS) return kv_v;      \
  } while (0)

inline Verdict check_rope(const void *x, const void *y, const int32_t *positions, const double *freq, int64_t tokens,
                          int64_t heads, int64_t dim, int64_t rotary, int64_t x_token, int64_t x_head, int64_t y_token,
                          int64_t y_head, int dtype) {
  KV_PASS(check_heads(tokens, heads, dim, dtype));
  KV_PASS(check_rotary(dim, rotary, tokens, heads));
  KV_PASS(check_stride(x_token, tokens));
  KV_PASS(check_stride(x_head, heads));
  KV_PASS(check_stride(y_token, tokens));
  KV_PASS(check_stride(y_head, heads));
  // rows of heads inside tokens or of tokens inside heads
  const bool inside = (heads <= 1 || y_head >= dim) && (tokens <= 1 || holds(y_token, heads, y_head, dim));
  const bool outside = (tokens <= 1 || y_token >= dim) && (heads <= 1 || holds(y_head, tokens, y_token, dim));
  KV_REQUIRE(inside || outside, "output heads overlap");
  if (tokens == 0) return fine();
  KV_REQUIRE(x != nullptr && y != nullptr && (rotary == 0 || (positions != nullptr && freq != nullptr)), "null operand");
  const uintptr_t size = type_bytes(dtype);
  KV_REQUIRE(aligned(x, size) && aligned(y, size) && aligned(positions, 4) && aligned(freq, 8), "misaligned operand");
  KV_REQUIRE(x != y || ((tokens <= 1 || x_token == y_token) && (heads <= 1 || x_head == y_head)), "in place with other strides");
  return fine();
}

inline Verdict check_append(const void *q, const void *q_out, const void *k, const void *v, const void *k_cache, const void *v_cache,
                            const int32_t *positions, const int32_t *slots, const double *freq, int64_t tokens, int64_t heads,
                            int64_t kv_heads, int64_t dim, int64_t rotary, int64_t q_token, int64_t q_out_token, int64_t k_token,
                            int64_t v_token, int64_t num_pages, int64_t page_size, int dtype) {
  KV_PASS(check_heads(tokens, heads, dim, dtype));
  KV_PASS(check_heads(tokens, kv_heads, dim, dtype));
  if ((heads + 2 * kv_heads) * dim > MOST) return unsupported("tensor too large");
  KV_PASS(check_rotary(dim, rotary, tokens, heads + 2 * kv_heads));
  KV_PASS(check_stride(q_token, tokens));
  KV_PASS(check_stride(k_token, tokens));
  KV_PASS(check_stride(v_token, tokens));
  KV_PASS(check_rows(tokens, q_out_token, heads * dim));
  KV_PASS(check_pool(num_pages, page_size, kv_heads, dim));
  if (tokens == 0) return fine();
  KV_REQUIRE(q != nullptr && q_out != nullptr && k != nullptr && v != nullptr && slots != nullptr &&
             (num_pages == 0 || (k_cache != nullptr && v_cache != nullptr)) &&
             (rotary == 0 || (positions != nullptr && freq != nullptr)), "null operand");
  const uintptr_t size = type_bytes(dtype);
  KV_REQUIRE(aligned(q, size) && aligned(q_out, size) && aligned(k, size) && aligned(v, size) && aligned(k_cache, size) &&
             aligned(v_cache, size) && aligned(positions, 4) && aligned(slots, 4) && aligned(freq, 8), "misaligned operand");
  KV_REQUIRE(q != q_out || tokens <= 1 || q_token == q_out_token, "in place with another stride");
  return fine();
}

inline Verdict check_attention(const void *q, const void *k_cache, const void *v_cache, const int32_t *table, const int32_t *lengths,
                               const void *out, const float *lse, const float *weights_in, const float *weights_out, int64_t batch,
                               int64_t heads, int64_t kv_heads, int64_t dim, int64_t q_stride, int64_t out_stride, int64_t num_pages,
                               int64_t page_size, int64_t max_pages, int64_t max_length, int64_t window, int64_t weights_stride,
                               int dtype) {
  KV_PASS(check_heads(batch, heads, dim, dtype));
  KV_PASS(check_heads(batch, kv_heads, dim, dtype));
  KV_REQUIRE(heads % kv_heads == 0, "heads must be a multiple of kv_heads");
  if (dim > 256) return unsupported("head_dim above 256");
  KV_PASS(check_stride(q_stride, batch));
  KV_PASS(check_rows(batch, out_stride, heads * dim));
  KV_PASS(check_pool(num_pages, page_size, kv_heads, dim));
  KV_REQUIRE(max_pages >= 0 && max_length >= 0 && window >= 0, "negative size");
  if (max_pages > MOST / page_size || max_length > MOST_SLOTS) return unsupported("more than 2^31 - 2^16 - 1 slots");
  if (batch * heads > MOST / 4) return unsupported("too many query heads");
  KV_REQUIRE(weights_in == nullptr || weights_out != nullptr, "weights_in without weights_out");
  KV_REQUIRE(weights_out == nullptr || (weights_stride >= longest_of(max_length, max_pages, page_size) && weights_stride <= MOST),
             "weights_stride below the longest sequence, or too large");
  if (weights_out != nullptr &&
      batch * kv_heads * ((longest_of(max_length, max_pages, page_size) + static_cast<int64_t>(WEIGHT_SLOTS) - 1) / WEIGHT_SLOTS) > MOST)
    return unsupported("too many slots");
  if (batch == 0) return fine();
  KV_REQUIRE(q != nullptr && out != nullptr && lengths != nullptr && (max_pages == 0 || table != nullptr) &&
             (num_pages == 0 || (k_cache != nullptr && v_cache != nullptr)), "null operand");
  const uintptr_t size = type_bytes(dtype);
  KV_REQUIRE(aligned(q, size) && aligned(out, size) && aligned(k_cache, size) && aligned(v_cache, size) && aligned(table, 4) &&
             aligned(lengths, 4) && aligned(lse, 4) && aligned(weights_in, 4) && aligned(weights_out, 4), "misaligned operand");
  // (a head's result is written when all blocks that read its query have: another sequence's may still be read)
  KV_REQUIRE(q != out || batch <= 1 || q_stride == out_stride, "in place with another stride");
  return fine();
}

// How eviction copies rows of `row_bytes`: in words of `word` bytes, as wide as every address in `bits` (which has the row's bytes
// among its own) allows, whole rows of at most COPY_WORDS words to a block.
constexpr int COPY_WORDS = 512;
struct CopyShape {
  int64_t word, words, rows;   // rows: of a block, 0 where not one fits
};
inline CopyShape copy_shape(uintptr_t bits, int64_t row_bytes) {
  const int64_t word = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 2;
  return {word, row_bytes / word, COPY_WORDS / (row_bytes / word)};
}
inline uintptr_t copy_bits(const void *k_src, const void *v_src, const void *k_dst, const void *v_dst, int64_t row_bytes) {
  return reinterpret_cast<uintptr_t>(k_src) | reinterpret_cast<uintptr_t>(v_src) | reinterpret_cast<uintptr_t>(k_dst) |
         reinterpret_cast<uintptr_t>(v_dst) | static_cast<uintptr_t>(row_bytes);
}

inline Verdict check_evict(const void *k_src, const void *v_src, const int32_t *src_table, const int32_t *lengths, const float *weights,
                           const void *k_dst, const void *v_dst, const int32_t *dst_table, const int32_t *dst_lengths,
                           const float *dst_weights, const int32_t *kept, int64_t batch, int64_t kv_heads, int64_t dim,
                           int64_t page_size, int64_t src_pages, int64_t src_max_pages, int64_t dst_pages, int64_t dst_max_pages,
                           int64_t max_length, int64_t weights_stride, int64_t budget, int64_t sinks, int64_t recent, int dtype,
                           int64_t dst_weights_stride = 0 /* rows of budget */) {
  KV_PASS(check_heads(batch, kv_heads, dim, dtype));
  KV_PASS(check_pool(src_pages, page_size, kv_heads, dim));
  KV_PASS(check_pool(dst_pages, page_size, kv_heads, dim));
  KV_REQUIRE(src_max_pages >= 0 && dst_max_pages >= 0 && max_length >= 0, "negative size");
  KV_REQUIRE(budget >= 1 && sinks >= 0 && recent >= 0 && sinks <= budget && recent <= budget - sinks,
             "budget must be at least 1 and at least sinks + recent");
  if (src_max_pages > MOST / page_size || dst_max_pages > MOST / page_size || max_length > MOST_SLOTS || budget > MOST_SLOTS)
    return unsupported("more than 2^31 - 2^16 - 1 slots");
  const int64_t longest = longest_of(max_length, src_max_pages, page_size), stays = budget < longest ? budget : longest;
  KV_REQUIRE(dst_max_pages * page_size >= stays, "the destination's table has no room for budget slots");
  KV_REQUIRE(weights_stride >= longest && weights_stride <= MOST, "weights_stride below the longest sequence, or too large");
  if (dst_weights_stride == 0) dst_weights_stride = budget;
  KV_REQUIRE(dst_weights_stride >= budget && dst_weights_stride <= MOST, "dst_weights_stride below budget, or too large");
  if (batch * kv_heads > MOST / 16 || batch * kv_heads > (MOST << 12) / budget) return unsupported("too many kv heads");
  if (batch == 0) return fine();
  KV_REQUIRE(lengths != nullptr && dst_lengths != nullptr && kept != nullptr && dst_weights != nullptr && weights != nullptr &&
             (src_max_pages == 0 || src_table != nullptr) && (dst_max_pages == 0 || dst_table != nullptr) &&
             (src_pages == 0 || (k_src != nullptr && v_src != nullptr)) && (dst_pages == 0 || (k_dst != nullptr && v_dst != nullptr)),
             "null operand");
  const uintptr_t size = type_bytes(dtype);
  KV_REQUIRE(aligned(k_src, size) && aligned(v_src, size) && aligned(k_dst, size) && aligned(v_dst, size) && aligned(src_table, 4) &&
             aligned(dst_table, 4) && aligned(lengths, 4) && aligned(dst_lengths, 4) && aligned(weights, 4) &&
             aligned(dst_weights, 4) && aligned(kept, 4), "misaligned operand");
  KV_REQUIRE(apart(weights, batch * kv_heads * weights_stride, dst_weights, batch * kv_heads * dst_weights_stride), "dst_weights may not lie in weights");
  const int64_t row_bytes = dim * type_bytes(dtype);
  const CopyShape copy = copy_shape(copy_bits(k_src, v_src, k_dst, v_dst, row_bytes), row_bytes);
  if (copy.rows == 0) return unsupported("head_dim too large");
  if (batch * kv_heads * (((stays < 1 ? 1 : stays) + copy.rows - 1) / copy.rows) > MOST) return unsupported("too many slots");
  return fine();
}

}  // namespace kv
