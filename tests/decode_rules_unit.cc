// Rules and limits of the decode-step operators that need no GPU: compiled and run by tests/test_decode_rules_cpu.py.
#include <cstdio>
#include <initializer_list>

#include "../mace_b200/csrc/mxfp4.h"

static int failures = 0;
#define EXPECT(cond)                                  \
  do {                                                \
    if (!(cond)) {                                    \
      std::printf("line %d: %s\n", __LINE__, #cond);  \
      ++failures;                                     \
    }                                                 \
  } while (0)

// Clusters of attention: never more slots to a block than its share, never more blocks than fit, never work above 64 MiB.
static void clusters() {
  const int64_t room[5] = {148, 146, 140, 128, 112}, twice[5] = {296, 296, 296, 296, 296};
  for (const int64_t *r : {room, twice})
    for (const int64_t share : {128, 256, 512, 1024})
      for (const int most : {8, 16})
        for (const int64_t bytes : {4, 256, 512, 1024, 2048})
          for (const int64_t units : {1ll, 2ll, 3ll, 7ll, 8ll, 9ll, 18ll, 19ll, 37ll, 74ll, 75ll, 148ll, 149ll, 1ll << 29})
            for (const int64_t longest : {0ll, 1ll, 127ll, 128ll, 129ll, 1000ll, 2048ll, 2049ll, 8192ll, 16384ll, 16385ll, 30000ll, 120000ll, (1ll << 31) - 65537}) {
              const int c = kv::cluster_of(units, longest, bytes, most, share, r);
              EXPECT(c >= 1 && c <= most && (c & (c - 1)) == 0);
              if (c == 1) continue;
              EXPECT(longest <= share * c);
              EXPECT(longest * bytes <= (64ll << 20) / units);
              int i = 0;
              while (1 << i < c) ++i;
              EXPECT(units * c <= r[i]);
              EXPECT(longest > kv::LEAST_RUN * (c / 2));
            }
  // eight heads of 1000 slots stay on clusters of 8; a single head of 120000 does not get 16 of 148 SMs
  EXPECT(kv::cluster_of(8, 1000, 512, 16, 1024, twice) == 8);
  EXPECT(kv::cluster_of(8, 8192, 512, 16, 1024, twice) == 16);
  EXPECT(kv::cluster_of(1, 120000, 512, 16, 1024, twice) == 1);
  EXPECT(kv::cluster_of(2, 60000, 512, 16, 1024, twice) == 1);
  EXPECT(kv::cluster_of(1, 30000, 2048, 8, 128, twice) == 1);
  EXPECT(kv::cluster_of(8, 2000, 1024, 16, 1024, room) == 8);
}

alignas(16) static char memory[64];
static const void *const X = memory;
static void *const Y = memory + 32;
static const int32_t *const I = reinterpret_cast<const int32_t *>(memory);
static float *const F = reinterpret_cast<float *>(memory);

// What attention with weights would refuse after its first kernel is refused before it.
static void weights_of_too_many_slots() {
  const auto code = [](int64_t batch, int64_t kv_heads, int64_t length, float *weights) {
    return kv::check_attention(X, X, X, I, I, Y, nullptr, nullptr, weights, batch, kv_heads, kv_heads, 8, kv_heads * 8, kv_heads * 8, 1 << 20, 16,
                               1 << 26, length, 0, length, MB_F16).code;
  };
  EXPECT(code(1 << 15, 1 << 8, 256 * 1024, F) == MB_UNSUPPORTED);
  EXPECT(code(1 << 15, 1 << 8, 255 * 1024, F) == MB_SUCCESS);
  EXPECT(code(1 << 15, 1 << 8, 255 * 1024 + 1, F) == MB_UNSUPPORTED);
  EXPECT(code(1 << 15, 1 << 8, 256 * 1024, nullptr) == MB_SUCCESS);
  EXPECT(code(0, 1 << 8, 256 * 1024, F) == MB_SUCCESS);
}

// What eviction would refuse between its two kernels is refused before the first.
static void rows_too_many_or_too_long() {
  const auto code = [](int64_t batch, int64_t dim, int64_t budget, const void *k) {
    return kv::check_evict(k, X, I, I, F, Y, Y, I, I, F + 16, I, batch, 1, dim, 16, 1 << 20, 1 << 20, 1 << 20, 1 << 20, budget, budget, budget, 0, 0,
                           MB_F32, budget).code;
  };
  // (weights that overlap would be refused first: 2^18 rows of 2^14 lie 2^32 values apart)
  const auto far = [&](int64_t batch, int64_t dim, int64_t budget, const void *k) {
    return kv::check_evict(k, X, I, I, F, Y, Y, I, I, reinterpret_cast<const float *>(uintptr_t{1} << 45), I, batch, 1, dim, 16, 1 << 20, 1 << 20, 1 << 20,
                           1 << 20, budget, budget, budget, 0, 0, MB_F32, budget).code;
  };
  EXPECT(far(1 << 18, 2048, 1 << 13, X) == MB_UNSUPPORTED);   // a row to a block, 2^31 of them
  EXPECT(far(1 << 18, 2048, (1 << 13) - 1, X) == MB_SUCCESS);
  EXPECT(far(1 << 18, 1024, 1 << 13, X) == MB_SUCCESS);
  EXPECT(far(1 << 18, 128, 1 << 13, memory + 4) == MB_SUCCESS);
  EXPECT(far(1 << 18, 512, 1 << 13, memory + 4) == MB_UNSUPPORTED);   // words of 4 bytes: as many blocks as of 2048 above
  EXPECT(code(1, 2048, 1, X) == MB_SUCCESS);
  EXPECT(code(1, 2052, 1, X) == MB_UNSUPPORTED);
  EXPECT(code(1, 512, 1, memory + 4) == MB_SUCCESS);
  EXPECT(code(1, 513, 1, memory + 4) == MB_UNSUPPORTED);
}

// Strides and extents up to the limits: no sum or product of them leaves 64 bits (the program is built with -fsanitize=undefined), and what
// overlaps or has no address is refused.
static void strides_at_the_limits() {
  const int64_t most = INT32_MAX, far = 1ll << 40, rows = (1ll << 31) - 8;
  const auto rope = [](int64_t tokens, int64_t heads, int64_t dim, int64_t xt, int64_t xh, int64_t yt, int64_t yh) {
    return kv::check_rope(X, Y, I, reinterpret_cast<const double *>(memory), tokens, heads, dim, dim, xt, xh, yt, yh, MB_BF16).code;
  };
  EXPECT(rope(2, 2, 64, 128, 64, 128, 64) == MB_SUCCESS);
  EXPECT(rope(2, 2, 64, 128, 64, 64, 128) == MB_SUCCESS);
  EXPECT(rope(2, 2, 64, 128, 64, 127, 64) == MB_INVALID_ARGS);
  EXPECT(rope(3, 2, 64, 128, 64, 64, 191) == MB_INVALID_ARGS);
  EXPECT(rope(3, 2, 64, 128, 64, 64, 192) == MB_SUCCESS);
  EXPECT(rope(2, 2, 64, 128, 64, far, 64) == MB_SUCCESS);
  EXPECT(rope(2, 2, 64, 0, 0, 64, far) == MB_SUCCESS);
  EXPECT(rope(2, 2, 64, 0, 0, far + 1, 64) == MB_INVALID_ARGS);
  // (heads - 1) * y_head alone would be 2^71
  EXPECT(rope(2, most / 2, 2, 0, 0, far, far) == MB_INVALID_ARGS);
  EXPECT(rope(most, 1, 2, far, 2, 2, 2) == MB_INVALID_ARGS);
  EXPECT(rope(most, 1, 2, 2, 2, far, 2) == MB_INVALID_ARGS);
  EXPECT(rope(1, most / 2, 2, 2, far, 2, 2) == MB_INVALID_ARGS);
  EXPECT(rope(1 << 19, 2, 2, far, 2, far, 2) == MB_SUCCESS);
  EXPECT(rope((1 << 19) + 2, 2, 2, far, 2, far, 2) == MB_INVALID_ARGS);
  for (const int64_t tokens : {1ll, 2ll, 1ll << 19, 1ll << 31})
    for (const int64_t heads : {1ll, 2ll, 1ll << 20, 1ll << 30})
      for (const int64_t a : {0ll, 1ll, 64ll, 1ll << 31, 1ll << 40, (1ll << 62)})
        for (const int64_t b : {0ll, 2ll, 64ll, 1ll << 20, 1ll << 40, (1ll << 62)}) rope(tokens, heads, 2, a, b, b, a);
  const auto append = [](int64_t tokens, int64_t q, int64_t q_out, int64_t k, int64_t v) {
    return kv::check_append(X, Y, X, X, Y, Y, I, I, reinterpret_cast<const double *>(memory), tokens, 1, 1, 8, 8, q, q_out, k, v, 10, 16, MB_F16).code;
  };
  EXPECT(append(1 << 19, far, far, far, far) == MB_SUCCESS);
  for (int i = 0; i < 4; ++i) EXPECT(append(rows, i == 0 ? far : 8, i == 1 ? far : 8, i == 2 ? far : 8, i == 3 ? far : 8) == MB_INVALID_ARGS);
  const auto attention = [](int64_t batch, int64_t q, int64_t out, int64_t kv_heads, int64_t pages, int64_t page) {
    return kv::check_attention(X, X, X, I, I, Y, nullptr, nullptr, nullptr, batch, kv_heads, kv_heads, 8, q, out, pages, page, 4, 64, 0, 0, MB_F16).code;
  };
  EXPECT(attention(1 << 19, far, far, 1, 10, 16) == MB_SUCCESS);
  EXPECT(attention(1 << 28, far, 8, 1, 10, 16) == MB_INVALID_ARGS);
  EXPECT(attention(1 << 28, 8, far, 1, 10, 16) == MB_INVALID_ARGS);
  EXPECT(attention(1, 8, 8, 1 << 27, 1 << 20, 1 << 10) == MB_UNSUPPORTED);   // a pool of 2^60 values
  EXPECT(attention(1, 8, 8, 1 << 27, 1 << 20, 1 << 9) == MB_SUCCESS);
  EXPECT(mx::check_tensor(X, X, X, rows, 32, far, MB_F16, false).code == MB_INVALID_ARGS);
  EXPECT(mx::check_tensor(X, X, X, 1 << 19, 32, far, MB_F16, true).code == MB_SUCCESS);
  EXPECT(mx::check_gemm(X, X, X, X, nullptr, Y, (1ll << 31) - 5000, 32, 32, far, MB_F16).code == MB_INVALID_ARGS);
}

static void attention_in_place() {
  const auto code = [](const void *out, int64_t batch, int64_t q_stride, int64_t out_stride) {
    return kv::check_attention(X, X, X, I, I, out, nullptr, nullptr, nullptr, batch, 8, 2, 64, q_stride, out_stride, 10, 16, 4, 64, 0, 0, MB_F16).code;
  };
  EXPECT(code(X, 2, 512, 512) == MB_SUCCESS);
  EXPECT(code(X, 2, 1024, 512) == MB_INVALID_ARGS);
  EXPECT(code(X, 1, 1024, 512) == MB_SUCCESS);
  EXPECT(code(Y, 2, 1024, 512) == MB_SUCCESS);
}

// Eviction's threads step through a sequence's first and last slots by as many as a cluster has, in 32 bits.
static void sequences_of_almost_2_31() {
  const int64_t most = kv::MOST_SLOTS;
  EXPECT(most + 16 * 1024 <= INT32_MAX);
  const auto evict = [](int64_t length, int64_t budget, int64_t sinks, int64_t recent) {
    return kv::check_evict(X, X, I, I, F, Y, Y, I, I, reinterpret_cast<const float *>(uintptr_t{1} << 45), I, 1, 1, 1, 1 << 16, (1 << 15) - 1, (1 << 15) - 1,
                           (1 << 15) - 1, (1 << 15) - 1, length, length, budget, sinks, recent, MB_F16, budget).code;
  };
  EXPECT(evict(most, most, most, 0) == MB_SUCCESS);
  EXPECT(evict(most, most, 0, most) == MB_SUCCESS);
  EXPECT(evict(INT32_MAX - 4096, 10, 0, 0) == MB_UNSUPPORTED);
  EXPECT(evict(1000, INT32_MAX - 4096, INT32_MAX - 4096, 0) == MB_UNSUPPORTED);
  EXPECT(evict(1000, most + 1, 0, most + 1) == MB_UNSUPPORTED);
  EXPECT(kv::check_attention(X, X, X, I, I, Y, nullptr, nullptr, nullptr, 1, 1, 1, 8, 8, 8, 10, 1 << 16, 1 << 14, most + 1, 0, 0, MB_F16).code == MB_UNSUPPORTED);
  EXPECT(kv::check_attention(X, X, X, I, I, Y, nullptr, nullptr, nullptr, 1, 1, 1, 8, 8, 8, 10, 1 << 16, 1 << 14, most, 0, 0, MB_F16).code == MB_SUCCESS);
}

int main() {
  sequences_of_almost_2_31();
  attention_in_place();
  clusters();
  weights_of_too_many_slots();
  rows_too_many_or_too_long();
  strides_at_the_limits();
  if (failures != 0) std::printf("%d failures\n", failures);
  return failures != 0;
}
