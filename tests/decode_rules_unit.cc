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
            for (const int64_t longest : {0ll, 1ll, 127ll, 128ll, 129ll, 1000ll, 2048ll, 2049ll, 8192ll, 16384ll, 16385ll, 30000ll, 120000ll,
                                          (1ll << 31) - 4097}) {
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

int main() {
  clusters();
  weights_of_too_many_slots();
  rows_too_many_or_too_long();
  if (failures != 0) std::printf("%d failures\n", failures);
  return failures != 0;
}
