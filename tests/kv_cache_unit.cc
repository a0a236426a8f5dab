// Page arithmetic and argument checks of the decode-step operators, without a GPU: compiled and run by tests/test_decode_cpu.py.
#include <cstdio>
#include <cstring>
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

alignas(16) static char memory[64];
static const void *const X = memory;
static void *const Y = memory + 32;
static const int32_t *const I = reinterpret_cast<const int32_t *>(memory);
static float *const F = reinterpret_cast<float *>(memory);
static const double *const D = reinterpret_cast<const double *>(memory);

struct Attention {
  const void *q = X, *k = X, *v = X, *out = Y;
  const int32_t *table = I, *lengths = I;
  const float *lse = F, *weights_in = nullptr, *weights_out = nullptr;
  int64_t batch = 2, heads = 8, kv_heads = 2, dim = 64, q_stride = 512, out_stride = 512, pages = 10, page = 16, max_pages = 4,
          max_length = 64, window = 0, weights_stride = 64;
  int dtype = MB_BF16;
  int code() const {
    return kv::check_attention(q, k, v, table, lengths, out, lse, weights_in, weights_out, batch, heads, kv_heads, dim, q_stride,
                               out_stride, pages, page, max_pages, max_length, window, weights_stride, dtype).code;
  }
};

struct Evict {
  const void *k = X, *v = X, *k_dst = Y, *v_dst = Y;
  const int32_t *table = I, *lengths = I, *dst_table = I, *dst_lengths = I, *kept = I;
  const float *weights = F, *dst_weights = F + 256;   // (2 x 2 x 64 weights)
  int64_t batch = 2, heads = 2, dim = 64, page = 16, pages = 10, max_pages = 4, dst_pages = 10, dst_max_pages = 2, max_length = 64,
          stride = 64, budget = 32, sinks = 4, recent = 8;
  int dtype = MB_F16;
  int code() const {
    return kv::check_evict(k, v, table, lengths, weights, k_dst, v_dst, dst_table, dst_lengths, dst_weights, kept, batch, heads, dim,
                           page, pages, max_pages, dst_pages, dst_max_pages, max_length, stride, budget, sinks, recent, dtype).code;
  }
};

struct Rope {
  const void *x = X, *y = Y;
  const int32_t *positions = I;
  const double *freq = D;
  int64_t tokens = 3, heads = 2, dim = 8, rotary = 8, xt = 16, xh = 8, yt = 16, yh = 8;
  int dtype = MB_F32;
  int code() const { return kv::check_rope(x, y, positions, freq, tokens, heads, dim, rotary, xt, xh, yt, yh, dtype).code; }
};

struct Append {
  const void *q = X, *q_out = Y, *k = X, *v = X, *kc = Y, *vc = Y;
  const int32_t *positions = I, *slots = I;
  const double *freq = D;
  int64_t tokens = 3, heads = 4, kv_heads = 2, dim = 8, rotary = 8, qt = 32, qot = 32, kt = 16, vt = 16, pages = 4, page = 2;
  int dtype = MB_F32;
  int code() const {
    return kv::check_append(q, q_out, k, v, kc, vc, positions, slots, freq, tokens, heads, kv_heads, dim, rotary, qt, qot, kt, vt, pages,
                            page, dtype).code;
  }
};

template <typename C, typename Change>
static int with(Change change) {
  C c;
  change(c);
  return c.code();
}

int main() {
  // ---- rows of pages: none outside the pool, and no offset that is cut to 32 bits
  EXPECT(kv::row_offset(0, 4, 2, 1, 16, 3, 8) == (1 * 16 + 3) * 8);
  EXPECT(kv::row_offset(3, 4, 2, 0, 16, 0, 8) == 3 * 2 * 16 * 8);
  EXPECT(kv::row_offset(4, 4, 2, 0, 16, 0, 8) == -1);
  EXPECT(kv::row_offset(-1, 4, 2, 0, 16, 0, 8) == -1);
  EXPECT(kv::row_offset(INT32_MIN, 4, 2, 0, 16, 0, 8) == -1);
  EXPECT(kv::row_offset(INT32_MAX, 4, 2, 0, 16, 0, 8) == -1);
  EXPECT(kv::row_offset(0, 0, 2, 0, 16, 0, 8) == -1);
  EXPECT(kv::row_offset(999999, 1000000, 8, 7, 64, 63, 128) == 1000000ll * 8 * 64 * 128 - 128);
  // ---- lengths
  bool bad;
  EXPECT(kv::usable_length(0, 64, &bad) == 0 && !bad);
  EXPECT(kv::usable_length(64, 64, &bad) == 64 && !bad);
  EXPECT(kv::usable_length(65, 64, &bad) == 64 && bad);
  EXPECT(kv::usable_length(-1, 64, &bad) == 0 && bad);
  EXPECT(kv::usable_length(INT32_MIN, 64, &bad) == 0 && bad);
  EXPECT(kv::longest_of(100, 4, 16) == 64 && kv::longest_of(10, 4, 16) == 10 && kv::longest_of(10, 0, 16) == 0);
  EXPECT(kv::window_begin(100, 0) == 0 && kv::window_begin(100, 100) == 0 && kv::window_begin(100, 30) == 70 && kv::window_begin(0, 5) == 0);

  // ---- attention
  EXPECT(Attention().code() == MB_SUCCESS);
  EXPECT(with<Attention>([](Attention &a) { a.batch = 0; a.q = a.out = nullptr; }) == MB_SUCCESS);
  EXPECT(with<Attention>([](Attention &a) { a.max_pages = 0; a.table = nullptr; }) == MB_SUCCESS);
  EXPECT(with<Attention>([](Attention &a) { a.dtype = 3; }) == MB_INVALID_ARGS);
  EXPECT(with<Attention>([](Attention &a) { a.dtype = -1; }) == MB_INVALID_ARGS);
  EXPECT(with<Attention>([](Attention &a) { a.heads = 7; a.q_stride = a.out_stride = 448; }) == MB_INVALID_ARGS);
  EXPECT(with<Attention>([](Attention &a) { a.kv_heads = 0; }) == MB_INVALID_ARGS);
  EXPECT(with<Attention>([](Attention &a) { a.dim = 0; }) == MB_INVALID_ARGS);
  EXPECT(with<Attention>([](Attention &a) { a.dim = 257; a.out_stride = 4096; }) == MB_UNSUPPORTED);
  EXPECT(with<Attention>([](Attention &a) { a.out_stride = 511; }) == MB_INVALID_ARGS);
  EXPECT(with<Attention>([](Attention &a) { a.q_stride = -512; }) == MB_INVALID_ARGS);
  EXPECT(with<Attention>([](Attention &a) { a.page = 0; }) == MB_INVALID_ARGS);
  EXPECT(with<Attention>([](Attention &a) { a.pages = 1ll << 28; }) == MB_UNSUPPORTED);
  EXPECT(with<Attention>([](Attention &a) { a.max_length = 1ll << 31; }) == MB_UNSUPPORTED);
  EXPECT(with<Attention>([](Attention &a) { a.max_length = -1; }) == MB_INVALID_ARGS);
  EXPECT(with<Attention>([](Attention &a) { a.window = -1; }) == MB_INVALID_ARGS);
  EXPECT(with<Attention>([](Attention &a) { a.weights_in = F; }) == MB_INVALID_ARGS);
  EXPECT(with<Attention>([](Attention &a) { a.weights_out = F; a.weights_stride = 63; }) == MB_INVALID_ARGS);
  EXPECT(with<Attention>([](Attention &a) { a.weights_out = F; }) == MB_SUCCESS);
  EXPECT(with<Attention>([](Attention &a) { a.lengths = nullptr; }) == MB_INVALID_ARGS);
  EXPECT(with<Attention>([](Attention &a) { a.k = nullptr; }) == MB_INVALID_ARGS);
  EXPECT(with<Attention>([](Attention &a) { a.v = memory + 1; }) == MB_INVALID_ARGS);
  EXPECT(with<Attention>([](Attention &a) { a.lse = reinterpret_cast<float *>(memory + 2); }) == MB_INVALID_ARGS);
  EXPECT(with<Attention>([](Attention &a) { a.batch = 1ll << 31; }) == MB_UNSUPPORTED);

  // ---- eviction
  EXPECT(Evict().code() == MB_SUCCESS);
  EXPECT(with<Evict>([](Evict &e) { e.sinks = 24; }) == MB_SUCCESS);
  EXPECT(with<Evict>([](Evict &e) { e.sinks = 25; }) == MB_INVALID_ARGS);
  EXPECT(with<Evict>([](Evict &e) { e.recent = 1ll << 62; }) == MB_INVALID_ARGS);
  EXPECT(with<Evict>([](Evict &e) { e.budget = 0; e.sinks = e.recent = 0; }) == MB_INVALID_ARGS);
  EXPECT(with<Evict>([](Evict &e) { e.sinks = -1; }) == MB_INVALID_ARGS);
  EXPECT(with<Evict>([](Evict &e) { e.budget = 33; }) == MB_INVALID_ARGS);                      // no room in the new table
  EXPECT(with<Evict>([](Evict &e) { e.budget = 33; e.max_length = 32; }) == MB_SUCCESS);        // nothing longer to keep
  EXPECT(with<Evict>([](Evict &e) { e.stride = 63; }) == MB_INVALID_ARGS);
  EXPECT(with<Evict>([](Evict &e) { e.dst_weights = F; }) == MB_INVALID_ARGS);
  EXPECT(with<Evict>([](Evict &e) { e.dst_weights = F + 255; }) == MB_INVALID_ARGS);
  EXPECT(with<Evict>([](Evict &e) { e.dst_weights = F - 127; }) == MB_INVALID_ARGS);              // (2 x 2 x 32 kept)
  EXPECT(with<Evict>([](Evict &e) { e.dst_weights = F - 128; }) == MB_SUCCESS);
  EXPECT(with<Evict>([](Evict &e) { e.kept = nullptr; }) == MB_INVALID_ARGS);
  EXPECT(with<Evict>([](Evict &e) { e.dst_table = nullptr; }) == MB_INVALID_ARGS);
  EXPECT(with<Evict>([](Evict &e) { e.k_dst = memory + 1; }) == MB_INVALID_ARGS);
  EXPECT(with<Evict>([](Evict &e) { e.dtype = 7; }) == MB_INVALID_ARGS);

  // ---- rotary positions
  EXPECT(Rope().code() == MB_SUCCESS);
  EXPECT(with<Rope>([](Rope &r) { r.y = X; }) == MB_SUCCESS);
  EXPECT(with<Rope>([](Rope &r) { r.y = X; r.xt = 32; }) == MB_INVALID_ARGS);
  EXPECT(with<Rope>([](Rope &r) { r.rotary = 3; }) == MB_INVALID_ARGS);
  EXPECT(with<Rope>([](Rope &r) { r.rotary = 10; }) == MB_INVALID_ARGS);
  EXPECT(with<Rope>([](Rope &r) { r.rotary = 0; r.freq = nullptr; r.positions = nullptr; }) == MB_SUCCESS);
  EXPECT(with<Rope>([](Rope &r) { r.freq = nullptr; }) == MB_INVALID_ARGS);
  EXPECT(with<Rope>([](Rope &r) { r.yt = 15; }) == MB_INVALID_ARGS);
  EXPECT(with<Rope>([](Rope &r) { r.yt = 8; r.yh = 24; }) == MB_SUCCESS);       // heads outside tokens
  EXPECT(with<Rope>([](Rope &r) { r.yt = 8; r.yh = 23; }) == MB_INVALID_ARGS);
  EXPECT(with<Rope>([](Rope &r) { r.xt = r.xh = 0; }) == MB_SUCCESS);           // one row read many times
  EXPECT(with<Rope>([](Rope &r) { r.xt = -16; }) == MB_INVALID_ARGS);
  EXPECT(with<Rope>([](Rope &r) { r.x = memory + 2; }) == MB_INVALID_ARGS);
  EXPECT(with<Rope>([](Rope &r) { r.freq = reinterpret_cast<const double *>(memory + 4); }) == MB_INVALID_ARGS);
  EXPECT(with<Rope>([](Rope &r) { r.tokens = -1; }) == MB_INVALID_ARGS);
  EXPECT(with<Rope>([](Rope &r) { r.heads = 0; }) == MB_INVALID_ARGS);
  EXPECT(with<Rope>([](Rope &r) { r.tokens = 0; r.x = nullptr; }) == MB_SUCCESS);

  // ---- append
  EXPECT(Append().code() == MB_SUCCESS);
  EXPECT(with<Append>([](Append &a) { a.kv_heads = 0; }) == MB_INVALID_ARGS);
  EXPECT(with<Append>([](Append &a) { a.qot = 31; }) == MB_INVALID_ARGS);
  EXPECT(with<Append>([](Append &a) { a.q_out = X; a.qt = 64; }) == MB_INVALID_ARGS);
  EXPECT(with<Append>([](Append &a) { a.slots = nullptr; }) == MB_INVALID_ARGS);
  EXPECT(with<Append>([](Append &a) { a.vc = nullptr; }) == MB_INVALID_ARGS);
  EXPECT(with<Append>([](Append &a) { a.pages = 0; a.kc = a.vc = nullptr; }) == MB_SUCCESS);
  EXPECT(with<Append>([](Append &a) { a.pages = 1ll << 30; }) == MB_UNSUPPORTED);

  // ---- 4-bit tensors: every byte of the scales has one place
  EXPECT(mx::blocks_of(1) == 1 && mx::blocks_of(32) == 1 && mx::blocks_of(33) == 2);
  EXPECT(mx::scale_bytes(128, 128) == 512 && mx::scale_bytes(129, 129) == 4 * 512 && mx::scale_bytes(1, 1) == 512);
  for (const long long rows : {1ll, 127ll, 300ll}) {
    const int64_t cols = 300, bytes = mx::scale_bytes(rows, cols);
    static unsigned char seen[1 << 14];
    std::memset(seen, 0, sizeof(seen));
    int64_t count = 0;
    for (int64_t r = 0; r < mx::tile_rows(rows) * 128; ++r)
      for (int64_t b = 0; b < mx::tile_cols(cols) * 4; ++b) {
        const int64_t at = mx::scale_at(r, b, mx::tile_cols(cols));
        EXPECT(at >= 0 && at < bytes && !seen[at]);
        seen[at] = 1;
        ++count;
      }
    EXPECT(count == bytes);
  }
  const auto tensor = [](const void *x, const void *codes, int64_t rows, int64_t cols, int64_t stride, int dtype, bool written) {
    return mx::check_tensor(x, codes, X, rows, cols, stride, dtype, written).code;
  };
  EXPECT(tensor(X, X, 3, 40, 40, MB_F32, true) == MB_SUCCESS);
  EXPECT(tensor(X, X, 3, 40, 0, MB_F32, false) == MB_SUCCESS);
  EXPECT(tensor(X, X, 3, 40, 39, MB_F32, true) == MB_INVALID_ARGS);
  EXPECT(tensor(X, memory + 8, 3, 40, 40, MB_F32, true) == MB_INVALID_ARGS);
  EXPECT(tensor(memory + 1, X, 3, 40, 40, MB_F16, true) == MB_INVALID_ARGS);
  EXPECT(tensor(nullptr, X, 3, 40, 40, MB_F16, true) == MB_INVALID_ARGS);
  EXPECT(tensor(nullptr, nullptr, 0, 40, 40, MB_F16, true) == MB_SUCCESS);
  EXPECT(tensor(X, X, -3, 40, 40, MB_F16, true) == MB_INVALID_ARGS);
  EXPECT(tensor(X, X, 1ll << 31, 40, 40, MB_F16, true) == MB_UNSUPPORTED);
  const auto gemm = [](const void *a, const float *bias, int64_t M, int64_t N, int64_t K, int64_t stride, int dtype) {
    return mx::check_gemm(a, X, X, X, bias, Y, M, N, K, stride, dtype).code;
  };
  EXPECT(gemm(X, F, 3, 5, 40, 5, MB_BF16) == MB_SUCCESS);
  EXPECT(gemm(X, F, 3, 5, 40, 4, MB_BF16) == MB_INVALID_ARGS);
  EXPECT(gemm(nullptr, F, 3, 5, 40, 5, MB_BF16) == MB_INVALID_ARGS);
  EXPECT(gemm(nullptr, F, 3, 5, 0, 5, MB_BF16) == MB_SUCCESS);   // an empty sum
  EXPECT(gemm(memory + 4, F, 3, 5, 40, 5, MB_BF16) == MB_INVALID_ARGS);
  EXPECT(gemm(X, reinterpret_cast<float *>(memory + 2), 3, 5, 40, 5, MB_BF16) == MB_INVALID_ARGS);
  EXPECT(gemm(X, F, 3, 5, 1ll << 31, 5, MB_BF16) == MB_UNSUPPORTED);
  EXPECT(gemm(X, F, 3, 5, 40, 5, 9) == MB_INVALID_ARGS);

  std::printf("%d failures\n", failures);
  return failures != 0;
}
