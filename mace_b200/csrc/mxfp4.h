// Layout of 4-bit microscaled operands and the checks of their calls; plain C++, tested on the host as well.
#pragma once

#include "kv_cache.h"

namespace mx {

constexpr int BLOCK = 32;        // values that share a scale
constexpr int TILE_ROWS = 128;   // scales: a tile is 128 rows x 4 blocks
constexpr int TILE_BLOCKS = 4;
constexpr int TILE_BYTES = 512;

MB_HD int64_t blocks_of(int64_t cols) { return (cols + BLOCK - 1) / BLOCK; }
MB_HD int64_t tile_rows(int64_t rows) { return (rows + TILE_ROWS - 1) / TILE_ROWS; }
MB_HD int64_t tile_cols(int64_t cols) { return (blocks_of(cols) + TILE_BLOCKS - 1) / TILE_BLOCKS; }
MB_HD int64_t scale_bytes(int64_t rows, int64_t cols) { return tile_rows(rows) * tile_cols(cols) * TILE_BYTES; }
// Where the scale of row r's block b lies, `tiles` tiles of blocks to a row of tiles.
MB_HD int64_t scale_at(int64_t r, int64_t b, int64_t tiles) {
  const uint32_t row = static_cast<uint32_t>(r), block = static_cast<uint32_t>(b);   // (both below 2^31)
  return (static_cast<int64_t>(row / TILE_ROWS) * tiles + block / TILE_BLOCKS) * TILE_BYTES + row % 32 * 16 + row / 32 % 4 * 4 +
         block % TILE_BLOCKS;
}

inline kv::Verdict check_tensor(const void *x, const void *codes, const void *scales, int64_t rows, int64_t cols, int64_t stride,
                                int dtype, bool written) {
  KV_REQUIRE(kv::is_type(dtype), "element type is not MB_F32, MB_F16 or MB_BF16");
  KV_REQUIRE(rows >= 0 && cols >= 0, "negative size");
  if (rows > kv::MOST || cols > kv::MOST - 4096) return kv::unsupported("tensor too large");
  KV_REQUIRE(stride >= 0 && stride <= kv::MOST_STRIDE && kv::reaches(rows, stride) && (!written || rows <= 1 || stride >= cols),
             "output rows overlap, or stride is negative or too large");
  if (rows == 0 || cols == 0) return kv::fine();
  KV_REQUIRE(x != nullptr && codes != nullptr && scales != nullptr, "null operand");
  KV_REQUIRE(kv::aligned(x, kv::type_bytes(dtype)) && kv::aligned(codes, 16) && kv::aligned(scales, 16),
             "codes and scales must be 16-byte aligned, values by their size");
  return kv::fine();
}

inline kv::Verdict check_gemm(const void *a, const void *a_scales, const void *b, const void *b_scales, const float *bias, const void *c,
                              int64_t M, int64_t N, int64_t K, int64_t stride, int dtype) {
  KV_REQUIRE(kv::is_type(dtype), "element type is not MB_F32, MB_F16 or MB_BF16");
  KV_REQUIRE(M >= 0 && N >= 0 && K >= 0, "negative size");
  if (M > kv::MOST - 4096 || N > kv::MOST - 4096 || K > (1 << 30)) return kv::unsupported("matrix too large");
  KV_REQUIRE(stride >= 0 && stride <= kv::MOST_STRIDE && kv::reaches(M, stride) && (M <= 1 || stride >= N), "output rows overlap, or stride is negative or too large");
  if (M == 0 || N == 0) return kv::fine();
  KV_REQUIRE(c != nullptr && (K == 0 || (a != nullptr && a_scales != nullptr && b != nullptr && b_scales != nullptr)), "null operand");
  KV_REQUIRE(kv::aligned(a, 16) && kv::aligned(a_scales, 16) && kv::aligned(b, 16) && kv::aligned(b_scales, 16) &&
             kv::aligned(bias, 4) && kv::aligned(c, kv::type_bytes(dtype)),
             "codes and scales must be 16-byte aligned, values by their size");
  return kv::fine();
}

}  // namespace mx
