// Quantization to 4-bit microscaled floating point (blocks of 32 E2M1 codes that share an E8M0 scale) and back.
//
// A thread has eight values at a time, so four neighbouring lanes have a block: its largest magnitude is two shuffles away, and its
// exponent field is the scale.  Dividing by a power of two is exact, and the conversion rounds to nearest even and saturates, so the
// result is the definition's bit for bit.
#include <algorithm>

#include "elements.cuh"
#include "mxfp4.h"

namespace {

constexpr int THREADS = 256;
constexpr int EACH = 8;    // values of a thread at a time
// Groups of them that a thread has, THREADS apart (TIMES, a template's argument): addresses are worked out once, and as many loads are
// in flight.  Four, or two where a row's end would leave half of a block without work.

struct MxParams {
  const void *x;
  void *y;
  uint8_t *codes, *scales;
  int64_t rows, stride;
  int cols, tiles;       // tiles of scales in a row of tiles
  int chunks;            // groups of EACH values in a row's tiles
  int vec;               // words of 16 bytes (fp32: two of them) are aligned
  int times;
  int block_rows, row_blocks;   // a block has block_rows rows at a time, or (row_blocks > 0) a row so many blocks
  uint32_t chunk_mul, chunk_shift, row_mul, row_shift;
};

// Eight values as they lie, zeros behind the row's end.
template <typename T>
struct Eight {
  uint32_t word[EACH * sizeof(T) / 4];
  // left: values of the row from here on
  __device__ __forceinline__ void load(const T *from, int left, bool vec) {
    constexpr int WORDS = sizeof(word) / 16;
    if (vec && left >= EACH) {
#pragma unroll
      for (int w = 0; w < WORDS; ++w) {
        const uint4 v = mb_load(reinterpret_cast<const uint4 *>(from) + w);
        word[4 * w] = v.x, word[4 * w + 1] = v.y, word[4 * w + 2] = v.z, word[4 * w + 3] = v.w;
      }
    } else {
      elem::Vec<T, 4 / sizeof(T)> pack;
#pragma unroll
      for (int w = 0; w < static_cast<int>(sizeof(word) / 4); ++w) {
        pack.word = 0;
#pragma unroll
        for (int i = 0; i < static_cast<int>(4 / sizeof(T)); ++i) {
          const int at = w * (4 / sizeof(T)) + i;
          if (at < left) pack.v[i] = mb_load(from + at);
        }
        word[w] = pack.word;
      }
    }
  }
  __device__ __forceinline__ float value(int i) const {
    elem::Vec<T, 4 / sizeof(T)> pack;
    pack.word = word[i * sizeof(T) / 4];
    return elem::widen(pack.v[i % (4 / sizeof(T))]);
  }
  // The largest magnitude as fp32 bits (a NaN's are larger than everything).
  __device__ __forceinline__ uint32_t top() const {
    if constexpr (sizeof(T) == 4) {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < EACH; ++i) m = max(m, word[i] & 0x7fffffffu);
      return m;
    } else {
      // magnitudes of 16-bit floats order as numbers, two at a time
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < EACH / 2; ++i) m = __vmaxu2(m, word[i] & 0x7fff7fffu);
      elem::Vec<T, 2> pack;
      pack.word = max(m & 0xffffu, m >> 16);
      return __float_as_uint(elem::widen(pack.v[0]));
    }
  }
};

// Eight codes: the first value in the low half of the first byte.
__device__ __forceinline__ uint32_t e2m1x8(const float (&v)[EACH]) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

// The values of two codes, as halves: every one is exact.
__device__ __forceinline__ float2 values_of(uint32_t byte) {
  uint32_t h;
  asm("{\n\t.reg .b8 c;\n\tcvt.u8.u32 c, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, c;\n\t}" : "=r"(h) : "r"(byte));
  return __half22float2(*reinterpret_cast<const __half2 *>(&h));
}

// Where a thread's groups lie.  WIDE: a row has one or more blocks, and the thread groups chunk, chunk + THREADS, .. of it; else a block
// has several rows, and the thread the same group of rows block_rows apart.
template <bool WIDE, int TIMES>
struct Span {
  int64_t row;
  int chunk;
  __device__ __forceinline__ explicit Span(const MxParams &p) {
    if (WIDE) {
      const int r = static_cast<int>(fast_div(blockIdx.x, p.row_mul, p.row_shift));
      row = r;
      chunk = (static_cast<int>(blockIdx.x) - r * p.row_blocks) * (THREADS * TIMES) + threadIdx.x;
    } else {
      const int r = static_cast<int>(fast_div(threadIdx.x, p.chunk_mul, p.chunk_shift));
      row = static_cast<int64_t>(blockIdx.x) * p.block_rows * TIMES + r;
      chunk = r < p.block_rows ? static_cast<int>(threadIdx.x) - r * p.chunks : p.chunks;
    }
  }
  __device__ __forceinline__ int64_t row_of(const MxParams &p, int i) const { return WIDE ? row : row + i * p.block_rows; }
  __device__ __forceinline__ int chunk_of(int i) const { return WIDE ? chunk + i * THREADS : chunk; }
  // Addresses of group i: with WIDE a constant behind the first one's.
  template <typename P>
  __device__ __forceinline__ P *values(const MxParams &p, P *first, int i) const {
    return WIDE ? first + i * THREADS * EACH : first + i * p.block_rows * p.stride;
  }
  __device__ __forceinline__ uint32_t *codes(const MxParams &p, uint32_t *first, int blocks, int i) const {
    return WIDE ? first + i * THREADS : first + static_cast<int64_t>(i) * p.block_rows * blocks * 4;
  }
  __device__ __forceinline__ uint8_t *scales(const MxParams &p, uint8_t *first, int i) const {
    static_assert(THREADS * EACH % (mx::BLOCK * mx::TILE_BLOCKS) == 0, "whole tiles");
    return WIDE ? first + i * (THREADS * EACH / (mx::BLOCK * mx::TILE_BLOCKS)) * mx::TILE_BYTES
                : p.scales + mx::scale_at(row_of(p, i), chunk / (mx::BLOCK / EACH), p.tiles);
  }
};

// Items are (row, group of eight) of the whole tiles: a lane whose block does not exist writes the tile's zeros.  Rows are whole groups
// of sixteen lanes, whose four scales leave as a word.
template <typename T, bool WIDE, int TIMES>
__global__ void __launch_bounds__(THREADS) quantize_mxfp4_kernel(const MxParams p) {
  mb_grid_dep_launch();
  mb_grid_dep_wait();
  const Span<WIDE, TIMES> at(p);
  const int blocks = static_cast<int>(mx::blocks_of(p.cols));
  const int64_t tile_rows = mx::tile_rows(p.rows) * mx::TILE_ROWS;
  const T *x0 = static_cast<const T *>(p.x) + at.row * p.stride + at.chunk * EACH;
  uint32_t *codes0 = reinterpret_cast<uint32_t *>(p.codes) + at.row * blocks * 4 + at.chunk;
  uint8_t *scales0 = p.scales + mx::scale_at(at.row, at.chunk / (mx::BLOCK / EACH), p.tiles);
  Eight<T> x[TIMES];
#pragma unroll
  for (int i = 0; i < TIMES; ++i) {
    const int left = p.cols - at.chunk_of(i) * EACH;
#pragma unroll
    for (uint32_t &w : x[i].word) w = 0;
    if (at.row_of(p, i) < p.rows && left > 0) x[i].load(at.values(p, x0, i), left, p.vec);
  }
#pragma unroll
  for (int i = 0; i < TIMES; ++i) {
    const int64_t row = at.row_of(p, i);
    const int chunk = at.chunk_of(i), block = chunk / (mx::BLOCK / EACH);
    // (all lanes take part in the exchange, also those of the last block whose groups lie behind the row)
    uint32_t top = x[i].top();
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // floor(log2 max) - 2, at least -127; the biased exponent is that plus 129, 0 for what is below 2^-126
    const int field = static_cast<int>(top >> 23);
    const int scale = field == 255 ? 255 : max(field - 2, 0);
    // times 2^(127 - scale): a field of 254 - scale, at scale 0 .. 252 always a normal number
    const float factor = __uint_as_float(static_cast<uint32_t>(254 - scale) << 23);
    float v[EACH];
#pragma unroll
    for (int j = 0; j < EACH; ++j) v[j] = x[i].value(j) * factor;
    const uint32_t word = scale == 255 ? 0 : e2m1x8(v);
    const bool there = row < p.rows && block < blocks;
    uint32_t four = there ? scale : 0;
    four |= __shfl_down_sync(0xffffffffu, four, 4, 16) << 8;
    four |= __shfl_down_sync(0xffffffffu, four, 8, 16) << 16;
    if (there) *at.codes(p, codes0, blocks, i) = word;
    if ((threadIdx.x & 15) == 0 && row < tile_rows && chunk < p.chunks)
      *reinterpret_cast<uint32_t *>(at.scales(p, scales0, i)) = four;
  }
}

template <typename T, bool WIDE, int TIMES>
__global__ void __launch_bounds__(THREADS) dequantize_mxfp4_kernel(const MxParams p) {
  mb_grid_dep_launch();
  mb_grid_dep_wait();
  const Span<WIDE, TIMES> at(p);
  const int blocks = static_cast<int>(mx::blocks_of(p.cols));
  T *y0 = static_cast<T *>(p.y) + at.row * p.stride + at.chunk * EACH;
  uint32_t *codes0 = reinterpret_cast<uint32_t *>(p.codes) + at.row * blocks * 4 + at.chunk;
  uint8_t *scales0 = p.scales + mx::scale_at(at.row, at.chunk / (mx::BLOCK / EACH), p.tiles);
  uint32_t word[TIMES];
  int scale[TIMES];
#pragma unroll
  for (int i = 0; i < TIMES; ++i) {
    const int64_t row = at.row_of(p, i);
    const int chunk = at.chunk_of(i);
    word[i] = scale[i] = 0;
    if (row < p.rows && chunk * EACH < p.cols) {
      word[i] = mb_load(at.codes(p, codes0, blocks, i));
      scale[i] = mb_load(at.scales(p, scales0, i));
    }
  }
#pragma unroll
  for (int i = 0; i < TIMES; ++i) {
    const int64_t row = at.row_of(p, i);
    const int col = at.chunk_of(i) * EACH;
    if (row >= p.rows || col >= p.cols) continue;
    // 2^(scale - 127): scale 0 is the subnormal 2^-127, 255 is NaN
    const float unit = __uint_as_float(scale[i] == 255 ? 0x7fc00000u : scale[i] == 0 ? 0x00400000u : static_cast<uint32_t>(scale[i]) << 23);
    T *to = at.values(p, y0, i);
    constexpr int W = 16 / sizeof(T);
    elem::Vec<T, W> out[EACH / W];
#pragma unroll
    for (int j = 0; j < EACH; j += 2) {
      const float2 v = values_of(word[i] >> (4 * j) & 0xffu);
      out[j / W].v[j % W] = elem::narrow<T>(v.x * unit);
      out[j / W].v[j % W + 1] = elem::narrow<T>(v.y * unit);
    }
    if (p.vec && col + EACH <= p.cols) {
#pragma unroll
      for (int w = 0; w < EACH / W; ++w) out[w].store(to + w * W);
    } else {
#pragma unroll
      for (int j = 0; j < EACH; ++j)
        if (col + j < p.cols) to[j] = out[j / W].v[j % W];
    }
  }
}

MxParams make(const void *x, void *y, uint8_t *codes, uint8_t *scales, int64_t rows, int64_t cols, int64_t stride, int dtype) {
  MxParams p = {};
  p.x = x; p.y = y; p.codes = codes; p.scales = scales; p.rows = rows; p.stride = stride;
  p.cols = static_cast<int>(cols);
  p.tiles = static_cast<int>(mx::tile_cols(cols));
  p.chunks = p.tiles * (mx::TILE_BLOCKS * mx::BLOCK / EACH);
  // a row of more than THREADS groups has blocks of its own; shorter ones share one
  p.block_rows = std::max(1, THREADS / p.chunks);
  const int fours = (p.chunks + 4 * THREADS - 1) / (4 * THREADS), twos = (p.chunks + 2 * THREADS - 1) / (2 * THREADS);
  p.times = p.chunks > THREADS && twos < 2 * fours ? 2 : 4;   // (4096 columns: 18.4 us with four for 4099 rows, 13.5 with two)
  p.row_blocks = p.chunks <= THREADS ? 0 : p.times == 2 ? twos : fours;
  fast_div_make(p.chunks, &p.chunk_mul, &p.chunk_shift);
  fast_div_make(p.row_blocks, &p.row_mul, &p.row_shift);
  const void *values = x != nullptr ? x : y;
  p.vec = kv::aligned(values, 16) && stride * kv::type_bytes(dtype) % 16 == 0;
  return p;
}

int64_t blocks_for(const MxParams &p, int64_t rows) {
  return p.row_blocks == 0 ? ceil_div64(rows, static_cast<int64_t>(p.block_rows) * p.times) : rows * p.row_blocks;
}

}  // namespace

extern "C" {

size_t mb_mxfp4_scale_bytes(int64_t rows, int64_t cols) {
  return rows <= 0 || cols <= 0 || rows > kv::MOST || cols > kv::MOST ? 0 : static_cast<size_t>(mx::scale_bytes(rows, cols));
}

int mb_quantize_mxfp4(mb_context *ctx, const void *x, uint8_t *codes, uint8_t *scales, int64_t rows, int64_t cols, int64_t stride,
                      int dtype) {
  if (ctx == nullptr) return MB_INVALID_ARGS;
  const kv::Verdict v = mx::check_tensor(x, codes, scales, rows, cols, stride, dtype, false);
  if (v.code != MB_SUCCESS) return mb_fail(ctx, v.code, "mb_quantize_mxfp4: %s", v.why);
  if (rows == 0 || cols == 0) return MB_SUCCESS;
  MB_CUDA(ctx, cudaSetDevice(ctx->device));
  const MxParams p = make(x, nullptr, codes, scales, rows, cols, stride, dtype);
  const int64_t blocks = blocks_for(p, mx::tile_rows(rows) * mx::TILE_ROWS);
  if (blocks > kv::MOST) return mb_fail(ctx, MB_UNSUPPORTED, "mb_quantize_mxfp4: tensor too large");
  MB_FOR_ELEMENT(dtype, MB_CUDA(ctx, mb_launch_chained(ctx, p.row_blocks == 0 ? quantize_mxfp4_kernel<T, false, 4> : p.times == 2 ? quantize_mxfp4_kernel<T, true, 2> : quantize_mxfp4_kernel<T, true, 4>,
                                                       dim3(static_cast<unsigned>(blocks)), dim3(THREADS), 0, p)));
  ctx->launches++;
  return MB_SUCCESS;
}

int mb_dequantize_mxfp4(mb_context *ctx, const uint8_t *codes, const uint8_t *scales, void *x, int64_t rows, int64_t cols,
                        int64_t stride, int dtype) {
  if (ctx == nullptr) return MB_INVALID_ARGS;
  const kv::Verdict v = mx::check_tensor(x, codes, scales, rows, cols, stride, dtype, true);
  if (v.code != MB_SUCCESS) return mb_fail(ctx, v.code, "mb_dequantize_mxfp4: %s", v.why);
  if (rows == 0 || cols == 0) return MB_SUCCESS;
  MB_CUDA(ctx, cudaSetDevice(ctx->device));
  const MxParams p = make(nullptr, x, const_cast<uint8_t *>(codes), const_cast<uint8_t *>(scales), rows, cols, stride, dtype);
  const int64_t blocks = blocks_for(p, rows);
  if (blocks > kv::MOST) return mb_fail(ctx, MB_UNSUPPORTED, "mb_dequantize_mxfp4: tensor too large");
  MB_FOR_ELEMENT(dtype, MB_CUDA(ctx, mb_launch_chained(ctx, p.row_blocks == 0 ? dequantize_mxfp4_kernel<T, false, 4> : p.times == 2 ? dequantize_mxfp4_kernel<T, true, 2> : dequantize_mxfp4_kernel<T, true, 4>,
                                                       dim3(static_cast<unsigned>(blocks)), dim3(THREADS), 0, p)));
  ctx->launches++;
  return MB_SUCCESS;
}

}  // extern "C"
