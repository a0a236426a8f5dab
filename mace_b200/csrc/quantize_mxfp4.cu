// Quantization to 4-bit microscaled floating point (blocks of 32 E2M1 codes that share an E8M0 scale) and back.
//
// A thread has eight values, so four neighbouring lanes have a block: its largest magnitude is two shuffles away, and its exponent
// field is the scale.  Dividing by a power of two is exact, and the conversion rounds to nearest even and saturates, so the result is
// the definition's bit for bit.
#include <algorithm>

#include "elements.cuh"
#include "mxfp4.h"

namespace {

constexpr int THREADS = 256;
constexpr int EACH = 8;   // values of a thread

struct MxParams {
  const void *x;
  void *y;
  uint8_t *codes, *scales;
  int64_t rows, stride;
  int cols, tiles;       // tiles of scales in a row of tiles
  int chunks;            // groups of EACH values in a row's tiles
  int vec;               // words of 16 bytes (fp32: two of them) are aligned
  int block_rows, row_blocks;   // a block has whole rows, or a row whole blocks
  uint32_t chunk_mul, chunk_shift, row_mul, row_shift;
};

template <typename T>
__device__ __forceinline__ void load_eight(const MxParams &p, const T *row, int col, float (&v)[EACH]) {
  if (p.vec && col + EACH <= p.cols) {
    constexpr int W = 16 / sizeof(T);
#pragma unroll
    for (int w = 0; w < EACH / W; ++w) {
      elem::Vec<T, W> word;
      word.load(row + col + w * W);
#pragma unroll
      for (int i = 0; i < W; ++i) v[w * W + i] = elem::widen(word.v[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < EACH; ++i) v[i] = col + i < p.cols ? elem::widen(mb_load(row + col + i)) : 0.f;
  }
}

// Two codes of a byte: lo in the low half.
__device__ __forceinline__ uint32_t e2m1x2(float lo, float hi) {
  uint16_t r;
  asm("{\n\t.reg .b8 c;\n\tcvt.rn.satfinite.e2m1x2.f32 c, %2, %1;\n\tcvt.u16.u8 %0, c;\n\t}" : "=h"(r) : "f"(lo), "f"(hi));
  return r;
}

// A thread's row and group of eight: with the whole tiles' groups of a row below THREADS a block has several rows, else a row
// several blocks.  chunk may lie behind the row's last.
__device__ __forceinline__ void place(const MxParams &p, int64_t *row, int *chunk) {
  if (p.row_blocks == 1) {
    const int r = static_cast<int>(fast_div(threadIdx.x, p.chunk_mul, p.chunk_shift));
    *row = static_cast<int64_t>(blockIdx.x) * p.block_rows + r;
    *chunk = r < p.block_rows ? static_cast<int>(threadIdx.x) - r * p.chunks : p.chunks;
  } else {
    const int r = static_cast<int>(fast_div(blockIdx.x, p.row_mul, p.row_shift));
    *row = r;
    *chunk = (static_cast<int>(blockIdx.x) - r * p.row_blocks) * THREADS + threadIdx.x;
  }
}

// Items are (row, group of eight) of the whole tiles: a lane whose block does not exist writes the tile's zeros.
template <typename T>
__global__ void __launch_bounds__(THREADS) quantize_mxfp4_kernel(const MxParams p) {
  mb_grid_dep_launch();
  mb_grid_dep_wait();
  int64_t row;
  int chunk;
  place(p, &row, &chunk);
  // (rows are whole groups of sixteen lanes, whose words of four scales leave together)
  if (chunk >= p.chunks || row >= mx::tile_rows(p.rows) * mx::TILE_ROWS) return;
  const int col = chunk * EACH;
  const bool there = row < p.rows;
  float v[EACH];
#pragma unroll
  for (int i = 0; i < EACH; ++i) v[i] = 0.f;
  if (there && col < p.cols) load_eight(p, static_cast<const T *>(p.x) + row * p.stride, col, v);
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
  const uint32_t lanes = 0xfu << (threadIdx.x & 28);
  top = max(top, __shfl_xor_sync(lanes, top, 1));
  top = max(top, __shfl_xor_sync(lanes, top, 2));
  // floor(log2 max) - 2, at least -127; the biased exponent is that plus 129, 0 for what is below 2^-126
  const int field = static_cast<int>(top >> 23);
  int scale = field == 255 ? 255 : max(field - 2, 0);
  uint32_t word = 0;
  if (scale != 255) {
    // times 2^(127 - scale): a field of 254 - scale, at scale 0 .. 252 always a normal number
    const float factor = __uint_as_float(static_cast<uint32_t>(254 - scale) << 23);
#pragma unroll
    for (int i = 0; i < EACH; i += 2) word |= e2m1x2(v[i] * factor, v[i + 1] * factor) << (4 * i);
  }
  const int64_t blocks = mx::blocks_of(p.cols);
  const int block = chunk / (mx::BLOCK / EACH);
  if (there && block < blocks) *reinterpret_cast<uint32_t *>(p.codes + row * blocks * 16 + chunk * 4) = word;
  // four blocks' scales make a word of their tile
  const uint32_t half = 0xffffu << (threadIdx.x & 16);
  uint32_t four = there && block < blocks ? scale : 0;
  four |= __shfl_down_sync(half, four, 4, 16) << 8;
  four |= __shfl_down_sync(half, four, 8, 16) << 16;
  if ((threadIdx.x & 15) == 0) *reinterpret_cast<uint32_t *>(p.scales + mx::scale_at(row, block, p.tiles)) = four;
}

template <typename T>
__global__ void __launch_bounds__(THREADS) dequantize_mxfp4_kernel(const MxParams p) {
  mb_grid_dep_launch();
  mb_grid_dep_wait();
  int64_t row;
  int chunk;
  place(p, &row, &chunk);
  const int col = chunk * EACH;
  if (row >= p.rows || col >= p.cols) return;
  const int64_t blocks = mx::blocks_of(p.cols);
  const uint32_t word = mb_load(reinterpret_cast<const uint32_t *>(p.codes + row * blocks * 16) + chunk);
  const int scale = mb_load(p.scales + mx::scale_at(row, chunk / (mx::BLOCK / EACH), p.tiles));
  // 2^(scale - 127): scale 0 is the subnormal 2^-127, 255 is NaN
  const float unit = __uint_as_float(scale == 255 ? 0x7fc00000u : scale == 0 ? 0x00400000u : static_cast<uint32_t>(scale) << 23);
  T *to = static_cast<T *>(p.y) + row * p.stride + col;
  T v[EACH];
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const uint32_t code = word >> (4 * i);
    // magnitude m (1 + half a bit) 2^(e - 1): bits e and mantissa put under a float's exponent, times 2^126; code 1 is a subnormal there
    const float value = __uint_as_float((code & 8u) << 28 | (code & 7u) << 22) * 8.507059173023461586e37f;
    v[i] = elem::narrow<T>(value * unit);
  }
  if (p.vec && col + EACH <= p.cols) {
    constexpr int W = 16 / sizeof(T);
#pragma unroll
    for (int w = 0; w < EACH / W; ++w) {
      elem::Vec<T, W> out;
#pragma unroll
      for (int i = 0; i < W; ++i) out.v[i] = v[w * W + i];
      out.store(to + w * W);
    }
  } else {
#pragma unroll
    for (int i = 0; i < EACH; ++i)
      if (col + i < p.cols) to[i] = v[i];
  }
}

MxParams make(const void *x, void *y, uint8_t *codes, uint8_t *scales, int64_t rows, int64_t cols, int64_t stride, int dtype) {
  MxParams p = {};
  p.x = x; p.y = y; p.codes = codes; p.scales = scales; p.rows = rows; p.stride = stride;
  p.cols = static_cast<int>(cols);
  p.tiles = static_cast<int>(mx::tile_cols(cols));
  p.chunks = p.tiles * (mx::TILE_BLOCKS * mx::BLOCK / EACH);
  p.block_rows = std::max(1, THREADS / p.chunks);
  p.row_blocks = (p.chunks + THREADS - 1) / THREADS;
  fast_div_make(p.chunks, &p.chunk_mul, &p.chunk_shift);
  fast_div_make(p.row_blocks, &p.row_mul, &p.row_shift);
  const void *values = x != nullptr ? x : y;
  p.vec = kv::aligned(values, 16) && stride * kv::type_bytes(dtype) % 16 == 0;
  return p;
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
  const int64_t blocks = ceil_div64(mx::tile_rows(rows) * mx::TILE_ROWS, p.block_rows) * p.row_blocks;
  if (blocks > kv::MOST) return mb_fail(ctx, MB_UNSUPPORTED, "mb_quantize_mxfp4: tensor too large");
  MB_FOR_ELEMENT(dtype, MB_CUDA(ctx, mb_launch_chained(ctx, quantize_mxfp4_kernel<T>, dim3(static_cast<unsigned>(blocks)), dim3(THREADS), 0, p)));
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
  const int64_t blocks = ceil_div64(rows, p.block_rows) * p.row_blocks;
  if (blocks > kv::MOST) return mb_fail(ctx, MB_UNSUPPORTED, "mb_dequantize_mxfp4: tensor too large");
  MB_FOR_ELEMENT(dtype, MB_CUDA(ctx, mb_launch_chained(ctx, dequantize_mxfp4_kernel<T>, dim3(static_cast<unsigned>(blocks)), dim3(THREADS), 0, p)));
  ctx->launches++;
  return MB_SUCCESS;
}

}  // extern "C"
