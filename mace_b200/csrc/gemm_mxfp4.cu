// Products of 4-bit microscaled matrices: C[m][n] = sum_k A[m][k] B[n][k] (+ bias[n]).
#include "elements.cuh"
#include "mxfp4.h"
#include "sm100_ptx.cuh"

namespace {

struct MxGemmParams {
  const uint8_t *a, *a_scales, *b, *b_scales;
  const float *bias;
  void *c;
  int64_t stride;
  int M, N, blocks, tiles;   // blocks of 32 and tiles of scales of a row
};

// ---- on CUDA cores ("tensor_cores" 0) --------------------------------------------------------------------------------------
//
// 64 x 64 of C a block, 4 x 4 a thread; a step is one block of 32, widened to fp32 in shared memory.
constexpr int CORE_TILE = 64;

__device__ __forceinline__ void widen_rows(const uint8_t *codes, const uint8_t *scales, int64_t row0, int rows, int block, int blocks,
                                           int tiles, float (*to)[CORE_TILE + 1]) {
  // 64 rows x 16 bytes: four threads a row, a word each
  const int r = threadIdx.x / 4, word = threadIdx.x % 4;
  const int64_t row = row0 + r;
  uint32_t bits = 0;
  float unit = 0.f;
  if (row < rows) {
    bits = mb_load(reinterpret_cast<const uint32_t *>(codes + (row * blocks + block) * 16) + word);
    const int s = mb_load(scales + mx::scale_at(row, block, tiles));
    unit = __uint_as_float(s == 255 ? 0x7fc00000u : s == 0 ? 0x00400000u : static_cast<uint32_t>(s) << 23);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t code = bits >> (4 * i);
    to[word * 8 + i][r] = __uint_as_float((code & 8u) << 28 | (code & 7u) << 22) * 8.507059173023461586e37f * unit;
  }
}

template <typename T>
__global__ void __launch_bounds__(256) gemm_mxfp4_cores_kernel(const MxGemmParams p) {
  __shared__ float as[mx::BLOCK][CORE_TILE + 1], bs[mx::BLOCK][CORE_TILE + 1];
  mb_grid_dep_launch();
  mb_grid_dep_wait();
  const int columns = (p.N + CORE_TILE - 1) / CORE_TILE;
  const int64_t m0 = static_cast<int64_t>(blockIdx.x / columns) * CORE_TILE, n0 = static_cast<int64_t>(blockIdx.x % columns) * CORE_TILE;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  float acc[4][4] = {};
  for (int block = 0; block < p.blocks; ++block) {
    __syncthreads();
    widen_rows(p.a, p.a_scales, m0, p.M, block, p.blocks, p.tiles, as);
    widen_rows(p.b, p.b_scales, n0, p.N, block, p.blocks, p.tiles, bs);
    __syncthreads();
    for (int k = 0; k < mx::BLOCK; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] += as[k][ty * 4 + i] * bs[k][tx + 16 * j];
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int64_t m = m0 + ty * 4 + i, n = n0 + tx + 16 * j;
      if (m < p.M && n < p.N)
        static_cast<T *>(p.c)[m * p.stride + n] = elem::narrow<T>(acc[i][j] + (p.bias != nullptr ? mb_load(p.bias + n) : 0.f));
    }
}

}  // namespace

extern "C" int mb_gemm_mxfp4(mb_context *ctx, const uint8_t *a_codes, const uint8_t *a_scales, const uint8_t *b_codes,
                             const uint8_t *b_scales, const float *bias, void *C, int64_t M, int64_t N, int64_t K, int64_t stride,
                             int dtype) {
  if (ctx == nullptr) return MB_INVALID_ARGS;
  const kv::Verdict v = mx::check_gemm(a_codes, a_scales, b_codes, b_scales, bias, C, M, N, K, stride, dtype);
  if (v.code != MB_SUCCESS) return mb_fail(ctx, v.code, "mb_gemm_mxfp4: %s", v.why);
  if (M == 0 || N == 0) return MB_SUCCESS;
  MB_CUDA(ctx, cudaSetDevice(ctx->device));
  MxGemmParams p = {};
  p.a = a_codes; p.a_scales = a_scales; p.b = b_codes; p.b_scales = b_scales; p.bias = bias; p.c = C; p.stride = stride;
  p.M = static_cast<int>(M); p.N = static_cast<int>(N);
  p.blocks = static_cast<int>(mx::blocks_of(K)); p.tiles = static_cast<int>(mx::tile_cols(K));
  const int64_t blocks = ceil_div64(M, CORE_TILE) * ceil_div64(N, CORE_TILE);
  if (blocks > kv::MOST) return mb_fail(ctx, MB_UNSUPPORTED, "mb_gemm_mxfp4: matrix too large");
  MB_FOR_ELEMENT(dtype, MB_CUDA(ctx, mb_launch_chained(ctx, gemm_mxfp4_cores_kernel<T>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, p)));
  ctx->launches++;
  return MB_SUCCESS;
}
