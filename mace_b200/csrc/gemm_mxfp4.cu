// Products of 4-bit microscaled matrices: C[m][n] = sum_k A[m][k] B[n][k] (+ bias[n]).
//
// tcgen05.mma kind::mxf4 multiplies E2M1 codes as they lie (two to a byte, 64 of the depth an instruction) and applies the block
// scales itself; products are exact, sums fp32 in tensor memory.  B's rows -- a layer's outputs -- are the MMA's 128 rows and A's --
// the tokens -- its columns: a lane of the accumulator is then one n, a warp's store 32 neighbouring values of a row of C, whatever
// C's stride, type and alignment, and a single token costs 16 columns instead of 128 rows.
#include <algorithm>

#include "elements.cuh"
#include "gemm_u8_cut.cuh"
#include "mxfp4.h"
#include "sm100_ptx.cuh"

int mb_make_map_u8(mb_context *ctx, CUtensorMap *map, const void *base, uint64_t inner, uint64_t rows, uint64_t batch,
                   uint64_t batch_stride_bytes, uint32_t box_inner, uint32_t box_rows, CUtensorMapSwizzle swizzle,
                   uint64_t row_pitch);

namespace {

struct MxGemmParams {
  const uint8_t *a, *a_scales, *b, *b_scales;
  const float *bias;
  void *c;
  int64_t stride;
  int M, N, blocks, tiles;   // blocks of 32 and tiles of scales of a row
  int tiles_n, count, splits;
  int words;         // C's rows are whole words of this many neighbouring values, aligned: 1, 2 or 4
  int *status;
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

// ---- on the tensor cores ---------------------------------------------------------------------------------------------------
//
// Ten warps: one requests a step's tiles (256 of the depth: 128 rows of B and BT of A by TMA with the 128-byte swizzle, their scales
// by bulk copies, as they lie in tiles), one copies the scales on to tensor memory and issues the MMAs, eight take accumulators
// out.  With as many tiles as SMs or more, CTAs walk over tiles; the eight warps first empty the accumulator into registers, so that
// the next tile's MMAs run while they convert and store.  With fewer tiles, the depth of each is cut over a cluster of `splits`
// CTAs, whose partial tiles are added through distributed shared memory, in the order of their ranks.
using namespace sm100;

constexpr int WORK_WARPS = 8, MMA_WARP = 8, TMA_WARP = 9, TC_THREADS = 320;
constexpr long long WAIT_BUDGET = 1ll << 31;  // ~1 s of SM clocks per wait

template <int BT>
struct Cfg {
  static constexpr int ROW_TILES = (BT + 127) / 128;            // of A's scales
  static constexpr int B_BYTES = 128 * 128, A_BYTES = BT * 128;
  static constexpr int B_SCALES = 2 * mx::TILE_BYTES, A_SCALES = ROW_TILES * 2 * mx::TILE_BYTES;
  static constexpr int STAGE_BYTES = B_BYTES + A_BYTES + B_SCALES + A_SCALES;
  static constexpr int STAGES = BT == 256 ? 4 : BT == 128 ? 6 : 8;
  static constexpr int RING = STAGES * STAGE_BYTES;
  static constexpr int SMEM_BYTES = RING + 1024 /*align*/ + 512 /*barriers*/;
  static constexpr int ACCUMULATORS = BT == 256 ? 1 : 2;
  static constexpr int ACC_COLUMNS = BT < 32 ? 32 : BT;         // of tensor memory, each accumulator
  static constexpr int SCALE_COLUMNS = 8 + 8 * ROW_TILES;       // ... each stage's scales
  static constexpr int TMEM = 512;
  static constexpr int HALF = BT / 2;                           // columns of an accumulator that a warp takes
  static_assert(STAGE_BYTES % 1024 == 0 && SMEM_BYTES <= 227 * 1024, "shared memory");
  static_assert(ACCUMULATORS * ACC_COLUMNS + STAGES * SCALE_COLUMNS <= TMEM, "tensor memory");
  static_assert(128 * BT * 4 <= RING, "a partial tile reuses the ring");
};

template <int COLUMNS>
__device__ __forceinline__ void take_columns(uint32_t taddr, uint32_t (&r)[COLUMNS]) {
  if constexpr (COLUMNS >= 32) {
#pragma unroll
    for (int i = 0; i < COLUMNS / 32; ++i) tmem_ld_32x32b_x32(taddr + i * 32, *reinterpret_cast<uint32_t(*)[32]>(&r[i * 32]));
  } else if constexpr (COLUMNS == 16) {
    tmem_ld_32x32b_x16(taddr, r);
  } else {
    tmem_ld_32x32b_x8(taddr, r);
  }
  tmem_ld_wait();
#pragma unroll
  for (int i = 0; i < COLUMNS; ++i) asm volatile("" : "+r"(r[i]));   // (values are there from here on)
}

template <typename T, int BT>
__global__ void __launch_bounds__(TC_THREADS, 1)
gemm_mxfp4_tc_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ MxGemmParams p) {
  using C = Cfg<BT>;
  constexpr int STAGES = C::STAGES;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t *smem = smem_raw + (smem_base - smem_u32(smem_raw));
  const uint32_t full_bar = smem_base + C::RING, empty_bar = full_bar + 8 * STAGES;
  const uint32_t done_bar = empty_bar + 8 * STAGES, taken_bar = done_bar + 8 * C::ACCUMULATORS;   // of an accumulator
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + C::RING + 16 * STAGES + 16 * C::ACCUMULATORS);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == MMA_WARP * 32) {
    prefetch_tensormap(&map_a);
    prefetch_tensormap(&map_b);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar + 8 * s, 1);
      mbar_init(empty_bar + 8 * s, 1);
    }
    for (int i = 0; i < C::ACCUMULATORS; ++i) {
      mbar_init(done_bar + 8 * i, 1);
      mbar_init(taken_bar + 8 * i, WORK_WARPS);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == TMA_WARP) {
    tmem_alloc(smem_u32(tmem_slot), C::TMEM);
    tmem_relinquish();
    mb_grid_dep_launch();  // (behind the allocation: common.cuh says why)
  }
  // this CTA's tiles, and its run of their depth
  const int rank = p.splits > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int first = blockIdx.x / p.splits, stride = gridDim.x / p.splits;
  const int steps_all = (p.blocks + 7) / 8;
  const int step0 = static_cast<int>(static_cast<int64_t>(steps_all) * rank / p.splits);
  const int steps = static_cast<int>(static_cast<int64_t>(steps_all) * (rank + 1) / p.splits) - step0;
  // The first tile's rows of B are asked for into L2 while the kernel in front, as a rule the tokens' quantization, still runs.  (Into L2
  // only: should that kernel write them after all, L2 is where its writes go.  One token through 24 layers of 4096 x 4096: 10.06 -> 9.69 us a layer.)
  if (warp == TMA_WARP && lane == 0)
    for (int i = 0; i < min(steps, STAGES); ++i) tma_prefetch_3d(&map_b, (step0 + i) * 128, first % p.tiles_n * 128, 0);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  mb_grid_dep_wait();
  const auto fail = [&](int code) {
    *abort_flag = 1;
    atomicCAS(p.status, 0, code);
  };

  if (warp == TMA_WARP) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 1;
      for (int tile = first; tile < p.count && *abort_flag == 0; tile += stride) {
        const int tn = tile % p.tiles_n, tm = tile / p.tiles_n;
        const int row_tiles = min(C::ROW_TILES, (p.M + 127) / 128 - tm * C::ROW_TILES);
        for (int i = 0; i < steps; ++i) {
          if (!mbar_wait(empty_bar + 8 * stage, phase, abort_flag, WAIT_BUDGET)) {
            fail(MB_DEV_TIMEOUT_PRODUCER);
            break;
          }
          const int step = step0 + i;
          const uint32_t fb = full_bar + 8 * stage, sb = smem_base + stage * C::STAGE_BYTES, sa = sb + C::B_BYTES;
          const uint32_t sbs = sa + C::A_BYTES, sas = sbs + C::B_SCALES;
          // (a row's last tile of scales may be the first of the step's two)
          const uint32_t scales = min(2, p.tiles - 2 * step) * mx::TILE_BYTES;
          mbar_arrive_expect_tx(fb, C::B_BYTES + C::A_BYTES + scales * (1 + row_tiles));
          tma_load_3d(sb, &map_b, fb, step * 128, tn * 128, 0);
          tma_load_3d(sa, &map_a, fb, step * 128, tm * BT, 0);
          bulk_load_1d(sbs, p.b_scales + (static_cast<int64_t>(tn) * p.tiles + 2 * step) * mx::TILE_BYTES, scales, fb);
          for (int r = 0; r < row_tiles; ++r)
            bulk_load_1d(sas + r * 2 * mx::TILE_BYTES,
                         p.a_scales + (static_cast<int64_t>(tm * C::ROW_TILES + r) * p.tiles + 2 * step) * mx::TILE_BYTES, scales, fb);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == MMA_WARP) {
    int stage = 0, acc = 0;
    uint32_t phase = 0, acc_phase = 1;
    const uint64_t k_major = make_smem_desc(0, 16, 1024, 2), scale_rows = make_smem_desc(0, 128, 128, 0);
    const auto at = [](uint64_t desc, uint32_t addr) { return desc | static_cast<uint64_t>((addr >> 4) & 0x3FFFu); };
    for (int tile = first; tile < p.count; tile += stride) {
      const int tm = tile / p.tiles_n;
      // (the last tokens: no more columns than they need)
      const int columns = min(BT, (p.M - tm * BT + 15) / 16 * 16);
      const uint32_t idesc0 = make_idesc_mxf4(128, columns, 0), idesc2 = make_idesc_mxf4(128, columns, 2);
      if (!mbar_wait_warp(taken_bar + 8 * acc, acc_phase, abort_flag, WAIT_BUDGET)) {
        fail(MB_DEV_TIMEOUT_MMA);
        break;
      }
      tc_fence_after_sync();
      const uint32_t d = tmem + acc * C::ACC_COLUMNS;
      bool ok = true;
      for (int i = 0; i < steps; ++i) {
        if (!mbar_wait_warp(full_bar + 8 * stage, phase, abort_flag, WAIT_BUDGET)) {
          fail(MB_DEV_TIMEOUT_MMA);
          ok = false;
          break;
        }
        tc_fence_after_sync();
        const uint32_t sb = smem_base + stage * C::STAGE_BYTES, sa = sb + C::B_BYTES, sbs = sa + C::A_BYTES, sas = sbs + C::B_SCALES;
        const uint32_t tb = tmem + C::ACCUMULATORS * C::ACC_COLUMNS + stage * C::SCALE_COLUMNS, ta = tb + 8;
        const int left = p.blocks - (step0 + i) * 8;   // blocks of the depth from here on: two to an MMA
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          if (4 * kt >= left) break;
          tmem_cp_32x128b_elect(tb + 4 * kt, at(scale_rows, sbs + kt * mx::TILE_BYTES));
#pragma unroll
          for (int r = 0; r < C::ROW_TILES; ++r)
            tmem_cp_32x128b_elect(ta + 4 * (kt * C::ROW_TILES + r), at(scale_rows, sas + (2 * r + kt) * mx::TILE_BYTES));
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            if (4 * kt + 2 * j >= left) break;
            mma_mxf4_ss_elect(d, at(k_major, sb + (2 * kt + j) * 32), at(k_major, sa + (2 * kt + j) * 32), j == 0 ? idesc0 : idesc2,
                              tb + 4 * kt, ta + 4 * kt * C::ROW_TILES, (i > 0 || kt > 0 || j > 0) ? 1u : 0u);
          }
        }
        mma_commit_elect(empty_bar + 8 * stage);
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (!ok) break;
      mma_commit_elect(done_bar + 8 * acc);
      if (++acc == C::ACCUMULATORS) {
        acc = 0;
        acc_phase ^= 1;
      }
    }
  } else {
    const int quarter = warp & 3, half = warp >> 2;
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int tile = first; tile < p.count; tile += stride) {
      const int tn = tile % p.tiles_n, tm = tile / p.tiles_n;
      const int64_t n = static_cast<int64_t>(tn) * 128 + quarter * 32 + lane;
      const float bias = p.bias != nullptr && n < p.N && rank == 0 ? mb_load(p.bias + n) : 0.f;
      if (!mbar_wait_warp(done_bar + 8 * acc, acc_phase, abort_flag, WAIT_BUDGET)) {
        fail(MB_DEV_TIMEOUT_EPILOGUE);
        break;
      }
      tc_fence_after_sync();
      uint32_t r[C::HALF];
      take_columns<C::HALF>(tmem + (static_cast<uint32_t>(quarter * 32) << 16) + acc * C::ACC_COLUMNS + half * C::HALF, r);
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(taken_bar + 8 * acc);
      if (++acc == C::ACCUMULATORS) {
        acc = 0;
        acc_phase ^= 1;
      }
      if (p.splits > 1) {
        // (every copy and MMA of this CTA's only tile is done: the ring is free)
        float *part = reinterpret_cast<float *>(smem) + half * C::HALF * 128 + quarter * 32 + lane;
#pragma unroll
        for (int c = 0; c < C::HALF; ++c) part[c * 128] = __uint_as_float(r[c]) + bias;
      } else {
        const int m0 = tm * BT + half * C::HALF, rows = p.M - m0;
        if (sizeof(T) == 2 && p.words > 1) {
          // two columns at a time: an even lane has the first one's values of itself and its neighbour, the odd one the second's
          // (64 bytes of two rows each a store instead of one's)
          const int odd = lane & 1;
          T *to = static_cast<T *>(p.c) + (m0 + odd) * p.stride + (n - odd);
#pragma unroll
          for (int c = 0; c < C::HALF; c += 2) {
            elem::Vec<T, 4 / sizeof(T)> mine;
            mine.v[0] = elem::narrow<T>(__uint_as_float(r[c]) + bias);
            mine.v[1 % (4 / sizeof(T))] = elem::narrow<T>(__uint_as_float(r[c + 1]) + bias);
            const uint32_t other = __shfl_xor_sync(0xffffffffu, mine.word, 1);
            const uint32_t word = odd ? __byte_perm(other, mine.word, 0x7632) : __byte_perm(mine.word, other, 0x5410);
            if (c + odd < rows && n < p.N) *reinterpret_cast<uint32_t *>(to) = word;
            to += 2 * p.stride;
          }
        } else if (n < p.N) {
          T *to = static_cast<T *>(p.c) + m0 * p.stride + n;
#pragma unroll
          for (int c = 0; c < C::HALF; ++c) {
            if (c < rows) *to = elem::narrow<T>(__uint_as_float(r[c]) + bias);
            to += p.stride;
          }
        }
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (*abort_flag != 0) {
    // copies and MMAs in flight must not outlive the memory they write (bounded: about 2 ms)
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);
  }
  if (p.splits > 1) {
    cluster_sync_all();
    const int tn = first % p.tiles_n, tm = first / p.tiles_n;
    const int rows = min(BT, p.M - tm * BT);
    const uint32_t mine = smem_u32(smem);
    // four neighbouring n at a time
    for (int i = rank * TC_THREADS + threadIdx.x; i < rows * 32; i += p.splits * TC_THREADS) {
      const int64_t n = static_cast<int64_t>(tn) * 128 + i % 32 * 4, m = static_cast<int64_t>(tm) * BT + i / 32;
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
      for (int s = 0; s < p.splits; ++s) {
        float v[4];
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(mapa_shared(mine + 16 * i, s)) : "memory");
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[j] += v[j];
      }
      T *to = static_cast<T *>(p.c) + m * p.stride + n;
      elem::Vec<T, 4> out;
#pragma unroll
      for (int j = 0; j < 4; ++j) out.v[j] = elem::narrow<T>(sum[j]);
      if (p.words == 4) {
        if (n < p.N) out.store(to);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n + j < p.N) to[j] = out.v[j];
      }
    }
    // no CTA of a cluster may leave while another still reads its tile
    cluster_sync_all();
  }
  if (warp == TMA_WARP) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, C::TMEM);
  }
}

template <typename T, int BT>
int launch_tc(mb_context *ctx, MxGemmParams &p, int splits, int type) {
  using C = Cfg<BT>;
  const auto kern = gemm_mxfp4_tc_kernel<T, BT>;
  const uint32_t bit = 1u << (type * 5 + (BT == 16 ? 0 : BT == 32 ? 1 : BT == 64 ? 2 : BT == 128 ? 3 : 4));
  if (!(ctx->mxfp4_attr_mask & bit)) {
    MB_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM_BYTES));
    ctx->mxfp4_attr_mask |= bit;
  }
  const uint64_t pitch = static_cast<uint64_t>(p.blocks) * 16;
  CUtensorMap ma, mb;
  MB_RETURN_IF_ERROR(mb_make_map_u8(ctx, &ma, p.a, pitch, p.M, 1, p.M * pitch, 128, BT, CU_TENSOR_MAP_SWIZZLE_128B, pitch));
  MB_RETURN_IF_ERROR(mb_make_map_u8(ctx, &mb, p.b, pitch, p.N, 1, p.N * pitch, 128, 128, CU_TENSOR_MAP_SWIZZLE_128B, pitch));
  const int64_t count = static_cast<int64_t>(p.tiles_n) * ceil_div64(p.M, BT);
  if (count * splits > kv::MOST) return mb_fail(ctx, MB_UNSUPPORTED, "mb_gemm_mxfp4: matrix too large");
  p.count = static_cast<int>(count);
  p.splits = splits;
  const unsigned grid = static_cast<unsigned>(splits > 1 ? count * splits : std::min<int64_t>(count, ctx->num_sms));
  MB_CUDA(ctx, mb_launch_clusters(ctx, kern, grid, TC_THREADS, C::SMEM_BYTES, splits, ma, mb, p));
  ctx->launches++;
  ctx->launches_tc++;
  return MB_SUCCESS;
}

template <typename T>
int gemm_tc(mb_context *ctx, MxGemmParams &p, int type) {
  // The tile width and cut with the smallest estimate, in nanoseconds.  Measured: a step's bytes come at 88 a nanosecond with every SM
  // asking; around a CTA's steps 3.5 us for a first round, 0.6 for a further one; joining a cluster's parts 0.8 us and 8 ns a token.
  // 4096 x 4096 weights: 1 token 5.8 us (16 x 4 CTAs a tile), 128 8.3, 512 9.8 (128 wide, uncut), 1000 11.4 (256 wide, uncut; 128 wide, two
  // rounds: 16.1).
  const int64_t steps = (p.blocks + 7) / 8;
  int bt = 256, splits = 1;
  int64_t best = -1;
  for (const int w : {16, 32, 64, 128, 256}) {
    if (w < 128 && p.M > w) continue;   // (narrower tiles than a tile of scales: one of them only)
    if (w > 16 && p.M <= w / 2) break;
    const int64_t tiles = p.tiles_n * ceil_div64(p.M, w);
    const int64_t step = (128 * 128 + w * 128 + 1024 + (w + 127) / 128 * 1024) / 88;
    for (const int s : {1, 2, 4, 8}) {
      if (s > steps) break;
      const int64_t rounds = ceil_div64(tiles * s, mb_resident_cluster_ctas(ctx, s));
      const int64_t cost = 3500 + (rounds - 1) * 600 + rounds * ceil_div64(steps, s) * step + (s > 1 ? rounds * (800 + 8 * w) : 0);
      if (best < 0 || cost < best) best = cost, bt = w, splits = s;
    }
  }
  switch (bt) {
    case 16: return launch_tc<T, 16>(ctx, p, splits, type);
    case 32: return launch_tc<T, 32>(ctx, p, splits, type);
    case 64: return launch_tc<T, 64>(ctx, p, splits, type);
    case 128: return launch_tc<T, 128>(ctx, p, splits, type);
    default: return launch_tc<T, 256>(ctx, p, splits, type);
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
  p.tiles_n = static_cast<int>(ceil_div64(N, 128));
  p.status = ctx->dev_status;
  const uintptr_t each = kv::type_bytes(dtype);
  p.words = N % 4 == 0 && stride % 4 == 0 && kv::aligned(C, 4 * each) ? 4 : N % 2 == 0 && stride % 2 == 0 && kv::aligned(C, 2 * each) ? 2 : 1;
  if (ctx->use_tensor_cores && ctx->encode_tiled != nullptr && K > 0) {
    int st = MB_SUCCESS;
    MB_FOR_ELEMENT(dtype, st = gemm_tc<T>(ctx, p, dtype));
    return st;
  }
  const int64_t blocks = ceil_div64(M, CORE_TILE) * ceil_div64(N, CORE_TILE);
  if (blocks > kv::MOST) return mb_fail(ctx, MB_UNSUPPORTED, "mb_gemm_mxfp4: matrix too large");
  MB_FOR_ELEMENT(dtype, MB_CUDA(ctx, mb_launch_chained(ctx, gemm_mxfp4_cores_kernel<T>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, p)));
  ctx->launches++;
  return MB_SUCCESS;
}
