// Product of two microscaled 4-bit operands on the sm_100a tensor cores:
//
//   out[i, j] = act( sum_k A[i, k] 2^(ea[i, k / 32]) B[j, k] 2^(eb[j, k / 32]) + bias[j] )
//
// A and B hold E2M1 numbers, two to a byte, with an E8M0 scale per 32 neighbours of a row, in the layout that
// microscaled.cu writes.  The MMA takes the scales itself (tcgen05.mma kind::mxf4, one scale per 32 elements), its
// products of two 4-bit numbers and two powers of two are exact, and the sums are fp32 in tensor memory.
//
// What bounds it.  Blocks of 128 x 256 sums load 48 KB of operands to a k-block (256 elements of depth), whose MMAs take 440 clocks,
// and L2 delivers some 75 bytes a clock to an SM: loads alone 158 us for 8192^3, MMAs alone 140, both 207.  Pairs of SMs
// with 256 x 256 sums load 32 KB each: 178 us, 6.2 PFLOP/s, the tensor pipe busy for 72 % of the time; a k-block takes 490
// clocks (11 tensor instructions issued by one thread), a tile 1300 more: the last MMAs run out, half of the sums are read,
// the next MMAs start.  Under sustained load the power limit lowers the clock: 4096 x 4096 x 8192 49 us in bursts, 61 in a loop
// of a tenth of a second.  2048 x 4096 x 4096 (15.7 us) has 128 tiles for 74 pairs: 1.7 rounds that take 2.
#include "fp4_mma.cuh"

namespace glowb200 {

int make_data_map(CUtensorMap *map, const void *base, int64_t rows, int64_t pitch, int box_rows) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return set_error(GLOWB200_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
  cuuint64_t dims[2] = {(cuuint64_t)pitch, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)pitch};
  cuuint32_t box[2] = {(cuuint32_t)kBlockK, (cuuint32_t)box_rows}, estr[2] = {1, 1};
  CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(GLOWB200_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
  return GLOWB200_OK;
}
int make_scale_map(CUtensorMap *map, const void *base, int64_t row_tiles, int64_t tiles, int box_tiles) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return set_error(GLOWB200_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
  cuuint64_t dims[2] = {(cuuint64_t)tiles * 128, (cuuint64_t)row_tiles}, strides[1] = {(cuuint64_t)tiles * 512};
  cuuint32_t box[2] = {256, (cuuint32_t)box_tiles}, estr[2] = {1, 1};
  CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void *>(base), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(GLOWB200_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
  return GLOWB200_OK;
}

namespace {

constexpr int kEpilogueWarps = 8;  // two to a lane quarter of tensor memory
constexpr int kThreads = 64 + 32 * kEpilogueWarps;

// Arrives on a barrier of another block of the cluster, for that block's tensor core to go on: what it waits for has been
// read into registers, no memory is handed over, and a release to the cluster would take a thousand clocks.
__device__ __forceinline__ void mbar_arrive_remote(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// Tensor memory (512 columns): two accumulators, then the scales of the k-blocks in flight.  Two accumulators of 256
// columns would leave no room for the scales, so they share kShared columns there: the epilogue empties those first, and
// the next tile's MMAs start as soon as it has.
template <int BLOCK_N, int STAGES, bool PAIR, typename Out>
struct Tile {
  static constexpr int kRows = PAIR ? 2 * kBlockM : kBlockM;  // of a tile
  static constexpr int kRowTiles = (BLOCK_N + 127) / 128;  // of the right operand's scales
  static constexpr int kBRows = PAIR ? BLOCK_N / 2 : BLOCK_N;  // that a block loads
  static constexpr int kABytes = kBlockM * kBlockK, kBBytes = kBRows * kBlockK;
  static constexpr int kSaBytes = 1024, kSbBytes = 1024 * kRowTiles;
  static constexpr int kStageBytes = kABytes + kBBytes + kSaBytes + kSbBytes;
  static constexpr int kChunk = 128 / (int)sizeof(Out);  // columns that a warp drains at a time: rows of 128 bytes
  static constexpr int kStaging = kEpilogueWarps * 32 * 128;
  static constexpr int kTotal = STAGES * kStageBytes + kStaging + 2 * BLOCK_N * 4 + 256 + 1024;
  static_assert(kTotal <= 232448, "more shared memory than a CTA can have");
  static constexpr int kShared = BLOCK_N == 256 ? 128 : 0;
  static constexpr uint32_t kScaleCols = 8 + 8 * kRowTiles;  // of one k-block
  static constexpr uint32_t kScalesAt = 2 * BLOCK_N - kShared;
  static_assert(kScalesAt + STAGES * kScaleCols <= 512 && kShared % kChunk == 0, "tensor memory");
};

__device__ __forceinline__ void tma_store_2d(const CUtensorMap *map, const void *src, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];"
               ::"l"(map), "r"(c0), "r"(c1), "r"(smem_u32(src))
               : "memory");
}

// Persistent: blocks, or pairs of them, walk the 128 x BLOCK_N (256 x BLOCK_N) tiles, row tile fastest (blocks that run
// together share weights).  Warp 0 loads, warp 1 (of a pair's even block) issues the copies of the scales and the MMAs,
// warps 2 to 9 drain.  The loads of a pair's two blocks are counted on the even one's barrier.
template <int BLOCK_N, int STAGES, bool PAIR, typename Out>
__global__ void __launch_bounds__(kThreads, 1)
fp4_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                const __grid_constant__ CUtensorMap map_sa, const __grid_constant__ CUtensorMap map_sb,
                const __grid_constant__ CUtensorMap map_out, const FcParams p) {
  using S = Tile<BLOCK_N, STAGES, PAIR, Out>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t *staging = smem + STAGES * (S::kABytes + S::kBBytes);
  uint8_t *scales = staging + S::kStaging;
  float *bias = reinterpret_cast<float *>(scales + STAGES * (S::kSaBytes + S::kSbBytes));  // [2][BLOCK_N]
  uint64_t *full = reinterpret_cast<uint64_t *>(bias + 2 * BLOCK_N);
  uint64_t *empty = full + STAGES;
  uint64_t *acc_full = empty + STAGES;  // [2]
  uint64_t *acc_empty = acc_full + 2;   // [2]
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(acc_empty + 2);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; s++) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; b++) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], (PAIR ? 2 : 1) * kEpilogueWarps);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x == 64) {
    prefetch_map(&map_a);
    prefetch_map(&map_sa);
    prefetch_map(&map_b);
    prefetch_map(&map_sb);
    prefetch_map(&map_out);
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      tmem_alloc_pair(tmem_slot, 512);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_slot, 512);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync();  // the partner's barriers exist before anything signals them
  tc_fence_after();
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  const int rank = PAIR ? (int)cluster_ctarank() : 0;
  const int64_t walker = PAIR ? blockIdx.x >> 1 : blockIdx.x, walkers = PAIR ? gridDim.x >> 1 : gridDim.x;
  const int m_tiles = (p.M + S::kRows - 1) / S::kRows, n_tiles = (p.N + BLOCK_N - 1) / BLOCK_N;
  const int64_t tiles = (int64_t)m_tiles * n_tiles;
  const int k_blocks = (p.k_steps + 3) >> 2;

  if (warp == 0) {
    Ring<STAGES> ring;
    bool live = true;
    for (int64_t t = walker; t < tiles && live; t += walkers) {
      const int n_tile = (int)(t / m_tiles), m0 = (int)(t - (int64_t)n_tile * m_tiles) * S::kRows + rank * kBlockM, n0 = n_tile * BLOCK_N;
      for (int kb = 0; kb < k_blocks; kb++, ring.next()) {
        const int s = ring.at;
        if (!warp_wait(&empty[s], ring.round ^ 1, abort_flag)) { live = false; break; }  // (passes at once the first time round)
        uint8_t *a = smem + s * (S::kABytes + S::kBBytes), *sa = scales + s * (S::kSaBytes + S::kSbBytes);
        if (elect_one()) {
          if constexpr (PAIR) {
            if (rank == 0) mbar_expect_tx(&full[s], 2 * S::kStageBytes);
            const uint32_t counted = map_to_cta(&full[s], 0);
            tma_load_2d_pair(sa, &map_sa, kb * 256, m0 >> 7, counted);
            tma_load_2d_pair(sa + S::kSaBytes, &map_sb, kb * 256, n0 >> 7, counted);
            tma_load_2d_pair(a, &map_a, kb * kBlockK, m0, counted);
            tma_load_2d_pair(a + S::kABytes, &map_b, kb * kBlockK, n0 + rank * S::kBRows, counted);
          } else {
            mbar_expect_tx(&full[s], S::kStageBytes);
            tma_load_2d(sa, &map_sa, kb * 256, m0 >> 7, &full[s]);
            tma_load_2d(sa + S::kSaBytes, &map_sb, kb * 256, n0 >> 7, &full[s]);
            tma_load_2d(a, &map_a, kb * kBlockK, m0, &full[s]);
            tma_load_2d(a + S::kABytes, &map_b, kb * kBlockK, n0, &full[s]);
          }
        }
        __syncwarp();
      }
    }
  } else if (warp == 1) {
    Ring<STAGES> ring;
    int lt = 0;
    bool live = rank == 0;
    for (int64_t t = walker; t < tiles && live; t += walkers, lt++) {
      const int buf = lt & 1;
      const int half_tile = BLOCK_N % 128 ? (int)(t / m_tiles) * BLOCK_N & 127 : 0;  // rows of the first scale tile in front of this tile's
      // The columns this tile's sums go to: of the shared ones the tile before has to be gone, else the one before that.
      if (S::kShared ? lt >= 1 && !warp_wait(&acc_empty[buf ^ 1], ((lt - 1) >> 1) & 1, abort_flag)
                     : lt >= 2 && !warp_wait(&acc_empty[buf], ((lt >> 1) - 1) & 1, abort_flag)) break;
      tc_fence_after();
      const uint32_t d_tmem = tmem_base + (uint32_t)(buf * (BLOCK_N - S::kShared));
      // The scales of a stage have columns of their own: a stage that is full again was empty, so the MMAs that read them are done.
      bool ready = mbar_try_wait(&full[ring.at], ring.round);
      // (Four MMAs whatever is left of the depth: what lies behind it is loaded as zeros under scales of 0.  Choosing among them
      // and not unrolling cost a sixteenth of a block's time where few blocks run.)
#pragma unroll 2
      for (int kb = 0; kb < k_blocks; kb++) {
        const int s = ring.at;
        if (!__all_sync(0xffffffffu, ready) && !warp_wait(&full[s], ring.round, abort_flag)) { live = false; break; }
        tc_fence_after();
        ring.next();
        ready = kb + 1 < k_blocks && mbar_try_wait(&full[ring.at], ring.round);  // (asked before this k-block's MMAs are issued)
        const uint32_t a_addr = smem_u32(smem + s * (S::kABytes + S::kBBytes));
        const uint32_t sa_addr = smem_u32(scales + s * (S::kSaBytes + S::kSbBytes)), sb_addr = sa_addr + S::kSaBytes;
        const uint64_t a_desc = smem_desc_sw128(a_addr), b_desc = smem_desc_sw128(a_addr + S::kABytes);
        const uint32_t t_sa = tmem_base + S::kScalesAt + (uint32_t)s * S::kScaleCols, t_sb = t_sa + 8;
        if (elect_one()) {
#pragma unroll
          for (int h = 0; h < 2; h++) {  // scale tiles: 128 elements of a row each
            tmem_copy_scales<PAIR>(t_sa + 4 * h, smem_desc_rows16(sa_addr + 512 * h));
#pragma unroll
            for (int r = 0; r < S::kRowTiles; r++)
              tmem_copy_scales<PAIR>(t_sb + (uint32_t)(4 * (h * S::kRowTiles + r)), smem_desc_rows16(sb_addr + 1024 * r + 512 * h));
          }
#pragma unroll
          for (int k = 0; k < 4; k++) {
            const uint32_t id = (uint32_t)(k & 1) * 2;  // which two of a scale word's four bytes
            umma_mxf4<PAIR>(d_tmem, a_desc + (uint64_t)(k * (kUmmaK >> 4)), b_desc + (uint64_t)(k * (kUmmaK >> 4)),
                            idesc_mxf4(S::kRows, BLOCK_N) | id << 4 | id << 29, t_sa + 4 * (k >> 1),
                            t_sb + (uint32_t)(4 * S::kRowTiles * (k >> 1) + (half_tile >> 5)), k != 0 ? 1u : (uint32_t)(kb != 0));
          }
          if constexpr (PAIR) umma_commit_pair(&empty[s]);
          else umma_commit(&empty[s]);
        }
        __syncwarp();
      }
      if (live && elect_one()) {
        if constexpr (PAIR) umma_commit_pair(&acc_full[buf]);
        else umma_commit(&acc_full[buf]);
      }
      __syncwarp();
    }
  } else {
    const int quarter = warp & 3, half = (warp - 2) >> 2, et = threadIdx.x - 64;
    constexpr int kChunks = BLOCK_N / S::kChunk;
    uint8_t *stage = staging + (warp - 2) * (32 * 128);  // 32 rows of 128 bytes, 16-byte pieces xor-ed with the row
    const uint32_t drained = PAIR ? map_to_cta(acc_empty, 0) : 0u;
    auto arrive_drained = [&](int buf) {
      if constexpr (PAIR) mbar_arrive_remote(drained + 8 * buf);
      else mbar_arrive(&acc_empty[buf]);
    };
    int lt = 0;
    bool dead = false;
    for (int64_t t = walker; t < tiles; t += walkers, lt++) {
      const int n_tile = (int)(t / m_tiles), m0 = (int)(t - (int64_t)n_tile * m_tiles) * S::kRows + rank * kBlockM, n0 = n_tile * BLOCK_N;
      const int buf = lt & 1;
      float *tile_bias = bias + buf * BLOCK_N;
      if (p.bias != nullptr) {
        if (et < BLOCK_N) tile_bias[et] = n0 + et < p.N ? p.bias[n0 + et] : 0.0f;
        asm volatile("bar.sync 1, %0;" ::"n"(kEpilogueWarps * 32) : "memory");
      }
      // A warp whose bounded wait gave up drains nothing any more, but walks on: the barrier counts every epilogue warp.
      if (!dead) dead = !warp_wait(&acc_full[buf], (lt >> 1) & 1, abort_flag);
      if (dead) continue;
      tc_fence_after();
      const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(buf * (BLOCK_N - S::kShared));
      // chunks whose draining frees what the next tile waits for: the shared columns, else all
      constexpr int kFirst = S::kShared ? S::kShared / S::kChunk : kChunks;
      const int last_of_first = kFirst - 1 < half ? -1 : (kFirst - 1 - half) / 2 * 2 + half;
      if (last_of_first < 0 && lane == 0) arrive_drained(buf);
#pragma unroll 1
      for (int i = half; i < kChunks; i += 2) {
        const int c = (S::kShared && buf == 0 ? kChunks - 1 - i : i) * S::kChunk;  // (the first accumulator shares its last columns)
        uint32_t acc[S::kChunk];
#pragma unroll
        for (int q = 0; q < S::kChunk; q += 16) tmem_ld_32x32b_x16(lane_addr + (uint32_t)(c + q), *reinterpret_cast<uint32_t(*)[16]>(acc + q));
        tmem_ld_wait();
        if (i == last_of_first) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_drained(buf);
        }
        if (n0 + c >= p.N) continue;
        if (p.bias != nullptr) {
#pragma unroll
          for (int q = 0; q < S::kChunk; q += 4) {
            const float4 b = *reinterpret_cast<const float4 *>(tile_bias + c + q);
            acc[q] = __float_as_uint(__uint_as_float(acc[q]) + b.x);
            acc[q + 1] = __float_as_uint(__uint_as_float(acc[q + 1]) + b.y);
            acc[q + 2] = __float_as_uint(__uint_as_float(acc[q + 2]) + b.z);
            acc[q + 3] = __float_as_uint(__uint_as_float(acc[q + 3]) + b.w);
          }
        }
        if (p.relu) {
#pragma unroll
          for (int q = 0; q < S::kChunk; q++) acc[q] = __uint_as_float(acc[q]) < 0.0f ? 0u : acc[q];
        }
        if (p.store_by_tma && lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        __syncwarp();  // the staging area is free again
#pragma unroll
        for (int q = 0; q < 8; q++) {
          uint4 w;
          if constexpr (sizeof(Out) == 4) {
            w = make_uint4(acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]);
          } else {
            uint32_t h[4];
#pragma unroll
            for (int e = 0; e < 4; e++) h[e] = pack2(__uint_as_float(acc[8 * q + 2 * e]), __uint_as_float(acc[8 * q + 2 * e + 1]), Out());
            w = make_uint4(h[0], h[1], h[2], h[3]);
          }
          *reinterpret_cast<uint4 *>(stage + lane * 128 + 16 * (q ^ (lane & 7))) = w;
        }
        if (p.store_by_tma) {
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0 && m0 + quarter * 32 < p.M) {
            tma_store_2d(&map_out, stage, n0 + c, m0 + quarter * 32);
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
        } else {  // rows off 16-byte boundaries
          __syncwarp();
          const int rows = min(32, p.M - m0 - quarter * 32), cols = min(S::kChunk, p.N - n0 - c);
          Out *out = reinterpret_cast<Out *>(p.out) + (size_t)(m0 + quarter * 32) * p.N + n0 + c;
          for (int r = 0; r < rows; r++)
            for (int j = lane; j < cols; j += 32)
              out[(size_t)r * p.N + j] = *reinterpret_cast<const Out *>(stage + r * 128 + ((j * (int)sizeof(Out)) ^ (16 * (r & 7))));
        }
      }
    }
    if (p.store_by_tma && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {  // a wait gave up: copies that are still on their way here get a bounded time to land
    if (threadIdx.x == 0 && p.status != nullptr) atomicOr(p.status, GLOWB200_STATUS_WAIT_TIMEOUT);
    const long long t0 = clock64();
    while (clock64() - t0 < 4000000ll) {
    }
    __syncthreads();
  }
  if constexpr (PAIR) cluster_sync();  // neither block leaves while its partner may read its tiles
  tc_fence_after();
  if (warp == 1) {
    if constexpr (PAIR) tmem_dealloc_pair(tmem_base, 512);
    else tmem_dealloc(tmem_base, 512);
  }
}

// the result [M, N]: boxes of 32 rows by 128 bytes, in the 128-byte swizzle
int make_out_map(CUtensorMap *map, const FcParams &p, int bytes) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return set_error(GLOWB200_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
  cuuint64_t dims[2] = {(cuuint64_t)p.N, (cuuint64_t)p.M}, strides[1] = {(cuuint64_t)p.N * bytes};
  cuuint32_t box[2] = {(cuuint32_t)(128 / bytes), 32}, estr[2] = {1, 1};
  CUresult r = fn(map, bytes == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, p.out, dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(GLOWB200_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
  return GLOWB200_OK;
}
template <int BLOCK_N, int STAGES, bool PAIR, typename Out>
int launch_tiles(const void *a, const void *sa, const void *b, const void *sb, int64_t K, FcParams p, cudaStream_t s) {
  using S = Tile<BLOCK_N, STAGES, PAIR, Out>;
  const int64_t pitch = mx_pitch(K), tiles = mx_tiles(K);
  CUtensorMap ma, mb, msa, msb, mout = {};
  if (int rc = make_data_map(&ma, a, p.M, pitch, kBlockM)) return rc;
  if (int rc = make_data_map(&mb, b, p.N, pitch, S::kBRows)) return rc;
  if (int rc = make_scale_map(&msa, sa, mx_row_tiles(p.M), tiles, 1)) return rc;
  if (int rc = make_scale_map(&msb, sb, mx_row_tiles(p.N), tiles, S::kRowTiles)) return rc;
  p.store_by_tma = aligned(p.out, 16) && (int64_t)p.N * sizeof(Out) % 16 == 0;
  if (p.store_by_tma)
    if (int rc = make_out_map(&mout, p, sizeof(Out))) return rc;
  auto kernel = fp4_gemm_kernel<BLOCK_N, STAGES, PAIR, Out>;
  GLOWB200_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kTotal));
  const int64_t work = (int64_t)((p.M + S::kRows - 1) / S::kRows) * ((p.N + BLOCK_N - 1) / BLOCK_N), most = sm_count() / (PAIR ? 2 : 1);
  const int64_t walkers = work < most ? work : most;
  if constexpr (!PAIR) {
    GLOWB200_CUDA_OK(launch_pdl(kernel, dim3((unsigned)walkers), kThreads, S::kTotal, s, ma, mb, msa, msb, mout, p));
  } else {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(2 * walkers));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = S::kTotal;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    GLOWB200_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, ma, mb, msa, msb, mout, static_cast<const FcParams>(p)));
  }
  return GLOWB200_OK;
}

template <typename Out>
int launch(const void *a, const void *sa, const void *b, const void *sb, int64_t K, const FcParams &p, cudaStream_t s) {
  // The tile whose rounds over the SMs take least: measured microseconds of a k-block and of what a tile costs beside its
  // k-blocks.  2048 x 4096 x 4096 takes 15.7 us in 256 x 256 tiles of pairs, 16.6 in 128 x 256, 22.3 in 128 x 128, 33 in
  // 128 x 64; 512 x 4096 x 4096 9.1, 9.1, 7.9, 11.2; 128 x 4096 x 37888 17.2, 13.8, 14.3, 20.4; 128 x 4096 x 256 8.4, 8.7, 7.0, 6.4.
  struct Kind {
    int rows, cols, sms;
    float block, tile;
  };
  constexpr Kind kKinds[4] = {{256, 256, 2, 0.33f, 1.6f}, {128, 256, 1, 0.37f, 1.7f}, {128, 128, 1, 0.265f, 0.9f}, {128, 64, 1, 0.235f, 0.5f}};
  int best = 0;
  float least = 0.0f;
  for (int i = 0; i < 4; i++) {
    const Kind &k = kKinds[i];
    const int64_t tiles = (int64_t)((p.M + k.rows - 1) / k.rows) * ((p.N + k.cols - 1) / k.cols), at_once = sm_count() / k.sms;
    const float cost = (float)((tiles + at_once - 1) / at_once) * ((float)((p.k_steps + 3) / 4) * k.block + k.tile);
    if (i == 0 || cost < least) {
      best = i;
      least = cost;
    }
  }
  switch (best) {
    case 0: return launch_tiles<256, 5, true, Out>(a, sa, b, sb, K, p, s);
    case 1: return launch_tiles<256, 3, false, Out>(a, sa, b, sb, K, p, s);
    case 2: return launch_tiles<128, 5, false, Out>(a, sa, b, sb, K, p, s);
    default: return launch_tiles<64, 7, false, Out>(a, sa, b, sb, K, p, s);
  }
}

int check_fc(const void *out, int out_type, const void *in, const void *weights, const void *weights_scales, int64_t M, int64_t K, int64_t N, int flags) {
  constexpr int64_t kMost = (1ll << 31) - 1024;  // (tiles reach beyond the last row and column)
  GLOWB200_REQUIRE(M >= 0 && N >= 0 && K > 0 && M <= kMost && N <= kMost && K <= kMost, "matrix dimensions out of range");
  GLOWB200_REQUIRE(out_type >= 0 && out_type <= 2, "float type %d is not GLOWB200_FLOAT32, _FLOAT16 or _BFLOAT16", out_type);
  GLOWB200_REQUIRE((flags & ~GLOWB200_FC_FUSE_RELU) == 0, "flags other than GLOWB200_FC_FUSE_RELU");
  if (M == 0 || N == 0) return GLOWB200_OK;
  GLOWB200_REQUIRE(out && in && weights && weights_scales, "NULL tensor pointer");
  GLOWB200_REQUIRE(aligned(weights, 16) && aligned(weights_scales, 16), "data and scales must start on 16-byte boundaries");
  GLOWB200_REQUIRE(aligned(out, float_type_bytes(out_type)), "the result is not aligned to its elements");
  return GLOWB200_OK;
}

// What is written (`name`: n bytes at p) beside weights and bias.
int check_beside(const char *name, const void *p, size_t n, const void *weights, const void *weights_scales, const float *bias, int64_t K, int64_t N) {
  GLOWB200_REQUIRE(apart(p, n, weights, (size_t)(N * mx_pitch(K))) && apart(p, n, weights_scales, glowb200_microscaled_fp4_scales_bytes(N, K)) &&
                       (bias == nullptr || apart(p, n, bias, (size_t)N * 4)),
                   "the %s lies over the weights or the bias", name);
  return GLOWB200_OK;
}

FcParams fc_params(void *out, const float *bias, int64_t M, int64_t K, int64_t N, int flags, int32_t *status) {
  return {out, bias, status, (int)M, (int)N, (int)((K + 63) / 64), (flags & GLOWB200_FC_FUSE_RELU) != 0, 0};
}

int run_fc(void *out, int out_type, const void *a, const void *sa, const void *b, const void *sb, const float *bias, int64_t M, int64_t K,
           int64_t N, int flags, int32_t *status, bool quantized, cudaStream_t s) {
  // The other kernel's time grows with the rows, which it adds up over a cluster, and shrinks with its splits of the depth: 64 rows
  // of 4096 x 4096 (K 1024, N 1024) 7.3 us (4.7) there and 6.3 (3.4) here, 32 rows 6.0 (4.1), 16 rows 5.2 (3.7), 64 rows of K
  // 16384, N 2048 8.1 and 13.6, 128 rows of it 15.7 and 16.8.  Behind a quantizing launch its clusters find their places
  // late: 33 rows of 4096 x 4096 12.6 us with the launch, 9.0 here, of K 16384, N 2048 11.0 and 19.
  const int64_t k_blocks = (K + 255) / 256;
  if ((M <= 16 && !quantized) || (M <= 32 && k_blocks >= 16 && !quantized) || (M <= kFewRows && k_blocks >= 32))
    return run_fp4_few_rows(fc_params(out, bias, M, K, N, flags, status), out_type, a, sa, -1, 0, b, sb, K, s);
  const FcParams p = fc_params(out, bias, M, K, N, flags, status);
  return with_float_type(out_type, [&](auto *t) {
    return launch<std::remove_pointer_t<decltype(t)>>(a, sa, b, sb, K, p, s);
  });
}

}  // namespace
}  // namespace glowb200

using namespace glowb200;

extern "C" int glowb200_microscaled_fp4_fc(void *out, int out_type, const uint8_t *in, const uint8_t *in_scales, const uint8_t *weights,
                                           const uint8_t *weights_scales, const float *bias, int64_t M, int64_t K, int64_t N, int flags,
                                           int32_t *status, glowb200_stream_t stream) {
  if (int rc = check_fc(out, out_type, in, weights, weights_scales, M, K, N, flags)) return rc;
  if (M == 0 || N == 0) return GLOWB200_OK;
  GLOWB200_REQUIRE(in_scales, "NULL tensor pointer");
  GLOWB200_REQUIRE(aligned(in, 16) && aligned(in_scales, 16), "data and scales must start on 16-byte boundaries");
  const size_t out_bytes = (size_t)(M * N) * float_type_bytes(out_type);
  GLOWB200_REQUIRE(apart(out, out_bytes, in, (size_t)(M * mx_pitch(K))) && apart(out, out_bytes, in_scales, glowb200_microscaled_fp4_scales_bytes(M, K)),
                   "the result lies over the input");
  if (int rc = check_beside("result", out, out_bytes, weights, weights_scales, bias, K, N)) return rc;
  return run_fc(out, out_type, in, in_scales, weights, weights_scales, bias, M, K, N, flags, status, false,
                reinterpret_cast<cudaStream_t>(stream));
}

extern "C" size_t glowb200_dynamic_microscaled_fp4_fc_workspace_bytes(int64_t M, int64_t K, int64_t N) {
  if (M < 0 || K < 0 || N < 0) return 0;
  return align_up((size_t)(M * mx_pitch(K)), 256) + glowb200_microscaled_fp4_scales_bytes(M, K);
}

extern "C" int glowb200_dynamic_microscaled_fp4_fc(void *out, int out_type, const void *in, int in_type, int64_t row_stride,
                                                   const uint8_t *weights, const uint8_t *weights_scales, const float *bias, int64_t M,
                                                   int64_t K, int64_t N, int flags, void *workspace, size_t workspace_bytes, int32_t *status,
                                                   glowb200_stream_t stream) {
  if (int rc = check_fc(out, out_type, in, weights, weights_scales, M, K, N, flags)) return rc;
  GLOWB200_REQUIRE(in_type >= 0 && in_type <= 2, "float type %d is not GLOWB200_FLOAT32, _FLOAT16 or _BFLOAT16", in_type);
  GLOWB200_REQUIRE(row_stride >= K || M <= 1, "a row stride of %lld elements for rows of %lld", (long long)row_stride, (long long)K);
  if (M == 0 || N == 0) return GLOWB200_OK;
  GLOWB200_REQUIRE(aligned(in, float_type_bytes(in_type)), "the input is not aligned to its elements");
  const size_t need = glowb200_dynamic_microscaled_fp4_fc_workspace_bytes(M, K, N);
  if (workspace == nullptr || workspace_bytes < need)
    return set_error(GLOWB200_ERR_WORKSPACE_TOO_SMALL, "workspace of %zu bytes given, %zu needed", workspace_bytes, need);
  GLOWB200_REQUIRE(aligned(workspace, 256), "workspace must be 256-byte aligned");
  const size_t out_bytes = (size_t)(M * N) * float_type_bytes(out_type), row_bytes = (size_t)K * float_type_bytes(in_type),
               stride_bytes = (size_t)row_stride * float_type_bytes(in_type);
  GLOWB200_REQUIRE(apart(out, out_bytes, in, row_bytes, M, stride_bytes) && apart(out, out_bytes, workspace, need) &&
                       apart(workspace, need, in, row_bytes, M, stride_bytes),
                   "result, input and workspace lie over one another");
  if (int rc = check_beside("result", out, out_bytes, weights, weights_scales, bias, K, N)) return rc;
  if (int rc = check_beside("workspace", workspace, need, weights, weights_scales, bias, K, N)) return rc;
  // Every tile of 128 columns quantizes all rows for itself: 8 rows of N 16384 8.6 us, in two launches 10; 16 rows 12.5 and
  // 10.4; 32 rows of N 4096 9.2 and 9.2.
  if (M <= kFewQuantizedRows && M * ((N + 127) / 128) <= 1024)
    return run_fp4_few_rows(fc_params(out, bias, M, K, N, flags, status), out_type, in, nullptr, in_type, row_stride, weights, weights_scales, K,
                            reinterpret_cast<cudaStream_t>(stream));
  uint8_t *data = reinterpret_cast<uint8_t *>(workspace), *scales = data + align_up((size_t)(M * mx_pitch(K)), 256);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (int rc = run_mx_quantize(in, in_type, M, K, row_stride, data, scales, s)) return rc;
  return run_fc(out, out_type, data, scales, weights, weights_scales, bias, M, K, N, flags, status, true, s);
}
