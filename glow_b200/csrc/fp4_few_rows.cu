// The microscaled product for few rows: a token, or a batch of decoding sequences.
//
// The weights are the MMA's 128-row operand and the rows of the input its columns, so that no more than 16 columns
// are computed for a token.  What bounds such a product is the weights' bytes and, at these sizes, latency: the depth is
// split over the blocks of a cluster, each of which has its k-blocks on their way at once, and their sums meet in shared
// memory, added in the blocks' order.  A float input is quantized by the block's own warps on its way to shared memory
// (eight warps, 256 columns of a row to a warp at a time): a launch of its own would cost more than the work does.
//
// One row of 4096 x 4096 takes 4.5 us, 8 float rows 5.3: 2.7 us are a launch's chain of map, load, scales, MMA and drain with
// one k-block, 0.9 a cluster's two barriers, the rest k-blocks, whose instructions take 0.2 us to issue.  The weights' bytes
// would take 1.4.  One row of K 4096, N 16384 moves 36 MB in 6.2 us, 5.8 TB/s.
#include "fp4_mma.cuh"

namespace glowb200 {
namespace {

constexpr int kWorkers = 8;  // warps that quantize and then drain, two to a lane quarter of tensor memory
constexpr int kThreads = 64 + 32 * kWorkers;
constexpr int kMostSplits = 8;

struct FewRowsParams {
  FcParams fc;
  const void *in;  // float input
  int64_t row_stride, cols;
  int splits, k_blocks;  // blocks of a cluster; k-blocks of a row
};

template <int NT>
struct FewRows {
  static constexpr int kStages = 4;
  static constexpr int kABytes = kBlockM * kBlockK, kBBytes = NT * kBlockK;
  static constexpr int kStageBytes = kABytes + kBBytes + 2048;
  static constexpr int kTotal = kStages * kStageBytes + 256 + 1024;
  static constexpr uint32_t kScaleCols = 16;  // of a stage: two tiles of either operand
  static constexpr uint32_t kTmemCols = NT + kStages * kScaleCols <= 128 ? 128 : 256;
  static constexpr int kAtOnce = NT <= 64 ? 2 : 1;  // blocks on an SM
  static_assert(NT + kStages * kScaleCols <= kTmemCols && kAtOnce * (kTotal + 1024) <= 233472 && kStages * kStageBytes >= NT * kBlockM * 4, "room");
};

__device__ __forceinline__ float4 ld_cluster(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
// In: void = packed input, loaded by TMA.
template <int NT, typename In, bool VEC, typename Out>
__global__ void __launch_bounds__(kThreads, FewRows<NT>::kAtOnce)
fp4_few_rows_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_sw,
                    const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_sx, const FewRowsParams p) {
  using S = FewRows<NT>;
  constexpr bool kPacked = std::is_void_v<In>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t *scales = smem + S::kStages * (S::kABytes + S::kBBytes);
  uint64_t *full = reinterpret_cast<uint64_t *>(scales + S::kStages * 2048);
  uint64_t *empty = full + S::kStages;
  uint64_t *acc_full = empty + S::kStages;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(acc_full + 1);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = p.splits > 1 ? (int)cluster_ctarank() : 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S::kStages; s++) {
      mbar_init(&full[s], kPacked ? 1 : 1 + p.fc.M);  // the loads and, of a float input, every row
      mbar_init(&empty[s], 1);
    }
    mbar_init(acc_full, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x == 32 * 2) {
    prefetch_map(&map_w);
    prefetch_map(&map_sw);
    if constexpr (kPacked) {
      prefetch_map(&map_x);
      prefetch_map(&map_sx);
    }
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, S::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  const int j0 = (int)(blockIdx.x / p.splits) * kBlockM;  // first of the tile's 128 rows of the weights
  // this block's k-blocks
  const int first = (int)((int64_t)p.k_blocks * rank / p.splits), last = (int)((int64_t)p.k_blocks * (rank + 1) / p.splits);

  if (warp == 0) {
    Ring<S::kStages> ring;
    for (int kb = first; kb < last; kb++, ring.next()) {
      const int s = ring.at;
      if (!warp_wait(&empty[s], ring.round ^ 1, abort_flag)) break;  // (passes at once the first time round)
      uint8_t *a = smem + s * (S::kABytes + S::kBBytes), *sa = scales + s * 2048;
      if (elect_one()) {
        mbar_expect_tx(&full[s], S::kABytes + 1024 + (kPacked ? S::kBBytes + 1024 : 0));
        tma_load_2d(a, &map_w, kb * kBlockK, j0, &full[s]);
        tma_load_2d(sa, &map_sw, kb * 256, j0 >> 7, &full[s]);
        if constexpr (kPacked) {
          tma_load_2d(a + S::kABytes, &map_x, kb * kBlockK, 0, &full[s]);
          tma_load_2d(sa + 1024, &map_sx, kb * 256, 0, &full[s]);
        }
      }
      __syncwarp();
    }
  } else if (warp == 1) {
    Ring<S::kStages> ring;
    bool ready = mbar_try_wait(&full[0], 0);
    for (int kb = first; kb < last; kb++) {
      const int s = ring.at;
      if (!__all_sync(0xffffffffu, ready) && !warp_wait(&full[s], ring.round, abort_flag)) break;
      tc_fence_after();
      ring.next();
      ready = kb + 1 < last && mbar_try_wait(&full[ring.at], ring.round);
      const uint32_t a_addr = smem_u32(smem + s * (S::kABytes + S::kBBytes)), sa_addr = smem_u32(scales + s * 2048);
      const uint64_t a_desc = smem_desc_sw128(a_addr), b_desc = smem_desc_sw128(a_addr + S::kABytes);
      const uint32_t t_sa = tmem_base + NT + (uint32_t)s * S::kScaleCols, t_sb = t_sa + 8;
      if (elect_one()) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
          tmem_copy_scales<false>(t_sa + 4 * h, smem_desc_rows16(sa_addr + 512 * h));
          tmem_copy_scales<false>(t_sb + 4 * h, smem_desc_rows16(sa_addr + 1024 + 512 * h));
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {  // (what lies behind the depth is zeros)
          const uint32_t id = (uint32_t)(k & 1) * 2;
          umma_mxf4<false>(tmem_base, a_desc + (uint64_t)(k * (kUmmaK >> 4)), b_desc + (uint64_t)(k * (kUmmaK >> 4)),
                           idesc_mxf4(kBlockM, NT) | id << 4 | id << 29, t_sa + 4 * (k >> 1), t_sb + 4 * (k >> 1), k != 0 ? 1u : (uint32_t)(kb != first));
        }
        if (kb + S::kStages < last) umma_commit(&empty[s]);  // (nobody waits for a stage that is not filled again)
        if (kb + 1 == last) umma_commit(acc_full);
      }
      __syncwarp();
    }
  } else {
    const int w = warp - 2;
    if constexpr (!kPacked) {
      // Rows of the input -> codes in the swizzled tile, scales in their tile.  Rows that are not there stay as they are:
      // each is a column of the product of its own, and nobody reads it.
      const In *in = reinterpret_cast<const In *>(p.in);
      constexpr int kBatch = sizeof(In) == 4 ? 2 : 4;  // rows of a warp on their way at once
      // (k-block, row), dealt in turn to so many warps that none skips kStages blocks: a wait by parity is one for the phase
      // before the present one at most, and a warp further ahead would find a stage empty that is two rounds behind.
      const int items = (last - first) * p.fc.M, dealt = min(kWorkers, S::kStages * p.fc.M);
      int block = 0, row = w;  // of the warp's next item; block: counted from the first
      for (; row >= p.fc.M; row -= p.fc.M) block++;
      bool live = true;
      for (int i0 = w < dealt ? w : items; i0 < items && live; i0 += kBatch * dealt) {
        Eight<VEC, In> x[kBatch];
        int blocks[kBatch], rows[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; i++) {
          blocks[i] = block;
          rows[i] = row;
          const int64_t col = (int64_t)(first + block) * 256 + lane * 8;
          x[i].load(in + (int64_t)row * p.row_stride + col, i0 + i * dealt < items ? p.cols - col : 0);
          for (row += dealt; row >= p.fc.M; row -= p.fc.M) block++;
        }
#pragma unroll
        for (int i = 0; i < kBatch; i++) {
          if (i0 + i * dealt >= items || !live) break;
          const int s = blocks[i] % S::kStages, r = rows[i];
          if (!warp_wait(&empty[s], (uint32_t)(blocks[i] / S::kStages & 1) ^ 1, abort_flag)) { live = false; break; }
          uint32_t byte;
          const uint32_t codes = mx_block(x[i], byte);
          *reinterpret_cast<uint32_t *>(smem + s * (S::kABytes + S::kBBytes) + S::kABytes + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4) = codes;
          if ((lane & 3) == 0) scales[s * 2048 + 1024 + (lane >> 4) * 512 + (r & 31) * 16 + (r >> 5) * 4 + ((lane >> 2) & 3)] = (uint8_t)byte;
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) mbar_arrive(&full[s]);
        }
      }
    }
    // The block's sums [row of the input][row of the weights], where its tiles were (all of them have been read).
    if (last > first && warp_wait(acc_full, 0, abort_flag)) {
      tc_fence_after();
      float *part = reinterpret_cast<float *>(smem);
      const int quarter = warp & 3;
#pragma unroll 1
      for (int c = 16 * (w >> 2); c < NT; c += 32) {
        if (c >= p.fc.M) break;
        uint32_t acc[16];
        tmem_ld_32x32b_x16(tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)c, acc);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; i++) part[(c + i) * kBlockM + quarter * 32 + lane] = __uint_as_float(acc[i]);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  const bool gave_up = *abort_flag != 0;
  if (gave_up) {  // copies that are still on their way here get a bounded time to land
    if (threadIdx.x == 0 && p.fc.status != nullptr) atomicOr(p.fc.status, GLOWB200_STATUS_WAIT_TIMEOUT);
    const long long t0 = clock64();
    while (clock64() - t0 < 4000000ll) {
    }
    __syncthreads();  // (each thread's loop ends for itself; what follows takes whole warps)
  }
  if (p.splits > 1) cluster_sync();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem_base, S::kTmemCols);
  if (!gave_up) {
    // Every block adds up its share of the tile, the parts in the blocks' order, four neighbours of a row to a thread.
    const int share = p.fc.M * (kBlockM / 4) / p.splits;
    const bool wide = (p.fc.N & 3) == 0 && (reinterpret_cast<uintptr_t>(p.fc.out) & (4 * sizeof(Out) - 1)) == 0;
#pragma unroll 2
    for (int e = rank * share + (int)threadIdx.x; e < (rank + 1) * share; e += kThreads) {
      const int i = e >> 5, j = j0 + (e & 31) * 4;
      const float4 *mine = reinterpret_cast<const float4 *>(smem) + e;
      float4 v[kMostSplits];
      if (p.splits == 1) {
        v[0] = *mine;
      } else {
#pragma unroll
        for (int r = 0; r < kMostSplits; r++)
          if (r < p.splits) v[r] = ld_cluster(map_to_cta(mine, (uint32_t)r));
      }
#pragma unroll
      for (int r = 1; r < kMostSplits; r++)
        if (r < p.splits) v[0] = make_float4(v[0].x + v[r].x, v[0].y + v[r].y, v[0].z + v[r].z, v[0].w + v[r].w);
      float sum[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
      __align__(16) Out w[4];
#pragma unroll
      for (int k = 0; k < 4; k++) {
        if (p.fc.bias != nullptr && j + k < p.fc.N) sum[k] += __ldg(p.fc.bias + j + k);
        if (p.fc.relu) sum[k] = sum[k] < 0.0f ? 0.0f : sum[k];
        w[k] = from_float<Out>(sum[k]);
      }
      Out *out = reinterpret_cast<Out *>(p.fc.out) + (size_t)i * p.fc.N + j;
      if (wide && j + 4 <= p.fc.N) {
        if constexpr (sizeof(Out) == 4) *reinterpret_cast<uint4 *>(out) = *reinterpret_cast<const uint4 *>(w);
        else *reinterpret_cast<uint2 *>(out) = *reinterpret_cast<const uint2 *>(w);
      } else {
#pragma unroll
        for (int k = 0; k < 4; k++)
          if (j + k < p.fc.N) out[k] = w[k];
      }
    }
  }
  __syncwarp();
  if (p.splits > 1) cluster_sync();  // no block leaves while another may read its sums
}

template <int NT, typename In, bool VEC, typename Out>
int launch(const CUtensorMap &mw, const CUtensorMap &msw, const void *in_scales, int64_t K, const FewRowsParams &p, cudaStream_t s) {
  using S = FewRows<NT>;
  CUtensorMap mx = {}, msx = {};
  if constexpr (std::is_void_v<In>) {
    if (int rc = make_data_map(&mx, p.in, p.fc.M, mx_pitch(K), NT)) return rc;
    if (int rc = make_scale_map(&msx, in_scales, 1, mx_tiles(K), 1)) return rc;
  }
  auto kernel = fp4_few_rows_kernel<NT, In, VEC, Out>;
  GLOWB200_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kTotal));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((p.fc.N + kBlockM - 1) / kBlockM * p.splits));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = S::kTotal;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)p.splits;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  GLOWB200_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, mw, msw, mx, msx, static_cast<const FewRowsParams>(p)));
  return GLOWB200_OK;
}

template <int NT, typename Out>
int launch_for_input(const CUtensorMap &mw, const CUtensorMap &msw, const void *in_scales, int in_type, int64_t K, const FewRowsParams &p,
                     cudaStream_t s) {
  if (in_type < 0) return launch<NT, void, false, Out>(mw, msw, in_scales, K, p, s);
  if constexpr (NT <= kFewQuantizedRows) {
    return with_float_type(in_type, [&](auto *t) {
      using T = std::remove_pointer_t<decltype(t)>;
      const bool vec = aligned(p.in, 16) && (p.row_stride * sizeof(T)) % 16 == 0;
      return vec ? launch<NT, T, true, Out>(mw, msw, in_scales, K, p, s) : launch<NT, T, false, Out>(mw, msw, in_scales, K, p, s);
    });
  }
  return set_error(GLOWB200_ERR_INVALID_ARGUMENT, "too many rows");
}

}  // namespace

int run_fp4_few_rows(const FcParams &fc, int out_type, const void *in, const void *in_scales, int in_type, int64_t row_stride,
                     const void *weights, const void *weights_scales, int64_t K, cudaStream_t s) {
  FewRowsParams p{fc, in, row_stride, K, 1, (fc.k_steps + 3) / 4};
  const int64_t tiles = (fc.N + kBlockM - 1) / kBlockM;
  // Blocks for the SMs once: one token of 4096 x 4096 takes 6.4, 5.5, 4.7 and 5.0 us in 1, 2, 4 and 8 splits (32 to 256 blocks), of
  // K 4096, N 16384 6.6 and 7.2 in 1 and 2, of 8192 x 8192 10.2, 7.5, 7.2 and 10.8.  Twice where a block has more than 32
  // pieces of rows to quantize: 16 rows of 4096 x 4096 7.0 and 6.6, 8 of N 16384 9.3 and 8.2 (8 of N 4096 5.3 and 5.8).
  auto fits = [&](int splits) {
    const bool much = in_type >= 0 && fc.M * (p.k_blocks / (splits / 2)) > 32;
    return splits <= kMostSplits && splits <= p.k_blocks && tiles * splits <= (much ? 2 : 1) * kB200Sms;
  };
  while (fits(p.splits * 2)) p.splits *= 2;
  CUtensorMap mw, msw;
  if (int rc = make_data_map(&mw, weights, fc.N, mx_pitch(K), kBlockM)) return rc;
  if (int rc = make_scale_map(&msw, weights_scales, mx_row_tiles(fc.N), mx_tiles(K), 1)) return rc;
  return with_float_type(out_type, [&](auto *o) {
    using Out = std::remove_pointer_t<decltype(o)>;
    if (fc.M <= 16) return launch_for_input<16, Out>(mw, msw, in_scales, in_type, K, p, s);
    if (fc.M <= 32) return launch_for_input<32, Out>(mw, msw, in_scales, in_type, K, p, s);
    if (fc.M <= 64) return launch_for_input<64, Out>(mw, msw, in_scales, in_type, K, p, s);
    return launch_for_input<128, Out>(mw, msw, in_scales, in_type, K, p, s);
  });
}

}  // namespace glowb200
