// Product of two microscaled 4-bit operands on the sm_100a tensor cores:
//
//   out[i, j] = act( sum_k A[i, k] 2^(ea[i, k / 32]) B[j, k] 2^(eb[j, k / 32]) + bias[j] )
//
// A and B hold E2M1 numbers, two to a byte, with an E8M0 scale per 32 neighbours of a row, in the layout that
// microscaled.cu writes.  The MMA takes the scales itself (tcgen05.mma kind::mxf4, one scale per 32 elements), its
// products of two 4-bit numbers and two powers of two are exact, and the sums are fp32 in tensor memory.
#include "microscaled.cuh"
#include "tcgen05.cuh"

namespace glowb200 {
namespace {

constexpr int kBlockM = 128;
constexpr int kBlockK = 128;  // bytes of a row per pipeline stage: 256 elements, one 128-byte swizzle atom
constexpr int kUmmaK = 32;    // bytes of a row per MMA: 64 elements, two scales
constexpr int kThreads = 192;

__device__ __forceinline__ void umma_mxf4(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t a_scales,
                                          uint32_t b_scales, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(a_scales), "r"(b_scales), "r"(accumulate)
      : "memory");
}
// 512 bytes of scales -> four columns of tensor memory, in each of the four lane quarters.
__device__ __forceinline__ void tmem_copy_scales(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
// Descriptor of 32 rows of 16 bytes, one behind the other (no swizzle): 8-row groups are 128 bytes apart.
__device__ __forceinline__ uint64_t smem_desc_rows16(uint32_t smem_addr) {
  return (uint64_t)((smem_addr & 0x3FFFFu) >> 4) | (uint64_t)1 << 16 | (uint64_t)(128 >> 4) << 32 | (uint64_t)1 << 46;
}
// Instruction descriptor for kind::mxf4: A = B = E2M1, both K-major, E8M0 scales, K 64.
__host__ __device__ constexpr uint32_t idesc_mxf4(int m, int n) {
  return (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(m >> 4) << 24);
}

struct FcParams {
  void *out;  // [M, N]
  const float *bias;
  int32_t *status;
  int M, N, k_steps;  // k_steps: MMAs to a row, 64 elements each
  int relu;
};

template <int BLOCK_N, int STAGES>
struct Smem {
  static constexpr int kRowTiles = (BLOCK_N + 127) / 128;
  static constexpr int kABytes = kBlockM * kBlockK, kBBytes = BLOCK_N * kBlockK;
  static constexpr int kSaBytes = 1024, kSbBytes = 1024 * kRowTiles;
  static constexpr int kStageBytes = kABytes + kBBytes + kSaBytes + kSbBytes;
  static constexpr int kTotal = STAGES * kStageBytes + 256 + 1024;
  static_assert(kTotal <= 232448, "more shared memory than a CTA can have");
};

template <int BLOCK_N, int STAGES, typename Out>
__global__ void __launch_bounds__(kThreads, 1)
fp4_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                const __grid_constant__ CUtensorMap map_sa, const __grid_constant__ CUtensorMap map_sb, const FcParams p) {
  using S = Smem<BLOCK_N, STAGES>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t *scales = smem + STAGES * (S::kABytes + S::kBBytes);
  uint64_t *full = reinterpret_cast<uint64_t *>(scales + STAGES * (S::kSaBytes + S::kSbBytes));
  uint64_t *empty = full + STAGES;
  uint64_t *acc_full = empty + STAGES;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(acc_full + 1);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
  constexpr uint32_t kScaleCols = 8 + 8 * S::kRowTiles;  // of one stage
  constexpr uint32_t kTmemCols = 512;
  static_assert(BLOCK_N + STAGES * kScaleCols <= kTmemCols, "tensor memory");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; s++) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(acc_full, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t tmem_base = *tmem_slot;
  const int m0 = blockIdx.x * kBlockM, n0 = blockIdx.y * BLOCK_N;
  const int k_blocks = (p.k_steps + 3) >> 2;

  if (warp == 0) {
    if (lane == 0) {
      for (int kb = 0; kb < k_blocks; kb++) {
        const int s = kb % STAGES;
        if (kb >= STAGES && !mbar_wait(&empty[s], ((kb / STAGES) - 1) & 1, abort_flag)) break;
        uint8_t *a = smem + s * (S::kABytes + S::kBBytes), *sa = scales + s * (S::kSaBytes + S::kSbBytes);
        mbar_expect_tx(&full[s], S::kStageBytes);
        tma_load_2d(a, &map_a, kb * kBlockK, m0, &full[s]);
        tma_load_2d(a + S::kABytes, &map_b, kb * kBlockK, n0, &full[s]);
        tma_load_2d(sa, &map_sa, kb * 256, m0 >> 7, &full[s]);
        tma_load_2d(sa + S::kSaBytes, &map_sb, kb * 256, n0 >> 7, &full[s]);
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      bool live = true;
      for (int kb = 0; kb < k_blocks; kb++) {
        const int s = kb % STAGES;
        if (!mbar_wait(&full[s], (kb / STAGES) & 1, abort_flag)) { live = false; break; }
        tc_fence_after();
        const uint32_t a_addr = smem_u32(smem + s * (S::kABytes + S::kBBytes));
        const uint32_t sa_addr = smem_u32(scales + s * (S::kSaBytes + S::kSbBytes)), sb_addr = sa_addr + S::kSaBytes;
        const uint64_t a_desc = smem_desc_sw128(a_addr), b_desc = smem_desc_sw128(a_addr + S::kABytes);
        const uint32_t t_sa = tmem_base + BLOCK_N + (uint32_t)s * kScaleCols, t_sb = t_sa + 8;
#pragma unroll
        for (int t = 0; t < 2; t++) {  // scale tiles: 128 elements of a row each
          tmem_copy_scales(t_sa + 4 * t, smem_desc_rows16(sa_addr + 512 * t));
#pragma unroll
          for (int r = 0; r < S::kRowTiles; r++)
            tmem_copy_scales(t_sb + (uint32_t)(4 * (t * S::kRowTiles + r)), smem_desc_rows16(sb_addr + 1024 * r + 512 * t));
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const uint32_t id = (uint32_t)(k & 1) * 2;  // which two of a scale word's four bytes
          umma_mxf4(tmem_base, a_desc + (uint64_t)(k * (kUmmaK >> 4)), b_desc + (uint64_t)(k * (kUmmaK >> 4)),
                    idesc_mxf4(kBlockM, BLOCK_N) | id << 4 | id << 29, t_sa + 4 * (k >> 1),
                    t_sb + (uint32_t)(4 * S::kRowTiles * (k >> 1)) + (BLOCK_N % 128 ? (uint32_t)((n0 & 127) >> 5) : 0u), (kb | k) != 0);
        }
        umma_commit(&empty[s]);
      }
      if (live) umma_commit(acc_full);
    }
  } else {
    const int quarter = warp & 3;
    const bool ok = __all_sync(0xffffffffu, mbar_wait(acc_full, 0, abort_flag));
    if (ok) {
      tc_fence_after();
      const int row = m0 + quarter * 32 + lane;
      const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16);
      Out *out = reinterpret_cast<Out *>(p.out) + (size_t)row * p.N;
#pragma unroll 1
      for (int c = 0; c < BLOCK_N; c += 16) {
        uint32_t acc[16];
        tmem_ld_32x32b_x16(lane_addr + (uint32_t)c, acc);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; i++) {
          const int j = n0 + c + i;
          if (row < p.M && j < p.N) {
            float v = __uint_as_float(acc[i]);
            if (p.bias) v += __ldg(p.bias + j);
            if (p.relu) v = v < 0.0f ? 0.0f : v;
            out[j] = from_float<Out>(v);
          }
        }
      }
    } else if (lane == 0 && p.status != nullptr) {
      atomicOr(p.status, GLOWB200_STATUS_WAIT_TIMEOUT);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem_base, kTmemCols);
}

// [rows, pitch] bytes, box of 128 bytes by box_rows, 128-byte swizzle.
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
// scale tiles [row tiles, tiles * 512 bytes] as words: a box is two tiles (256 words) of box_tiles row tiles.
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

template <int BLOCK_N, int STAGES, typename Out>
int launch(const void *a, const void *sa, const void *b, const void *sb, int64_t K, const FcParams &p, cudaStream_t s) {
  using S = Smem<BLOCK_N, STAGES>;
  const int64_t pitch = mx_pitch(K), tiles = mx_tiles(K);
  CUtensorMap ma, mb, msa, msb;
  if (int rc = make_data_map(&ma, a, p.M, pitch, kBlockM)) return rc;
  if (int rc = make_data_map(&mb, b, p.N, pitch, BLOCK_N)) return rc;
  if (int rc = make_scale_map(&msa, sa, mx_row_tiles(p.M), tiles, 1)) return rc;
  if (int rc = make_scale_map(&msb, sb, mx_row_tiles(p.N), tiles, S::kRowTiles)) return rc;
  auto kernel = fp4_gemm_kernel<BLOCK_N, STAGES, Out>;
  GLOWB200_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kTotal));
  GLOWB200_CUDA_OK(launch_pdl(kernel, dim3((p.M + kBlockM - 1) / kBlockM, (p.N + BLOCK_N - 1) / BLOCK_N), kThreads, S::kTotal, s, ma, mb, msa, msb, p));
  return GLOWB200_OK;
}

int check_fc(const void *out, int out_type, const void *in, const void *weights, const void *weights_scales, int64_t M, int64_t K, int64_t N, int flags) {
  GLOWB200_REQUIRE(M >= 0 && N >= 0 && K > 0 && M < (1ll << 31) && N < (1ll << 31) && K < (1ll << 31), "matrix dimensions out of range");
  GLOWB200_REQUIRE(out_type >= 0 && out_type <= 2, "float type %d is not GLOWB200_FLOAT32, _FLOAT16 or _BFLOAT16", out_type);
  GLOWB200_REQUIRE((flags & ~GLOWB200_FC_FUSE_RELU) == 0, "flags other than GLOWB200_FC_FUSE_RELU");
  if (M == 0 || N == 0) return GLOWB200_OK;
  GLOWB200_REQUIRE(out && in && weights && weights_scales, "NULL tensor pointer");
  GLOWB200_REQUIRE(aligned(weights, 16) && aligned(weights_scales, 16), "data and scales must start on 16-byte boundaries");
  GLOWB200_REQUIRE(aligned(out, float_type_bytes(out_type)), "the result is not aligned to its elements");
  return GLOWB200_OK;
}

int run_fc(void *out, int out_type, const void *a, const void *sa, const void *b, const void *sb, const float *bias, int64_t M, int64_t K,
           int64_t N, int flags, int32_t *status, cudaStream_t s) {
  const FcParams p{out, bias, status, (int)M, (int)N, (int)((K + 63) / 64), (flags & GLOWB200_FC_FUSE_RELU) != 0};
  return with_float_type(out_type, [&](auto *t) {
    return launch<256, 4, std::remove_pointer_t<decltype(t)>>(a, sa, b, sb, K, p, s);
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
  return run_fc(out, out_type, in, in_scales, weights, weights_scales, bias, M, K, N, flags, status, reinterpret_cast<cudaStream_t>(stream));
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
  uint8_t *data = reinterpret_cast<uint8_t *>(workspace), *scales = data + align_up((size_t)(M * mx_pitch(K)), 256);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (int rc = run_mx_quantize(in, in_type, M, K, row_stride, data, scales, s)) return rc;
  return run_fc(out, out_type, data, scales, weights, weights_scales, bias, M, K, N, flags, status, s);
}
