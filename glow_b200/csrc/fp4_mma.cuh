// What the two kernels of the microscaled product share: MMA and scale copies, descriptors, tensor maps.
#pragma once
#include "microscaled.cuh"
#include "tcgen05.cuh"

namespace glowb200 {

constexpr int kBlockM = 128;
constexpr int kBlockK = 128;  // bytes of a row per pipeline stage: 256 elements, one 128-byte swizzle atom
constexpr int kUmmaK = 32;    // bytes of a row per MMA: 64 elements, two scales

struct FcParams {
  void *out;  // [M, N]
  const float *bias;
  int32_t *status;
  int M, N, k_steps;  // k_steps: MMAs to a row, 64 elements each
  int relu, store_by_tma;
};

// fp4_few_rows.cu: a product of at most kFewRows rows.  `in` is packed (in_type < 0), or a float matrix of in_type with
// at most kFewQuantizedRows rows.
constexpr int kFewRows = 128, kFewQuantizedRows = 32;
int run_fp4_few_rows(const FcParams &p, int out_type, const void *in, const void *in_scales, int in_type, int64_t row_stride,
                     const void *weights, const void *weights_scales, int64_t K, cudaStream_t s);

// ---- tensor maps (fp4_gemm.cu) ----
// [rows, pitch] bytes: boxes of 128 bytes by box_rows, 128-byte swizzle.
int make_data_map(CUtensorMap *map, const void *base, int64_t rows, int64_t pitch, int box_rows);
// Scale tiles [row tiles, tiles * 512 bytes] as words: a box is two tiles (256 words) of box_tiles row tiles.
int make_scale_map(CUtensorMap *map, const void *base, int64_t row_tiles, int64_t tiles, int box_tiles);

// PAIR: one MMA over the two SMs of a cluster of two blocks, 256 rows: each has its own 128 rows of A and of the
// result, its own scales and half of B's rows.
template <bool PAIR>
__device__ __forceinline__ void umma_mxf4(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t a_scales,
                                          uint32_t b_scales, uint32_t accumulate) {
  if constexpr (PAIR)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(a_scales), "r"(b_scales), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(a_scales), "r"(b_scales), "r"(accumulate)
        : "memory");
}
// 512 bytes of scales -> four columns of tensor memory, in each of the four lane quarters (PAIR: in both blocks, each
// from its own shared memory).
template <bool PAIR>
__device__ __forceinline__ void tmem_copy_scales(uint32_t taddr, uint64_t desc) {
  if constexpr (PAIR) asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
  else asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
// Descriptor of 32 rows of 16 bytes, one behind the other (no swizzle): 8-row groups are 128 bytes apart.
__device__ __forceinline__ uint64_t smem_desc_rows16(uint32_t smem_addr) {
  return (uint64_t)((smem_addr & 0x3FFFFu) >> 4) | (uint64_t)1 << 16 | (uint64_t)(128 >> 4) << 32 | (uint64_t)1 << 46;
}
// Instruction descriptor for kind::mxf4: A = B = E2M1, both K-major, E8M0 scales, K 64.
__host__ __device__ constexpr uint32_t idesc_mxf4(int m, int n) {
  return (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(m >> 4) << 24);
}

// One lane of a warp that runs together.  The loops that issue TMA loads and MMAs are walked by whole warps and only the
// instructions are this lane's: their operands then stay in uniform registers.  In a loop of one lane of a divergent
// warp every tcgen05 instruction took 60 to 95 clocks to issue, 1100 to 1270 a k-block, whatever the MMAs' size.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}

// Descriptors of tensor maps come from memory the first time; this needs no wait for the kernel before.
__device__ __forceinline__ void prefetch_map(const CUtensorMap *map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }

// mbar_wait by a whole warp, whose lanes agree on the outcome.
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, volatile int *abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag));
}

// Position in a ring of N places, and how often (even or odd) it has come round.
template <int N>
struct Ring {
  int at = 0;
  uint32_t round = 0;
  __device__ __forceinline__ void next() {
    if (++at == N) {
      at = 0;
      round ^= 1;
    }
  }
};

}  // namespace glowb200
