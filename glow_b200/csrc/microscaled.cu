// The microscaled 4-bit format: quantizing float rows and back.
//
// A block of 32 neighbours of a row shares the scale 2^e, e = floor(log2(max |x|)) - 2, so that its largest element is
// 4 to 8 times the scale and the E2M1 numbers (up to 6) are used whole; elements are x * 2^-e, an exact product, rounded
// to the nearest E2M1 number.
#include "microscaled.cuh"

namespace glowb200 {
namespace {

constexpr int kQuantThreads = 256;

// A block takes a scale tile: 128 rows by 128 columns.  Eight neighbours of a row to a lane, so four lanes share a scale;
// a warp has two rows at a time.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kQuantThreads) mx_quantize_kernel(const T *__restrict__ in, int64_t rows, int64_t cols, int64_t row_stride,
                                                                    int64_t tiles, uint8_t *__restrict__ data, uint8_t *__restrict__ scales) {
  __shared__ __align__(16) uint8_t tile[512];
  pdl_wait();
  pdl_launch_dependents();
  const int64_t row_tile = blockIdx.x / tiles, col_tile = blockIdx.x - row_tile * tiles;
  if (threadIdx.x < 32) reinterpret_cast<uint4 *>(tile)[threadIdx.x] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  const int lane = threadIdx.x & 31, first = threadIdx.x >> 4;  // 16 threads to a row
  const int64_t col = col_tile * 128 + (lane & 15) * 8, pitch = 16 * ((cols + 31) / 32);
#pragma unroll 4
  for (int i = 0; i < 8; i++) {
    const int r = i * 16 + first;
    const int64_t row = row_tile * 128 + r;
    if (row_tile * 128 + i * 16 + (first & ~1) >= rows) break;  // (of the warp's two rows the first: all lanes leave together)
    const bool real = row < rows;
    Eight<VEC, T> x;
    x.load(in + row * row_stride + col, real ? cols - col : 0);
    uint32_t byte;
    const uint32_t codes = mx_block(x, byte);
    if (real && col / 2 < pitch) {  // (pitch: whole blocks)
      *reinterpret_cast<uint32_t *>(data + row * pitch + col / 2) = codes;
      if ((lane & 3) == 0) tile[(r & 31) * 16 + (r >> 5) * 4 + ((lane & 15) >> 2)] = (uint8_t)byte;
    }
  }
  __syncthreads();
  if (threadIdx.x < 32)
    reinterpret_cast<uint4 *>(scales + (size_t)blockIdx.x * 512)[threadIdx.x] = reinterpret_cast<const uint4 *>(tile)[threadIdx.x];
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) mx_dequantize_kernel(const uint8_t *__restrict__ data, const uint8_t *__restrict__ scales, int64_t rows,
                                                            int64_t cols, int64_t tiles, T *__restrict__ out) {
  pdl_wait();
  pdl_launch_dependents();
  const int64_t chunks = (cols + 7) / 8, pitch = 16 * ((cols + 31) / 32);
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < rows * chunks; i += gridDim.x * 256ll) {
    const int64_t row = i / chunks, col = (i - row * chunks) * 8;
    const uint32_t codes = *reinterpret_cast<const uint32_t *>(data + row * pitch + col / 2);
    const float scale = mx_scale(scales[mx_scale_at(row, col >> 5, tiles)]);
    __align__(16) T w[8];
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const float2 n = mx_numbers((codes >> (8 * k)) & 0xFFu);
      w[2 * k] = from_float<T>(n.x * scale);
      w[2 * k + 1] = from_float<T>(n.y * scale);
    }
    T *o = out + row * cols + col;
    if (VEC) {
#pragma unroll
      for (int k = 0; k < (int)(8 * sizeof(T) / 16); k++) reinterpret_cast<uint4 *>(o)[k] = reinterpret_cast<const uint4 *>(w)[k];
    } else {
#pragma unroll
      for (int k = 0; k < 8; k++)
        if (col + k < cols) o[k] = w[k];
    }
  }
}

int check_matrix(int64_t rows, int64_t cols) {
  GLOWB200_REQUIRE(rows >= 0 && cols > 0 && rows < (1ll << 31) && cols < (1ll << 31), "matrix dimensions out of range");
  return GLOWB200_OK;
}

}  // namespace

int run_mx_quantize(const void *in, int in_type, int64_t rows, int64_t cols, int64_t row_stride, uint8_t *data, uint8_t *scales,
                    cudaStream_t s) {
  const int64_t tiles = mx_tiles(cols), blocks = mx_row_tiles(rows) * tiles;
  GLOWB200_REQUIRE(blocks < (1ll << 31), "the matrix has more than 2^31 tiles of 128 x 128");
  return with_float_type(in_type, [&](auto *t) {
    using T = std::remove_pointer_t<decltype(t)>;
    const bool vec = aligned(in, 16) && (row_stride * sizeof(T)) % 16 == 0;
    auto kernel = vec ? mx_quantize_kernel<T, true> : mx_quantize_kernel<T, false>;
    GLOWB200_CUDA_OK(launch_pdl(kernel, dim3((unsigned)blocks), kQuantThreads, 0, s, reinterpret_cast<const T *>(in), rows, cols, row_stride,
                                tiles, data, scales));
    return GLOWB200_OK;
  });
}

}  // namespace glowb200

using namespace glowb200;

extern "C" size_t glowb200_microscaled_fp4_scales_bytes(int64_t rows, int64_t cols) {
  if (rows < 0 || cols < 0) return 0;
  return (size_t)(mx_row_tiles(rows) * mx_tiles(cols) * 512);
}

extern "C" int glowb200_microscaled_fp4_quantize(const void *in, int in_type, int64_t rows, int64_t cols, int64_t row_stride, uint8_t *data,
                                                 uint8_t *scales, glowb200_stream_t stream) {
  if (int rc = check_matrix(rows, cols)) return rc;
  GLOWB200_REQUIRE(in_type >= 0 && in_type <= 2, "float type %d is not GLOWB200_FLOAT32, _FLOAT16 or _BFLOAT16", in_type);
  GLOWB200_REQUIRE(row_stride >= cols || rows <= 1, "a row stride of %lld elements for rows of %lld", (long long)row_stride, (long long)cols);
  if (rows == 0) return GLOWB200_OK;
  GLOWB200_REQUIRE(in && data && scales, "NULL tensor pointer");
  GLOWB200_REQUIRE(aligned(in, float_type_bytes(in_type)), "the input is not aligned to its elements");
  GLOWB200_REQUIRE(aligned(data, 16) && aligned(scales, 16), "data and scales must start on 16-byte boundaries");
  return run_mx_quantize(in, in_type, rows, cols, row_stride, data, scales, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int glowb200_microscaled_fp4_dequantize(const uint8_t *data, const uint8_t *scales, int64_t rows, int64_t cols, void *out,
                                                   int out_type, glowb200_stream_t stream) {
  if (int rc = check_matrix(rows, cols)) return rc;
  GLOWB200_REQUIRE(out_type >= 0 && out_type <= 2, "float type %d is not GLOWB200_FLOAT32, _FLOAT16 or _BFLOAT16", out_type);
  if (rows == 0) return GLOWB200_OK;
  GLOWB200_REQUIRE(data && scales && out, "NULL tensor pointer");
  GLOWB200_REQUIRE(aligned(data, 16) && aligned(scales, 16), "data and scales must start on 16-byte boundaries");
  GLOWB200_REQUIRE(aligned(out, float_type_bytes(out_type)), "the result is not aligned to its elements");
  const int64_t chunks = rows * ((cols + 7) / 8), most = (int64_t)sm_count() * 32, blocks = (chunks + 255) / 256;
  return with_float_type(out_type, [&](auto *t) {
    using T = std::remove_pointer_t<decltype(t)>;
    const bool vec = aligned(out, 16) && cols % 8 == 0;
    auto kernel = vec ? mx_dequantize_kernel<T, true> : mx_dequantize_kernel<T, false>;
    GLOWB200_CUDA_OK(launch_pdl(kernel, dim3((unsigned)(blocks < most ? blocks : most)), 256, 0, reinterpret_cast<cudaStream_t>(stream), data,
                                scales, rows, cols, mx_tiles(cols), reinterpret_cast<T *>(out)));
    return GLOWB200_OK;
  });
}
