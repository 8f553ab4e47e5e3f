// The microscaled 4-bit format: quantizing float rows and back.
//
// A block of 32 neighbours of a row shares the scale 2^e, e = floor(log2(max |x|)) - 2, so that its largest element is
// 4 to 8 times the scale and the E2M1 numbers (up to 6) are used whole; elements are x * 2^-e, an exact product, rounded
// to the nearest E2M1 number.
#include "microscaled.cuh"

namespace glowb200 {
namespace {

constexpr int kThreads = 256;

// Both kernels: a block takes a scale tile, 128 rows by 128 columns; eight neighbours of a row to a lane, so four lanes share
// a scale, a warp has two rows at a time and a thread eight places.  All of a thread's loads are asked for before the
// first is used.
struct TilePlace {
  int64_t row0, col;  // of the block; of the thread's eight columns
  int first, rows;    // the thread's first row of the block; rows that are there
  __device__ __forceinline__ TilePlace(int64_t all_rows, unsigned tiles) {
    const unsigned row_tile = blockIdx.x / tiles;
    row0 = (int64_t)row_tile * 128;
    col = (int64_t)(blockIdx.x - row_tile * tiles) * 128 + (threadIdx.x & 15) * 8;
    first = (int)(threadIdx.x >> 4);
    rows = (int)min((int64_t)128, all_rows - row0);
  }
};

// RAGGED: rows off 16-byte boundaries, or whose last eight columns are not all there.  Their elements come one to a lane, 32
// neighbours at a time, and change places in shared memory: eight single loads to a lane would ask for eight times as
// many lines.
template <typename T, bool RAGGED>
__global__ void __launch_bounds__(kThreads) mx_quantize_kernel(const T *__restrict__ in, int64_t rows, int64_t cols, int64_t row_stride,
                                                               unsigned tiles, uint8_t *__restrict__ data, uint8_t *__restrict__ scales) {
  __shared__ __align__(16) uint8_t tile[512];
  __shared__ __align__(16) T staged[RAGGED ? kThreads * 8 : 8];
  pdl_wait();
  pdl_launch_dependents();
  const TilePlace at(rows, tiles);
  const int lane = threadIdx.x & 31;
  if (threadIdx.x < 32) reinterpret_cast<uint4 *>(tile)[threadIdx.x] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  const int64_t pitch = 16 * ((cols + 31) / 32);
  const T *x = in + (at.row0 + at.first) * row_stride + at.col;
  const int64_t left = cols - at.col;
  // (row r = 16 i + first of the block: r % 32 and r / 32 of its place in the scale tile are i's alone but for `first`)
  uint8_t *out = data + (at.row0 + at.first) * pitch + at.col / 2, *out_scale = tile + at.first * 16 + ((lane & 15) >> 2);
  const int mine = at.col / 2 < pitch ? at.rows - at.first : 0;  // (pitch: whole blocks)
  auto finish = [&](int i, const Eight<true, T> &v) {
    uint32_t byte;
    const uint32_t codes = mx_block(v, byte);
    if (i * 16 < mine) {
      *reinterpret_cast<uint32_t *>(out) = codes;
      if ((lane & 3) == 0) out_scale[(i & 1) * 256 + (i >> 1) * 4] = (uint8_t)byte;
    }
    out += 16 * pitch;
  };
  constexpr int kAtOnce = sizeof(T) == 4 ? 4 : 8;
#pragma unroll
  for (int i0 = 0; i0 < 8; i0 += kAtOnce) {
    if (i0 * 16 >= at.rows) break;
    Eight<true, T> v[kAtOnce];
    if constexpr (!RAGGED) {
#pragma unroll
      for (int i = 0; i < kAtOnce; i++) v[i].load(x + (int64_t)(i0 + i) * 16 * row_stride, (i0 + i) * 16 + at.first < at.rows ? left : 0);
#pragma unroll
      for (int i = 0; i < kAtOnce; i++)
        if ((i0 + i) * 16 < at.rows) finish(i0 + i, v[i]);
    } else {
      // the warp's two rows of 128 columns, 32 at a time: element e of them is row e / 128, column e % 128
      T *mine = staged + (threadIdx.x & ~31) * 8;
      const int64_t col0 = at.col - (lane & 15) * 8;
      const int row = (at.first & ~1);
      T w[kAtOnce][8];
#pragma unroll
      for (int i = 0; i < kAtOnce; i++)
#pragma unroll
        for (int k = 0; k < 8; k++) {
          const int r = (i0 + i) * 16 + row + (k >> 2);
          const int64_t c = col0 + (k & 3) * 32 + lane;
          w[i][k] = r < at.rows && c < cols ? in[(at.row0 + r) * row_stride + c] : from_float<T>(0.0f);
        }
#pragma unroll
      for (int i = 0; i < kAtOnce; i++)
        if ((i0 + i) * 16 < at.rows) {
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 8; k++) mine[k * 32 + lane] = w[i][k];
          __syncwarp();
#pragma unroll
          for (int k = 0; k < (int)(8 * sizeof(T) / 16); k++)
            reinterpret_cast<uint4 *>(v[i].w)[k] = reinterpret_cast<const uint4 *>(mine + lane * 8)[k];
          finish(i0 + i, v[i]);
        }
    }
  }
  __syncthreads();
  if (threadIdx.x < 32)
    reinterpret_cast<uint4 *>(scales + (size_t)blockIdx.x * 512)[threadIdx.x] = reinterpret_cast<const uint4 *>(tile)[threadIdx.x];
}

template <typename T, bool RAGGED>
__global__ void __launch_bounds__(kThreads) mx_dequantize_kernel(const uint8_t *__restrict__ data, const uint8_t *__restrict__ scales, int64_t rows,
                                                                 int64_t cols, unsigned tiles, T *__restrict__ out) {
  __shared__ __align__(16) uint8_t tile[512];
  __shared__ __align__(16) T staged[RAGGED ? kThreads * 8 : 8];
  pdl_wait();
  pdl_launch_dependents();
  const TilePlace at(rows, tiles);
  const int lane = threadIdx.x & 31;
  const int64_t pitch = 16 * ((cols + 31) / 32);
  const uint8_t *d = data + (at.row0 + at.first) * pitch + at.col / 2;
  uint32_t codes[8];
#pragma unroll
  for (int i = 0; i < 8; i++)
    codes[i] = i * 16 + at.first < at.rows && at.col < cols ? __ldg(reinterpret_cast<const uint32_t *>(d + (int64_t)i * 16 * pitch)) : 0u;
  if (threadIdx.x < 32)
    reinterpret_cast<uint4 *>(tile)[threadIdx.x] = __ldg(reinterpret_cast<const uint4 *>(scales + (size_t)blockIdx.x * 512) + threadIdx.x);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; i++) {
    if (i * 16 >= at.rows) break;
    const int r = i * 16 + at.first;
    const float scale = mx_scale(tile[at.first * 16 + ((lane & 15) >> 2) + (i & 1) * 256 + (i >> 1) * 4]);
    float v[8];
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const float2 n = mx_numbers((codes[i] >> (8 * k)) & 0xFFu);
      v[2 * k] = n.x * scale;
      v[2 * k + 1] = n.y * scale;
    }
    uint32_t w[2 * sizeof(T)];
#pragma unroll
    for (int k = 0; k < (int)(2 * sizeof(T)); k++) {
      if constexpr (sizeof(T) == 4) w[k] = __float_as_uint(v[k]);
      else w[k] = pack2(v[2 * k], v[2 * k + 1], T());
    }
    if constexpr (!RAGGED) {
      if (r < at.rows && at.col < cols) {
        T *o = out + (at.row0 + r) * cols + at.col;
#pragma unroll
        for (int k = 0; k < (int)(sizeof(T) / 2); k++)
          reinterpret_cast<uint4 *>(o)[k] = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
      }
    } else {
      T *mine = staged + (threadIdx.x & ~31) * 8;
      __syncwarp();
#pragma unroll
      for (int k = 0; k < (int)(sizeof(T) / 2); k++)
        reinterpret_cast<uint4 *>(mine + lane * 8)[k] = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
      __syncwarp();
      const int64_t col0 = at.col - (lane & 15) * 8;
#pragma unroll
      for (int k = 0; k < 8; k++) {
        const int rr = i * 16 + (at.first & ~1) + (k >> 2);
        const int64_t c = col0 + (k & 3) * 32 + lane;
        if (rr < at.rows && c < cols) out[(at.row0 + rr) * cols + c] = mine[k * 32 + lane];
      }
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
    const bool whole = aligned(in, 16) && (row_stride * sizeof(T)) % 16 == 0 && cols % 8 == 0;
    auto kernel = whole ? mx_quantize_kernel<T, false> : mx_quantize_kernel<T, true>;
    GLOWB200_CUDA_OK(launch_pdl(kernel, dim3((unsigned)blocks), kThreads, 0, s, reinterpret_cast<const T *>(in), rows, cols, row_stride,
                                (unsigned)tiles, data, scales));
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
  const int64_t tiles = mx_tiles(cols), blocks = mx_row_tiles(rows) * tiles;
  GLOWB200_REQUIRE(blocks < (1ll << 31), "the matrix has more than 2^31 tiles of 128 x 128");
  return with_float_type(out_type, [&](auto *t) {
    using T = std::remove_pointer_t<decltype(t)>;
    auto kernel = aligned(out, 16) && cols % 8 == 0 ? mx_dequantize_kernel<T, false> : mx_dequantize_kernel<T, true>;
    GLOWB200_CUDA_OK(launch_pdl(kernel, dim3((unsigned)blocks), kThreads, 0, reinterpret_cast<cudaStream_t>(stream), data, scales, rows, cols,
                                (unsigned)tiles, reinterpret_cast<T *>(out)));
    return GLOWB200_OK;
  });
}
