// The microscaled 4-bit format: quantizing float rows and back.
//
// A block of 32 neighbours of a row shares the scale 2^e, e = floor(log2(max |x|)) - 2, so that its largest element is
// 4 to 8 times the scale and the E2M1 numbers (up to 6) are used whole; elements are x * 2^-e, an exact product, rounded
// to the nearest E2M1 number.
//
// 8192 x 4096 rows: fp32 quantized in 24.4 us (6.2 TB/s, the rate of a copy), fp16 in 15.7 (5.4 TB/s; the arithmetic, 88
// instructions to eight numbers, fills two thirds of the issue slots), and back to bf16 in 11.4.  Few rows: 2.1 and 1.5 us,
// a launch.  Rows of odd width, by single elements: 16384 x 2001 fp16 24.6 (2002, by pairs: 17.5; 2000: 17.1) and 17.8 (13.6; 11.5).
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

// Rows off 16-byte boundaries, or whose last eight columns are not all there, come in words W of four bytes or two, one to a
// lane, neighbours to neighbouring lanes, and change places in shared memory: loads of a lane's own eight elements would ask
// for as many lines eight times.  (W void: whole rows, 16 bytes to a lane.)
template <typename T, typename W>
struct Words {
  static constexpr int kRow = 128 * sizeof(T) / sizeof(W) / 32, kBoth = 2 * kRow;  // words of a lane: of a row, of the warp's two
  static constexpr int kElements = sizeof(W) / sizeof(T) > 0 ? sizeof(W) / sizeof(T) : 1;
  bool in[kRow];       // the word's column is there
  int rows;            // of the block from the warp's first row on
  __device__ __forceinline__ Words(const TilePlace &at, int64_t cols) {
    const int64_t first = at.col - (threadIdx.x & 15) * 8;
#pragma unroll
    for (int k = 0; k < kRow; k++) in[k] = first + (k * 32 + (int)(threadIdx.x & 31)) * kElements < cols;
    rows = at.rows - (at.first & ~1);
  }
  // the lane's first word of the warp's first row
  template <typename P>
  static __device__ __forceinline__ P *start(P *base, const TilePlace &at, int64_t stride) {
    return base + (at.row0 + (at.first & ~1)) * stride + at.col - (threadIdx.x & 15) * 8 + (threadIdx.x & 31) * kElements;
  }
};
template <typename T>
struct Words<T, void> {
  static constexpr int kBoth = 1;
};

template <typename T, typename W>
__global__ void __launch_bounds__(kThreads) mx_quantize_kernel(const T *__restrict__ in, int64_t rows, int64_t cols, int64_t row_stride,
                                                               unsigned tiles, uint8_t *__restrict__ data, uint8_t *__restrict__ scales) {
  constexpr bool kWhole = std::is_void_v<W>;
  __shared__ __align__(16) uint8_t tile[512];
  __shared__ __align__(16) T staged[kWhole ? 8 : kThreads * 8];
  pdl_wait();
  pdl_launch_dependents();
  const TilePlace at(rows, tiles);
  const int lane = threadIdx.x & 31;
  if (threadIdx.x < 32) reinterpret_cast<uint4 *>(tile)[threadIdx.x] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  const int64_t pitch = 16 * ((cols + 31) / 32);
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
  if constexpr (kWhole) {
    const T *x = in + (at.row0 + at.first) * row_stride + at.col;
    const int64_t left = cols - at.col;
#pragma unroll
    for (int i0 = 0; i0 < 8; i0 += kAtOnce) {
      if (i0 * 16 >= at.rows) break;
      Eight<true, T> v[kAtOnce];
#pragma unroll
      for (int i = 0; i < kAtOnce; i++) v[i].load(x + (int64_t)(i0 + i) * 16 * row_stride, (i0 + i) * 16 + at.first < at.rows ? left : 0);
#pragma unroll
      for (int i = 0; i < kAtOnce; i++)
        if ((i0 + i) * 16 < at.rows) finish(i0 + i, v[i]);
    }
  } else {
    using S = Words<T, W>;
    const S words(at, cols);
    const T *x = S::start(in, at, row_stride);
    W *mine_here = reinterpret_cast<W *>(staged + (threadIdx.x & ~31) * 8);
#pragma unroll
    for (int i0 = 0; i0 < 8; i0 += kAtOnce) {
      if (i0 * 16 >= at.rows) break;
      W w[kAtOnce][S::kBoth];
#pragma unroll
      for (int i = 0; i < kAtOnce; i++) {
#pragma unroll
        for (int k = 0; k < S::kBoth; k++)
          w[i][k] = words.in[k % S::kRow] && (i0 + i) * 16 + k / S::kRow < words.rows
                        ? __ldg(reinterpret_cast<const W *>(x + (k / S::kRow) * row_stride + (k % S::kRow) * 32 * S::kElements))
                        : W(0);
        x += 16 * row_stride;
      }
#pragma unroll
      for (int i = 0; i < kAtOnce; i++)
        if ((i0 + i) * 16 < at.rows) {
          __syncwarp();
#pragma unroll
          for (int k = 0; k < S::kBoth; k++) mine_here[k * 32 + lane] = w[i][k];
          __syncwarp();
          Eight<true, T> v;
#pragma unroll
          for (int k = 0; k < (int)(8 * sizeof(T) / 16); k++)
            reinterpret_cast<uint4 *>(v.w)[k] = reinterpret_cast<const uint4 *>(staged + threadIdx.x * 8)[k];
          finish(i0 + i, v);
        }
    }
  }
  __syncthreads();
  if (threadIdx.x < 32)
    reinterpret_cast<uint4 *>(scales + (size_t)blockIdx.x * 512)[threadIdx.x] = reinterpret_cast<const uint4 *>(tile)[threadIdx.x];
}

template <typename T, typename W>
__global__ void __launch_bounds__(kThreads) mx_dequantize_kernel(const uint8_t *__restrict__ data, const uint8_t *__restrict__ scales, int64_t rows,
                                                                 int64_t cols, unsigned tiles, T *__restrict__ out) {
  constexpr bool kWhole = std::is_void_v<W>;
  __shared__ __align__(16) uint8_t tile[512];
  __shared__ __align__(16) T staged[kWhole ? 8 : kThreads * 8];
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
  const uint8_t *my_scale = tile + at.first * 16 + ((lane & 15) >> 2);
  auto numbers = [&](int i, uint32_t (&w)[2 * sizeof(T)]) {
    const float scale = mx_scale(my_scale[(i & 1) * 256 + (i >> 1) * 4]);
    float v[8];
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const float2 n = mx_numbers((codes[i] >> (8 * k)) & 0xFFu);
      v[2 * k] = n.x * scale;
      v[2 * k + 1] = n.y * scale;
    }
#pragma unroll
    for (int k = 0; k < (int)(2 * sizeof(T)); k++) {
      if constexpr (sizeof(T) == 4) w[k] = __float_as_uint(v[k]);
      else w[k] = pack2(v[2 * k], v[2 * k + 1], T());
    }
  };
  auto put = [](T *to, const uint32_t (&w)[2 * sizeof(T)]) {
#pragma unroll
    for (int k = 0; k < (int)(sizeof(T) / 2); k++)
      reinterpret_cast<uint4 *>(to)[k] = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
  };
  uint32_t w[2 * sizeof(T)];
  if constexpr (kWhole) {
    T *o = out + (at.row0 + at.first) * cols + at.col;
    const int mine = at.col < cols ? at.rows - at.first : 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      if (i * 16 >= at.rows) break;
      numbers(i, w);
      if (i * 16 < mine) put(o, w);
      o += 16 * cols;
    }
  } else {
    using S = Words<T, W>;
    const S words(at, cols);
    T *o = S::start(out, at, cols);
    const W *mine_here = reinterpret_cast<const W *>(staged + (threadIdx.x & ~31) * 8);
#pragma unroll
    for (int i = 0; i < 8; i++) {
      if (i * 16 >= at.rows) break;
      numbers(i, w);
      __syncwarp();
      put(staged + threadIdx.x * 8, w);
      __syncwarp();
#pragma unroll
      for (int k = 0; k < S::kBoth; k++)
        if (words.in[k % S::kRow] && i * 16 + k / S::kRow < words.rows)
          *reinterpret_cast<W *>(o + (k / S::kRow) * cols + (k % S::kRow) * 32 * S::kElements) = mine_here[k * 32 + lane];
      o += 16 * cols;
    }
  }
}

// Calls f with a null pointer of the word that rows `stride` elements of T apart, `cols` of them there, are taken in.
template <typename T, typename F>
int with_word(const void *base, int64_t stride, int64_t cols, F f) {
  if (aligned(base, 16) && stride * sizeof(T) % 16 == 0 && cols % 8 == 0) return f(static_cast<void *>(nullptr));
  if constexpr (sizeof(T) == 2)
    if (!aligned(base, 4) || stride % 2 != 0 || cols % 2 != 0) return f(static_cast<uint16_t *>(nullptr));
  return f(static_cast<uint32_t *>(nullptr));
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
    return with_word<T>(in, row_stride, cols, [&](auto *w) {
      GLOWB200_CUDA_OK(launch_pdl(mx_quantize_kernel<T, std::remove_pointer_t<decltype(w)>>, dim3((unsigned)blocks), kThreads, 0, s,
                                  reinterpret_cast<const T *>(in), rows, cols, row_stride, (unsigned)tiles, data, scales));
      return GLOWB200_OK;
    });
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
  const size_t bytes = (size_t)float_type_bytes(in_type), data_bytes = (size_t)(rows * mx_pitch(cols)), scale_bytes = glowb200_microscaled_fp4_scales_bytes(rows, cols);
  GLOWB200_REQUIRE(apart(data, data_bytes, in, cols * bytes, rows, row_stride * bytes) && apart(scales, scale_bytes, in, cols * bytes, rows, row_stride * bytes) &&
                       apart(data, data_bytes, scales, scale_bytes),
                   "a result lies over the input or the other result");
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
  const size_t out_bytes = (size_t)(rows * cols) * float_type_bytes(out_type);
  GLOWB200_REQUIRE(apart(out, out_bytes, data, (size_t)(rows * mx_pitch(cols))) && apart(out, out_bytes, scales, glowb200_microscaled_fp4_scales_bytes(rows, cols)),
                   "the result lies over the input");
  const int64_t tiles = mx_tiles(cols), blocks = mx_row_tiles(rows) * tiles;
  GLOWB200_REQUIRE(blocks < (1ll << 31), "the matrix has more than 2^31 tiles of 128 x 128");
  return with_float_type(out_type, [&](auto *t) {
    using T = std::remove_pointer_t<decltype(t)>;
    return with_word<T>(out, cols, cols, [&](auto *w) {
      GLOWB200_CUDA_OK(launch_pdl(mx_dequantize_kernel<T, std::remove_pointer_t<decltype(w)>>, dim3((unsigned)blocks), kThreads, 0,
                                  reinterpret_cast<cudaStream_t>(stream), data, scales, rows, cols, (unsigned)tiles, reinterpret_cast<T *>(out)));
      return GLOWB200_OK;
    });
  });
}
