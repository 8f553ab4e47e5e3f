// Group norm of channels-last activations with the activation behind it.
//
//   y[n, p, c] = act((x[n, p, c] - mean[n, g]) / sqrt(var[n, g] + eps) * gamma[c] + beta[c]),   g = c / (C / G)
//
// mean and var over the C / G channels of the group and all pixels of the image.  Variances come from squares of
// differences from a mean, never from a difference of two large sums: a chunk of the group is read twice (the second
// time from cache), and chunks are joined by n, mean, M2 (the sum of squared differences) of both:
//   M2 = M2a + M2b + (mean_b - mean_a)^2 na nb / (na + nb).
#include "microscaled.cuh"

namespace glowb200 {
namespace {

struct NormParams {
  const void *in;
  void *out;
  int8_t *out_i8;
  const float *gamma, *beta;
  float2 *partial;  // [images][groups][chunks] mean, M2
  float2 *stats;    // [images][groups] mean, 1 / sqrt(var + eps)
  int64_t images, pixels;
  int channels, groups, chunks;
  int64_t chunk_pixels;
  float eps, quant_scale;
  int32_t quant_offset;
  int act;
};

__device__ __forceinline__ float block_sum(float v, float *shared) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0f;
  for (int i = 0; i < (int)(blockDim.x >> 5); i++) v += shared[i];
  return v;
}

// A block takes a chunk of the pixels of one group of one image.
template <typename T>
__global__ void __launch_bounds__(256) norm_chunk_kernel(const NormParams p) {
  __shared__ float shared[8];
  pdl_wait();
  pdl_launch_dependents();
  const int64_t chunk = blockIdx.x % p.chunks, ng = blockIdx.x / p.chunks, n = ng / p.groups;
  const int g = (int)(ng - n * p.groups), width = p.channels / p.groups;
  const int64_t first = chunk * p.chunk_pixels, last = min(first + p.chunk_pixels, p.pixels), count = (last - first) * width;
  const T *x = reinterpret_cast<const T *>(p.in) + (n * p.pixels + first) * p.channels + g * width;
  float sum = 0.0f;
  for (int64_t i = threadIdx.x; i < count; i += 256) sum += to_float(x[i / width * p.channels + i % width]);
  const float mean = block_sum(sum, shared) / (float)count;
  float squares = 0.0f;
  for (int64_t i = threadIdx.x; i < count; i += 256) {
    const float d = to_float(x[i / width * p.channels + i % width]) - mean;
    squares += d * d;
  }
  squares = block_sum(squares, shared);
  if (threadIdx.x == 0) p.partial[blockIdx.x] = make_float2(mean, squares);
}

// A thread joins the chunks of one group of one image.
__global__ void __launch_bounds__(128) norm_join_kernel(const NormParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int64_t ng = blockIdx.x * 128ll + threadIdx.x;
  if (ng >= p.images * p.groups) return;
  const int width = p.channels / p.groups;
  float count = 0.0f, mean = 0.0f, squares = 0.0f;
  for (int c = 0; c < p.chunks; c++) {
    const float2 part = p.partial[ng * p.chunks + c];
    const float more = (float)((min((c + 1) * p.chunk_pixels, p.pixels) - c * p.chunk_pixels) * width), all = count + more;
    const float d = part.x - mean;
    mean += d * (more / all);
    squares += part.y + d * d * (count * (more / all));
    count = all;
  }
  p.stats[ng] = make_float2(mean, 1.0f / sqrtf(squares / count + p.eps));
}

template <typename T, typename Out>
__global__ void __launch_bounds__(256) norm_apply_kernel(const NormParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int64_t total = p.images * p.pixels * p.channels, image = p.pixels * p.channels;
  const int width = p.channels / p.groups;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const int64_t n = i / image;
    const int c = (int)(i % p.channels);
    const float2 s = p.stats[n * p.groups + c / width];
    float y = (to_float(reinterpret_cast<const T *>(p.in)[i]) - s.x) * s.y;
    y = y * (p.gamma ? p.gamma[c] : 1.0f) + (p.beta ? p.beta[c] : 0.0f);
    if (p.act == GLOWB200_NORM_ACT_RELU) y = y < 0.0f ? 0.0f : y;
    else if (p.act == GLOWB200_NORM_ACT_SWISH) y = y / (1.0f + expf(-y));
    if constexpr (sizeof(Out) == 1) {  // quantization::quantize<int8_t>, as the Quantize node
      const long long v = (long long)rintf(__fadd_rn(__fdiv_rn(y, p.quant_scale), (float)p.quant_offset));
      p.out_i8[i] = (int8_t)(v < -128 ? -128 : (v > 127 ? 127 : v));
    } else {
      reinterpret_cast<Out *>(p.out)[i] = from_float<Out>(y);
    }
  }
}

// Chunks of an image's pixels: enough blocks to fill the GPU a few times over, a thousand elements or more in each.
int64_t chunk_count(int64_t images, int64_t pixels, int64_t channels, int64_t groups) {
  const int64_t want = (8 * kB200Sms + images * groups - 1) / (images * groups), most = pixels * (channels / groups) / 1024;
  const int64_t chunks = want < most ? want : most;
  return chunks < 1 ? 1 : chunks > pixels ? pixels : chunks;
}

}  // namespace
}  // namespace glowb200

using namespace glowb200;

extern "C" size_t glowb200_group_norm_workspace_bytes(int64_t images, int64_t pixels, int64_t channels, int64_t groups) {
  if (images <= 0 || pixels <= 0 || channels <= 0 || groups <= 0) return 0;
  return align_up((size_t)(images * groups) * 8, 256) + (size_t)(images * groups * chunk_count(images, pixels, channels, groups)) * 8;
}

extern "C" int glowb200_group_norm(void *out, int out_type, int8_t *out_i8, float quant_scale, int32_t quant_offset, const void *in, int in_type,
                                   const float *gamma, const float *beta, int64_t images, int64_t pixels, int64_t channels, int64_t groups,
                                   float eps, int act, void *workspace, size_t workspace_bytes, glowb200_stream_t stream) {
  GLOWB200_REQUIRE(images >= 0 && pixels >= 0 && channels > 0 && groups > 0 && images < (1ll << 31) && pixels < (1ll << 31) &&
                       channels < (1ll << 31) && images * groups < (1ll << 31),
                   "dimensions out of range");
  GLOWB200_REQUIRE(channels % groups == 0, "%lld channels do not fall into %lld equal groups", (long long)channels, (long long)groups);
  GLOWB200_REQUIRE(in_type >= 0 && in_type <= 2 && (out_i8 != nullptr || (out_type >= 0 && out_type <= 2)),
                   "a float type is not GLOWB200_FLOAT32, _FLOAT16 or _BFLOAT16");
  GLOWB200_REQUIRE(act >= GLOWB200_NORM_ACT_NONE && act <= GLOWB200_NORM_ACT_SWISH, "activation %d is none of GLOWB200_NORM_ACT_*", act);
  GLOWB200_REQUIRE(eps >= 0.0f, "eps must not be negative");
  if (images == 0 || pixels == 0) return GLOWB200_OK;
  GLOWB200_REQUIRE(in && (out != nullptr) != (out_i8 != nullptr), "NULL tensor pointer, or both results are given");
  GLOWB200_REQUIRE(aligned(in, float_type_bytes(in_type)) && (out_i8 != nullptr || aligned(out, float_type_bytes(out_type))),
                   "a tensor is not aligned to its elements");
  const size_t need = glowb200_group_norm_workspace_bytes(images, pixels, channels, groups);
  if (workspace == nullptr || workspace_bytes < need)
    return set_error(GLOWB200_ERR_WORKSPACE_TOO_SMALL, "workspace of %zu bytes given, %zu needed", workspace_bytes, need);
  GLOWB200_REQUIRE(aligned(workspace, 256), "workspace must be 256-byte aligned");
  NormParams p{};
  p.in = in, p.out = out, p.out_i8 = out_i8, p.gamma = gamma, p.beta = beta;
  p.stats = reinterpret_cast<float2 *>(workspace);
  p.partial = reinterpret_cast<float2 *>(reinterpret_cast<uint8_t *>(workspace) + align_up((size_t)(images * groups) * 8, 256));
  p.images = images, p.pixels = pixels, p.channels = (int)channels, p.groups = (int)groups;
  const int64_t chunks = chunk_count(images, pixels, channels, groups);
  p.chunk_pixels = (pixels + chunks - 1) / chunks;
  p.chunks = (int)((pixels + p.chunk_pixels - 1) / p.chunk_pixels);
  p.eps = eps, p.quant_scale = quant_scale, p.quant_offset = quant_offset, p.act = act;
  GLOWB200_REQUIRE(images * groups * p.chunks < (1ll << 31), "more than 2^31 groups");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return with_float_type(in_type, [&](auto *t) {
    using T = std::remove_pointer_t<decltype(t)>;
    GLOWB200_CUDA_OK(launch_pdl(norm_chunk_kernel<T>, dim3((unsigned)(images * groups * p.chunks)), 256, 0, s, p));
    GLOWB200_CUDA_OK(launch_pdl(norm_join_kernel, dim3((unsigned)((images * groups + 127) / 128)), 128, 0, s, p));
    const int64_t blocks = (images * pixels * channels + 255) / 256, most = (int64_t)sm_count() * 32;
    const dim3 grid((unsigned)(blocks < most ? blocks : most));
    if (out_i8 != nullptr) {
      GLOWB200_CUDA_OK(launch_pdl(norm_apply_kernel<T, int8_t>, grid, 256, 0, s, p));
      return GLOWB200_OK;
    }
    return with_float_type(out_type, [&](auto *o) {
      GLOWB200_CUDA_OK(launch_pdl(norm_apply_kernel<T, std::remove_pointer_t<decltype(o)>>, grid, 256, 0, s, p));
      return GLOWB200_OK;
    });
  });
}
