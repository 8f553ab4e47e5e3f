// Group norm of channels-last activations with the activation behind it.
//
//   y[n, p, c] = act((x[n, p, c] - mean[n, g]) / sqrt(var[n, g] + eps) * gamma[c] + beta[c]),   g = c / (C / G)
//
// mean and var over the C / G channels of the group and all pixels of the image.  Variances come from squares of
// differences from a mean, never from a difference of two large sums: a thread takes a few pixels at a time, with their
// own mean, and what two parts of a group know of themselves (n, mean, M2 = the sum of squared differences) is joined by
//   M2 = M2a + M2b + (mean_b - mean_a)^2 na nb / (na + nb),
// in an order that depends on the sizes alone.
//
// Bound by bytes, or by launches.  Small inputs take one launch: a block has some groups of one image and reads their
// pixels twice, the second time from cache.  Others take two: statistics of chunks of pixels, all channels to a block, then
// a pass that joins them and normalises, from the last chunk to the first: what the first pass read last is still in L2
// (126 MB).
#include <cstdlib>

#include "microscaled.cuh"

namespace glowb200 {
namespace {

constexpr int kNormThreads = 512;

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
  int slices, slice, rows;  // single launch: slices of an image, channels of one; rows: pixels that a block takes side by side
  float eps, quant_scale;
  int32_t quant_offset;
  int act;
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}
// A warp joins parts of one group, of which at(i) gives mean, M2 and, by `n`, the number: all lanes get mean and M2 of the
// whole.  (The mean first, then what the parts' own means differ from it: no quotient but the one.)
template <typename At>
__device__ __forceinline__ float2 join_parts(int count, float total, At at) {
  const int lane = threadIdx.x & 31;
  float sum = 0.0f, squares = 0.0f, n;
  for (int i = lane; i < count; i += 32) {
    const float2 v = at(i, n);
    sum = fmaf(n, v.x, sum);
    squares += v.y;
  }
  const float mean = warp_sum(sum) / total;
  for (int i = lane; i < count; i += 32) {
    const float2 v = at(i, n);
    const float d = v.x - mean;
    squares = fmaf(n * d, d, squares);
  }
  return make_float2(mean, warp_sum(squares));
}

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};
template <typename P>
__device__ __forceinline__ P load_pack(const P *p) {
  P r;
  if constexpr (sizeof(P) == 16) *reinterpret_cast<uint4 *>(&r) = *reinterpret_cast<const uint4 *>(p);
  else if constexpr (sizeof(P) == 8) *reinterpret_cast<uint2 *>(&r) = *reinterpret_cast<const uint2 *>(p);
  else if constexpr (sizeof(P) == 4) *reinterpret_cast<uint32_t *>(&r) = *reinterpret_cast<const uint32_t *>(p);
  else r = *p;
  return r;
}
// (read for the last time)
template <typename P>
__device__ __forceinline__ P load_last(const P *p) {
  P r;
  if constexpr (sizeof(P) == 16) *reinterpret_cast<uint4 *>(&r) = __ldcs(reinterpret_cast<const uint4 *>(p));
  else if constexpr (sizeof(P) == 4) *reinterpret_cast<uint32_t *>(&r) = __ldcs(reinterpret_cast<const uint32_t *>(p));
  else r = load_pack(p);
  return r;
}
// (not read again here)
template <typename P>
__device__ __forceinline__ void store_pack(P *p, const P &r) {
  if constexpr (sizeof(P) == 32) {
    __stcs(reinterpret_cast<uint4 *>(p), reinterpret_cast<const uint4 *>(&r)[0]);
    __stcs(reinterpret_cast<uint4 *>(p) + 1, reinterpret_cast<const uint4 *>(&r)[1]);
  } else if constexpr (sizeof(P) == 16) {
    __stcs(reinterpret_cast<uint4 *>(p), *reinterpret_cast<const uint4 *>(&r));
  } else if constexpr (sizeof(P) == 8) {
    __stcs(reinterpret_cast<uint2 *>(p), *reinterpret_cast<const uint2 *>(&r));
  } else if constexpr (sizeof(P) == 4) {
    __stcs(reinterpret_cast<uint32_t *>(p), *reinterpret_cast<const uint32_t *>(&r));
  } else {
    *p = r;
  }
}

// Statistics of `groups` groups of `width` channels over `pixels` pixels: x is the first of them, in pixels of `channels`
// channels.  Thread t of the first columns * rows has VEC channels (column t % columns) of every rows-th pixel; UNIT: how
// many neighbours of them lie in one group.  Lane 0 of the warp that gets a group calls done(group, {mean, M2}).
template <typename T, int VEC, int UNIT, typename Done>
__device__ __forceinline__ void group_parts(const T *x, int pixels, int channels, int groups, int width, int rows, float2 *shared, Done done) {
  constexpr int kBatch = VEC >= 8 ? 4 : 8, kUnits = VEC / UNIT;
  const int columns = groups * width / VEC, t = threadIdx.x, row = t / columns, column = t - row * columns;
  const int base = pixels / rows, extra = pixels - base * rows;  // row r has base pixels, the first `extra` rows one more
  if (row < rows) {
    float mean[VEC], squares[VEC], n = 0.0f;
#pragma unroll
    for (int k = 0; k < VEC; k++) mean[k] = squares[k] = 0.0f;
    const T *at = x + (int64_t)row * channels + column * VEC;
    const int64_t step = (int64_t)rows * channels;
    int left = base + (row < extra ? 1 : 0);
    auto take = [&](const Pack<T, VEC> *p, auto count_tag) {
      constexpr int kCount = decltype(count_tag)::value;
      const float share = __fdividef((float)kCount, n + (float)kCount), cross = n * share;
#pragma unroll
      for (int k = 0; k < VEC; k++) {
        float v[kCount], m = 0.0f, q = 0.0f;
#pragma unroll
        for (int i = 0; i < kCount; i++) {
          v[i] = to_float(p[i].v[k]);
          m += v[i];
        }
        m *= 1.0f / (float)kCount;
#pragma unroll
        for (int i = 0; i < kCount; i++) {
          const float d = v[i] - m;
          q = fmaf(d, d, q);
        }
        const float d = m - mean[k];
        mean[k] = fmaf(d, share, mean[k]);
        squares[k] += fmaf(d * d, cross, q);
      }
      n += (float)kCount;
    };
    for (; left >= kBatch; left -= kBatch) {
      Pack<T, VEC> p[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; i++) p[i] = load_pack(reinterpret_cast<const Pack<T, VEC> *>(at + i * step));
      at += kBatch * step;
      take(p, std::integral_constant<int, kBatch>());
    }
    {
      Pack<T, VEC> p[kBatch - 1];
#pragma unroll
      for (int i = 0; i < kBatch - 1; i++)
        if (i < left) p[i] = load_pack(reinterpret_cast<const Pack<T, VEC> *>(at + i * step));
#pragma unroll
      for (int i = 0; i < kBatch - 1; i++)
        if (i < left) take(p + i, std::integral_constant<int, 1>());
    }
    // the channels of a unit, n numbers each: M2 = sum of theirs + n * (sum of squared differences of their means)
#pragma unroll
    for (int u = 0; u < kUnits; u++) {
      float m = 0.0f, q = 0.0f, sum = 0.0f;
#pragma unroll
      for (int k = 0; k < UNIT; k++) m += mean[u * UNIT + k];
      m *= 1.0f / (float)UNIT;
#pragma unroll
      for (int k = 0; k < UNIT; k++) {
        const float d = mean[u * UNIT + k] - m;
        sum += squares[u * UNIT + k];
        q = fmaf(d, d, q);
      }
      shared[t * kUnits + u] = make_float2(m, fmaf(n, q, sum));
    }
  }
  __syncthreads();
  const int per_row = columns * kUnits, of_group = width / UNIT, warps = blockDim.x >> 5, lane = t & 31;
  // units of a group, row by row: a lane walks them 32 at a time
  const int first_row = lane / of_group, first_unit = lane - first_row * of_group, more_rows = 32 / of_group, more_units = 32 - more_rows * of_group;
  const float few = (float)base * (float)UNIT, many = (float)(base + 1) * (float)UNIT, total = (float)pixels * (float)width;
  for (int g = t >> 5; g < groups; g += warps) {
    int r = 0, u = 0;
    const float2 part = join_parts(rows * of_group, total, [&](int i, float &n) {
      if (i == lane) {
        r = first_row;
        u = first_unit;
      } else {
        r += more_rows;
        u += more_units;
        if (u >= of_group) {
          u -= of_group;
          r++;
        }
      }
      n = r < extra ? many : few;
      return shared[r * per_row + g * of_group + u];
    });
    if (lane == 0) done(g, part);
  }
}

template <typename Out>
__device__ __forceinline__ Out norm_result(float y, const NormParams &p) {
  if (p.act == GLOWB200_NORM_ACT_RELU) {
    y = y < 0.0f ? 0.0f : y;
  } else if (p.act == GLOWB200_NORM_ACT_SWISH) {
    // (16-bit results: the fast exponential and quotient are off by some 2^-21)
    if constexpr (sizeof(Out) == 2) y = __fdividef(y, 1.0f + __expf(-y));
    else y = y / (1.0f + expf(-y));
  }
  if constexpr (sizeof(Out) == 1) {  // quantization::quantize<int8_t>, as the Quantize node
    const long long v = (long long)rintf(__fadd_rn(__fdiv_rn(y, p.quant_scale), (float)p.quant_offset));
    return (int8_t)(v < -128 ? -128 : (v > 127 ? 127 : v));
  } else {
    return from_float<Out>(y);
  }
}

// Normalises the same pixels; stats: mean and 1 / sqrt(var + eps) of the groups; c0: their first channel.
template <typename T, int VEC, int UNIT, typename Out>
__device__ __forceinline__ void normalise(const NormParams &p, const T *x, Out *y, int pixels, int groups, int width, int c0,
                                          const float2 *stats) {
  constexpr int kBatch = VEC >= 8 ? 4 : 8;
  const int columns = groups * width / VEC, t = threadIdx.x, row = t / columns, column = t - row * columns;
  if (row >= p.rows) return;
  float mean[VEC], gain[VEC], shift[VEC];
#pragma unroll
  for (int u = 0; u < VEC; u += UNIT) {
    const float2 s = stats[(column * VEC + u) / width];
#pragma unroll
    for (int k = u; k < u + UNIT; k++) {
      const int c = c0 + column * VEC + k;
      mean[k] = s.x;
      gain[k] = s.y * (p.gamma ? __ldg(p.gamma + c) : 1.0f);
      shift[k] = p.beta ? __ldg(p.beta + c) : 0.0f;
    }
  }
  int64_t at = (int64_t)row * p.channels + column * VEC;
  int left = row < pixels ? (pixels - row + p.rows - 1) / p.rows : 0;
  const int64_t step = (int64_t)p.rows * p.channels;
  auto one = [&](const Pack<T, VEC> &in, int64_t to) {
    Pack<Out, VEC> out;
#pragma unroll
    for (int k = 0; k < VEC; k++) out.v[k] = norm_result<Out>(fmaf(to_float(in.v[k]) - mean[k], gain[k], shift[k]), p);
    store_pack(reinterpret_cast<Pack<Out, VEC> *>(y + to), out);
  };
  for (; left >= kBatch; left -= kBatch) {
    Pack<T, VEC> in[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; i++) in[i] = load_last(reinterpret_cast<const Pack<T, VEC> *>(x + at + i * step));
#pragma unroll
    for (int i = 0; i < kBatch; i++) one(in[i], at + i * step);
    at += kBatch * step;
  }
  Pack<T, VEC> in[kBatch - 1];
#pragma unroll
  for (int i = 0; i < kBatch - 1; i++)
    if (i < left) in[i] = load_last(reinterpret_cast<const Pack<T, VEC> *>(x + at + i * step));
#pragma unroll
  for (int i = 0; i < kBatch - 1; i++)
    if (i < left) one(in[i], at + i * step);
}

__device__ __forceinline__ float2 to_stats(float2 part, float n, float eps) { return make_float2(part.x, 1.0f / sqrtf(part.y / n + eps)); }
template <typename Out>
__device__ __forceinline__ Out *result(const NormParams &p) {
  if constexpr (sizeof(Out) == 1) return reinterpret_cast<Out *>(p.out_i8);
  else return reinterpret_cast<Out *>(p.out);
}

// A block takes p.slice channels (whole groups) of one image.
template <typename T, int VEC, int UNIT, typename Out>
__global__ void __launch_bounds__(kNormThreads) norm_single_kernel(const NormParams p) {
  extern __shared__ float2 norm_shared[];
  pdl_wait();
  pdl_launch_dependents();
  const int width = p.channels / p.groups, groups = p.slice / width;
  const int64_t n = blockIdx.x / p.slices;
  const int c0 = (int)(blockIdx.x - n * p.slices) * p.slice;
  const T *x = reinterpret_cast<const T *>(p.in) + n * p.pixels * p.channels + c0;
  float2 *stats = norm_shared;
  const float total = (float)p.pixels * (float)width;
  group_parts<T, VEC, UNIT>(x, (int)p.pixels, p.channels, groups, width, p.rows, norm_shared + groups,
                            [&](int g, float2 part) { stats[g] = to_stats(part, total, p.eps); });
  __syncthreads();
  normalise<T, VEC, UNIT, Out>(p, x, result<Out>(p) + n * p.pixels * p.channels + c0, (int)p.pixels, groups, width, c0, stats);
}

// A block takes a chunk of one image's pixels, all channels.
template <typename T, int VEC, int UNIT>
__global__ void __launch_bounds__(kNormThreads) norm_stats_kernel(const NormParams p) {
  extern __shared__ float2 norm_shared[];
  pdl_wait();
  pdl_launch_dependents();
  const int64_t n = blockIdx.x / p.chunks, chunk = blockIdx.x - n * p.chunks, first = chunk * p.chunk_pixels;
  group_parts<T, VEC, UNIT>(reinterpret_cast<const T *>(p.in) + (n * p.pixels + first) * p.channels,
                            (int)min(p.chunk_pixels, p.pixels - first), p.channels, p.groups, p.channels / p.groups, p.rows, norm_shared,
                            [&](int g, float2 part) { p.partial[(n * p.groups + g) * p.chunks + chunk] = part; });
}

template <typename T, int VEC, int UNIT, typename Out>
__global__ void __launch_bounds__(kNormThreads) norm_chunks_kernel(const NormParams p) {
  extern __shared__ float2 norm_shared[];
  pdl_wait();
  pdl_launch_dependents();
  const int64_t block = gridDim.x - 1 - blockIdx.x, n = block / p.chunks, chunk = block - n * p.chunks, first = chunk * p.chunk_pixels;
  const int width = p.channels / p.groups, lane = threadIdx.x & 31;
  const float most = (float)p.chunk_pixels * (float)width, rest = (float)(p.pixels - (p.chunks - 1) * p.chunk_pixels) * (float)width,
              total = (float)p.pixels * (float)width;
  for (int g = threadIdx.x >> 5; g < p.groups; g += blockDim.x >> 5) {
    const float2 *parts = p.partial + (n * p.groups + g) * p.chunks;
    const float2 part = join_parts(p.chunks, total, [&](int i, float &count) {
      count = i + 1 < p.chunks ? most : rest;
      return parts[i];
    });
    if (lane == 0) norm_shared[g] = to_stats(part, total, p.eps);
  }
  __syncthreads();
  const int64_t at = (n * p.pixels + first) * p.channels;
  normalise<T, VEC, UNIT, Out>(p, reinterpret_cast<const T *>(p.in) + at, result<Out>(p) + at, (int)min(p.chunk_pixels, p.pixels - first),
                               p.groups, width, 0, norm_shared);
}

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

// ---- any number of channels: one group to a block, a thread to an element ----
// A block takes a chunk of the pixels of one group of one image.
template <typename T>
__global__ void __launch_bounds__(256) norm_any_parts_kernel(const NormParams p) {
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
__global__ void __launch_bounds__(128) norm_any_join_kernel(const NormParams p) {
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
__global__ void __launch_bounds__(256) norm_any_apply_kernel(const NormParams p) {
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
    result<Out>(p)[i] = norm_result<Out>(y, p);
  }
}

// The kernels of any number of channels: enough blocks to fill the GPU a few times over, a thousand elements or more in each.
int64_t any_chunks(int64_t images, int64_t pixels, int64_t channels, int64_t groups) {
  const int64_t want = (8 * kB200Sms + images * groups - 1) / (images * groups), most = pixels * (channels / groups) / 1024;
  const int64_t chunks = want < most ? want : most;
  return chunks < 1 ? 1 : chunks > pixels ? pixels : chunks;
}
// The two launches: blocks of 16 pixels to a thread or more (of 256 threads, 16 bytes of a pixel each), but as many
// blocks as the GPU runs at once where there are pixels for them.
int64_t image_chunks(int64_t images, int64_t pixels, int64_t channels) {
  const int64_t rows = 2048 / channels > 1 ? 2048 / channels : 1;
  const int64_t least = (4 * kB200Sms + images - 1) / images, by_work = pixels / (16 * rows), most = (pixels + 2 * rows - 1) / (2 * rows);
  int64_t chunks = by_work > least ? by_work : least < most ? least : most;
  return chunks > 256 ? 256 : chunks < 1 ? 1 : chunks;
}

// Elements that a thread takes side by side: as many as 16 bytes hold, or four bytes, or one.
int side_by_side(const void *in, const void *out, int in_bytes, int out_bytes, int64_t channels) {
  for (int vec : {16 / in_bytes, 4 / in_bytes})
    if (vec > 1 && channels % vec == 0 && aligned(in, vec * in_bytes) && aligned(out, vec * out_bytes > 16 ? 16 : vec * out_bytes)) return vec;
  return 1;
}
// Channels of a slice of the single launch: the fewest whole groups of 64 bytes or more a pixel.  0: none suits.
int64_t pick_slice(int64_t channels, int64_t groups, int vec, int in_bytes) {
  const int64_t width = channels / groups;
  for (int64_t k = 1; k <= groups; k++)
    if (groups % k == 0 && width * k % vec == 0 && (width * k * in_bytes >= 64 || k == groups)) return width * k / vec <= kNormThreads ? width * k : 0;
  return 0;
}

// Threads of a block: enough for a pixel's columns; rows of them side by side, no more than there are pixels.
int threads_for(int64_t columns) { return columns <= 128 ? 256 : kNormThreads; }
int rows_for(int64_t columns, int64_t pixels) {
  const int64_t rows = threads_for(columns) / columns;
  return (int)(rows < pixels ? rows : pixels);
}

template <typename T, int VEC, int UNIT, typename Out>
int launch_unit(NormParams p, int64_t slice, cudaStream_t s) {
  const int width = p.channels / p.groups;
  const int64_t columns = (slice > 0 ? slice : p.channels) / VEC;
  p.rows = rows_for(columns, slice > 0 ? p.pixels : p.chunk_pixels);
  const unsigned threads = (unsigned)((columns * p.rows + 31) / 32 * 32);
  const size_t parts = (size_t)(columns * p.rows * (VEC / UNIT)) * sizeof(float2);
  if (slice > 0) {
    p.slice = (int)slice;
    p.slices = (int)(p.channels / slice);
    GLOWB200_CUDA_OK(launch_pdl(norm_single_kernel<T, VEC, UNIT, Out>, dim3((unsigned)(p.images * p.slices)), threads,
                                parts + (size_t)(slice / width) * sizeof(float2), s, p));
    return GLOWB200_OK;
  }
  const dim3 grid((unsigned)(p.images * p.chunks));
  GLOWB200_CUDA_OK(launch_pdl(norm_stats_kernel<T, VEC, UNIT>, grid, threads, parts, s, p));
  GLOWB200_CUDA_OK(launch_pdl(norm_chunks_kernel<T, VEC, UNIT, Out>, grid, threads, (size_t)p.groups * sizeof(float2), s, p));
  return GLOWB200_OK;
}
template <typename T, int VEC, typename Out>
int launch_vec(const NormParams &p, int64_t slice, cudaStream_t s) {
  const int width = p.channels / p.groups;
  if constexpr (VEC == 8)
    if (width % 8 == 0) return launch_unit<T, VEC, 8, Out>(p, slice, s);
  if constexpr (VEC >= 4)
    if (width % 4 == 0) return launch_unit<T, VEC, 4, Out>(p, slice, s);
  if constexpr (VEC >= 2)
    if (width % 2 == 0) return launch_unit<T, VEC, 2, Out>(p, slice, s);
  return launch_unit<T, VEC, 1, Out>(p, slice, s);
}

template <typename T, typename Out>
int launch(NormParams p, cudaStream_t s) {
  const void *out = sizeof(Out) == 1 ? static_cast<const void *>(p.out_i8) : p.out;
  const int vec = side_by_side(p.in, out, sizeof(T), sizeof(Out), p.channels);
  int64_t slice = pick_slice(p.channels, p.groups, vec, sizeof(T));
  const char *e = getenv("GN_MODE");
  const bool single = slice > 0 && (e ? e[0] == 's' : p.pixels * slice * (int64_t)sizeof(T) <= 65536);
  if (single || p.channels / vec <= kNormThreads) {
    const int64_t chunks = image_chunks(p.images, p.pixels, p.channels);
    p.chunk_pixels = (p.pixels + chunks - 1) / chunks;
    p.chunks = (int)((p.pixels + p.chunk_pixels - 1) / p.chunk_pixels);
    if (!single) slice = 0;
    if (vec == 1) return launch_vec<T, 1, Out>(p, slice, s);
    if constexpr (sizeof(T) == 4) return launch_vec<T, 4, Out>(p, slice, s);
    else return vec == 8 ? launch_vec<T, 8, Out>(p, slice, s) : launch_vec<T, 2, Out>(p, slice, s);
  }
  const int64_t chunks = any_chunks(p.images, p.pixels, p.channels, p.groups), blocks = (p.images * p.pixels * p.channels + 255) / 256;
  p.chunk_pixels = (p.pixels + chunks - 1) / chunks;
  p.chunks = (int)((p.pixels + p.chunk_pixels - 1) / p.chunk_pixels);
  GLOWB200_CUDA_OK(launch_pdl(norm_any_parts_kernel<T>, dim3((unsigned)(p.images * p.groups * p.chunks)), 256, 0, s, p));
  GLOWB200_CUDA_OK(launch_pdl(norm_any_join_kernel, dim3((unsigned)((p.images * p.groups + 127) / 128)), 128, 0, s, p));
  const int64_t most = (int64_t)sm_count() * 32;
  GLOWB200_CUDA_OK(launch_pdl(norm_any_apply_kernel<T, Out>, dim3((unsigned)(blocks < most ? blocks : most)), 256, 0, s, p));
  return GLOWB200_OK;
}

}  // namespace
}  // namespace glowb200

using namespace glowb200;

extern "C" size_t glowb200_group_norm_workspace_bytes(int64_t images, int64_t pixels, int64_t channels, int64_t groups) {
  if (images <= 0 || pixels <= 0 || channels <= 0 || groups <= 0) return 0;
  if (channels % groups != 0) return 0;
  const int64_t a = any_chunks(images, pixels, channels, groups), b = image_chunks(images, pixels, channels);
  return align_up((size_t)(images * groups) * 8, 256) + (size_t)(images * groups * (a > b ? a : b)) * 8;
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
  p.eps = eps, p.quant_scale = quant_scale, p.quant_offset = quant_offset, p.act = act;
  GLOWB200_REQUIRE(images * groups * any_chunks(images, pixels, channels, groups) < (1ll << 31) && images * image_chunks(images, pixels, channels) < (1ll << 31),
                   "more than 2^31 groups");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return with_float_type(in_type, [&](auto *t) {
    using T = std::remove_pointer_t<decltype(t)>;
    if (out_i8 != nullptr) return launch<T, int8_t>(p, s);
    return with_float_type(out_type, [&](auto *o) { return launch<T, std::remove_pointer_t<decltype(o)>>(p, s); });
  });
}
