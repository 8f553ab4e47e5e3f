// Group norm of channels-last activations with the activation behind it.
//
//   y[n, p, c] = act((x[n, p, c] - mean[n, g]) / sqrt(var[n, g] + eps) * gamma[c] + beta[c]),   g = c / (C / G)
//
// mean and var over the C / G channels of the group and all pixels of the image.  Variances come from squares of
// differences from a mean, never from a difference of two large sums: a thread takes a few pixels at a time, with their
// own mean (norm_any_*: a block its share of a group, in two passes), and what two parts of a group know of themselves
// (n, mean, M2 = the sum of squared differences) is joined by
//   M2 = M2a + M2b + (mean_b - mean_a)^2 na nb / (na + nb),
// in an order that depends on the sizes and on the tensors' alignment alone.
//
// Three ways, by size:
//   - one launch (norm_single_kernel) where a slice of 64 bytes of every pixel, whole groups, of one image lies in the shared
//     memory of one to eight blocks: they form a cluster, tell one another what they know of the groups, and read their
//     pixels once.  Bound by latency (one image of 14 x 14 x 1024 fp16: 4.0 us) or by issue slots: some 70 instructions to
//     16 bytes and 590 to a warp beside them (64 x 56 x 56 x 256 fp16 48 us, 4.3 TB/s of 205 MB that have to move; its two
//     launches 60).  128 bytes of a pixel take 52 there, 32 bytes 56, twice the blocks 57.
//   - two launches (norm_stats_kernel, norm_chunks_kernel) for larger images: statistics of chunks of whole pixels, then a
//     pass that joins them and normalises, from the last chunk and the last pixels to the first: what the first pass read
//     last is still in L2 (126 MB).  8 x 256 x 256 x 128 fp16 70 us, 24 of them the statistics; Swish adds 5.  Bound by latency
//     rather than by bytes or issue slots: on 4 images the passes move 3.7 and 3.1 TB/s of DRAM with 40 % of the issue slots used.  An SM has two
//     blocks of 256 threads (registers, and the ring's shared memory), which wait for their stages (3.3 and 4.0 of 9.8 cycles to
//     an instruction), and none at all for a quarter of the time, at either end of a launch.
//   - any number of channels a pixel (norm_any_*): three plain launches, an element to a thread at a time, whose 64-bit quotients
//     for places bound them: 8 x 32 x 32 x 8192 fp16 679 us, of which the bytes would take 42.
// An int8 result costs a division and a conversion by 64 bits to an element, as the Quantize node rounds: 64 x 56 x 56 x 256 fp16
// 169 us (float 48), 8 x 256 x 256 x 128 bf16 with Swish 204 (75); quotients of the zeros that Relu leaves are the slowest (247).
#include "group_norm_plan.h"
#include "microscaled.cuh"
#include "tcgen05.cuh"

namespace glowb200 {
namespace {

constexpr int kMostShared = 232448;  // bytes that a block can have: what kernels are allowed, whatever a launch takes (calls may overlap)

struct NormParams {
  const void *in;
  void *out;
  int8_t *out_i8;
  const float *gamma, *beta;
  float2 *partial;  // [images][groups][chunks] mean, M2
  float2 *stats;    // [images][groups] mean, 1 / sqrt(var + eps)
  int32_t *status;
  int64_t images, pixels;
  int channels, groups, chunks;
  int64_t chunk_pixels;
  int slices, slice, rows;  // single launch: slices of an image, channels of one; rows: pixels that a block takes side by side
  int held_at;              // ... where its pixels lie in shared memory
  int width, columns, of_group;  // channels of a group; pieces of a pixel that a block takes; units of a group
  uint32_t by_width, by_columns, by_rows, by_group;  // (for fast_div)
  float eps, quant_scale;
  int32_t quant_offset;
  int act;
};

// Two floats in a register pair, for the two-lane instructions.
struct Two {
  uint64_t v;
  __device__ __forceinline__ Two() {}
  __device__ __forceinline__ Two(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
  __device__ __forceinline__ float2 both() const {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
  }
};
__device__ __forceinline__ Two operator+(Two a, Two b) {
  Two r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two operator*(Two a, Two b) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
// Two 16-bit numbers of a word, widened: fp16 through the mixed-precision add (conversions issue at an eighth of its rate),
// bf16 by its place.
__device__ __forceinline__ Two widen(uint32_t w, __half) {
  float a, b;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tadd.rn.f32.f16 %0, l, %3;\n\tadd.rn.f32.f16 %1, h, %3;\n\t}" : "=f"(a), "=f"(b) : "r"(w), "f"(-0.0f));
  return Two(a, b);
}
__device__ __forceinline__ Two widen(uint32_t w, __nv_bfloat16) { return Two(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)); }

template <int N>
struct Known {  // a number known when compiled, and one that is not (value 0)
  static constexpr int value = N;
  __device__ __forceinline__ constexpr operator int() const { return N; }
};
struct Count {
  static constexpr int value = 0;
  int n;
  __device__ __forceinline__ operator int() const { return n; }
};
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}
// A warp joins parts of one group, of which at(i, n) gives mean and M2 and sets the number: all lanes get mean and M2 of the
// whole.  (The mean first, then what the parts' own means differ from it: no quotient but the one.)  MOST: parts of a
// lane that are asked for before the first is used; more come twice.
template <int MOST, typename At>
__device__ __forceinline__ float2 join_parts(int count, float total, At at) {
  const int lane = threadIdx.x & 31;
  float sum = 0.0f, squares = 0.0f, n[MOST];
  float2 v[MOST];
#pragma unroll
  for (int k = 0; k < MOST; k++) {
    n[k] = 0.0f;
    v[k] = make_float2(0.0f, 0.0f);
    if (lane + 32 * k < count) v[k] = at(lane + 32 * k, n[k]);
  }
#pragma unroll
  for (int k = 0; k < MOST; k++) {
    sum = fmaf(n[k], v[k].x, sum);
    squares += v[k].y;
  }
  for (int i = lane + 32 * MOST; i < count; i += 32) {
    float m;
    const float2 w = at(i, m);
    sum = fmaf(m, w.x, sum);
    squares += w.y;
  }
  const float mean = warp_sum(sum) / total;
#pragma unroll
  for (int k = 0; k < MOST; k++) {
    const float d = v[k].x - mean;
    if (n[k] > 0.0f) squares = fmaf(n[k] * d, d, squares);
  }
  for (int i = lane + 32 * MOST; i < count; i += 32) {
    float m;
    const float2 w = at(i, m);
    const float d = w.x - mean;
    squares = fmaf(m * d, d, squares);
  }
  return make_float2(mean, warp_sum(squares));
}

// VEC neighbours, as they are loaded and stored: words, or one element.
template <typename T, int VEC>
struct Pack {
  static constexpr int kWords = sizeof(T) * VEC / 4 > 0 ? sizeof(T) * VEC / 4 : 1, kTwos = (VEC + 1) / 2;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const T *p) {
    if constexpr (kWords == 4) {
      const uint4 r = *reinterpret_cast<const uint4 *>(p);
      w[0] = r.x, w[1] = r.y, w[2] = r.z, w[3] = r.w;
    } else if constexpr (sizeof(T) * VEC == 4) {
      w[0] = *reinterpret_cast<const uint32_t *>(p);
    } else {
      w[0] = *reinterpret_cast<const uint16_t *>(p);
    }
  }
  __device__ __forceinline__ Two two(int i) const {  // elements 2i and 2i + 1 (of one element: it and 0)
    if constexpr (sizeof(T) == 4) return Two(__uint_as_float(w[VEC > 1 ? 2 * i : 0]), VEC > 1 ? __uint_as_float(w[2 * i + (VEC > 1)]) : 0.0f);
    else return widen(w[i], T());
  }
};
// What follows the normalisation of some numbers.
template <typename Out, int N>
__device__ __forceinline__ void activate(float (&y)[N], int act) {
  if (act == GLOWB200_NORM_ACT_RELU) {
#pragma unroll
    for (int k = 0; k < N; k++) asm("max.NaN.f32 %0, %0, %1;" : "+f"(y[k]) : "f"(0.0f));
  } else if (act == GLOWB200_NORM_ACT_SWISH) {
    if constexpr (sizeof(Out) == 2) {
      // (16-bit results: exponential and reciprocal are approximate, off by some 2^-21 of the result, and the product in front of
      // them is rounded, which is |y| 2^-24 of it: 2^-18 at y = -80.  Both are lost in the rounding to come, 2^-9 or 2^-12.)
#pragma unroll
      for (int k = 0; k < N; k++) {
        float e;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(y[k] * -1.4426950408889634f));
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(1.0f + e));
        y[k] *= e;
      }
    } else {
#pragma unroll
      for (int k = 0; k < N; k++) y[k] = y[k] / (1.0f + expf(-y[k]));
    }
  }
}

// max(x, 0) of two 16-bit numbers, NaN staying NaN
__device__ __forceinline__ uint32_t relu2(uint32_t w, __half) {
  asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(w) : "r"(0u));
  return w;
}
__device__ __forceinline__ uint32_t relu2(uint32_t w, __nv_bfloat16) {
  asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(w) : "r"(0u));
  return w;
}
// (results: not read again here)
template <typename Out, int VEC>
__device__ __forceinline__ void store_results(Out *p, float (&y)[VEC], const NormParams &q, int act) {
  constexpr bool kPairs = sizeof(Out) == 2 && VEC > 1;  // Relu after the rounding, two at a time
  if (act == GLOWB200_NORM_ACT_SWISH || (!kPairs && act == GLOWB200_NORM_ACT_RELU)) activate<Out>(y, act);
  if constexpr (sizeof(Out) == 1) {  // quantization::quantize<int8_t>, as the Quantize node
    uint32_t w[(VEC + 3) / 4] = {};
#pragma unroll
    for (int k = 0; k < VEC; k++) {
      const long long v = (long long)rintf(__fadd_rn(__fdiv_rn(y[k], q.quant_scale), (float)q.quant_offset));
      w[k / 4] |= (uint32_t)(uint8_t)(v < -128 ? -128 : (v > 127 ? 127 : v)) << (8 * (k % 4));
    }
    if constexpr (VEC == 8) *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
    else if constexpr (VEC == 4) *reinterpret_cast<uint32_t *>(p) = w[0];
    else if constexpr (VEC == 2) *reinterpret_cast<uint16_t *>(p) = (uint16_t)w[0];
    else *reinterpret_cast<uint8_t *>(p) = (uint8_t)w[0];
  } else if constexpr (VEC == 1) {
    *p = from_float<Out>(y[0]);
  } else if constexpr (sizeof(Out) == 2) {
    uint32_t w[VEC / 2];
#pragma unroll
    for (int k = 0; k < VEC / 2; k++) w[k] = pack2(y[2 * k], y[2 * k + 1], Out());
    if (act == GLOWB200_NORM_ACT_RELU) {
#pragma unroll
      for (int k = 0; k < VEC / 2; k++) w[k] = relu2(w[k], Out());
    }
    if constexpr (VEC == 8) __stcs(reinterpret_cast<uint4 *>(p), make_uint4(w[0], w[1], w[2], w[3]));
    else if constexpr (VEC == 4) __stcs(reinterpret_cast<uint2 *>(p), make_uint2(w[0], w[1]));
    else *reinterpret_cast<uint32_t *>(p) = w[0];
  } else if constexpr (VEC == 2) {
    *reinterpret_cast<float2 *>(p) = make_float2(y[0], y[1]);
  } else {
#pragma unroll
    for (int k = 0; k < VEC; k += 4) __stcs(reinterpret_cast<float4 *>(p + k), make_float4(y[k], y[k + 1], y[k + 2], y[k + 3]));
  }
}

// Which pixels of a block are this thread's: every rows-th from `row` on, in the column's channels.
struct Place {
  int row, column, base, extra;  // row r has `base` pixels, the first `extra` rows one more
  __device__ __forceinline__ Place(const NormParams &p, int pixels) {
    row = fast_div((int)threadIdx.x, p.columns, p.by_columns);
    column = (int)threadIdx.x - row * p.columns;
    base = fast_div(pixels, p.rows, p.by_rows);
    extra = pixels - base * p.rows;
  }
  __device__ __forceinline__ int pixels(const NormParams &p) const { return row < p.rows ? base + (row < extra ? 1 : 0) : 0; }
};

// A block's pixels by plain loads: calls body(pixels, how many, the first one's place) for those of this thread, `left` from
// `at` on.
template <typename T, int VEC>
struct Loads {
  static constexpr int kBatch = 4;
  const T *at;
  int64_t step;
  int left;
  template <typename Body>
  __device__ __forceinline__ void each(Body body) {
    Pack<T, VEC> p[kBatch];
    for (int first = 0; first < left; first += kBatch) {
#pragma unroll
      for (int i = 0; i < kBatch; i++)
        if (first + i < left) p[i].load(at + i * step);
      at += kBatch * step;
      body(p, min(left - first, kBatch), first);
    }
  }
};

// The same for at most kNormHeld pixels of a thread that stay in shared memory, so that they come from memory once: asynchronous
// copies of 16 bytes, four commit groups of four (each thread reads what it copied itself).
template <typename T, int VEC>
struct Held {
  static constexpr bool kCan = VEC * sizeof(T) == 16;
  static constexpr int kBatch = 4;
  __host__ __device__ static constexpr int bytes(int threads, int pixels) { return threads * 16 * pixels; }  // pixels of a thread, a multiple of 4
  uint32_t place;
  int left;
  bool first;  // still on their way
  __device__ __forceinline__ Held(const Loads<T, VEC> &from, void *shared)
      : place((uint32_t)__cvta_generic_to_shared(shared) + 16 * threadIdx.x), left(from.left), first(true) {
    const T *at = from.at;
#pragma unroll
    for (int g = 0; g < kNormHeld / kBatch; g++) {
#pragma unroll
      for (int i = 0; i < kBatch; i++)
        if (g * kBatch + i < left) {
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(place + (g * kBatch + i) * 16 * blockDim.x), "l"(at) : "memory");
          at += from.step;
        }
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
  }
  template <typename Body>
  __device__ __forceinline__ void each(Body body) const {
    Pack<T, VEC> p[kBatch];
#pragma unroll 1
    for (int at = 0; at < left; at += kBatch) {
      if (first) {
        if (at == 0) asm volatile("cp.async.wait_group 3;" ::: "memory");
        else if (at == kBatch) asm volatile("cp.async.wait_group 2;" ::: "memory");
        else if (at == 2 * kBatch) asm volatile("cp.async.wait_group 1;" ::: "memory");
        else asm volatile("cp.async.wait_group 0;" ::: "memory");
      }
#pragma unroll
      for (int i = 0; i < kBatch; i++)
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(p[i].w[0]), "=r"(p[i].w[1]), "=r"(p[i].w[2]), "=r"(p[i].w[3])
                     : "r"(place + (at + i) * 16 * blockDim.x)
                     : "memory");  // (what is behind the last is old, and not used)
      body(p, min(kBatch, left - at), at);
    }
  }
};

// The same for whole pixels, which lie one behind the other: bulk copies bring eight of every thread at a time into a ring
// in shared memory, ahead of the arithmetic.  Pieces of 16 bytes only.  What bounds these kernels beside the bytes is issue
// slots: few warps with eight pixels at a time pay less of them for waiting and joining than many with four.
constexpr int kStages = 3;
template <typename T, int VEC>
struct Stream {
  static constexpr bool kCan = VEC * sizeof(T) == 16;
  static constexpr int kBatch = 8;
  __host__ __device__ static constexpr int bytes(int threads) { return kCan ? kStages * threads * 16 * kBatch + 128 : 0; }
  const uint8_t *x;
  uint8_t *ring;
  uint64_t *full, *empty;
  volatile int *gave_up;
  int pixels, rows, columns, mine, stages, stage_bytes;  // mine: pixels of this thread
  uint32_t pixel_bytes;
  bool backwards;  // from the last stage to the first

  __device__ __forceinline__ int stage_of(int j) const { return backwards ? stages - 1 - j : j; }
  __device__ __forceinline__ void ask(int j) const {  // (by one thread)
    const int first = stage_of(j) * kBatch * rows, slot = j % kStages;
    const uint32_t size = (uint32_t)min(kBatch * rows, pixels - first) * pixel_bytes;
    mbar_expect_tx(&full[slot], size);
    // The second half of a chunk is to be found in L2 by the second pass, which begins there (8 x 256 x 256 x 128 78 -> 75 us).
    uint64_t policy;
    if (backwards || 2 * first < pixels) asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
    else asm volatile("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(policy));
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;"
                 ::"r"(smem_u32(ring + slot * stage_bytes)), "l"(x + (int64_t)first * pixel_bytes), "r"(size), "r"(smem_u32(&full[slot])), "l"(policy)
                 : "memory");
  }
  // By all threads: barriers, and the first stages on their way.
  __device__ __forceinline__ Stream(const NormParams &p, const T *from, int pixels, const Place &place, void *shared, bool backwards)
      : x(reinterpret_cast<const uint8_t *>(from)), ring(reinterpret_cast<uint8_t *>(shared)), pixels(pixels), rows(p.rows), columns(p.columns),
        mine(place.pixels(p)), stages((place.base + (place.extra ? 1 : 0) + kBatch - 1) / kBatch), stage_bytes(blockDim.x * 16 * kBatch),
        pixel_bytes(p.channels * (uint32_t)sizeof(T)), backwards(backwards) {
    full = reinterpret_cast<uint64_t *>(ring + kStages * stage_bytes);
    empty = full + kStages;
    gave_up = reinterpret_cast<volatile int *>(empty + kStages);
    if (threadIdx.x == 0) {
      for (int s = 0; s < kStages; s++) {
        mbar_init(&full[s], 1);
        mbar_init(&empty[s], blockDim.x >> 5);
      }
      *gave_up = 0;
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
      for (int j = 0; j < kStages && j < stages; j++) ask(j);
    }
    __syncthreads();
  }
  // body(pixels, how many, the first one's place among this thread's)
  template <typename Body>
  __device__ __forceinline__ void each(Body body) {
    const int t = threadIdx.x;
    const uint32_t place = smem_u32(ring) + 16 * t, apart = 16 * rows * columns;
    int slot = 0;
    uint32_t round = 0;
    for (int j = 0; j < stages; j++) {
      if (!__all_sync(0xffffffffu, mbar_wait(&full[slot], round, gave_up))) return;
      const int first = stage_of(j) * kBatch, count = min(kBatch, mine - first);
      Pack<T, VEC> p[kBatch];
      auto read = [&](int i) {
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(p[i].w[0]), "=r"(p[i].w[1]), "=r"(p[i].w[2]), "=r"(p[i].w[3])
                     : "r"(place + slot * stage_bytes + i * apart)
                     : "memory");
      };
      if (count == kBatch) {
#pragma unroll
        for (int i = 0; i < kBatch; i++) read(i);
      } else {
#pragma unroll
        for (int i = 0; i < kBatch; i++)
          if (i < count) read(i);
      }
      __syncwarp();
      if ((t & 31) == 0) mbar_arrive(&empty[slot]);
      // the stage before this one is filled again once every warp has read it
      if (t < 32 && j > 0 && j - 1 + kStages < stages) {
        const int before = slot == 0 ? kStages - 1 : slot - 1;
        if (!__all_sync(0xffffffffu, mbar_wait(&empty[before], slot == 0 ? round ^ 1 : round, gave_up))) return;
        if (t == 0) ask(j - 1 + kStages);
        __syncwarp();
      }
      if (count > 0) body(p, count, first);
      if (++slot == kStages) {
        slot = 0;
        round ^= 1;
      }
    }
  }
  // By all threads, at the end: a wait that gave up is reported, copies on their way get a bounded time to land.
  __device__ __forceinline__ void finish(int32_t *status) const {
    __syncthreads();
    if (*gave_up) {
      if (threadIdx.x == 0 && status != nullptr) atomicOr(status, GLOWB200_STATUS_WAIT_TIMEOUT);
      const long long t0 = clock64();
      while (clock64() - t0 < 4000000ll) {
      }
      __syncthreads();
    }
  }
};

// Statistics of `groups` groups of `width` channels over `pixels` pixels, which `source` hands out.  Thread t of the first columns * rows has VEC channels (column t % columns) of every
// rows-th pixel; UNIT: how many neighbours of them lie in one group.  Lane 0 of the warp that gets a group calls done(group, {mean, M2}).
template <typename T, int VEC, int UNIT, typename Source, typename Done>
__device__ __forceinline__ void group_parts(const NormParams &p, Source source, int pixels, const Place &place, int groups, float2 *shared,
                                            Done done) {
  // A unit's numbers are one sum; units of one channel come two to a register pair.
  constexpr int kBatch = Source::kBatch, kUnits = VEC / UNIT, kTwos = Pack<T, VEC>::kTwos, kSums = UNIT > 1 ? kUnits : kTwos, kEach = UNIT > 1 ? UNIT / 2 : 1;
  const int t = threadIdx.x;
  {
    Two mean[kSums], squares[kSums];  // (UNIT > 1: both halves of a mean are the same, those of M2 are to be added)
    float n = 0.0f;
#pragma unroll
    for (int k = 0; k < kSums; k++) mean[k] = squares[k] = Two(0.0f, 0.0f);
    // `count` of kBatch pixels: their mean, the squares of what they differ from it, and those joined to what was before.
    auto take = [&](const auto &from, auto count) {
      const float many = (float)count, numbers = many * (float)UNIT;
      const float each = decltype(count)::value ? 1.0f / (float)(decltype(count)::value * UNIT) : __fdividef(1.0f, numbers);
      const float share = __fdividef(many, n + many), cross = (UNIT > 1 ? 0.5f : 1.0f) * n * share * (float)UNIT;
      const Two minus_share(-share, -share), crosses(cross, cross);
#pragma unroll
      for (int u = 0; u < kSums; u++) {
        Two x[kBatch][kEach], sum, q;
#pragma unroll
        for (int i = 0; i < kBatch; i++)
          if (i < count) {
#pragma unroll
            for (int k = 0; k < kEach; k++) {
              x[i][k] = from[i].two(u * kEach + k);
              sum = i == 0 && k == 0 ? x[i][k] : sum + x[i][k];
            }
          }
        const float2 halves = sum.both();
        const Two less = UNIT > 1 ? Two(-each * (halves.x + halves.y), -each * (halves.x + halves.y)) : Two(-each * halves.x, -each * halves.y);
#pragma unroll
        for (int i = 0; i < kBatch; i++)
          if (i < count) {
#pragma unroll
            for (int k = 0; k < kEach; k++) {
              const Two d = x[i][k] + less;
              q = i == 0 && k == 0 ? d * d : fma2(d, d, q);
            }
          }
        const Two d = mean[u] + less;
        mean[u] = fma2(d, minus_share, mean[u]);
        squares[u] = squares[u] + fma2(d * d, crosses, q);
      }
      n += many;
    };
    source.each([&](const auto &x, int count, int) {
      if (count == kBatch) take(x, Known<kBatch>());
      else take(x, Count{count});
    });
    if (place.row < p.rows)
#pragma unroll
    for (int u = 0; u < kSums; u++) {
      const float2 m = mean[u].both(), q = squares[u].both();
      if constexpr (UNIT > 1) {
        shared[t * kUnits + u] = make_float2(m.x, q.x + q.y);
      } else {
        shared[t * kUnits + 2 * u] = make_float2(m.x, q.x);
        if (VEC > 1) shared[t * kUnits + 2 * u + (VEC > 1)] = make_float2(m.y, q.y);
      }
    }
  }
  __syncthreads();
  const int per_row = p.columns * kUnits, warps = blockDim.x >> 5, lane = t & 31;
  const float few = (float)place.base * (float)UNIT, many = (float)(place.base + 1) * (float)UNIT, total = (float)pixels * (float)p.width;
  for (int g = t >> 5; g < groups; g += warps) {
    const float2 part = join_parts<4>(p.rows * p.of_group, total, [&](int i, float &n) {  // units of the group, row by row
      const int r = fast_div(i, p.of_group, p.by_group);
      n = r < place.extra ? many : few;
      return shared[r * per_row + g * p.of_group + (i - r * p.of_group)];
    });
    if (lane == 0) done(g, part);
  }
}

// Normalises the same pixels; stats: mean and 1 / sqrt(var + eps) of the groups; c0: their first channel.
template <typename T, int VEC, int UNIT, typename Out, typename Source>
__device__ __forceinline__ void normalise(const NormParams &p, Source source, Out *y, const Place &place, int c0, const float2 *stats) {
  constexpr int kTwos = Pack<T, VEC>::kTwos;
  const int column = place.column;
  // (x - mean) * gain + shift, the difference first: where a group's numbers hardly differ, gains are large
  constexpr int kMeans = UNIT > 1 ? VEC / UNIT : kTwos, kEach = UNIT > 1 ? UNIT / 2 : 1;  // of register pairs
  float less[VEC / UNIT + 1] = {}, gain[2 * kTwos] = {}, shift[2 * kTwos] = {};
  if (place.row < p.rows)
#pragma unroll
  for (int u = 0; u < VEC; u += UNIT) {
    const float2 s = stats[fast_div(column * VEC + u, p.width, p.by_width)];
    less[u / UNIT] = -s.x;
#pragma unroll
    for (int k = u; k < u + UNIT; k++) {
      const int c = c0 + column * VEC + k;
      gain[k] = s.y * (p.gamma ? __ldg(p.gamma + c) : 1.0f);
      shift[k] = p.beta ? __ldg(p.beta + c) : 0.0f;
    }
  }
  Two lesses[kMeans], gains[kTwos], shifts[kTwos];
#pragma unroll
  for (int k = 0; k < kMeans; k++) lesses[k] = UNIT > 1 ? Two(less[k], less[k]) : Two(less[2 * k], less[2 * k + 1 <= VEC ? 2 * k + 1 : 2 * k]);
#pragma unroll
  for (int k = 0; k < kTwos; k++) {
    gains[k] = Two(gain[2 * k], gain[2 * k + 1]);
    shifts[k] = Two(shift[2 * k], shift[2 * k + 1]);
  }
  const int64_t first = (int64_t)place.row * p.channels + column * VEC, step = (int64_t)p.rows * p.channels;
  const int act = p.act;
  source.each([&](const auto &in, int count, int from) {
    Out *to = y + first + from * step;
#pragma unroll
    for (int i = 0; i < Source::kBatch; i++)
      if (i < count) {
        float v[VEC];
#pragma unroll
        for (int k = 0; k < kTwos; k++) {
          const float2 r = fma2(in[i].two(k) + lesses[k / kEach], gains[k], shifts[k]).both();
          v[2 * k] = r.x;
          if (2 * k + 1 < VEC) v[2 * k + (VEC > 1)] = r.y;
        }
        store_results(to + i * step, v, p, act);
      }
  });
}

__device__ __forceinline__ float2 to_stats(float2 part, float n, float eps) { return make_float2(part.x, 1.0f / sqrtf(part.y / n + eps)); }
template <typename Out>
__device__ __forceinline__ Out *result(const NormParams &p) {
  if constexpr (sizeof(Out) == 1) return reinterpret_cast<Out *>(p.out_i8);
  else return reinterpret_cast<Out *>(p.out);
}

// A thread's pixels of a block, by plain loads.
template <typename T, int VEC>
__device__ __forceinline__ Loads<T, VEC> loads_of(const NormParams &p, const T *x, const Place &place) {
  return {x + (int64_t)place.row * p.channels + place.column * VEC, (int64_t)p.rows * p.channels, place.pixels(p)};
}

__device__ __forceinline__ float2 ld_cluster2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}

// A cluster's blocks (one to eight) take p.slice channels (whole groups) of one image, chunk_pixels pixels each, and tell one
// another what they know of the groups.
template <typename T, int VEC, int UNIT, typename Out>
__global__ void __launch_bounds__(kNormThreads) norm_single_kernel(const NormParams p) {
  extern __shared__ __align__(16) float2 norm_shared[];
  pdl_wait();
  pdl_launch_dependents();
  const int width = p.width, groups = fast_div(p.slice, width, p.by_width), warps = blockDim.x >> 5, lane = threadIdx.x & 31;
  const unsigned unit = blockIdx.x / (unsigned)p.chunks, n = unit / (unsigned)p.slices;
  const int64_t first = (int64_t)(blockIdx.x - unit * p.chunks) * p.chunk_pixels;
  const int c0 = (int)(unit - n * p.slices) * p.slice, pixels = (int)max((int64_t)0, min(p.chunk_pixels, p.pixels - first));
  const int64_t at = ((int64_t)n * p.pixels + first) * p.channels + c0;
  const Place place(p, pixels);
  float2 *mine = norm_shared, *stats = mine + groups, *parts = stats + groups;
  const Loads<T, VEC> loads = loads_of<T, VEC>(p, reinterpret_cast<const T *>(p.in) + at, place);
  auto run = [&](auto source) {
    group_parts<T, VEC, UNIT>(p, source, pixels, place, groups, parts, [&](int g, float2 part) { mine[g] = part; });
    __syncthreads();
    if (p.chunks > 1) cluster_sync();
    const float most = (float)p.chunk_pixels * (float)width, total = (float)p.pixels * (float)width;
    for (int g = threadIdx.x >> 5; g < groups; g += warps) {
      const float2 part = join_parts<1>(p.chunks, total, [&](int i, float &count) {
        const int64_t left = p.pixels - i * p.chunk_pixels;
        count = left >= p.chunk_pixels ? most : left > 0 ? (float)left * (float)width : 0.0f;
        if (left <= 0) return make_float2(0.0f, 0.0f);
        return p.chunks > 1 ? ld_cluster2(map_to_cta(&mine[g], (uint32_t)i)) : mine[g];
      });
      if (lane == 0) stats[g] = to_stats(part, total, p.eps);
    }
    __syncthreads();
    if (p.chunks > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // this block has read the others' parts
    if constexpr (Held<T, VEC>::kCan) source.first = false;
    normalise<T, VEC, UNIT, Out>(p, source, result<Out>(p) + at, place, c0, stats);
    __syncwarp();
    if (p.chunks > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // none leaves before it is read
  };
  if constexpr (Held<T, VEC>::kCan) run(Held<T, VEC>(loads, reinterpret_cast<uint8_t *>(norm_shared) + p.held_at));
  else run(loads);
}

// A block takes a chunk of one image's pixels, all channels.
template <typename T, int VEC, int UNIT>
__global__ void __launch_bounds__(kNormThreads) norm_stats_kernel(const NormParams p) {
  extern __shared__ __align__(16) float2 norm_shared[];
  pdl_wait();
  pdl_launch_dependents();
  const int64_t n = blockIdx.x / (unsigned)p.chunks, chunk = blockIdx.x - n * p.chunks, first = chunk * p.chunk_pixels;
  const T *x = reinterpret_cast<const T *>(p.in) + (n * p.pixels + first) * p.channels;
  const int pixels = (int)min(p.chunk_pixels, p.pixels - first);
  const Place place(p, pixels);
  auto done = [&](int g, float2 part) { p.partial[(n * p.groups + g) * p.chunks + chunk] = part; };
  float2 *parts = norm_shared + Stream<T, VEC>::bytes(blockDim.x) / sizeof(float2);
  if constexpr (Stream<T, VEC>::kCan) {
    Stream<T, VEC> stream(p, x, pixels, place, norm_shared, false);
    group_parts<T, VEC, UNIT>(p, stream, pixels, place, p.groups, parts, done);
    stream.finish(p.status);
  } else {
    group_parts<T, VEC, UNIT>(p, loads_of<T, VEC>(p, x, place), pixels, place, p.groups, parts, done);
  }
}

template <typename T, int VEC, int UNIT, typename Out>
__global__ void __launch_bounds__(kNormThreads) norm_chunks_kernel(const NormParams p) {
  extern __shared__ __align__(16) float2 norm_shared[];
  pdl_wait();
  pdl_launch_dependents();
  const unsigned block = gridDim.x - 1 - blockIdx.x;
  const int64_t n = block / (unsigned)p.chunks, chunk = block - n * p.chunks, first = chunk * p.chunk_pixels;
  const int width = p.width, lane = threadIdx.x & 31, pixels = (int)min(p.chunk_pixels, p.pixels - first);
  const int64_t at = (n * p.pixels + first) * p.channels;
  const T *x = reinterpret_cast<const T *>(p.in) + at;
  const Place place(p, pixels);
  float2 *stats = norm_shared + Stream<T, VEC>::bytes(blockDim.x) / sizeof(float2);
  auto join = [&]() {
    const float most = (float)p.chunk_pixels * (float)width, rest = (float)(p.pixels - (p.chunks - 1) * p.chunk_pixels) * (float)width,
                total = (float)p.pixels * (float)width;
    for (int g = threadIdx.x >> 5; g < p.groups; g += blockDim.x >> 5) {
      const float2 *parts = p.partial + (n * p.groups + g) * p.chunks;
      const float2 part = join_parts<10>(p.chunks, total, [&](int i, float &count) {
        count = i + 1 < p.chunks ? most : rest;
        return parts[i];
      });
      if (lane == 0) stats[g] = to_stats(part, total, p.eps);
    }
    __syncthreads();
  };
  if constexpr (Stream<T, VEC>::kCan) {
    Stream<T, VEC> stream(p, x, pixels, place, norm_shared, true);
    join();
    normalise<T, VEC, UNIT, Out>(p, stream, result<Out>(p) + at, place, 0, stats);
    stream.finish(p.status);
  } else {
    join();
    normalise<T, VEC, UNIT, Out>(p, loads_of<T, VEC>(p, x, place), result<Out>(p) + at, place, 0, stats);
  }
}

// ---- any number of channels: one group to a block, a thread to an element ----
__device__ __forceinline__ float block_sum(float v, float *shared) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0f;
  for (int i = 0; i < (int)(blockDim.x >> 5); i++) v += shared[i];
  return v;
}

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
  // What the numbers less `from` and their squares add up to, 64 elements of a thread at a time: a long group is not one long chain.
  auto sums_from = [&](float from) {
    float2 sums = make_float2(0.0f, 0.0f);
    for (int64_t i = threadIdx.x; i < count;) {
      float2 few = make_float2(0.0f, 0.0f);
      for (int k = 0; k < 64 && i < count; k++, i += 256) {
        const float d = to_float(x[i / width * p.channels + i % width]) - from;
        few.x += d;
        few.y += d * d;
      }
      sums.x += few.x;
      sums.y += few.y;
    }
    return make_float2(block_sum(sums.x, shared), block_sum(sums.y, shared));
  };
  // `about` is off by its sum's roundings, the same way in every thread where numbers hardly differ; what the differences from it add
  // up to takes that out of the mean, and out of the squares (which are never fewer than its share).
  const float about = sums_from(0.0f).x / (float)count;
  const float2 sums = sums_from(about);
  const float rest = sums.x / (float)count, share = sums.x * rest, mean = about + rest, squares = sums.y <= share ? 0.0f : sums.y - share;
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
    float y[1] = {fmaf(to_float(reinterpret_cast<const T *>(p.in)[i]) - s.x, s.y * (p.gamma ? p.gamma[c] : 1.0f), p.beta ? p.beta[c] : 0.0f)};
    store_results(result<Out>(p) + i, y, p, p.act);
  }
}

// The kernels of any number of channels: enough blocks to fill the GPU a few times over, a thousand elements or more in each.
int64_t any_chunks(int64_t images, int64_t pixels, int64_t channels, int64_t groups) {
  const int64_t want = (8 * kB200Sms + images * groups - 1) / (images * groups), most = pixels * (channels / groups) / 1024;
  const int64_t chunks = want < most ? want : most;
  return chunks < 1 ? 1 : chunks > pixels ? pixels : chunks;
}
// The two launches: two blocks to an SM at once, in the fewest rounds that leave few SMs idle; what a block does beside its
// pixels takes as long as some twenty pixels to a thread do.
int64_t image_chunks(int64_t images, int64_t pixels, int64_t channels) {
  const int64_t at_once = 2 * kB200Sms, rows = 2048 / channels > 1 ? 2048 / channels : 1, most = (pixels + 8 * rows - 1) / (8 * rows);
  int64_t best = 1;
  float used = 0.0f;
  for (int64_t rounds = 1; rounds <= 4; rounds++) {
    int64_t chunks = at_once * rounds / images;
    chunks = chunks > most ? most : chunks < 1 ? 1 : chunks;
    const float u = (float)(images * chunks) / (float)((images * chunks + at_once - 1) / at_once * at_once);
    if (u > used + 0.04f) {
      best = chunks;
      used = u;
    }
  }
  return best;
}

// Elements that a thread takes side by side: as many as 16 bytes hold, or four bytes, or one.
int side_by_side(const void *in, const void *out, int in_bytes, int out_bytes, int64_t channels) {
  for (int vec : {16 / in_bytes, 4 / in_bytes})
    if (vec > 1 && channels % vec == 0 && aligned(in, vec * in_bytes) && aligned(out, vec * out_bytes > 16 ? 16 : vec * out_bytes)) return vec;
  return 1;
}

template <typename T, int VEC, int UNIT, typename Out>
int launch_unit(NormParams p, int64_t slice, cudaStream_t s) {
  const int width = p.channels / p.groups;
  const int64_t columns = (slice > 0 ? slice : p.channels) / VEC;
  if (slice == 0) p.rows = norm_rows(columns, p.chunk_pixels);
  auto reciprocal = [](int64_t d) { return 0xffffffffu / (uint32_t)d; };
  p.width = width, p.columns = (int)columns, p.of_group = width / UNIT;
  p.by_width = reciprocal(width), p.by_columns = reciprocal(columns), p.by_rows = reciprocal(p.rows), p.by_group = reciprocal(p.of_group);
  const unsigned threads = (unsigned)((columns * p.rows + 31) / 32 * 32);
  const size_t parts = (size_t)(columns * p.rows * (VEC / UNIT)) * sizeof(float2);
  if (slice > 0) {
    p.slice = (int)slice;
    p.slices = (int)(p.channels / slice);
    const size_t own = parts + 2 * (size_t)(slice / width) * sizeof(float2);
    p.held_at = (int)align_up(own, 16);
    const int64_t each = (p.chunk_pixels + p.rows - 1) / p.rows;
    GLOWB200_REQUIRE(each <= kNormHeld, "more pixels to a thread than stay in shared memory");
    const size_t shared = Held<T, VEC>::kCan ? p.held_at + Held<T, VEC>::bytes((int)threads, (int)align_up((size_t)each, 4)) : own;
    auto kernel = norm_single_kernel<T, VEC, UNIT, Out>;
    GLOWB200_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostShared));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(p.images * p.slices * p.chunks));
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = shared;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)p.chunks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    GLOWB200_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, static_cast<const NormParams>(p)));
    return GLOWB200_OK;
  }
  auto run = [&](auto kernel, size_t shared) {
    GLOWB200_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostShared));
    GLOWB200_CUDA_OK(launch_pdl(kernel, dim3((unsigned)(p.images * p.chunks)), threads, shared, s, p));
    return GLOWB200_OK;
  };
  if (int rc = run(norm_stats_kernel<T, VEC, UNIT>, Stream<T, VEC>::bytes((int)threads) + parts)) return rc;
  return run(norm_chunks_kernel<T, VEC, UNIT, Out>, Stream<T, VEC>::bytes((int)threads) + (size_t)p.groups * sizeof(float2));
}
template <typename T, int VEC, typename Out>
int launch_vec(const NormParams &p, int64_t slice, cudaStream_t s) {
  const int width = p.channels / p.groups;
  if constexpr (VEC >= 4)
    if (width % 4 == 0) return launch_unit<T, VEC, 4, Out>(p, slice, s);
  if constexpr (VEC >= 2)
    if (width % 2 == 0) return launch_unit<T, VEC, 2, Out>(p, slice, s);
  return launch_unit<T, VEC, 1, Out>(p, slice, s);
}

template <typename T, typename Out>
int launch_width(const NormParams &p, int vec, int64_t slice, cudaStream_t s) {
  if (vec == 1) return launch_vec<T, 1, Out>(p, slice, s);
  if constexpr (sizeof(T) == 4) return launch_vec<T, 4, Out>(p, slice, s);
  else return vec == 8 ? launch_vec<T, 8, Out>(p, slice, s) : launch_vec<T, 2, Out>(p, slice, s);
}

template <typename T, typename Out>
int launch(NormParams p, cudaStream_t s) {
  const void *out = sizeof(Out) == 1 ? static_cast<const void *>(p.out_i8) : p.out;
  const int vec = side_by_side(p.in, out, sizeof(T), sizeof(Out), p.channels);
  const int64_t slice = norm_slice(p.channels, p.groups, vec, sizeof(T));
  const NormSingle single = norm_single(slice, vec, p.pixels);
  if (single.blocks > 0) {
    p.chunks = single.blocks, p.rows = single.rows, p.chunk_pixels = single.chunk_pixels;
    return launch_width<T, Out>(p, vec, slice, s);
  }
  if (p.channels / vec <= kNormThreads) {
    const int64_t chunks = image_chunks(p.images, p.pixels, p.channels);
    p.chunk_pixels = (p.pixels + chunks - 1) / chunks;
    p.chunks = (int)((p.pixels + p.chunk_pixels - 1) / p.chunk_pixels);
    return launch_width<T, Out>(p, vec, 0, s);
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
  if (channels % groups != 0 || norm_always_single(pixels, channels, groups)) return 0;
  const int64_t a = any_chunks(images, pixels, channels, groups), b = image_chunks(images, pixels, channels);
  return align_up((size_t)(images * groups) * 8, 256) + (size_t)(images * groups * (a > b ? a : b)) * 8;
}

extern "C" int glowb200_group_norm(void *out, int out_type, int8_t *out_i8, float quant_scale, int32_t quant_offset, const void *in, int in_type,
                                   const float *gamma, const float *beta, int64_t images, int64_t pixels, int64_t channels, int64_t groups,
                                   float eps, int act, void *workspace, size_t workspace_bytes, int32_t *status, glowb200_stream_t stream) {
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
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return set_error(GLOWB200_ERR_WORKSPACE_TOO_SMALL, "workspace of %zu bytes given, %zu needed", workspace_bytes, need);
  GLOWB200_REQUIRE(aligned(workspace, 256), "workspace must be 256-byte aligned");
  const void *result = out_i8 != nullptr ? out_i8 : out;
  const int in_bytes = float_type_bytes(in_type), out_bytes = out_i8 != nullptr ? 1 : float_type_bytes(out_type);
  const size_t count = (size_t)(images * pixels * channels);
  GLOWB200_REQUIRE((result == in && in_bytes == out_bytes) || apart(result, count * out_bytes, in, count * in_bytes), "the result lies over a part of the input");
  GLOWB200_REQUIRE((gamma == nullptr || apart(result, count * out_bytes, gamma, (size_t)channels * 4)) &&
                       (beta == nullptr || apart(result, count * out_bytes, beta, (size_t)channels * 4)) &&
                       (need == 0 || (apart(workspace, need, in, count * in_bytes) && apart(workspace, need, result, count * out_bytes) &&
                                      (gamma == nullptr || apart(workspace, need, gamma, (size_t)channels * 4)) &&
                                      (beta == nullptr || apart(workspace, need, beta, (size_t)channels * 4)))),
                   "the result or the workspace lies over another tensor");
  NormParams p{};
  p.in = in, p.out = out, p.out_i8 = out_i8, p.gamma = gamma, p.beta = beta;
  p.stats = reinterpret_cast<float2 *>(workspace);
  p.partial = reinterpret_cast<float2 *>(reinterpret_cast<uint8_t *>(workspace) + align_up((size_t)(images * groups) * 8, 256));
  p.images = images, p.pixels = pixels, p.channels = (int)channels, p.groups = (int)groups;
  p.eps = eps, p.quant_scale = quant_scale, p.quant_offset = quant_offset, p.act = act, p.status = status;
  GLOWB200_REQUIRE(images * groups * any_chunks(images, pixels, channels, groups) < (1ll << 31) && images * image_chunks(images, pixels, channels) < (1ll << 31),
                   "more than 2^31 groups");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return with_float_type(in_type, [&](auto *t) {
    using T = std::remove_pointer_t<decltype(t)>;
    if (out_i8 != nullptr) return launch<T, int8_t>(p, s);
    return with_float_type(out_type, [&](auto *o) { return launch<T, std::remove_pointer_t<decltype(o)>>(p, s); });
  });
}
