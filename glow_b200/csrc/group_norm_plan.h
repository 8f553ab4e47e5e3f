// How the one launch of a channels-last group norm falls into blocks and threads.  Host code without CUDA, which a test walks.
#pragma once
#include <cstdint>

namespace glowb200 {

constexpr int kNormThreads = 512;
constexpr int kNormHeld = 16;  // pixels of a thread that stay in shared memory

// Channels of a slice of the single launch: the fewest whole groups of 64 bytes or more a pixel.  0: none suits.
inline int64_t norm_slice(int64_t channels, int64_t groups, int vec, int in_bytes) {
  const int64_t width = channels / groups;
  for (int64_t k = 1; k <= groups && width * k / vec <= kNormThreads; k++)
    if (groups % k == 0 && width * k % vec == 0 && (width * k * in_bytes >= 64 || k == groups)) return width * k;
  return 0;
}

// Pixels that a block takes side by side: of 256 threads' pieces; 512 where a pixel has more, 128 where those hold a whole slice
// (64 x 7 x 7 x 2048 17.6 -> 10.2 us, one image of 14 x 14 x 1024 4.2 -> 4.0; in clusters 8 x 28 x 28 x 512 6.0 -> 6.4).
inline int norm_rows(int64_t columns, int64_t pixels) {
  const int64_t rows = (columns <= 64 && columns * pixels <= 128 * (kNormHeld - 1) ? 128 : columns <= 256 ? 256 : kNormThreads) / columns;
  return (int)(rows < pixels ? rows : pixels);
}

// The one launch over a slice: blocks of its cluster (as few as hold the slice's pixels, eight at most; 0: they do not), pixels
// of a block, and those that a block takes side by side: no thread has more than kNormHeld.  Half of a cluster's pixels
// may go into 128 threads where all of them did not; where too many of those stay idle behind the last whole pixel
// (columns that do not divide 128), the block keeps the pixels side by side that the cluster was chosen for.
struct NormSingle {
  int blocks, rows;
  int64_t chunk_pixels;
};
inline NormSingle norm_single(int64_t slice, int vec, int64_t pixels) {
  if (slice <= 0) return {0, 0, 0};
  const int64_t columns = slice / vec;
  const int rows = norm_rows(columns, pixels);
  for (int blocks = 1; blocks <= 8; blocks *= 2)
    if (blocks * (int64_t)rows * (kNormHeld - 1) >= pixels) {
      const int64_t chunk = (pixels + blocks - 1) / blocks;
      const int fewer = norm_rows(columns, chunk);
      return {blocks, fewer * (int64_t)kNormHeld >= chunk ? fewer : rows, chunk};
    }
  return {0, 0, 0};
}
// Whether every type and alignment of such an input takes the one launch, which needs no workspace.
inline bool norm_always_single(int64_t pixels, int64_t channels, int64_t groups) {
  for (int bytes : {2, 4})
    for (int vec : {16 / bytes, 4 / bytes, 1})
      if (channels % vec == 0 && norm_single(norm_slice(channels, groups, vec, bytes), vec, pixels).blocks == 0) return false;
  return true;
}

}  // namespace glowb200
