"""How group norm's one launch falls into blocks and threads: the host code that decides it, walked on the CPU."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

WALK = r"""
#include <cstdio>
#include <initializer_list>
#include "group_norm_plan.h"
using namespace glowb200;
static long plans, bad;
static void check(int64_t columns, int64_t pixels, NormSingle p, const char *what, long a, long b, long c) {
  if (p.blocks == 0) return;
  plans++;
  const bool right = p.rows >= 1 && columns * p.rows <= kNormThreads && (p.blocks & (p.blocks - 1)) == 0 && p.blocks <= 8 &&
                     p.chunk_pixels == (pixels + p.blocks - 1) / p.blocks && (p.chunk_pixels + p.rows - 1) / p.rows <= kNormHeld;
  if (!right && bad++ < 20)
    printf("%s %ld %ld %ld: %ld columns, %ld pixels, %d blocks of %ld, %d rows, %ld pixels to a thread\n", what, a, b, c, (long)columns,
           (long)pixels, p.blocks, (long)p.chunk_pixels, p.rows, (long)((p.chunk_pixels + p.rows - 1) / p.rows));
}
int main() {
  // every number of pieces a slice can have, and every number of pixels that fits
  for (int64_t columns = 1; columns <= kNormThreads; columns++)
    for (int64_t pixels = 1; pixels <= 8 * (kNormHeld - 1) * (kNormThreads / columns) + 1; pixels++)
      check(columns, pixels, norm_single(columns * 8, 8, pixels), "slice", (long)columns, 0, 0);
  // channels, groups and types, as a call gives them
  for (int64_t groups : {1, 2, 3, 4, 5, 7, 8, 9, 16, 24, 32, 64})
    for (int64_t width = 1; width <= 256; width++)
      for (int bytes : {2, 4})
        for (int vec : {16 / bytes, 4 / bytes, 1}) {
          const int64_t channels = groups * width, slice = channels % vec ? 0 : norm_slice(channels, groups, vec, bytes);
          if (slice == 0) continue;
          if (slice % width || channels % slice || slice % vec) bad++;
          for (int64_t pixels = 1; pixels <= 1300; pixels++)
            check(slice / vec, pixels, norm_single(slice, vec, pixels), "channels, groups, bytes", (long)channels, (long)groups, bytes);
        }
  printf("%ld plans, %ld wrong\n", plans, bad);
  return bad != 0;
}
"""


def test_no_thread_has_more_pixels_than_stay_in_shared_memory(tmp_path):
    """A thread copies 16 pixels at most; one more would be read from shared memory that nobody wrote."""
    src, exe = tmp_path / "walk.cpp", tmp_path / "walk"
    src.write_text(WALK)
    subprocess.run([os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-I", os.path.join(ROOT, "glow_b200", "csrc"), str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
    assert int(r.stdout.split(" plans")[0].split()[-1]) > 100000
