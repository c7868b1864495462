"""How attention over shared prefixes divides its tall tiles among workgroups
(csrc/qkv_kv8_frame.h, built for the CPU): whatever the fp32 sums of a plan come to, there is a
workgroup for each range, and the ranges have each tile's steps once, in as many parts as the
join counts."""

import ctypes
import os
import random
import shutil
import subprocess

import numpy as np
import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "quashkv_amd", "csrc")

# A plan as the kernels make it, from the fp32 sums given; then each workgroup's range as share8
# goes over it.  0: sound; else the place that is not.
SHIM = r"""
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <vector>
#define __device__
#define __forceinline__ inline
using std::max;
using std::min;
namespace qkv_kv8 { constexpr int kWaves = 4; }
#include "qkv_kv8_frame.h"
using namespace qkv_kv8;

extern "C" int check(int target, int n, const int* tiles, const int* steps, float steps_sum,
                     float tiles_sum, float short_sum, int32_t* frame) {
  Frame F = frame_of(target, 1.f / target, steps_sum, tiles_sum, short_sum, [&](int R) {
    int64_t parts = 0;
    for (int i = 0; i < n; ++i) parts += int64_t(tiles[i]) * div_up(steps[i], R);
    return static_cast<int>(min(parts, int64_t(INT32_MAX)));
  });
  const int most = F.tall;
  int64_t total = 0, rows = 0, slots = 0;
  std::vector<int> at(n + 1);
  for (int i = 0; i < n; ++i) {
    at[i] = static_cast<int>(total);
    total += int64_t(tiles[i]) * extent(F, steps[i]);
  }
  if (total >= INT32_MAX) return 1;
  at[n] = static_cast<int>(total);
  fit_ranges(F, at[n]);
  frame[0] = F.range, frame[1] = F.tall, frame[2] = F.setup, frame[3] = most;
  if (F.tall > most || most > target) return 2;
  if (int64_t(target) * F.range >= INT32_MAX || int64_t(F.tall) * F.range < total) return 3;
  // partial rows: an item's tiles have these at most, beyond two a tile 128 rows a range
  for (int i = 0; i < n; ++i) {
    const int64_t k = F.setup < 0 ? div_up(steps[i], F.range)
                      : F.tall < 2 ? 1 : (steps[i] + F.setup - 2) / F.range + 2;
    rows += tiles[i];
    slots += tiles[i] * k;
  }
  if (slots > 2 * rows + target) return 4;
  int item = 0, tile = 0, done = 0, parts = 0;   // of the tile at hand
  for (int j = 0; j < F.tall; ++j)
    for (int x = j * F.range, end = min(x + F.range, at[n]); x < end;) {
      int i = static_cast<int>(std::upper_bound(at.begin(), at.end(), x) - at.begin()) - 1;
      const int E = extent(F, steps[i]), p = (x - at[i]) / E, in = x - at[i] - p * E;
      const int m = min(E - in, end - x);
      const int from = cut_at(F, steps[i], in), to = in + m == E ? steps[i] : cut_at(F, steps[i], in + m);
      if (in == 0) item = i, tile = p, done = parts = 0;
      if (i != item || p != tile) return 5;
      if (from < to) {
        int none;
        const int k = (x - in) / F.range;
        const int of = parts_at(F, steps[i], x - in - k * F.range, none);
        if (from != done || j - k - none != parts || parts >= of) return 6;
        done = to;
        ++parts;
      }
      x += m;
      if (in + m == E) {
        int none;
        if (done != steps[i]) return 7;
        if (parts != parts_at(F, steps[i], (at[i] + p * E) % F.range, none)) return 8;
      }
    }
  return 0;
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("needs g++")
    at = tmp_path_factory.mktemp("frame")
    src, so = at / "frame.cpp", at / "frame.so"
    src.write_text(SHIM)
    subprocess.run([gxx, "-std=c++17", "-O2", "-Wall", "-ffp-contract=off", "-shared", "-fPIC",
                    f"-I{CSRC}", str(src), "-o", str(so)], check=True)
    fn = ctypes.CDLL(str(so)).check
    i32, f32 = ctypes.POINTER(ctypes.c_int32), ctypes.c_float
    fn.argtypes = [ctypes.c_int, ctypes.c_int, i32, i32, f32, f32, f32, i32]
    return fn


def wave_sum(v):
    """Lane 63 of the scan over 64 lanes, fp32 in the order of its steps."""
    v = np.asarray(v, dtype=np.float32).reshape(4, 16).copy()
    for s in (1, 2, 4, 8):
        w = v.copy()
        w[:, s:] = v[:, s:] + v[:, :-s]
        v = w
    r = v[:, 15]
    return (r[3] + r[2]) + (r[1] + r[0])


def sums(items):
    """(steps, tiles) of the plan's fp32 sums, an item a lane, or 16 waves of them and more."""
    n = len(items)
    lanes = max(64, 1024 if n > 64 else 64)
    st, ti = np.zeros(lanes, np.float32), np.zeros(lanes, np.float32)
    for i, (t, s) in enumerate(items):
        st[i % lanes] += np.float32(t) * np.float32(s)
        ti[i % lanes] += np.float32(t)
    waves = [[wave_sum(x[64 * w:64 * w + 64]) for w in range(lanes // 64)] for x in (st, ti)]
    if lanes == 64:
        return waves[0][0], waves[1][0]
    return tuple(wave_sum(w + [0] * 48) for w in waves)


def run(lib, target, items, steps, tiles, short=0.0):
    t = np.array([i[0] for i in items], np.int32)
    s = np.array([i[1] for i in items], np.int32)
    frame = np.zeros(4, np.int32)
    p = lambda a: a.ctypes.data_as(ctypes.POINTER(ctypes.c_int32))
    rc = lib(target, len(items), p(t), p(s), float(steps), float(tiles), float(short), p(frame))
    assert rc == 0, (rc, target, items[:8], frame.tolist(),
                     sum(a * (b + max(int(frame[2]), 0)) for a, b in items))
    return frame


# workgroups of a kv head, and tall tiles and steps of requests whose places' fp32 sum falls short
EXAMPLES = [
    (42, [(458, 30318), (325, 18861), (179, 13111), (302, 24962), (329, 12382)]),
    (51, [(4093, 282), (8565, 4002)]),
    (25, [(7906, 4453), (754, 4401)]),
    (42, [(13395, 7067), (3408, 5005), (6363, 1793), (15099, 922)]),
]


@pytest.mark.parametrize("target,items", EXAMPLES)
def test_sums_above_2_24(lib, target, items):
    run(lib, target, items, *sums(items))
    for off in (2.0 ** -24, 2.0 ** -22, 2.0 ** -20):     # other orders of the additions
        for sign in (-1, 1):
            steps, tiles = sums(items)
            run(lib, target, items, np.float32(steps * (1 + sign * off)), tiles)


@pytest.mark.parametrize("target", [1, 2, 4, 8, 16, 21, 25, 32, 42, 51, 64, 85, 128, 256])
def test_ranges_have_workgroups(lib, target):
    rng = random.Random(target)
    for size in range(8, 30):
        for n in (1, 2, 3, 5, 20, 64, 65, 300, 1500):
            if n << 2 > 1 << size:
                continue
            # items of like and of unlike sizes, of together about 2^size places; tiles as
            # many as rows x query heads below 2^28 make
            each = 2.0 ** size / n
            items = []
            for _ in range(n):
                tiles = int(min(2 ** rng.uniform(0, 13), each / 4, 120000 / n)) + 1
                steps = int(min(max(each * rng.choice([0.3, 1.0, 1.7]) / tiles, 1), 2 ** 25 - 1))
                items.append((tiles, steps))
            if sum(t * (s + 8) for t, s in items) >= 1 << 30:
                continue
            steps, tiles = sums(items)
            short = rng.choice([0.0, 0.0, float(steps) * rng.random(), 4.0])
            run(lib, target, items, steps, tiles, short)
            run(lib, target, items, np.float32(steps * (1 - 2.0 ** -20)), tiles, short)
