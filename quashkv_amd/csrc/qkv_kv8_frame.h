// How share8 (qkv_kv8_shared.hip) divides a kv head's work: arithmetic on numbers of steps alone,
// which a CPU compiler takes, too.
#pragma once

namespace qkv_kv8 {

// Set-up and end of a tall tile, in its steps (0.8 us at d = 128), and the least that a range
// takes of one; a step of a short tile; places of a kv head's tall tiles, at most.
constexpr int kSetUp = 8, kCut = 2;
constexpr float kShortStep = 0.5f;
constexpr float kMostPlaces = 0x1p30f;

// How a kv head's work is divided: its tall tiles have places, one behind the other, which are cut
// into ranges.  Where tiles are few and long each has whole ranges (aligned); else a tile has
// its steps and `setup` more, so that a range of many short tiles is no longer than one of a
// part of a long one.
struct Frame {
  int32_t range;      // places of a range
  int32_t tall;       // ranges (from frame_of: as many as there may be, see fit_ranges)
  int32_t setup;      // -1: aligned
  int32_t least;      // steps of a part of a short tile
  int32_t fours;      // parts of short tiles
  int32_t lates;      // tiles of the second launch
};

__device__ __forceinline__ int div_up(int a, int b) {
  return static_cast<int>((static_cast<uint32_t>(a) + b - 1) / static_cast<uint32_t>(b));
}
__device__ __forceinline__ int extent(const Frame& F, int steps) {
  return F.setup < 0 ? div_up(steps, F.range) * F.range : steps + F.setup;
}

// steps, tiles, fours: sums over the items of tall tiles' steps, their number, and short tiles'
// steps, in fp32, rounded above 2^24; count(R): of the tall tiles' parts if each were cut into R
// steps by itself.
template <typename Count>
__device__ __forceinline__ Frame frame_of(int target, float per_target, float steps, float tiles,
                                          float fours, Count count) {
  Frame F{1, 0, 0, 0, 0, 0};
  const float few = kShortStep * fours, all = (steps + few) * per_target + kSetUp;
  if (steps > 0.f && steps + kSetUp * tiles < kMostPlaces) {
    int n = target - static_cast<int>(few / all + 0.5f);
    if (few > 0.f && n == target) --n;
    n = max(n, 1);
    const float each = steps / static_cast<float>(n);
    F.setup = static_cast<int>(fminf(0.25f * each, static_cast<float>(kSetUp))) & ~1;
    F.tall = n;
    F.range = max(static_cast<int>((steps + tiles * F.setup) / static_cast<float>(n)) + 1, 4);
    // aligned: the shortest parts, as near as eighths, that are no more than n; then a range has
    // one set-up, where else one that spans tiles has two
    int R = max((static_cast<int>(ceilf(each)) + 1) & ~1, 4), parts = 0;
#pragma unroll 1
    for (int k = 0; k < 8; ++k) {
      if (R > F.range + kSetUp) break;
      parts = count(R);
      if (parts <= n) break;
      R += max(2, (R / 8) & ~1);
    }
    if (parts <= n && R <= F.range + kSetUp) {
      F.range = R;
      F.setup = -1;
    }
  }
  F.least = static_cast<int>(fminf(all, 1e9f)) / kWaves * kWaves + kWaves;
  return F;
}

// The step of a tall tile of `steps` at which a range that ends at place p of it cuts it: not next
// to its ends, and between rounds of two steps.
__device__ __forceinline__ int cut_at(const Frame& F, int steps, int p) {
  if (F.setup < 0) return min(p, steps);
  const int s = p - F.setup;
  return s < kCut ? 0 : steps - s < kCut ? steps : s & ~1;
}
// Of a tile whose places begin at place a of a range: the parts that it is in, and the ranges from
// that one on that have no step of it.
__device__ __forceinline__ int parts_at(const Frame& F, int steps, int a, int& none) {
  none = 0;
  if (F.setup < 0) return div_up(steps, F.range);
  const int E = steps + F.setup, R = F.range, ends = (a + E - 1) / R;
  none = min(ends, (F.setup + kCut - 1 + a) / R);
  return ends + 1 - none - (ends > none && ends * R - a > E - kCut);
}

// Counts the ranges of the tall tiles' places (all extents, exactly) in F, which frame_of made: no
// more than the workgroups that it has for them.  Where the sums that it went by were rounded (above
// 2^24) and its ranges are too short by that, they are made longer.  (Aligned tiles never ask for
// it: their parts were counted exactly, and their extents go by the range.)
__device__ __forceinline__ void fit_ranges(Frame& F, int places) {
  const int most = F.tall;
  F.tall = div_up(places, F.range);
  if (F.tall > most) {
    F.range = div_up(places, most);
    F.tall = div_up(places, F.range);
  }
}

}  // namespace qkv_kv8
