// Attention over the 8-bit paged cache (qkv_kv8.h) of a batch in groups whose requests share
// a prefix (C ABI: qkv_kv8_attention_shared): the prefix is read once for all rows of a group.
//
// Mathematics: decode8's (qkv_kv8_decode.h), whose partial results over parts of a row's tokens
// -- maximum m, sum l, values o, all relative to 2^m -- join as
//   M = max m_i,  out = sum 2^(m_i - M) o_i / sum 2^(m_i - M) l_i.
// So the rows of a group, one behind the other as its requests are, are one set of rows over the
// prefix' tokens, without a mask, and each request's rows are a set over its own tokens.
//
// A request takes part in its group's prefix if its queries all see it; the prefix is read
// from the first of these.  The others, and those of groups for which sharing does not pay (see
// pays), go over all of their tokens by themselves.
//
// Work.  Three kinds of such sets (items): of more than 32 rows, in tall tiles of 128
// (prefill_piece); of fewer, in tiles of 16 (decode_piece); and, of these, requests' own few
// tokens.  The first launch (share8) has the first two, on a workgroup of 8 waves per CU, each of
// which knows its part from the lengths alone: the tall tiles' steps, tile behind tile, are cut
// into equal ranges, one a workgroup, so that all end together wherever tiles end (1131 rows,
// 7 query heads a kv head, over 250 steps: 124 tiles on 256 CUs), and the other workgroups take
// the short tiles, two at a time, four waves each, cut where they are long.  The second launch
// (share_rest) takes the few own tokens, joining them with the prefix' partial results as it
// goes, and joins whatever else was cut.
//
// Measured (a call; attention_kv8 over the same tables): 60 rows of requests of up to 500 own tokens
// behind 8192, 32 / 8 heads, d = 128, bf16: 41 us (95); behind 32,000 78 (340); 56 rows of six
// groups, up to 5003 + 700, 24 / 8 heads, d = 96, e4m3: 28 (45); seven requests' 1131 rows behind
// 16,001, 14 / 2 heads, d = 64, fp32 results: 139 (240), bf16 124 (209); 256 requests of up to 300
// behind 8192: 95 (353).
// Of the first's 41: the plan 3.6 us (loads of the lengths, then some 1000 instructions of one
// wave), a tile's place, queries and first codes 4.5, four rounds of 128 tokens 13 (prefill8's
// loop, see there; 10.3 with weights of 11 bits), halves' join and 16.8 MB of partial results 3.1, a
// gap of 3 between the launches, and the second one 8 (13 the longest): own tokens' chain of
// lengths - page - codes - results.
// Many tall tiles are bound by that loop's issue: of the 1131 rows' 133 us the SIMDs spend
// 53 % on VALU work and 27 % on products (pairs of weights: 98 GFLOP).  Two workgroups a CU, which
// d = 64 has LDS for, are slower (155 us: 45 registers spilled, and twice the partial results).
//
// Tried: the plan in a launch of its own (9 us, and a gap) with short tiles in the first launch
// (a tile by one wave: 8 us each, one behind the other; 47 us in all); ranges that do not count
// set-up (a range of 33 tiles of 5 steps: 272 us for the 140 above); in the second launch a word of
// each line of a step's codes loaded a step before them (39.4 -> 40.5, six groups 29.1 -> 29.6).
#include <algorithm>
#include <atomic>

#include "qkv_kv8_decode.h"
#include "qkv_kv8_frame.h"
#include "qkv_kv8_prefill.h"
#include "qkv_pages_dev.h"

namespace {

using namespace qkv_kv8;

constexpr int kFew = 32;        // rows of an item up to which its tiles have 16 rows, else 128
constexpr int kLate = 16;       // own steps of few rows that are left to the second launch
constexpr int kMaxGroups = 2048;
constexpr int kSmall = 64;      // requests, and groups, up to which every workgroup plans for itself
constexpr int kItems = 2 * kSmall;

// Rows of a request, or of a group, over steps [s0, s0 + steps) of request `table`'s tokens.
struct Item {
  int32_t q0, ql, kv, s0, steps;
  int32_t rows;       // ql x query heads of a kv head, within the buffer; 0: nothing to do
  int32_t table;
  bool group;
  bool part;          // whether its rows have other items, too
  bool pairs;         // whether some of its requests have weights of 22 bits (share8)
  __device__ __forceinline__ bool tall() const { return rows > kFew; }
  __device__ __forceinline__ bool late() const {
    return !group && rows > 0 && !tall() && steps <= kLate;
  }
  __device__ __forceinline__ bool four() const { return rows > 0 && !tall() && !late(); }
  __device__ __forceinline__ int tiles() const {
    return tall() ? (rows + kPreRows - 1) / kPreRows : (rows + kRows - 1) / kRows;
  }
};

// Where items lie: for N items (groups, then requests) the sums before each, and what pieces need.
// In LDS (every workgroup's own) or in the workspace (share_plan's).
struct Places {
  int32_t* tall;      // [N + 1] places of tall tiles
  int32_t* fours;     // [N + 1] parts
  int4* geo;          // two each: q0, ql (0: nothing to do), kv, s0; steps, 4 table + 2 pairs +
                      // causal, slot, rows
};

struct Share {
  const int32_t* group_start;
  const int32_t* prefix_lens;
  int32_t groups;
  int32_t always;     // groups of two members share, whatever that costs
  int32_t small;      // whether workgroups plan for themselves
  Frame* frame;       // the plan, for the second launch and, not small, for the first
  Places at;          // not small
  int4* meta;         // three a request: its own item as the join needs it (join_of) and its
                      // group's; first rows of both, -, ql
  int4* lates;        // three a tile of the second launch: its group's item; request, tile, first
                      // row, ql; kv, s0, rows, rows of the group before
  int32_t late_cap;   // tiles that it holds
  int32_t* row_req;   // not small: a row's request, -1: none
};

__device__ __forceinline__ int steps_of(int kv) { return (kv + kStep - 1) / kStep; }
__device__ __forceinline__ int rows_of(const Att& A, const Req& r) { return r.q0 < 0 ? 0 : r.rows(A); }
// whole steps of a group's prefix
__device__ __forceinline__ int prefix_of(const Share& S, int g) {
  return max(S.prefix_lens[g], 0) & ~(kStep - 1);
}
// Whether all of a request's queries see the prefix: its first one does.
__device__ __forceinline__ bool takes_part(const Att& A, const Req& r, int prefix) {
  const int64_t sees = int64_t(r.kv) - (A.causal ? r.ql - 1 : 0);
  return prefix > 0 && rows_of(A, r) > 0 && sees >= prefix;
}
// Twice what a step of an item of so many rows costs, in steps of a tall tile.
__device__ __forceinline__ int cost_of(int rows) {
  return rows > kFew ? 2 * ((rows + kPreRows - 1) / kPreRows) : (rows + kRows - 1) / kRows;
}
// Whether a group shares its prefix of `steps`: if its rows in one cost less than its requests'
// each (`alone`, summed), by more than what the partial results of the prefix cost: the join, and
// each tile's set-up once more.  Requests of whole tall tiles never do: 16 x 64 rows, 4 query heads a
// kv head, over 8000 tokens: 229 us shared, 157 alone.
__device__ __forceinline__ bool pays(const Share& S, int members, int alone, int rows, int steps) {
  return members > 1 && (S.always || int64_t(alone) * steps > int64_t(cost_of(rows)) * (steps + 2 * kSetUp));
}
__device__ __forceinline__ Item no_item() { return Item{0, 0, 0, 0, 0, 0, 0, false, false, false}; }
__device__ __forceinline__ Item own_item(const Att& A, const Req& r, int b, int prefix) {
  const int s0 = prefix / kStep, rows = rows_of(A, r) * A.G;
  return Item{r.q0, r.ql, r.kv, s0, max(1, steps_of(r.kv) - s0), rows, b, false, prefix > 0, false};
}
__device__ __forceinline__ Item group_item(const Att& A, int prefix, int lead, int row0, int row1,
                                           bool pairs) {
  const int ql = max(row1 - row0, 0);
  return Item{row0, ql, prefix, 0, prefix / kStep, ql * A.G, lead, true, true, pairs};
}

// Parts that an item's tile is cut into at most, and its partial rows.
__device__ __forceinline__ int most_parts(const Item& it, const Frame& F) {
  if (it.late()) return 1;
  if (it.four()) return div_up(it.steps, F.least);
  if (F.setup < 0) return div_up(it.steps, F.range);
  return F.tall < 2 ? 1 : (it.steps + F.setup - 2) / F.range + 2;
}
__device__ __forceinline__ int64_t slots_of(const Item& it, const Frame& F) {
  if (it.rows == 0 || it.late()) return 0;
  const int n = most_parts(it, F);
  return it.part || n > 1 ? int64_t(it.rows) * n : 0;
}

// The tiles of an item in the order of its places: from both ends in turn, so that of a causal
// request's tiles any few neighbours have the same work.
__device__ __forceinline__ int tile_at(int p, int n) { return p & 1 ? n - 1 - p / 2 : p / 2; }
__device__ __forceinline__ int place_of(int t, int n) {
  return t < (n + 1) / 2 ? 2 * t : 2 * (n - 1 - t) + 1;
}

// What the join needs of an item: its first partial row, rows (0: nothing to join), and for tall
// tiles their steps and the first one's place in its range; else 0 and the parts.
__device__ __forceinline__ int4 join_of(const Item& it, const Frame& F, int64_t slots, int64_t slot,
                                        int at) {
  if (slots == 0) return make_int4(0, 0, 0, 0);
  return it.tall() ? make_int4(static_cast<int>(slot), it.rows, it.steps, at % F.range)
                   : make_int4(static_cast<int>(slot), it.rows, 0, most_parts(it, F));
}
// Parts of the tile of row rr of a joined item.
__device__ __forceinline__ int parts_of(const int4& j, const Frame& F, int rr) {
  if (rr < 0 || rr >= j.y) return 0;  // (lengths that do not fit q_start)
  if (j.z == 0) return j.w;
  int none, a = 0;
  if (F.setup >= 0) {
    const int n = div_up(j.y, kPreRows);
    a = (j.w + place_of(rr / kPreRows, n) * (j.z + F.setup)) % F.range;
  }
  return parts_at(F, j.z, a, none);
}

__device__ __forceinline__ void put_item(const Places& P, int i, const Item& it, bool causal,
                                         int tall, int fours, int64_t slot, int64_t slots,
                                         bool fits) {
  P.tall[i] = tall;
  P.fours[i] = fours;
  P.geo[2 * i] = make_int4(it.q0, fits ? it.ql : 0, it.kv, it.s0);
  P.geo[2 * i + 1] = make_int4(it.steps, 4 * it.table + 2 * it.pairs + causal,
                               slots > 0 ? static_cast<int>(slot) : -1, it.rows);
}
// What the second launch needs of request b: own, group: its items' joins; q0: the group's first
// row; late: its tiles of that launch before.
__device__ __forceinline__ void put_request(const Att& A, const Share& S, int b, const Item& it,
                                            const int4& own, const int4& group, int q0, int late) {
  S.meta[3 * b] = own;
  S.meta[3 * b + 1] = group;
  S.meta[3 * b + 2] = make_int4(it.q0, q0, 0, it.ql);
  // (lengths that do not fit q_start may ask for more tiles than there are)
  for (int t = 0; it.late() && t < it.tiles() && late + t < S.late_cap; ++t) {
    int4* const to = S.lates + 3 * (late + t);
    to[0] = group;
    to[1] = make_int4(b, t, it.q0, it.ql);
    to[2] = make_int4(it.kv, it.s0, it.rows, (it.q0 - q0) * A.G);
  }
}

// Inclusive sum over a wave's lanes.
__device__ __forceinline__ int64_t scan64(int64_t v) {
  using qkv_pages::dpp;
  v += dpp<0x111, 0xf>(v);  // row_shr 1, 2, 4, 8
  v += dpp<0x112, 0xf>(v);
  v += dpp<0x114, 0xf>(v);
  v += dpp<0x118, 0xf>(v);
  v += dpp<0x142, 0xa>(v);  // row_bcast 15, 31
  v += dpp<0x143, 0xc>(v);
  return v;
}

__device__ __forceinline__ uint64_t bits_below(int n) {
  return n >= 64 ? ~uint64_t(0) : (uint64_t(1) << n) - 1;
}
// Inclusive maximum over a wave's lanes.
__device__ __forceinline__ int max_scan(int v) {
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x111, 0xf, 0xf, false));  // as wave_scan
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x112, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x114, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x118, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x142, 0xa, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x143, 0xc, 0xf, false));
  return v;
}

// The plan of up to 64 requests and groups by one wave, a lane each; to LDS, and what the second
// launch needs to the workspace where `tell`.
__device__ __forceinline__ Frame plan_wave(const Att& A, const Share& S, const Places& P, bool tell) {
  const int lane = threadIdx.x & 63;
  int start = 0, end = 0, prefix = 0;
  if (lane < S.groups) {
    start = S.group_start[lane];
    end = S.group_start[lane + 1];
    prefix = prefix_of(S, lane);
  }
  Req r{0, 0, 0};
  if (lane < A.B) r = request(A, lane);
  const int rows = lane < A.B ? rows_of(A, r) : 0;
  // A lane is a group and a request.  Its request's group is the last one that begins at it or
  // before; all of a group's lanes, as bits, are its range's part of those that take part.
  // (One group at a time: 0.4 us each.)
  int* const at = P.tall;
  at[lane] = -1;
  __builtin_amdgcn_wave_barrier();
  if (start >= 0 && start < min(end, kSmall)) at[start] = lane;
  __builtin_amdgcn_wave_barrier();
  const int named = max_scan(at[lane]), of = max(named, 0);
  const int theirs_end = __shfl(end, of, 64), theirs_prefix = __shfl(prefix, of, 64);
  const bool in = named >= 0 && lane < theirs_end && lane < A.B && takes_part(A, r, theirs_prefix);
  const int lo = min(max(start, 0), kSmall), hi = min(max(end, lo), kSmall);
  const uint64_t mine = __ballot(in) & (bits_below(hi) & ~bits_below(lo));
  const int first = mine ? __builtin_ctzll(mine) : 0, last = mine ? 63 - __builtin_clzll(mine) : 0;
  const int cost = in ? cost_of(rows * A.G) : 0, costs = wave_scan(cost);
  const int row0 = __shfl(r.q0, first, 64), row1 = __shfl(r.q0 + rows, last, 64);
  const int alone = __shfl(costs, last, 64) - __shfl(costs - cost, first, 64);
  const bool pairs = (__ballot(rows * A.G <= kFew) & mine) != 0;
  // the lane's group, its request
  Item it[2] = {group_item(A, prefix, first, row0, row1, pairs), no_item()};
  const bool does = mine != 0 && pays(S, __popcll(mine), alone, it[0].rows, it[0].steps);
  if (!does) it[0] = no_item();
  const uint64_t sharing = __ballot(does);
  const int group = in && (sharing >> of & 1) ? of : -1;
  const int shares = group < 0 ? 0 : theirs_prefix;
  if (lane < A.B) it[1] = own_item(A, r, lane, shares);
  // sums over all items; and over those before the lane's, groups first
  auto total = [&](auto f) { return lane_value(wave_scan(f(it[0]) + f(it[1])), 63); };
  auto before = [&](auto f, int* to) {
    const int v = f(it[0]), w = f(it[1]);
    const int a = wave_scan(v), b = wave_scan(w) + lane_value(a, 63);
    to[0] = a - v;
    to[1] = b - w;
    return lane_value(b, 63);
  };
  auto steps_as = [](const Item& x, bool on) {
    return on ? static_cast<float>(x.tiles()) * static_cast<float>(x.steps) : 0.f;
  };
  Frame F = frame_of(
      A.target, A.per_target, total([&](const Item& x) { return steps_as(x, x.tall()); }),
      total([](const Item& x) { return x.tall() ? static_cast<float>(x.tiles()) : 0.f; }),
      total([&](const Item& x) { return steps_as(x, x.four()); }),
      [&](int R) {
        return total([&](const Item& x) { return x.tall() ? x.tiles() * div_up(x.steps, R) : 0; });
      });
  int tall[2] = {0, 0}, fours[2] = {0, 0}, late[2], tall_all = 0;
  if (F.range > 1) {
    tall_all = before([&](const Item& x) {
      return x.tall() ? x.tiles() * extent(F, x.steps) : 0;
    }, tall);
    fit_ranges(F, tall_all);
  }
  if (__any(it[0].four() || it[1].four()))
    F.fours = before([&](const Item& x) { return x.four() ? x.tiles() * most_parts(x, F) : 0; },
                     fours);
  F.lates = min(before([](const Item& x) { return x.late() ? x.tiles() : 0; }, late), S.late_cap);
  // (lengths that do not fit q_start may ask for more rows than there are: such sums, modulo 2^32,
  // may be anything, but no item's rows leave the workspace)
  uint32_t slots[2], slot[2];
  bool fits[2];
#pragma unroll
  for (int k = 0; k < 2; ++k)
    slots[k] = static_cast<uint32_t>(qkv_pages::imin(slots_of(it[k], F), int64_t(A.nslots) + 1));
  slot[0] = wave_scan(slots[0]);
  slot[1] = wave_scan(slots[1]) + lane_value(slot[0], 63);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    fits[k] = slot[k] <= static_cast<uint32_t>(A.nslots) && slot[k] >= slots[k];
    slot[k] -= slots[k];
  }
#pragma unroll
  for (int k = 0; k < 2; ++k)
    put_item(P, k * kSmall + lane, it[k], k == 1 && A.causal, tall[k], fours[k], slot[k], slots[k],
             fits[k]);
  if (lane == 0) {
    P.tall[kItems] = tall_all;
    P.fours[kItems] = F.fours;
  }
  if (tell) {
    if (lane == 0) *S.frame = F;
    int4 j[2];
#pragma unroll
    for (int k = 0; k < 2; ++k)
      j[k] = fits[k] ? join_of(it[k], F, slots[k], slot[k], tall[k]) : make_int4(0, 0, 0, 0);
    auto theirs = [&](int x) {
      const int u = __shfl(x, max(group, 0), 64);
      return group < 0 ? 0 : u;
    };
    const int4 g = make_int4(theirs(j[0].x), theirs(j[0].y), theirs(j[0].z), theirs(j[0].w));
    const int q0 = theirs(it[0].q0);
    if (lane < A.B) put_request(A, S, lane, it[1], j[1], g, q0, late[1]);
  }
  return F;
}

constexpr int kW = kPlanThr / 64;
static_assert(kW == 16, "a wave's sums are a lane of 16");

// Inclusive sums of K <= 4 values over the workgroup; `total` those of all.  The waves' sums meet
// in the lanes of each: 16 k + w has wave w's of value k.
template <int K>
__device__ __forceinline__ void block_sums(int64_t* v, int64_t* part, int64_t* total) {
  using qkv_pages::dpp;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = scan64(v[k]);
  __syncthreads();  // (part's last readers)
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (lane == 63) part[kW * k + wave] = v[k];
  __syncthreads();
  int64_t u = lane < kW * K ? part[lane] : 0;
  const int64_t own = u;
  u += dpp<0x111, 0xf>(u);  // row_shr 1, 2, 4, 8
  u += dpp<0x112, 0xf>(u);
  u += dpp<0x114, 0xf>(u);
  u += dpp<0x118, 0xf>(u);
  auto at = [](int64_t x, int l) {
    return (static_cast<int64_t>(lane_value(static_cast<int>(x >> 32), l)) << 32) |
           static_cast<uint32_t>(lane_value(static_cast<int>(x), l));
  };
#pragma unroll
  for (int k = 0; k < K; ++k) {
    v[k] += at(u - own, kW * k + wave);
    total[k] = at(u, kW * k + kW - 1);
  }
}

// Inclusive sum over 16 lanes.
__device__ __forceinline__ float row_scan(float v) {
  auto add = [&](auto ctrl) {
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v),
                                                               decltype(ctrl)::value, 0xf, 0xf, false));
  };
  using std::integral_constant;
  add(integral_constant<int, 0x111>{});  // row_shr 1, 2, 4, 8
  add(integral_constant<int, 0x112>{});
  add(integral_constant<int, 0x114>{});
  add(integral_constant<int, 0x118>{});
  return v;
}

constexpr int32_t kPairs = 1 << 30;  // (requests are fewer)

// The same of more requests or groups, by a workgroup, into the workspace.  ONE: a thread has
// one item, and keeps it.  (Up to 256 requests by plan_wave, four a lane: 3 us less a call at 96 to 200
// requests, none at 256, and 0.4 to 0.8 more for those up to 64, whose plan shares the code.)
template <bool ONE>
__global__ __launch_bounds__(kPlanThr) void share_plan(Att A, Share S) {
  extern __shared__ __align__(16) int32_t sh[];
  __shared__ int64_t part[kW * 4];
  const int tid = threadIdx.x, Gr = S.groups, items = Gr + A.B;
  int4* const joins = reinterpret_cast<int4*>(sh);  // ONE: [Gr]
  int32_t* const start = sh + (ONE ? 4 * Gr : 0);   // [Gr + 1]
  int32_t* const lead = start + Gr + 1; // [Gr]: the first request that takes part,
  int32_t* const many = lead + Gr;      // how many do, and kPairs where one has few rows,
  int32_t* const row0 = many + Gr;      // their first row and the end of their last one,
  int32_t* const row1 = row0 + Gr;
  int32_t* const cost = row1 + Gr;      // and what they cost alone; then whether they share
  int32_t* const whole = cost + Gr;     // prefix_of
  // f(i) for the thread's items of [from, to)
  auto each = [&](int from, int to, auto f) {
    if (ONE) {
      if (tid >= from && tid < to) f(tid);
    } else {
      for (int i = from + tid; i < to; i += kPlanThr) f(i);
    }
  };
  Req kept{0, 0, 0};
  if (ONE && tid >= Gr && tid < items) kept = request(A, tid - Gr);
  auto req = [&](int b) { return ONE ? kept : request(A, b); };
  const int rows_end = A.q_start && tid == 0 ? A.q_start[A.B] : 0;
  for (int g = tid; g <= Gr && Gr > 0; g += kPlanThr) {
    start[g] = S.group_start[g];
    if (g < Gr) {
      lead[g] = row0[g] = INT32_MAX;
      many[g] = row1[g] = cost[g] = 0;
      whole[g] = prefix_of(S, g);
    }
  }
  __syncthreads();
  auto group_of = [&](int b) {  // -1: in none
    if (Gr == 0 || b < start[0] || b >= start[Gr]) return -1;
    int lo = 0, hi = Gr;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (start[mid] <= b) lo = mid;
      else hi = mid;
    }
    return start[lo] <= b && b < start[lo + 1] ? lo : -1;
  };
  int mine = -1;  // ONE: the request's group, where it takes part
  each(Gr, items, [&](int i) {
    const int b = i - Gr, g = group_of(b);
    if (g < 0) return;
    const Req r = req(b);
    const int p = whole[g];
    if (!takes_part(A, r, p)) return;
    mine = g;
    atomicMin(&lead[g], b);
    atomicAdd(&many[g], 1);
    if (rows_of(A, r) * A.G <= kFew) atomicOr(&many[g], kPairs);
    atomicAdd(&cost[g], cost_of(rows_of(A, r) * A.G));
    atomicMin(&row0[g], r.q0);
    atomicMax(&row1[g], r.q0 + rows_of(A, r));
  });
  __syncthreads();
  each(0, Gr, [&](int g) {
    cost[g] = pays(S, many[g] & ~kPairs, cost[g], max(row1[g] - row0[g], 0) * A.G, whole[g] / kStep);
  });
  __syncthreads();
  auto make = [&](int i, int& g) {
    if (i < Gr) {
      g = i;
      return cost[i] ? group_item(A, whole[i], lead[i], row0[i], row1[i], (many[i] & kPairs) != 0)
                     : no_item();
    }
    const int b = i - Gr;
    const Req r = req(b);
    g = ONE ? mine : group_of(b);
    if (g >= 0 && (!cost[g] || !(ONE || takes_part(A, r, whole[g])))) g = -1;
    return own_item(A, r, b, g >= 0 ? whole[g] : 0);
  };
  Item own = no_item();
  int own_g = -1;
  if (ONE && tid < items) own = make(tid, own_g);
  auto item = [&](int i, int& g) {
    if (!ONE) return make(i, g);
    g = own_g;
    return own;
  };
  // steps and number of tall tiles, steps of short ones
  float sum[3] = {0.f, 0.f, 0.f};
  each(0, items, [&](int i) {
    int g;
    const Item it = item(i, g);
    const float n = static_cast<float>(it.tiles()), st = n * static_cast<float>(it.steps);
    sum[0] += it.tall() ? st : 0.f;
    sum[1] += it.tall() ? n : 0.f;
    sum[2] += it.four() ? st : 0.f;
  });
  float* const fpart = reinterpret_cast<float*>(part);
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const float v = wave_scan(sum[k]);
    if ((tid & 63) == 63) fpart[kW * k + (tid >> 6)] = v;
  }
  __syncthreads();
  {
    const float v = row_scan((tid & 63) < 3 * kW ? fpart[tid & 63] : 0.f);
#pragma unroll
    for (int k = 0; k < 3; ++k) sum[k] = lane_value(v, kW * k + kW - 1);
  }
  Frame F = frame_of(A.target, A.per_target, sum[0], sum[1], sum[2], [&](int R) {
    int64_t n = 0, all;
    each(0, items, [&](int i) {
      int g;
      const Item it = item(i, g);
      if (it.tall()) n += it.tiles() * div_up(it.steps, R);
    });
    block_sums<1>(&n, part, &all);
    return static_cast<int>(min(all, int64_t(INT32_MAX)));
  });
  const bool runs = F.range > 1;
  // (how many ranges there are decides whether tiles are cut at all)
  if (runs) {
    int64_t n = 0, all;
    each(0, items, [&](int i) {
      int g;
      const Item it = item(i, g);
      if (it.tall()) n += int64_t(it.tiles()) * extent(F, it.steps);
    });
    block_sums<1>(&n, part, &all);
    fit_ranges(F, static_cast<int>(all));
  }
  const int4 none = make_int4(0, 0, 0, 0);
  int4 join = none;
  int late = 0;
  int64_t base[4] = {0, 0, 0, 0};  // places of tall tiles, parts, tiles of the second launch, rows
  for (int i0 = 0; i0 < items; i0 += kPlanThr) {
    const int i = i0 + tid;
    Item it = no_item();
    int g = -1;
    if (i < items) it = item(i, g);
    const int64_t n[4] = {runs && it.tall() ? int64_t(it.tiles()) * extent(F, it.steps) : 0,
                          it.four() ? it.tiles() * most_parts(it, F) : 0,
                          it.late() ? it.tiles() : 0, slots_of(it, F)};
    int64_t v[4] = {n[0], n[1], n[2], n[3]}, total[4];
    block_sums<4>(v, part, total);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[k] += base[k] - n[k];
      base[k] += total[k];
    }
    if (i >= items) continue;
    const bool fits = v[3] + n[3] <= A.nslots;
    put_item(S.at, i, it, i >= Gr && A.causal, static_cast<int>(v[0]), static_cast<int>(v[1]), v[3],
             n[3], fits);
    join = fits ? join_of(it, F, n[3], v[3], static_cast<int>(v[0])) : none;
    late = static_cast<int>(v[2]);
    // (requests' entries follow when all groups' are known; without ONE theirs wait behind)
    if (i < Gr) {
      if (ONE) joins[i] = join;
      else S.meta[3 * A.B + i] = join;
    } else if (!ONE) {
      S.meta[3 * (i - Gr)] = join;
      S.meta[3 * (i - Gr) + 2] = make_int4(late, 0, 0, 0);
    }
  }
  if (tid == 0) {
    S.at.tall[items] = static_cast<int32_t>(base[0]);
    S.at.fours[items] = static_cast<int32_t>(base[1]);
    F.fours = static_cast<int32_t>(base[1]);
    F.lates = min(static_cast<int32_t>(base[2]), S.late_cap);
    *S.frame = F;
  }
  __syncthreads();
  each(Gr, items, [&](int i) {
    const int b = i - Gr;
    int g;
    const Item it = item(i, g);
    int4 theirs = none;
    if (!ONE) {
      join = S.meta[3 * b];
      late = S.meta[3 * b + 2].x;
      if (g >= 0) theirs = S.meta[3 * A.B + g];
    } else if (g >= 0) {
      theirs = joins[g];
    }
    put_request(A, S, b, it, join, theirs, g >= 0 ? row0[g] : 0, late);
  });
  // ---- the rows' requests
  if (A.q_start == nullptr) {
    for (int r = tid; r < A.rows; r += kPlanThr) S.row_req[r] = r / A.uniform_q;
    return;
  }
  __syncthreads();
  int32_t* const lens = sh + A.B + 1;  // ONE
  if (ONE) {
    if (tid >= Gr && tid < items) {
      sh[tid - Gr] = kept.q0;
      lens[tid - Gr] = kept.ql;
    }
  } else {
    for (int b = tid; b < A.B; b += kPlanThr) sh[b] = A.q_start[b];
  }
  if (tid == 0) sh[A.B] = rows_end;
  __syncthreads();
  for (int r = tid; r < A.rows; r += kPlanThr) {
    int lo = 0, hi = A.B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (sh[mid] <= r) lo = mid;
      else hi = mid;
    }
    const int in = r - sh[lo];
    const int ql = ONE ? lens[lo] : A.q_lens ? A.q_lens[lo] : sh[lo + 1] - sh[lo];
    S.row_req[r] = in >= 0 && in < ql ? lo : -1;
  }
}

// The last i < n with key[i] <= x (key[0] <= x < key[n], ascending), by a wave, 64 keys at a time.
__device__ __forceinline__ int find_wave(const int32_t* key, int n, int x) {
  const int lane = threadIdx.x & 63;
  int lo = 0;
  while (n > 1) {
    const int step = (n + 63) / 64, i = lane * step;
    const uint64_t m = __ballot(i < n && key[lo + min(i, n - 1)] <= x);
    const int at = (__popcll(m) - 1) * step;
    lo += at;
    n = min(step, n - at);
  }
  return lo;
}

__device__ __forceinline__ int same(int v) { return __builtin_amdgcn_readfirstlane(v); }
// What share8 is called with, read anew where it is needed: held in registers from the kernel's
// start on, arguments and the loops' state take more SGPRs than there are (80 spilled).
struct Args {
  Att a;
  Share s;
};
__device__ __forceinline__ const Args& args_anew() {
  auto p = __builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const Args*)p;
}

// threadIdx.x, for what is computed from it to stay within a loop's pass.
__device__ __forceinline__ int thread_anew() {
  int t = threadIdx.x;
  asm volatile("" : "+v"(t));
  return t;
}

// Workgroup (j, h), j < target: the j-th range of kv head h's tall tiles, where there is one, then
// short tiles, two at a time, in turn with the other workgroups that take these.
//
// Weights are f16 pairs (22 bits) but, without PLO (bf16 results of 16-bit queries), those of
// requests of more than kFew rows, of which qkv_kv8_attention's result has 11 bits, too: their own
// tall tiles', and the prefix' where no request of fewer rows shares it.
template <int D, bool FP8, bool QLO, bool PLO>
__global__ __launch_bounds__(kPreThr, 2) void share8(Args) {
  __shared__ v4f sbuf[2][2][4];
  __shared__ int32_t sh_tall[kItems + 1], sh_fours[kItems + 1];
  __shared__ int4 sh_geo[2 * kItems];
  __shared__ Frame sh_frame;
  __shared__ int32_t sh_x;
  extern __shared__ __align__(16) uint8_t lds[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  {
    const Args C = args_anew();  // (a copy: its loads are one batch)
    if (wave == 0) {
      Frame F;
      if (C.s.small) F = plan_wave(C.a, C.s, Places{sh_tall, sh_fours, sh_geo}, blockIdx.x == 0);
      else F = *C.s.frame;
      if (threadIdx.x == 0) {
        sh_frame = F;
        const int j = blockIdx.x / C.a.H;
        sh_x = j < F.tall ? j * F.range : 0;  // (ranges end below 2^31)
      }
    }
    __syncthreads();
  }
  // the last item whose places begin at x or before, and the place; then its geometry
  auto find = [&](const Share& S, int items, const int32_t* mine, const int32_t* theirs, int x,
                  int& first) {
    int i;
    if (S.small) {
      i = find_wave(mine, kItems, x);
      first = same(mine[i]);
    } else {
      i = find_wave(theirs, items, x);
      first = same(theirs[i]);
    }
    return i;
  };
  auto piece = [&](const Share& S, int i, int& s0, int& steps, int& rows, bool& pairs) {
    int4 x, y;
    if (S.small) {
      x = sh_geo[2 * i];
      y = sh_geo[2 * i + 1];
    } else {
      x = S.at.geo[2 * i];
      y = S.at.geo[2 * i + 1];
    }
    Piece P{};
    P.r = Req{same(x.x), same(x.y), same(x.z)};
    s0 = same(x.w);
    steps = same(y.x);
    P.b = same(y.y) >> 2;
    pairs = same(y.y) & 2;
    P.causal = same(y.y) & 1;
    P.slot = same(y.z);
    rows = same(y.w);
    return P;
  };
  while (true) {
    const Args& C = args_anew();
    const int items = C.s.groups + C.a.B, h = blockIdx.x % C.a.H, j = blockIdx.x / C.a.H;
    Frame F;
    F.range = same(sh_frame.range);
    F.setup = same(sh_frame.setup);
    if (j >= same(sh_frame.tall)) break;
    const int x = same(sh_x), total = same(C.s.small ? sh_tall[kItems] : C.s.at.tall[items]);
    const int end = min((j + 1) * F.range, total);
    __syncthreads();  // (sh_x is read)
    if (x >= end) break;
    int first, s0, steps, rows;
    const int i = find(C.s, items, sh_tall, C.s.at.tall, x, first);
    bool pairs;
    Piece P = piece(C.s, i, s0, steps, rows, pairs);
    const int E = extent(F, steps), p = (x - first) / E, in = x - first - p * E;
    const int n = min(E - in, end - x);
    if (threadIdx.x == 0) sh_x = x + n;
    const int from = cut_at(F, steps, in), to = in + n == E ? steps : cut_at(F, steps, in + n);
    if (from < to) {
      P.rt = tile_at(p, (rows + kPreRows - 1) / kPreRows);
      P.s0 = s0 + from;
      P.s1 = min(s0 + to, steps_of(P.r.kv));  // (an item without tokens counts a step)
      // the part of the tile: ranges before this one that have steps of it
      if (P.slot >= 0) {
        int none;
        const int k = (x - in) / F.range;
        parts_at(F, steps, x - in - k * F.range, none);
        P.slot += (j - k - none) * rows;
      }
      if (PLO || pairs) prefill_piece<D, FP8, QLO, true, true>(C.a, P, h, thread_anew(), lds, sbuf);
      else prefill_piece<D, FP8, QLO, false, true>(C.a, P, h, thread_anew(), lds, sbuf);
    }
    __syncthreads();
  }
  // short tiles' workgroups: those without a tall range, the last one at least
  int u, units, every;
  {
    const Args& C = args_anew();
    units = (same(sh_frame.fours) + 1) / 2;
    const int from = min(same(sh_frame.tall), C.a.target - 1);
    every = C.a.target - from;
    u = static_cast<int>(blockIdx.x / C.a.H) - from;
  }
  if (u < 0) return;
  for (; u < units; u += every) {
    const Args& C = args_anew();
    const int items = C.s.groups + C.a.B, h = blockIdx.x % C.a.H;
    const int half = wave >> 2, k = 2 * u + half;
    // (without a piece of its own the half takes the other's barriers, and has no row or step)
    Piece P{};
    P.slot = -1;
    if (k < same(sh_frame.fours)) {
      int first, s0, steps, rows;
      const int i = find(C.s, items, sh_fours, C.s.at.fours, k, first);
      bool pairs;
      P = piece(C.s, i, s0, steps, rows, pairs);
      const int least = same(sh_frame.least), parts = (steps + least - 1) / least;
      const int in = k - first;
      P.rt = in / parts;
      P.part = in % parts;
      P.s0 = s0 + P.part * least;
      P.s1 = min(min(s0 + steps, P.s0 + least), steps_of(P.r.kv));
      if (P.slot >= 0) P.slot += P.part * rows;
    }
    float* const mine = reinterpret_cast<float*>(lds) + half * kWaves * kRows * (D + 6);
    decode_piece<D, FP8, QLO, true>(
        C.a, P, h, thread_anew() & 255, reinterpret_cast<float(*)[kRows][D + 4]>(mine),
        reinterpret_cast<float(*)[kRows][2]>(mine + kWaves * kRows * (D + 4)));
    __syncthreads();  // (the buffers' last readers)
  }
}

// Partial results of a row on their way: four parts of one item.
struct Parts {
  float m[4], l[4];
  v4f v[4][2];
};
// Parts p0, p0 + every, ... of `parts`: a lane has coordinates d0 .. d0 + 7 (on: of the row's).
template <int D>
__device__ __forceinline__ Parts load_parts(const Att& A, int64_t first, int rows, int p0, int every,
                                            int parts, bool on, int d0) {
  Parts r;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int p = p0 + every * k;
    r.m[k] = -INFINITY;
    r.l[k] = 0.f;
    r.v[k][0] = r.v[k][1] = v4f{0.f, 0.f, 0.f, 0.f};
    if (p < parts) {
      const int64_t at = first + int64_t(p) * rows;
      r.m[k] = A.part_ml[2 * at];
      r.l[k] = A.part_ml[2 * at + 1];
      const v4f* const src = reinterpret_cast<const v4f*>(A.part_o + at * D + (on ? d0 : 0));
      r.v[k][0] = src[0];
      r.v[k][1] = src[1];
    }
  }
  return r;
}
__device__ __forceinline__ void fold(const Parts& r, float& M, float& L, float* x) {
  float mn = M;
#pragma unroll
  for (int k = 0; k < 4; ++k) mn = fmaxf(mn, r.m[k]);
  const float ref = mn == -INFINITY ? 0.f : mn, e0 = __builtin_amdgcn_exp2f(M - ref);
  L = fall(L, M - ref);
  M = mn;
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] *= e0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float e = __builtin_amdgcn_exp2f(r.m[k] - ref);
    L += fall(r.l[k], r.m[k] - ref);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = fmaf(r.v[k][j >> 2][j & 3], e, x[j]);
  }
}
// All of a row's parts from p0 on.
template <int D>
__device__ __forceinline__ void add_parts(const Att& A, int64_t first, int rows, int p0, int every,
                                          int parts, bool on, int d0, float& M, float& L, float* x) {
  for (; __any(p0 < parts); p0 += 4 * every)
    fold(load_parts<D>(A, first, rows, p0, every, parts, on, d0), M, L, x);
}

// Waves of a tile of the second launch: four, or as many as the card's two workgroups a CU have for
// each.  A call with four / two / one, 8192 shared tokens, 8 kv heads, 4 query heads each, by requests
// and their own tokens: 64 + 500 us 39.2 / 40.6 / 47.8, 96 + 300 54.9 / 52.7 / 55.3, 128 + 300 59.6 /
// 57.0 / 58.7, 256 + 100 88 / 80 / 77, 256 + 300 91 / 85 / 83; but 256 + 1000 109 / 110 / 114.  (With
// the prefix' weights in 11 bits; their 22 take 3 to 11 us of the first launch alike.)
__device__ __forceinline__ int waves_of(const Att& A, int tiles) {
  const int most = 2 * kWaves * A.target;  // of a kv head
  return kWaves * tiles <= most ? kWaves : 2 * tiles <= most ? 2 : 1;
}

// The second launch.  Its first workgroups take a tile of 16 rows each of the requests that have
// few own tokens: the prefix' partial results, which are there, dealt to the waves by rows and
// parts, then the own tokens as a piece of four waves, then all in LDS.  The others join what else
// the first launch left, a row (query and head) on D / 8 lanes of 8 or 16: where there are few
// rows (deal) a workgroup takes a wave's rows, its waves every fourth part, and they meet in LDS,
// else a wave takes its rows by itself.
template <int D, bool FP8, bool QLO>
__global__ __launch_bounds__(kThr, 2) void share_rest(Att A, Share S, int deal) {
  constexpr int LPR = D > 64 ? 16 : 8, RW = 64 / LPR;  // lanes of a row, rows of a wave
  __shared__ float red_o[kWaves][kRows][D + 4];
  __shared__ float red_ml[kWaves][kRows][2];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane >> 4, d0 = 8 * (lane & 15);
  const bool on = d0 < D;
  const Frame F = *S.frame;
  const int tiles = same(F.lates), W = waves_of(A, tiles), T = kWaves / W;
  const int lates = div_up(tiles, T) * A.H;
  if (static_cast<int>(blockIdx.x) < lates) {
    const int u = blockIdx.x / A.H, h = blockIdx.x - u * A.H, t = u * T + wave / W, turn = wave % W;
    // (a wave without a tile has no row or step, and takes the others' barriers)
    int4 pre = make_int4(0, 0, 0, 0), q = pre, kv = pre;
    if (t < tiles) {
      pre = S.lates[3 * t];
      q = S.lates[3 * t + 1];
      kv = S.lates[3 * t + 2];
    }
    Piece P{};
    P.b = same(q.x);
    P.rt = same(q.y);
    P.r = Req{same(q.z), same(q.w), same(kv.x)};
    P.causal = A.causal;
    P.slot = -1;
    P.s0 = same(kv.y);
    P.s1 = steps_of(P.r.kv);
    // sets of 4 rows, `at_once` of them by `each` waves, which deal out the parts
    const int rows = min(kRows, same(kv.z) - P.rt * kRows), sets = (rows + 3) / 4;
    const int at_once = min(W, sets <= 1 ? 1 : sets == 2 ? 2 : 4), each = W / at_once;
    const int p0 = turn % each;
    int parts = 0;
    int64_t first = 0;
    Parts some;
    auto parts_from = [&](int set) {
      const int rr = P.rt * kRows + 4 * set + r, rp = rr + same(kv.w);
      parts = 4 * set + r < rows ? parts_of(pre, F, rp) : 0;
      first = int64_t(h) * A.nslots + pre.x + rp;
      some = load_parts<D>(A, first, pre.y, p0, each, parts, on, d0);
    };
    // (the first parts are on their way while the own tokens are gone over)
    decode_steps<D, FP8, QLO>(A, P, h, tid, turn, W, red_o, red_ml, [&] { parts_from(turn / each); });
    if (same(pre.y) > 0) {
      for (int set = turn / each; set < sets; set += at_once) {
        if (set >= at_once) parts_from(set);
        float* const o = &red_o[wave][4 * set + r][on ? d0 : 0];
        float* const ml = red_ml[wave][4 * set + r];
        float M = ml[0], L = ml[1], x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = o[j];
        fold(some, M, L, x);
        add_parts<D>(A, first, pre.y, p0 + 4 * each, each, parts, on, d0, M, L, x);
        if (on) {
#pragma unroll
          for (int j = 0; j < 8; ++j) o[j] = x[j];
        }
        if (d0 == 0) {
          ml[0] = M;
          ml[1] = L;
        }
      }
    }
    __syncthreads();
    constexpr int PER = D / 8;
    for (int i = 64 * turn + lane; i < rows * PER; i += 64 * W) {
      const int k = i / PER, e0 = 8 * (i % PER), w0 = wave - turn;
      float M = -INFINITY, L = 0.f, x[8] = {};
      for (int w = 0; w < W; ++w) M = fmaxf(M, red_ml[w0 + w][k][0]);
      const float ref = M == -INFINITY ? 0.f : M;
      for (int w = 0; w < W; ++w) {
        const float m = red_ml[w0 + w][k][0] - ref, f = __builtin_amdgcn_exp2f(m);
        const float* const o = &red_o[w0 + w][k][e0];
        L += fall(red_ml[w0 + w][k][1], m);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = fmaf(o[j], f, x[j]);
      }
      const int rr = P.rt * kRows + k, qi = rr / A.G;
      const int64_t row = int64_t(P.r.q0) + qi;
      if (qi < P.r.ql && row >= 0 && row < A.rows) {
        const float inv = inverse(L);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] *= inv;
        store8(A.out, (row * A.Hq + h * A.G + rr - qi * A.G) * D + e0, x, A.out_dtype, A.out_vec);
      }
    }
    return;
  }
  const int e0 = 8 * (lane % LPR), rw = lane / LPR;
  const bool in = e0 < D;
  int4 rows_req = make_int4(0, 0, 0, 0);  // small: the lane's request's rows
  if (S.small && lane < A.B) rows_req = S.meta[3 * lane + 2];
  const int all = A.rows * A.Hq, unit = deal ? RW : RW * kWaves;  // (all < 2^28)
  const int every = unit * (static_cast<int>(gridDim.x) - lates);
  for (int u = unit * (static_cast<int>(blockIdx.x) - lates); u < all; u += every) {
    const int f0 = u + (deal ? 0 : RW * wave);
    const int f = min(f0 + rw, all - 1), row = f / A.Hq, hq = f - row * A.Hq, h = hq / A.G;
    int b = -1;
    if (S.small) {
      const int last = lane_value(row, 63);
      for (int x = lane_value(row, 0); x <= last; ++x) {
        const uint64_t m = __ballot(lane < A.B && x >= rows_req.x && x - rows_req.x < rows_req.w);
        if (row == x && m != 0) b = __builtin_ctzll(m);
      }
    } else {
      b = S.row_req[row];
    }
    int4 own = make_int4(0, 0, 0, 0), pre = own, q0 = own;
    if (b >= 0) {  // (own.y 0: its result is there already)
      own = S.meta[3 * b];
      pre = S.meta[3 * b + 1];
      q0 = S.meta[3 * b + 2];
    }
    const int gq = hq - h * A.G, ro = (row - q0.x) * A.G + gq, rp = (row - q0.y) * A.G + gq;
    const int no = f0 + rw < all ? parts_of(own, F, ro) : 0;
    const int np = no > 0 ? parts_of(pre, F, rp) : 0;
    if (!__any(no > 0)) continue;  // (deal: the same in all waves)
    const int64_t base = int64_t(h) * A.nslots;
    float M = -INFINITY, L = 0.f, x[8] = {};
    const int p0 = deal ? wave : 0, step = deal ? kWaves : 1;
    add_parts<D>(A, base + pre.x + rp, pre.y, p0, step, np, in, e0, M, L, x);
    add_parts<D>(A, base + own.x + ro, own.y, p0, step, no, in, e0, M, L, x);
    if (!deal) {
      if (no == 0 || !in) continue;
      const float inv = inverse(L);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] *= inv;
      store8(A.out, int64_t(f) * D + e0, x, A.out_dtype, A.out_vec);
      continue;
    }
    __syncthreads();  // (the arrays' last readers)
    if (in) {
      *reinterpret_cast<v4f*>(&red_o[wave][rw][e0]) = v4f{x[0], x[1], x[2], x[3]};
      *reinterpret_cast<v4f*>(&red_o[wave][rw][e0 + 4]) = v4f{x[4], x[5], x[6], x[7]};
    }
    if (e0 == 0) {
      red_ml[wave][rw][0] = M;
      red_ml[wave][rw][1] = L;
    }
    __syncthreads();
    if (wave != 0 || no == 0 || !in) continue;
    M = -INFINITY;
    L = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) M = fmaxf(M, red_ml[w][rw][0]);
    const float ref = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float e = __builtin_amdgcn_exp2f(red_ml[w][rw][0] - ref);
      L += fall(red_ml[w][rw][1], red_ml[w][rw][0] - ref);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = fmaf(red_o[w][rw][e0 + j], e, x[j]);
    }
    const float inv = inverse(L);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] *= inv;
    store8(A.out, int64_t(f) * D + e0, x, A.out_dtype, A.out_vec);
  }
}

// Workgroups per kv head: one per CU, and no more (a second one would wait for a first to end).
int32_t target_of(int32_t H) { return std::max(1, qkv_num_cus() / H); }

// The workspace.  Each row is in two items at most, its group's prefix and its own tokens.
// An item of tall tiles has partial rows for (places - 2) / range + 2 parts, all beyond the two
// within a tile per range; one of short tiles for its parts, those beyond one within 16 rows per
// part of `least` steps, 2 target of them at most.
struct Layout {
  int64_t rows;           // partial rows of a kv head
  int64_t late;           // tiles of the second launch, at most
  int64_t meta, lates, row_req, tall, fours, geo, ml, o, bytes;
};
Layout layout(int64_t B, int64_t groups, int64_t rows, int32_t G, int32_t H, int32_t d) {
  Layout L;
  const int64_t t = target_of(H), all = 2 * rows * G, items = B + groups;
  const bool high = rows * G > kFew;  // there may be items of tall tiles
  L.rows = high ? 2 * all + (kPreRows + 2 * kRows) * t : all + 2 * kRows * t;
  const bool small = B <= kSmall && groups <= kSmall;
  auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
  L.meta = 256;
  L.late = std::min(2 * std::min(B, rows), rows * G / kRows + std::min(B, rows));
  L.lates = L.meta + up(48 * B + 16 * groups);
  L.row_req = L.lates + up(48 * L.late);
  L.tall = L.row_req + (small ? 0 : up(4 * rows));
  L.fours = L.tall + (small ? 0 : up(4 * (items + 1)));
  L.geo = L.fours + (small ? 0 : up(4 * (items + 1)));
  L.ml = L.geo + (small ? 0 : up(32 * items));
  L.o = L.ml + up(8 * H * L.rows);
  L.bytes = L.o + up(4 * H * L.rows * d);
  return L;
}

template <int D, bool FP8, bool QLO, bool PLO>
void start(const Att& A, const Share& S, hipStream_t s) {
  constexpr int smem = std::max(kPreLds<D>, 2 * kWaves * kRows * (D + 6) * 4);
  // more LDS than a kernel has by default, asked for once per device (a failure is the
  // launch's, which the caller reports)
  static std::atomic<uint64_t> asked{0};
  int dev = 0;
  (void)hipGetDevice(&dev);
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (!(asked.load(std::memory_order_relaxed) & bit)) {
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(&share8<D, FP8, QLO, PLO>),
                              hipFuncAttributeMaxDynamicSharedMemorySize, smem);
    asked.fetch_or(bit, std::memory_order_relaxed);
  }
  share8<D, FP8, QLO, PLO><<<A.target * A.H, kPreThr, smem, s>>>(Args{A, S});
}

// Both launches; the second one of `rest` workgroups.
template <int D, bool FP8>
void run(const Att& A, const Share& S, uint32_t rest, int deal, hipStream_t s) {
  if (A.q_dtype == QKV_F32) start<D, FP8, true, true>(A, S, s);
  else if (A.out_dtype != QKV_BF16) start<D, FP8, false, true>(A, S, s);
  else start<D, FP8, false, false>(A, S, s);
  if (A.q_dtype == QKV_F32) share_rest<D, FP8, true><<<rest, kThr, 0, s>>>(A, S, deal);
  else share_rest<D, FP8, false><<<rest, kThr, 0, s>>>(A, S, deal);
}

// Calls whose requests would read little all the same go to qkv_kv8_attention.  us of it / shared,
// 8 kv heads, d = 128, 4 query heads a kv head, by requests x prefix (and the bytes that they
// would read): 4 x 8000 (69 MB) 20 / 27, 16 x 2000 (84) 21 / 25, 64 x 500 (134) 15 / 28;
// 4 x 32,000 (266) 41 / 31, 16 x 8000 (277) 43 / 28, 64 x 2000 (336) 38 / 29.  With 2 kv heads of
// d = 64: 64 x 500 15 / 22, 16 x 8000 19 / 22; 64 x 8000 34 / 30.  The host knows the table's
// width for it, not the lengths: under a table of room for much more than they are, short requests do
// not count as small.  Nor does it know of calls of many rows a request whether a group will share:
// 8 x 210 rows, 7 query heads, over 16,001 207 / 172; those that do not have lost the plan and the second
// launch, 8 x 256 rows over 8000, 7 query heads, d = 64 113.5 / 115.5, 4 x 64, d = 128 60 / 61,
// 16 x 64 160 / 173.
constexpr double kLittle = 192e6;
bool little(int64_t B, int64_t rows, int32_t G, int32_t H, int32_t d, int64_t width, int32_t page) {
  return rows * G <= kFew * B && double(B) * width * page * H * 2 * d <= kLittle;
}
// Calls whose tall tiles' places, were every request as long as the table is wide, are more than a
// plan counts: they go there, too.
bool too_wide(int64_t B, int64_t groups, int64_t rows, int32_t G, int64_t width, int32_t page) {
  const double tiles = 2.0 * rows * G / kPreRows + std::min<double>(B + groups, 2.0 * rows * G / kFew);
  const double longest = std::min(double(width) * page, double(QKV_PAGED_TOKENS)) / kStep;
  return tiles * (longest + 1 + kSetUp) >= kMostPlaces;
}
// The longest request's rows for that call, as far as their number tells (a hint; who knows a
// bound of them, of a batch with padding rows, say, makes that call instead)
int64_t longest_of(int64_t B, int64_t rows, int32_t G) {
  return rows > 2 * B ? rows : std::max<int64_t>(1, kFew / G);
}

}  // namespace

extern "C" int64_t qkv_kv8_attention_shared_workspace_bytes(int32_t B, int32_t groups, int64_t rows,
                                                            int32_t Hq, int32_t Hkv, int32_t d) {
  if (Hkv < 1 || d < 1) return 0;
  if (B < 1 || rows < 1) return 256;
  const int32_t G = Hq / Hkv;
  return std::max(layout(B, std::max(groups, 0), rows, G, Hkv, d).bytes,
                  qkv_kv8_attention_workspace_bytes(B, rows, Hq, Hkv, d, longest_of(B, rows, G)));
}

extern "C" int64_t qkv_kv8_attention_shared_plain(int32_t B, int32_t groups, int64_t rows, int32_t Hq,
                                                  int32_t Hkv, int32_t d, int32_t pages_per_seq,
                                                  int32_t page_tokens) {
  if (B < 1 || B > kMaxB || groups < 0 || groups > kMaxGroups || rows < 1 || Hkv < 1 || Hq < Hkv ||
      rows * Hq >= (1 << 28))
    return 0;  // (nothing to do, or refused)
  const int32_t G = Hq / Hkv;
  return too_wide(B, groups, rows, G, pages_per_seq, page_tokens) ||
                 little(B, rows, G, Hkv, d, pages_per_seq, page_tokens)
             ? longest_of(B, rows, G) : 0;
}

extern "C" int qkv_kv8_attention_shared(
    const void* q, int32_t q_dtype, int64_t q_row_stride, int64_t q_head_stride, int64_t rows,
    const void* kpool, const float* kscale, const void* vpool, const float* vscale, int32_t fmt,
    int32_t num_pages, int32_t page_tokens, const int32_t* table, int32_t pages_per_seq,
    const int32_t* group_start, const int32_t* prefix_lens, int32_t groups, int32_t always,
    const int32_t* q_start,
    const int32_t* q_lens, const int32_t* kv_lens, int32_t B, int32_t Hq, int32_t Hkv, int32_t d,
    float scale, int32_t causal, void* out, int32_t out_dtype, void* workspace, int64_t ws_bytes,
    void* stream) {
  const int st = qkv_kv8_check(fmt, num_pages, page_tokens, Hkv, d);
  if (st != QKV_OK) return st;
  QKV_REQUIRE(qkv_dtype_ok(q_dtype) && qkv_dtype_ok(out_dtype), "unknown element type %d / %d",
              q_dtype, out_dtype);
  QKV_REQUIRE(Hq >= 1 && Hq % Hkv == 0, "query heads (%d) must be a multiple of kv heads (%d)", Hq,
              Hkv);
  QKV_REQUIRE(B >= 0 && B <= kMaxB && pages_per_seq >= 1,
              "batch %d must lie in [0, %d], pages_per_seq %d be positive", B, kMaxB, pages_per_seq);
  QKV_REQUIRE(groups >= 0 && groups <= kMaxGroups, "groups must lie in [0, %d]; got %d", kMaxGroups,
              groups);
  const int32_t G = Hq / Hkv;
  QKV_REQUIRE(rows >= 0 && rows * Hq < (1 << 28), "rows x query heads must lie in [0, 2^28); got "
              "%lld x %d", static_cast<long long>(rows), Hq);
  if (rows == 0 || B == 0) return QKV_OK;
  QKV_REQUIRE(q_start || !q_lens, "q_lens needs q_start");
  QKV_REQUIRE(q_start || rows % B == 0, "without q_start the rows (%lld) must be B (%d) times one "
              "length", static_cast<long long>(rows), B);
  QKV_REQUIRE(q && kpool && kscale && vpool && vscale && table && kv_lens && out &&
                  (groups == 0 || (group_start && prefix_lens)),
              "qkv_kv8_attention_shared: null pointer");
  QKV_REQUIRE(qkv_aligned(kpool, 16) && qkv_aligned(vpool, 16),
              "the pools must be 16-byte aligned");
  const Layout L = layout(B, groups, rows, G, Hkv, d);
  const int64_t need = qkv_kv8_attention_shared_workspace_bytes(B, groups, rows, Hq, Hkv, d);
  QKV_REQUIRE(workspace && qkv_aligned(workspace, 256) && ws_bytes >= need,
              "qkv_kv8_attention_shared: workspace too small or not 256-byte aligned");
  const bool wide = too_wide(B, groups, rows, G, pages_per_seq, page_tokens);
  if (!always && (wide || little(B, rows, G, Hkv, d, pages_per_seq, page_tokens)))
    return qkv_kv8_attention(q, q_dtype, q_row_stride, q_head_stride, rows, kpool, kscale, vpool,
                             vscale, fmt, num_pages, page_tokens, table, pages_per_seq, q_start,
                             q_lens, kv_lens, B, Hq, Hkv, d, longest_of(B, rows, G), scale, causal,
                             out, out_dtype, workspace, ws_bytes, stream);
  QKV_REQUIRE(!wide && L.rows < INT32_MAX &&
                  L.late * Hkv < (1 << 23),  // (a launch has fewer than 2^32 threads)
              "%lld rows of %d query heads a kv head over a table of %d pages are too large for one "
              "call", static_cast<long long>(rows), G, pages_per_seq);
  const int qb = q_dtype == QKV_F32 ? 4 : 2, ob = out_dtype == QKV_F32 ? 4 : 2;
  char* const ws = static_cast<char*>(workspace);
  Att A{};
  A.q = q;
  A.q_ts = q_row_stride;
  A.q_hs = q_head_stride;
  A.q_dtype = q_dtype;
  A.q_vec = qkv_aligned(q, 16) && q_row_stride * qb % 16 == 0 && q_head_stride * qb % 16 == 0;
  A.rows = static_cast<int32_t>(rows);
  A.kpool = static_cast<const uint8_t*>(kpool);
  A.kscale = kscale;
  A.vpool = static_cast<const uint8_t*>(vpool);
  A.vscale = vscale;
  A.npages = num_pages;
  A.lg = qkv_page_lg(page_tokens);
  A.table = table;
  A.width = pages_per_seq;
  A.q_start = q_start;
  A.q_lens = q_lens;
  A.kv_lens = kv_lens;
  A.B = B;
  A.Hq = Hq;
  A.H = Hkv;
  A.G = G;
  A.uniform_q = static_cast<int32_t>(rows / B);
  A.scale = scale;
  A.causal = causal;
  A.out = out;
  A.out_dtype = out_dtype;
  A.out_vec = qkv_aligned(out, 16) && d * ob % 16 == 0;
  A.target = target_of(Hkv);
  A.per_target = 1.f / A.target;
  A.nslots = static_cast<int32_t>(L.rows);
  A.part_ml = reinterpret_cast<float*>(ws + L.ml);
  A.part_o = reinterpret_cast<float*>(ws + L.o);
  Share S{};
  S.group_start = group_start;
  S.prefix_lens = prefix_lens;
  S.groups = groups;
  S.always = always;
  S.small = B <= kSmall && groups <= kSmall;
  S.frame = reinterpret_cast<Frame*>(ws);
  S.at = Places{reinterpret_cast<int32_t*>(ws + L.tall), reinterpret_cast<int32_t*>(ws + L.fours),
                reinterpret_cast<int4*>(ws + L.geo)};
  S.lates = reinterpret_cast<int4*>(ws + L.lates);
  S.meta = reinterpret_cast<int4*>(ws + L.meta);
  S.late_cap = static_cast<int32_t>(L.late);
  S.row_req = reinterpret_cast<int32_t*>(ws + L.row_req);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (!S.small) {
    if (groups + B <= kPlanThr)
      share_plan<true><<<1, kPlanThr, std::max(11 * groups + 1, 2 * B + 1) * sizeof(int32_t), s>>>(A, S);
    else
      share_plan<false><<<1, kPlanThr, std::max(7 * groups + 1, B + 1) * sizeof(int32_t), s>>>(A, S);
    QKV_LAUNCHED();
  }
  // the second launch: a workgroup per tile that may be its own, and some that join the rest, few
  // where rows tell that most requests have few of them (each reads lengths before it ends)
  const int deal = rows * Hq < 8192;
  const int64_t joins = std::min<int64_t>((rows * Hq + 3) / 4, rows * G > kFew * int64_t(B) ? 2048 : 256);
  const uint32_t rest = static_cast<uint32_t>(L.late * Hkv + joins);
  if (fmt == QKV_CODES_I8) {
    if (d == 128) run<128, false>(A, S, rest, deal, s);
    else if (d == 96) run<96, false>(A, S, rest, deal, s);
    else run<64, false>(A, S, rest, deal, s);
  } else {
    if (d == 128) run<128, true>(A, S, rest, deal, s);
    else if (d == 96) run<96, true>(A, S, rest, deal, s);
    else run<64, true>(A, S, rest, deal, s);
  }
  QKV_LAUNCHED();
  return QKV_OK;
}
