// Attention over the 8-bit paged cache (qkv_kv8.h) of a batch in groups whose requests share
// a prefix (C ABI: qkv_kv8_attention_shared): the prefix is read once for all rows of a group.
//
// Mathematics: decode8's (qkv_kv8_decode.h), whose partial results over parts of a row's tokens
// -- maximum m, sum l, values o, all relative to 2^m -- join as
//   M = max m_i,  out = sum 2^(m_i - M) o_i / sum 2^(m_i - M) l_i.
// So the rows of a group, one behind the other as its requests are, are one set of rows over the
// prefix' tokens, without a mask, and each request's rows are a set over its own tokens: items
// of both kinds are cut into pieces, run in one launch, and are joined row by row.
//
// A request takes part in its group's prefix if its queries all lie behind it (causal), or it
// holds the prefix at all; the prefix is read from the first of these.  The others, and those
// of a group with one such request, go over all of their tokens by themselves.
//
// Three launches: the plan (one workgroup: items, pieces, where partial results go), the
// attention, the join.
#include <algorithm>
#include <atomic>

#include "qkv_kv8_decode.h"
#include "qkv_kv8_prefill.h"

namespace {

using namespace qkv_kv8;

constexpr int kFew = 32;        // rows of an item up to which its tiles have 16 rows, else 128
constexpr int kLeast = 4;       // steps of the shortest piece
constexpr int kMaxGroups = 2048;

// What the plan leaves for the other two launches.
struct Share {
  const int32_t* group_start;
  const int32_t* prefix_lens;
  int32_t groups;
  int32_t* head;      // [0], [1]: tall and short pieces
  int4* pieces;       // two each; tall ones from 0, short ones from cap_tall on
  int32_t cap_tall, cap_short;
  int4* meta;         // two a request: first row, first partial row of its own tokens, their
                      // parts, rows; the same of the prefix (rows' distance last).  No parts
                      // of its own: nothing to join
  int32_t* row_req;   // a row's request, -1: none
};

// Rows of one piece of work over steps [s0, s1) of one request's tokens.
struct Item {
  int32_t q0, ql, kv, s0, s1;
  int32_t rows;       // ql x query heads of a kv head, within the buffer
  __device__ __forceinline__ bool tall() const { return rows > kFew; }
  __device__ __forceinline__ int tiles() const {
    return tall() ? (rows + kPreRows - 1) / kPreRows : (rows + kRows - 1) / kRows;
  }
  __device__ __forceinline__ int steps() const { return rows > 0 ? max(1, s1 - s0) : 0; }
};

__device__ __forceinline__ int steps_of(int kv) { return (kv + kStep - 1) / kStep; }

constexpr int kW = kPlanThr / 64;

// Inclusive sums of two values over the workgroup; `total` those of all.
__device__ __forceinline__ void block_sums(int64_t v[2], int64_t (*part)[2], int64_t total[2]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
      const int64_t u = __shfl_up(static_cast<long long>(v[k]), o, 64);
      if (lane >= o) v[k] += u;
    }
  __syncthreads();  // (part's last readers)
  if (lane == 63) {
    part[wave][0] = v[0];
    part[wave][1] = v[1];
  }
  __syncthreads();
  total[0] = total[1] = 0;
#pragma unroll
  for (int w = 0; w < kW; ++w)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int64_t u = part[w][k];
      if (w < wave) v[k] += u;
      total[k] += u;
    }
}

__global__ __launch_bounds__(kPlanThr) void share_plan(Att A, Share S) {
  extern __shared__ int32_t sh[];
  __shared__ int64_t part[kW][2];
  __shared__ float sums[kW];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, Gr = S.groups;
  int32_t* const start = sh;            // [Gr + 1]
  int32_t* const lead = start + Gr + 1; // [Gr]: the first request that takes part,
  int32_t* const many = lead + Gr;      // how many do,
  int32_t* const row0 = many + Gr;      // their first row and the end of their last one;
  int32_t* const row1 = row0 + Gr;
  int32_t* const cuts = row1 + Gr;      // parts of the prefix, its first partial row
  int32_t* const slots = cuts + Gr;
  for (int g = tid; g <= Gr && Gr > 0; g += kPlanThr) {
    start[g] = S.group_start[g];
    if (g < Gr) {
      lead[g] = row0[g] = INT32_MAX;
      many[g] = row1[g] = 0;
    }
  }
  __syncthreads();
  // the prefix of a group in whole steps
  auto prefix_of = [&](int g) { return max(S.prefix_lens[g], 0) & ~(kStep - 1); };
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
  auto rows_of = [&](const Req& r) { return r.q0 < 0 ? 0 : r.rows(A); };
  auto takes_part = [&](const Req& r, int prefix) {
    const int64_t sees = int64_t(r.kv) - (A.causal ? r.ql - 1 : 0);  // its first query
    return prefix > 0 && rows_of(r) > 0 && sees >= prefix;
  };
  for (int b = tid; b < A.B; b += kPlanThr) {
    const int g = group_of(b);
    if (g < 0) continue;
    const Req r = request(A, b);
    if (!takes_part(r, prefix_of(g))) continue;
    atomicMin(&lead[g], b);
    atomicAdd(&many[g], 1);
    atomicMin(&row0[g], r.q0);
    atomicMax(&row1[g], r.q0 + rows_of(r));
  }
  __syncthreads();
  // items: g of groups, then b of requests
  auto group_item = [&](int g) {
    Item it{0, 0, 0, 0, 0, 0};
    if (many[g] < 2) return it;
    it.kv = prefix_of(g);
    it.q0 = row0[g];
    it.ql = row1[g] - row0[g];
    it.s1 = it.kv / kStep;
    it.rows = it.ql * A.G;
    return it;
  };
  auto own_item = [&](int b, int& g) {
    const Req r = request(A, b);
    g = group_of(b);
    if (g >= 0 && (many[g] < 2 || !takes_part(r, prefix_of(g)))) g = -1;
    Item it{r.q0, r.ql, r.kv, g >= 0 ? prefix_of(g) / kStep : 0, steps_of(r.kv), rows_of(r) * A.G};
    return it;
  };
  const int items = Gr + A.B;
  float sum = 0.f;
  for (int i = tid; i < items; i += kPlanThr) {
    int g;
    const Item it = i < Gr ? group_item(i) : own_item(i - Gr, g);
    sum += (it.tall() ? 1.f : 0.5f) * it.tiles() * it.steps();
  }
  sum = wave_scan(sum);
  if (lane == 63) sums[wave] = sum;
  __syncthreads();
  sum = 0.f;
#pragma unroll
  for (int w = 0; w < kW; ++w) sum += sums[w];
  const int C0 = static_cast<int>(fminf(sum * A.per_target, 1e9f)) + 1;
  const int Ct = max(kLeast, (C0 + 1) & ~1), Cs = max(kLeast, (C0 + kWaves - 1) & ~(kWaves - 1));
  int64_t base[2] = {0, 0};  // pieces (tall ones in the high half), partial rows
  for (int i0 = 0; i0 < items; i0 += kPlanThr) {
    const int i = i0 + tid;
    Item it{0, 0, 0, 0, 0, 0};
    int g = -1;
    if (i < items) it = i < Gr ? group_item(i) : own_item(i - Gr, g);
    const int C = it.tall() ? Ct : Cs;
    const int tiles = it.tiles(), parts = (it.steps() + C - 1) / C;
    const bool join = it.rows > 0 && (i < Gr || g >= 0 || parts > 1);
    const int64_t n = int64_t(tiles) * parts;
    int64_t v[2] = {it.tall() ? n << 32 : n, join ? int64_t(it.rows) * parts : 0}, total[2];
    const int64_t own0 = v[0], own1 = v[1];
    block_sums(v, part, total);
    const int64_t before = base[0] + v[0] - own0, slot = base[1] + v[1] - own1;
    base[0] += total[0];
    base[1] += total[1];
    if (i >= items) continue;
    // (lengths that do not fit q_start may ask for more than there is)
    const int64_t first = it.tall() ? before >> 32 : before & 0xffffffff;
    const bool fits = slot + own1 <= A.nslots && first + n <= (it.tall() ? S.cap_tall : S.cap_short);
    const int32_t at = join && fits ? static_cast<int32_t>(slot) : -1;
    const bool runs = fits && it.rows > 0;
    if (runs) {
      int4* to = S.pieces + 2 * (first + (it.tall() ? 0 : S.cap_tall));
      const int table = i < Gr ? lead[i] : i - Gr, causal = i >= Gr && A.causal;
      for (int t = tiles - 1; t >= 0; --t)
        for (int p = 0; p < parts; ++p) {
          const int s0 = it.s0 + p * C;
          *to++ = make_int4(table, it.q0, it.ql, it.kv);
          *to++ = make_int4(2 * t + causal, s0, min(it.s1, s0 + C), join ? at + p * it.rows : -1);
        }
    }
    if (i < Gr) {
      cuts[i] = runs ? parts : 0;
      slots[i] = at;
    } else {
      S.meta[2 * (i - Gr)] = make_int4(it.q0, at, runs && join ? parts : 0, it.rows);
    }
  }
  if (tid == 0) {
    S.head[0] = static_cast<int32_t>(min(base[0] >> 32, int64_t(S.cap_tall)));
    S.head[1] = static_cast<int32_t>(min(base[0] & 0xffffffff, int64_t(S.cap_short)));
  }
  __syncthreads();
  for (int b = tid; b < A.B; b += kPlanThr) {
    int g;
    const Item it = own_item(b, g);
    int4 m = make_int4(0, 0, 0, 0);
    if (g >= 0) m = make_int4(slots[g], cuts[g], (row1[g] - row0[g]) * A.G, (it.q0 - row0[g]) * A.G);
    S.meta[2 * b + 1] = m;
  }
  // ---- the rows' requests
  if (A.q_start == nullptr) {
    for (int r = tid; r < A.rows; r += kPlanThr) S.row_req[r] = r / A.uniform_q;
    return;
  }
  __syncthreads();
  for (int b = tid; b <= A.B; b += kPlanThr) sh[b] = A.q_start[b];
  __syncthreads();
  for (int r = tid; r < A.rows; r += kPlanThr) {
    int lo = 0, hi = A.B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (sh[mid] <= r) lo = mid;
      else hi = mid;
    }
    const int in = r - sh[lo], ql = A.q_lens ? A.q_lens[lo] : sh[lo + 1] - sh[lo];
    S.row_req[r] = in >= 0 && in < ql ? lo : -1;
  }
}

// A workgroup per (tall piece, kv head), or per two short pieces: four waves each.
template <int D, bool FP8, bool QLO, bool PLO>
__global__ __launch_bounds__(kPreThr, 2) void share8(Att A, Share S) {
  __shared__ v4f sbuf[2][2][4];
  extern __shared__ __align__(16) uint8_t lds[];
  const int tall = S.head[0] * A.H, h = blockIdx.x % A.H;
  auto piece = [&](int at) {
    const int4 x = S.pieces[2 * at], y = S.pieces[2 * at + 1];
    auto same = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    Piece P{};
    P.b = same(x.x);
    P.r = Req{same(x.y), same(x.z), same(x.w)};
    P.rt = same(y.x) >> 1;
    P.causal = same(y.x) & 1;
    P.s0 = same(y.y);
    P.s1 = same(y.z);
    P.slot = same(y.w);
    return P;
  };
  if (static_cast<int>(blockIdx.x) < tall) {
    const Piece P = piece(blockIdx.x / A.H);
    prefill_piece<D, FP8, QLO, PLO, true>(A, P, h, lds, sbuf);
  } else {
    const int half = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
    const int at = 2 * ((blockIdx.x - tall) / A.H) + half, n = S.head[1];
    if (at - half >= n) return;
    // (without a piece of its own the half takes the other's barriers, and has no row or step)
    Piece P{};
    P.slot = -1;
    if (at < n) P = piece(S.cap_tall + at);
    float* const mine = reinterpret_cast<float*>(lds) + half * kWaves * kRows * (D + 6);
    decode_piece<D, FP8, QLO, true>(
        A, P, h, threadIdx.x & 255, reinterpret_cast<float(*)[kRows][D + 4]>(mine),
        reinterpret_cast<float(*)[kRows][2]>(mine + kWaves * kRows * (D + 4)));
  }
}

// Joins the partial results of 4 rows (a query and head each) a workgroup, 16 lanes a row with
// 8 coordinates each; its waves take every fourth part and meet in LDS.
template <int D>
__global__ __launch_bounds__(kThr) void share_join(Att A, Share S) {
  __shared__ float acc[kWaves][4][D + 4], ml[kWaves][4][2];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane >> 4, d0 = 8 * (lane & 15);
  const bool on = d0 < D;
  const int all = A.rows * A.Hq;  // (< 2^28)
  for (int f0 = 4 * blockIdx.x; f0 < all; f0 += 4 * gridDim.x) {
    const int f = min(f0 + r, all - 1), row = f / A.Hq, hq = f - row * A.Hq;
    const int h = hq / A.G, b = S.row_req[row];
    int4 own = make_int4(0, 0, 0, 0), pre = own;
    if (b >= 0) {
      own = S.meta[2 * b];
      pre = S.meta[2 * b + 1];
    }
    const int parts = f0 + r < all && own.z > 0 ? own.z + pre.y : 0;
    const int rr = (row - own.x) * A.G + hq - h * A.G;
    const int64_t base = int64_t(h) * A.nslots + rr;
    float M = -INFINITY, L = 0.f, x[8] = {};
    for (int p0 = wave; __any(p0 < parts); p0 += 4 * kWaves) {
      float m[4], l[4];
      v4f v[4][2];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int p = p0 + kWaves * k;
        m[k] = -INFINITY;
        l[k] = 0.f;
        v[k][0] = v[k][1] = v4f{0.f, 0.f, 0.f, 0.f};
        if (p < parts) {
          const int64_t at = base + (p < own.z ? own.y + p * own.w
                                               : pre.x + (p - own.z) * pre.z + pre.w);
          m[k] = A.part_ml[2 * at];
          l[k] = A.part_ml[2 * at + 1];
          const v4f* const src = reinterpret_cast<const v4f*>(A.part_o + at * D + (on ? d0 : 0));
          v[k][0] = src[0];
          v[k][1] = src[1];
        }
      }
      float mn = M;
#pragma unroll
      for (int k = 0; k < 4; ++k) mn = fmaxf(mn, m[k]);
      const float ref = mn == -INFINITY ? 0.f : mn, e0 = __builtin_amdgcn_exp2f(M - ref);
      L = fall(L, M - ref);
      M = mn;
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] *= e0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float e = __builtin_amdgcn_exp2f(m[k] - ref);
        L += fall(l[k], m[k] - ref);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = fmaf(v[k][j >> 2][j & 3], e, x[j]);
      }
    }
    __syncthreads();  // (the arrays' last readers)
    if (on) {
      *reinterpret_cast<v4f*>(&acc[wave][r][d0]) = v4f{x[0], x[1], x[2], x[3]};
      *reinterpret_cast<v4f*>(&acc[wave][r][d0 + 4]) = v4f{x[4], x[5], x[6], x[7]};
    }
    if (d0 == 0) {
      ml[wave][r][0] = M;
      ml[wave][r][1] = L;
    }
    __syncthreads();
    // wave w: row w
    const int joins = __builtin_amdgcn_readlane(parts, 16 * wave), c = 2 * lane;
    if (c >= D || joins == 0) continue;
    float mx = -INFINITY, sum = 0.f, y0 = 0.f, y1 = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) mx = fmaxf(mx, ml[w][wave][0]);
    const float ref = mx == -INFINITY ? 0.f : mx;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float e = __builtin_amdgcn_exp2f(ml[w][wave][0] - ref);
      sum += fall(ml[w][wave][1], ml[w][wave][0] - ref);
      y0 = fmaf(acc[w][wave][c], e, y0);
      y1 = fmaf(acc[w][wave][c + 1], e, y1);
    }
    const float inv = inverse(sum);
    const int64_t to = int64_t(f0 + wave) * D + c;
    qkv_store(A.out, to, y0 * inv, A.out_dtype);
    qkv_store(A.out, to + 1, y1 * inv, A.out_dtype);
  }
}

// Pieces that a launch aims at, per kv head: one workgroup per CU.
int32_t target_of(int32_t H) { return std::max(1, (qkv_num_cus() + H - 1) / H); }

// Bounds of a launch and its workspace.  Each row is in two items, its group's prefix and its own
// tokens; items of more than kFew rows have tall tiles.  The steps (a short tile's count half)
// are cut so that pieces beyond one a tile are within the target, 2 target for short ones.
struct Layout {
  int64_t tall, shorts;   // pieces
  int64_t rows;           // partial rows of a kv head
  int64_t meta, row_req, pieces, ml, o, bytes;
};
Layout layout(int64_t B, int64_t groups, int64_t rows, int32_t G, int32_t H, int32_t d) {
  Layout L;
  const int64_t t = target_of(H), all = 2 * rows * G;
  const int64_t items = std::min(B + groups, 2 * rows);
  const int64_t high = std::min(items, all / (kFew + 1));   // items of tall tiles
  L.tall = high > 0 ? all / kPreRows + high + t : 0;
  L.shorts = std::min(2 * items, all / kRows + items) + 2 * t;
  L.rows = all + (high > 0 ? kPreRows * t : 0) + 2 * kRows * t;
  auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
  L.meta = 256;
  L.row_req = L.meta + up(32 * B);
  L.pieces = L.row_req + up(4 * rows);
  L.ml = L.pieces + up(32 * (L.tall + L.shorts));
  L.o = L.ml + up(8 * H * L.rows);
  L.bytes = L.o + up(4 * H * L.rows * d);
  return L;
}

template <int D, bool FP8, bool QLO, bool PLO>
void start(const Att& A, const Share& S, uint32_t grid, hipStream_t s) {
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
  share8<D, FP8, QLO, PLO><<<grid, kPreThr, smem, s>>>(A, S);
}

template <int D, bool FP8>
void run(const Att& A, const Share& S, uint32_t grid, hipStream_t s) {
  if (A.q_dtype == QKV_F32) start<D, FP8, true, true>(A, S, grid, s);
  else if (A.out_dtype != QKV_BF16) start<D, FP8, false, true>(A, S, grid, s);
  else start<D, FP8, false, false>(A, S, grid, s);
}

}  // namespace

extern "C" int64_t qkv_kv8_attention_shared_workspace_bytes(int32_t B, int32_t groups, int64_t rows,
                                                            int32_t Hq, int32_t Hkv, int32_t d) {
  if (Hkv < 1 || d < 1) return 0;
  if (B < 1 || rows < 1) return 256;
  return layout(B, std::max(groups, 0), rows, Hq / Hkv, Hkv, d).bytes;
}

extern "C" int qkv_kv8_attention_shared(
    const void* q, int32_t q_dtype, int64_t q_row_stride, int64_t q_head_stride, int64_t rows,
    const void* kpool, const float* kscale, const void* vpool, const float* vscale, int32_t fmt,
    int32_t num_pages, int32_t page_tokens, const int32_t* table, int32_t pages_per_seq,
    const int32_t* group_start, const int32_t* prefix_lens, int32_t groups, const int32_t* q_start,
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
  QKV_REQUIRE(workspace && qkv_aligned(workspace, 256) && ws_bytes >= L.bytes,
              "qkv_kv8_attention_shared: workspace too small or not 256-byte aligned");
  QKV_REQUIRE(L.rows < INT32_MAX && (L.tall + L.shorts) * Hkv < INT32_MAX,
              "batch of %d requests and %lld rows is too large for one call", B,
              static_cast<long long>(rows));
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
  Share S{group_start,
          prefix_lens,
          groups,
          reinterpret_cast<int32_t*>(ws),
          reinterpret_cast<int4*>(ws + L.pieces),
          static_cast<int32_t>(L.tall),
          static_cast<int32_t>(L.shorts),
          reinterpret_cast<int4*>(ws + L.meta),
          reinterpret_cast<int32_t*>(ws + L.row_req)};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const uint32_t lds = std::max(7 * groups + 1, B + 1) * sizeof(int32_t);
  share_plan<<<1, kPlanThr, lds, s>>>(A, S);
  QKV_LAUNCHED();
  const uint32_t grid = static_cast<uint32_t>((L.tall + (L.shorts + 1) / 2) * Hkv);
  if (fmt == QKV_CODES_I8) {
    if (d == 128) run<128, false>(A, S, grid, s);
    else if (d == 96) run<96, false>(A, S, grid, s);
    else run<64, false>(A, S, grid, s);
  } else {
    if (d == 128) run<128, true>(A, S, grid, s);
    else if (d == 96) run<96, true>(A, S, grid, s);
    else run<64, true>(A, S, grid, s);
  }
  QKV_LAUNCHED();
  const uint32_t joins = static_cast<uint32_t>(std::min<int64_t>((rows * Hq + 3) / 4, 2048));
  if (d == 128) share_join<128><<<joins, kThr, 0, s>>>(A, S);
  else if (d == 96) share_join<96><<<joins, kThr, 0, s>>>(A, S);
  else share_join<64><<<joins, kThr, 0, s>>>(A, S);
  QKV_LAUNCHED();
  return QKV_OK;
}
