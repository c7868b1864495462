// What decode8 (qkv_kv8_attn.hip) and prefill8 (qkv_kv8_prefill.hip) share.
#pragma once

#include <algorithm>
#include <type_traits>

#include "qkv_kv8.h"

namespace qkv_kv8 {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));

constexpr int kStep = 64;        // tokens of a wave's step
constexpr int kRows = 16;        // query rows of a decode tile
constexpr int kPreRows = 128;    // and of a prefill tile
constexpr int kWaves = 4;
constexpr int kThr = 64 * kWaves;
constexpr float kHead = 8.f;     // the running maximum may lag by 2^8 before a rescale
constexpr float kUp = 7.f;       // largest weight in f16: 2^(kUp + kHead) at most, 2^kUp at least,
                                 // so that f16's smallest step is 2^-31 of it
// The sum of weights p' / vs is kept times this.  (The weights take it, not 1 / vs, which at
// the largest scales, 2^121, would leave the normal fp32.)  With weights from 2^kUp to
// 2^(kUp + kHead) it lies between 2^(kUp - 10 - 121) and tokens x 2^(kUp + kHead - 10) / vs:
// in range for 2^22 tokens at the smallest scale, 2^-100, and for 2^31 at 2^-91.
// Weights below 2^-126 are 0.  They are relative to the largest p vs, so the sum is whole where
// the value scales of a request and head, other than 0, lie within 2^80 of each other: of
// 2^22 tokens that together are 2^-24 of the sum, each at a scale 2^80 smaller is
// 2^(kUp - 46 - 80) = 2^-119.  (fp16 values are within 2^40.)
constexpr float kSum = 0x1p-10f;
// Below this a value scale counts as that of a block of zeros: append makes none but 0, yet
// what lies behind the cached tokens may be anything, and 1 / scale has to be finite.
constexpr float kLeast = 0x1p-126f;
constexpr float kZero = 100.f;   // see stand_in
constexpr float kLog2e = 1.44269504088896340736f;

struct Att {
  const void* q;
  int64_t q_ts, q_hs;
  int32_t q_dtype, q_vec;
  int32_t rows;
  const uint8_t* kpool;
  const float* kscale;
  const uint8_t* vpool;
  const float* vscale;
  int32_t npages, lg;
  const int32_t* table;
  int32_t width;
  const int32_t* q_start;
  const int32_t* q_lens;
  const int32_t* kv_lens;
  int32_t B, Hq, H, G, uniform_q;
  float scale;
  int32_t causal;
  void* out;
  int32_t out_dtype, out_vec;
  int32_t few;      // requests of up to this many rows (queries x G) are decode8's
  int32_t least;    // steps of the shortest piece, INT32_MAX / 2: nothing is cut
  int32_t target;   // pieces that a launch aims at, per kv head
  float per_target; // 1 / target
  int32_t nslots;   // partial results that the workspace holds
  int32_t* used;    // [0]: of them, per kv head, in this launch; [1], [2]: pieces and C (plan)
  int4* desc;       // [slot][H]: whose they are
  int4* plan;       // [piece]: request, piece of it, its first slot; null: the kernels' own
  float* part_o;    // [slot][H][row][D]
  float* part_ml;   // [slot][H][row][2]
};

// Request b's rows, as its lengths have them, and its tokens.  Rows behind the buffer are no
// part of any tile: they would push others' tiles out of the grid.
struct Req {
  int32_t q0, ql, kv;
  __device__ __forceinline__ int rows(const Att& A) const {
    return max(0, min(ql, A.rows - max(q0, 0)));
  }
};

__device__ __forceinline__ Req request(const Att& A, int b) {
  Req r;
  if (A.q_start == nullptr) {
    r.q0 = b * A.uniform_q;
    r.ql = A.uniform_q;
  } else {
    r.q0 = A.q_start[b];
    r.ql = A.q_lens ? A.q_lens[b] : A.q_start[b + 1] - r.q0;
    r.ql = max(r.ql, 0);
  }
  int64_t room = int64_t(A.width) << A.lg;
  if (room > QKV_PAGED_TOKENS) room = QKV_PAGED_TOKENS;
  const int64_t kv = A.kv_lens[b];
  r.kv = static_cast<int32_t>(kv < 0 ? 0 : kv < room ? kv : room);
  return r;
}

// One workgroup's part of the launch: steps [s0, s1) of tile `rt` of request b.
struct Piece {
  Req r;
  int32_t b, rt, s0, s1;
  int32_t slot;   // of its partial result, -1: the tile is not cut
  int32_t part, parts;
};

// Inclusive sum over a wave's lanes.
template <typename T>
__device__ __forceinline__ T wave_scan(T v) {
  auto add = [&](auto ctrl, auto mask) {
    const int u = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), decltype(ctrl)::value,
                                              decltype(mask)::value, 0xf, false);
    v += __builtin_bit_cast(T, u);
  };
  using std::integral_constant;
  add(integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{});  // row_shr 1, 2, 4, 8
  add(integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{});
  add(integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{});
  add(integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{});
  add(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});  // row_bcast 15, 31
  add(integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});
  return v;
}
template <typename T>
__device__ __forceinline__ T lane_value(T v, int lane) {
  return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}

// How a launch's work is cut.  A launch has the tiles of ROWS query rows of the requests that
// are its own (rows up to A.few: decode8's 16-row tiles; more: prefill8's).  A tile's steps
// are cut into pieces of C, the smallest C that keeps the launch near its target of pieces;
// so long requests are shared by many workgroups and short ones are not cut.  (prefill8 cuts
// nothing where the tiles alone reach the target: its partial results cost more.)
template <int ROWS>
struct Cut {
  static constexpr bool PRE = ROWS == kPreRows;
  static constexpr int ROUND = PRE ? 2 : kWaves;  // steps that a workgroup takes at once
  static __device__ __forceinline__ void cost(const Att& A, const Req& r, int& tiles, int& steps) {
    const int n = r.rows(A) * A.G;
    tiles = (n > A.few) == PRE ? (n + ROWS - 1) / ROWS : 0;
    steps = max(1, (r.kv + kStep - 1) / kStep);
  }
  // sum: of tiles times steps (rounded alike in every workgroup; C is above its share in
  // any case), all: tiles
  static __device__ __forceinline__ int length(const Att& A, float sum, int all) {
    if (PRE && all >= A.target) return INT32_MAX / 2;
    const int c = static_cast<int>(fminf(sum * A.per_target, 1e9f)) + 1;
    return max(A.least, (c + ROUND - 1) / ROUND * ROUND);
  }
  // whole prefill tiles: the last ones first, of a causal prompt the longest
  static __device__ __forceinline__ bool reversed(int C) { return PRE && C == INT32_MAX / 2; }
};

// Piece number `want` of the launch.  Up to 64 requests every wave finds it by prefix sums
// over them, so that no launch and no host knowledge of the lengths is needed, and
// workgroup 0 tells the join how many partial results there are.  More requests are
// planned by a launch of their own (plan8).
template <int ROWS>
__device__ __forceinline__ bool locate(const Att& A, int want, Piece& P) {
  using K = Cut<ROWS>;
  const int lane = threadIdx.x & 63;
  int C, in, slot0, steps;
  if (A.plan == nullptr) {
    Req r{0, 0, 0};
    int tiles = 0, st = 1;
    if (lane < A.B) {
      r = request(A, lane);
      K::cost(A, r, tiles, st);
    }
    const float sum = lane_value(wave_scan(static_cast<float>(tiles) * st), 63);
    const int all = K::PRE ? lane_value(wave_scan(tiles), 63) : 0;
    C = K::length(A, sum, all);
    // prefill8's workgroups have a CU each, and one piece too many would run behind all others
    // (4 chunks of 400 rows over 1500 tokens, 14 / 2 heads: 49 -> 27 us): C grows until
    // the pieces are within the target, as at last they are, being the tiles
    if (K::PRE && all < A.target)
      while (lane_value(wave_scan(tiles * ((st + C - 1) / C)), 63) > A.target)
        C += max(K::ROUND, C / 8 / K::ROUND * K::ROUND);
    if (K::reversed(C)) want = want < all ? all - 1 - want : INT32_MAX;
    const int per = (st + C - 1) / C, mine = tiles * per, cut = per > 1 ? mine : 0;
    const int end = wave_scan(mine), cuts = wave_scan(cut);
    if (blockIdx.x == 0 && threadIdx.x == 0) A.used[0] = lane_value(cuts, 63);
    const uint64_t hit = __ballot(want >= end - mine && want < end);
    if (hit == 0) return false;
    P.b = __builtin_ctzll(hit);
    in = want - lane_value(end - mine, P.b);
    slot0 = lane_value(cuts - cut, P.b);
    steps = lane_value(st, P.b);
    P.r = Req{lane_value(r.q0, P.b), lane_value(r.ql, P.b), lane_value(r.kv, P.b)};
  } else {
    if (want >= A.used[1]) return false;
    const int4 e = A.plan[want];
    C = A.used[2];
    P.b = __builtin_amdgcn_readfirstlane(e.x);
    in = __builtin_amdgcn_readfirstlane(e.y);
    slot0 = __builtin_amdgcn_readfirstlane(e.z);
    P.r = request(A, P.b);
    int tiles;
    K::cost(A, P.r, tiles, steps);
  }
  P.parts = (steps + C - 1) / C;
  P.rt = in / P.parts;
  P.part = in - P.rt * P.parts;
  P.s0 = P.part * C;
  P.s1 = min(steps, P.s0 + C);
  P.slot = P.parts > 1 ? slot0 + in : -1;
  return true;
}

constexpr int kPlanThr = 1024;
constexpr int kMaxB = 16000;  // requests of a call (their prefix sums fit 64 KiB of LDS)

// Lists the pieces of a launch, at most `cap`, for more requests than a wave has lanes: one
// workgroup.  (Every workgroup summing over all requests for itself took 147 us at 1000
// requests of 100 tokens, 8 kv heads, d = 128.)
template <int ROWS>
__global__ __launch_bounds__(kPlanThr) void plan8(Att A, int cap) {
  using K = Cut<ROWS>;
  constexpr int W = kPlanThr / 64;
  extern __shared__ int32_t ends[];  // [B + 1] pieces of the requests before b
  __shared__ float sums[W];
  __shared__ int32_t part[W][2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  float sum = 0.f;
  int all = 0;
  for (int b = tid; b < A.B; b += kPlanThr) {
    int tiles, st;
    K::cost(A, request(A, b), tiles, st);
    sum += static_cast<float>(tiles) * st;
    all += tiles;
  }
  sum = wave_scan(sum);
  all = wave_scan(all);
  if (lane == 63) {
    sums[wave] = sum;
    part[wave][0] = all;
  }
  if (tid == 0) ends[0] = 0;
  __syncthreads();
  sum = 0.f;
  all = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    sum += sums[w];
    all += part[w][0];
  }
  const int C = K::length(A, sum, all);
  int base[2] = {0, 0};  // pieces, pieces of cut tiles
  for (int b0 = 0; b0 < A.B; b0 += kPlanThr) {
    const int b = b0 + tid;
    int own[2] = {0, 0}, v[2];
    if (b < A.B) {
      int tiles, st;
      K::cost(A, request(A, b), tiles, st);
      const int per = (st + C - 1) / C;
      own[0] = tiles * per;
      own[1] = per > 1 ? own[0] : 0;
    }
    __syncthreads();  // (part's last readers)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      v[k] = wave_scan(own[k]);
      if (lane == 63) part[wave][k] = v[k];
    }
    __syncthreads();
    int tot[2] = {0, 0};
#pragma unroll
    for (int w = 0; w < W; ++w)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (w < wave) v[k] += part[w][k];
        tot[k] += part[w][k];
      }
    // a request's first piece carries its first slot until all are listed
    if (b < A.B) {
      ends[b + 1] = base[0] + v[0];
      const int first = base[0] + v[0] - own[0];
      if (own[0] > 0 && first < cap) A.plan[first].w = base[1] + v[1] - own[1];
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) base[k] += tot[k];
  }
  __syncthreads();
  const int total = min(base[0], cap);
  if (tid == 0) {
    A.used[0] = base[1];
    A.used[1] = total;
    A.used[2] = C;
  }
  for (int p = tid; p < total; p += kPlanThr) {
    int lo = 0, hi = A.B;  // ends[lo] <= p < ends[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (ends[mid] <= p) lo = mid;
      else hi = mid;
    }
    int4* const to = A.plan + (K::reversed(C) ? total - 1 - p : p);
    const int slot0 = K::reversed(C) ? 0 : A.plan[ends[lo]].w;
    to->x = lo;
    to->y = p - ends[lo];
    to->z = slot0;
  }
}

// Where the piece's partial result goes, in units of [slot][H], or -1 past the workspace.
__device__ __forceinline__ int64_t place(const Att& A, const Piece& P, int h) {
  const int64_t at = int64_t(P.slot) * A.H + h;
  if (at >= A.nslots) return -1;
  if (threadIdx.x == 0) A.desc[at] = make_int4(P.part == 0 ? P.parts : 0, P.r.q0, P.r.ql, P.rt);
  return at;
}

// Two codes as f16, of bytes 0 and 1 (or 2 and 3) of a dword.
template <bool FP8>
__device__ __forceinline__ void widen(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (FP8) {
    lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false));
    hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true));
  } else {
    // 0x6400 | u is the f16 1024 + u; u = code + 128
    const uint32_t u = w ^ 0x80808080u;
    const v2h off = {static_cast<_Float16>(-1152.f), static_cast<_Float16>(-1152.f)};
    lo = __builtin_bit_cast(
        uint32_t, __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) + off);
    hi = __builtin_bit_cast(
        uint32_t, __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) + off);
  }
}

template <bool FP8>
__device__ __forceinline__ v8h widen8(uint32_t a, uint32_t b) {
  v4u r;
  uint32_t x, y;
  widen<FP8>(a, x, y);
  r[0] = x;
  r[1] = y;
  widen<FP8>(b, x, y);
  r[2] = x;
  r[3] = y;
  return __builtin_bit_cast(v8h, r);
}

__device__ __forceinline__ uint32_t pk(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f{a, b}), v2h));
}

// x as f16 hi + lo, both rounded to nearest.
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = pk(a, b);
  const v2h h = __builtin_bit_cast(v2h, hi);
  lo = pk(a - static_cast<float>(h[0]), b - static_cast<float>(h[1]));
}

__device__ __forceinline__ v4f mfma(v8h a, v8h b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// A lane's part of its query row (element `at` on; 8 values from col(k) on for each product
// step k) as f16, times a power of two that brings the row's largest into [2^9, 2^10):
// 16-bit types are exact so, fp32 takes lo beside it.  Lanes FIRST and 32 apart share a row.
// c: what turns a score of these into an exponent of 2.  stage: THR * 8 KS floats of LDS.
template <int KS, bool LO, int THR, int FIRST, typename Col>
__device__ __forceinline__ void load_query(const Att& A, int64_t at, bool live, Col col,
                                           float* stage, v8h* qh, v8h* ql, float& c) {
  float x[KS][8];
  if (A.q_vec && A.q_dtype != QKV_F32) {
    v4u w[KS];
#pragma unroll
    for (int k = 0; k < KS; ++k)
      w[k] = live ? *reinterpret_cast<const v4u*>(static_cast<const uint16_t*>(A.q) + at + col(k))
                  : v4u{0, 0, 0, 0};
    if (A.q_dtype == QKV_BF16) {
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int j = 0; j < 8; ++j)
          x[k][j] = __uint_as_float(j & 1 ? w[k][j >> 1] & 0xffff0000u : w[k][j >> 1] << 16);
    } else {
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int j = 0; j < 8; ++j)
          x[k][j] = static_cast<float>(__builtin_bit_cast(v8h, w[k])[j]);
    }
  } else if (A.q_vec) {
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const v4f* const p = reinterpret_cast<const v4f*>(static_cast<const float*>(A.q) + at + col(k));
      const v4f a = live ? p[0] : v4f{0.f, 0.f, 0.f, 0.f}, b = live ? p[1] : v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < 8; ++j) x[k][j] = j < 4 ? a[j & 3] : b[j & 3];
    }
  } else {  // (rolled, through LDS: it runs once, and unrolled it would be most of the code)
    float* const t = stage + threadIdx.x;
#pragma unroll 1
    for (int k = 0; k < KS; ++k)
#pragma unroll 1
      for (int j = 0; j < 8; ++j)
        t[(8 * k + j) * THR] = live ? qkv_load(A.q, at + col(k) + j, A.q_dtype) : 0.f;
#pragma unroll
    for (int i = 0; i < 8 * KS; ++i) x[i >> 3][i & 7] = t[i * THR];
    __syncthreads();
  }
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 8 * KS; ++i) amax = fmaxf(amax, fabsf(x[i >> 3][i & 7]));
#pragma unroll
  for (int o = FIRST; o < 64; o *= 2) amax = fmaxf(amax, __shfl_xor(amax, o, 64));
  int ex = 0;
  if (amax > 0.f && amax < INFINITY) frexpf(amax, &ex);
  ex = max(ex, -110);
  const float up = ldexpf(1.f, 10 - ex);
  c = ldexpf(A.scale * kLog2e, ex - 10);
#pragma unroll
  for (int k = 0; k < KS; ++k) {
    v4u hi, lo;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t a, b;
      split2(x[k][2 * j] * up, x[k][2 * j + 1] * up, a, b);
      hi[j] = a;
      lo[j] = b;
    }
    qh[k] = __builtin_bit_cast(v8h, hi);
    if constexpr (LO) ql[k] = __builtin_bit_cast(v8h, lo);
  }
}

// Tokens below this are seen by query qi of the piece's request.
__device__ __forceinline__ int limit(const Att& A, const Req& r, int qi) {
  return A.causal ? min(r.kv, r.kv - r.ql + qi + 1) : r.kv;
}

// What a block whose scale counts as 0 takes in place of log2(scale).  Its values are 0, so
// its weights are part of the sum alone, and any number does that keeps them in range.  One
// for all blocks does not: beside blocks of small scales it raises the maximum until their
// f16 weights vanish (scale 1 beside values of 1e-6: 1e-2 off), beside large ones its own
// weights vanish from the sum.  So a lane takes what brings the largest of its weights
// (exponent `top`) to the maximum m of the blocks so far and of the step's others, within
// [-kZero, kZero]: the maximum is raised only by a block 2^kZero above it, or by the first one.
__device__ __forceinline__ float stand_in(float top, float m) {
  return m == -INFINITY ? -kZero : fminf(fmaxf(m - top, -kZero), kZero);
}

// l times 2^d, d <= 0, in two factors: of zero blocks alone, l may be 2^kZero above a sum
// beside large scales, and d below the exponents of fp32.
__device__ __forceinline__ float fall(float l, float d) {
  return l * __builtin_amdgcn_exp2f(fminf(d + kZero, 0.f)) *
         __builtin_amdgcn_exp2f(fmaxf(d, -kZero));
}

// Of a sum of weights: 0 of a row that saw nothing, and a query's NaN is the result's.  (It
// leaves m at -inf; the joins take such parts too, whose 2^(m - M) = 0 keeps a NaN.)
__device__ __forceinline__ float inverse(float l) { return l == 0.f ? 0.f : kSum / l; }

// Eight consecutive results to element `at` of out.
__device__ __forceinline__ void store8(void* out, int64_t at, const float* x, int dt, bool vec) {
  if (!vec) {
#pragma unroll
    for (int j = 0; j < 8; ++j) qkv_store(out, at + j, x[j], dt);
  } else if (dt == QKV_F32) {
    v4f* p = reinterpret_cast<v4f*>(static_cast<float*>(out) + at);
    p[0] = v4f{x[0], x[1], x[2], x[3]};
    p[1] = v4f{x[4], x[5], x[6], x[7]};
  } else if (dt == QKV_F16) {
    *reinterpret_cast<v4u*>(static_cast<uint16_t*>(out) + at) =
        v4u{pk(x[0], x[1]), pk(x[2], x[3]), pk(x[4], x[5]), pk(x[6], x[7])};
  } else {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      w[j] = qkv_f32_to_bf16(x[2 * j]) | uint32_t(qkv_f32_to_bf16(x[2 * j + 1])) << 16;
    *reinterpret_cast<v4u*>(static_cast<uint16_t*>(out) + at) = v4u{w[0], w[1], w[2], w[3]};
  }
}

// Four of them.
__device__ __forceinline__ void store4(void* out, int64_t at, const float* x, int dt, bool vec) {
  if (!vec) {
#pragma unroll
    for (int j = 0; j < 4; ++j) qkv_store(out, at + j, x[j], dt);
  } else if (dt == QKV_F32) {
    *reinterpret_cast<v4f*>(static_cast<float*>(out) + at) = v4f{x[0], x[1], x[2], x[3]};
  } else if (dt == QKV_F16) {
    *reinterpret_cast<v2u*>(static_cast<uint16_t*>(out) + at) = v2u{pk(x[0], x[1]), pk(x[2], x[3])};
  } else {
    *reinterpret_cast<v2u*>(static_cast<uint16_t*>(out) + at) =
        v2u{qkv_f32_to_bf16(x[0]) | uint32_t(qkv_f32_to_bf16(x[1])) << 16,
            qkv_f32_to_bf16(x[2]) | uint32_t(qkv_f32_to_bf16(x[3])) << 16};
  }
}

// Joins the pieces of cut tiles, 4 rows of a tile a wave, 8 coordinates a lane.  Decode
// tiles have many pieces and few rows: a workgroup takes 4 rows, its waves every fourth
// piece, and they meet in LDS.  Prefill tiles have many rows and few pieces: a workgroup
// takes 16 rows.
// (workgroup `block` of `blocks`)
template <int D, int ROWS>
__device__ __forceinline__ void join_tiles(const Att& A, int block, int blocks) {
  constexpr bool DEAL = ROWS == kRows;  // pieces to the waves
  constexpr int UR = DEAL ? 4 : 4 * kWaves, GR = ROWS / UR;
  __shared__ float acc[DEAL ? kWaves : 1][4][D + 4], ml[DEAL ? kWaves : 1][4][2];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane >> 4, d0 = 8 * (lane & 15);
  const bool on = d0 < D;
  const int64_t units = int64_t(min(*A.used, A.nslots / A.H)) * A.H * GR;
  for (int64_t u = block; u < units; u += blocks) {
    const int64_t at = u / GR;  // slot * H + h
    const int4 t = A.desc[at];
    const int parts = t.x, h = static_cast<int>(at % A.H);
    const int rr0 = UR * static_cast<int>(u % GR) + (DEAL ? 0 : 4 * wave);
    // (0: not the tile's first piece; lengths that do not fit q_start may leave a slot unset)
    if (parts <= 0 || parts > A.nslots || t.w < 0 || int64_t(t.w) * ROWS > int64_t(A.rows) * A.G ||
        (t.w * ROWS + rr0) / A.G >= t.z)
      continue;
    float M = -INFINITY, L = 0.f, x[8] = {};
    constexpr int EVERY = DEAL ? kWaves : 1;
    for (int p = DEAL ? wave : 0; p < parts; p += 4 * EVERY) {
      float m[4], l[4];
      v4f v[4][2];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int q = p + EVERY * k;
        const int64_t s = at + int64_t(q < parts ? q : p) * A.H;
        const int64_t row = (s < A.nslots ? s : at) * ROWS + rr0 + r;
        m[k] = q < parts ? A.part_ml[2 * row] : -INFINITY;
        l[k] = A.part_ml[2 * row + 1];
        const v4f* const src =
            reinterpret_cast<const v4f*>(A.part_o + row * D + (on ? d0 : 0));
        v[k][0] = src[0];
        v[k][1] = src[1];
      }
      float mn = M;
#pragma unroll
      for (int k = 0; k < 4; ++k) mn = fmaxf(mn, m[k]);
      const float ref = mn == -INFINITY ? 0.f : mn, f = __builtin_amdgcn_exp2f(M - ref);
      L = fall(L, M - ref);
      M = mn;
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] *= f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float e = __builtin_amdgcn_exp2f(m[k] - ref);
        L += fall(l[k], m[k] - ref);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = fmaf(v[k][j >> 2][j & 3], e, x[j]);
      }
    }
    if constexpr (!DEAL) {
      const int rr = t.w * ROWS + rr0 + r, qi = rr / A.G;
      const int64_t row = int64_t(t.y) + qi;
      if (!on || qi >= t.z || row < 0 || row >= A.rows) continue;
      const float inv = inverse(L);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] *= inv;
      store8(A.out, (row * A.Hq + h * A.G + rr - qi * A.G) * D + d0, x, A.out_dtype, A.out_vec);
    } else {
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
      const int rr = t.w * ROWS + rr0 + wave, qi = rr / A.G, c = 2 * lane;
      const int64_t row = int64_t(t.y) + qi;
      if (c >= D || qi >= t.z || row < 0 || row >= A.rows) continue;
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
      const int64_t to = (row * A.Hq + h * A.G + rr - qi * A.G) * D + c;
      qkv_store(A.out, to, y0 * inv, A.out_dtype);
      qkv_store(A.out, to + 1, y1 * inv, A.out_dtype);
    }
  }
}

template <int D, int ROWS>
__global__ __launch_bounds__(kThr) void join8(Att A) {
  join_tiles<D, ROWS>(A, blockIdx.x, gridDim.x);
}

// Both kernels' tiles in one launch, the first `split` workgroups decode8's.  (12 requests,
// chunks of up to 301 rows beside decoding ones: 6.1 us instead of 3 + 5 and a launch; the call
// 27.1 -> 24.6, now 25.1.)
template <int D>
__global__ __launch_bounds__(kThr) void join_both8(Att A, Att P, int split) {
  const int b = blockIdx.x;
  if (b < split) join_tiles<D, kRows>(A, b, split);
  else join_tiles<D, kPreRows>(P, b - split, gridDim.x - split);
}

// Workgroups of a join: the units are counted on the device.
inline uint32_t join_grid(const Att& A, int rows) {
  const int64_t units = int64_t(A.nslots) * (rows == kRows ? kRows / 4 : rows / (4 * kWaves));
  return static_cast<uint32_t>(std::min<int64_t>(units, 1024));
}

}  // namespace qkv_kv8

// Launches prefill8 over up to `pieces` pieces (a bound) per kv head.
void qkv_kv8_prefill(const qkv_kv8::Att& A, int32_t d, bool fp8, uint32_t pieces,
                     hipStream_t s);
