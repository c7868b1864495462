// Attention of a ragged batch of queries over the 8-bit paged cache (qkv_kv8.h).
//
// Mathematics.  With block scales ks, vs (16 tokens and a head each), codes kc, vc and
// c = scale log2(e):  y_t = c ks (q . kc_t) + log2(vs),  p'_t = 2^(y_t - m),
//   out = (sum p'_t vc_t) / (sum p'_t / vs):
// the value scale enters the softmax's exponent, where it costs an addend of a
// multiply-add instead of a product per weight, and the running maximum m is taken
// over y, so that a weight's 16 bits are spent where |p v| is large.  Codes are exact
// in f16, and so are 16-bit queries times a power of two per row; fp32 queries and the weights
// are f16 pairs hi + lo (22 bits).  (Weights of one f16 for bf16 results were no faster:
// 32 x 8192 tokens 87.0 us, with pairs 86.0.)
//
// Layout.  Scores are S^T = K Q^T on v_mfma_f32_16x16x32_f16 (rows tokens, columns the
// query rows that share a kv head), values O^T = V^T P^T.  Row m of score tile i is token
// 16 (m / 4) + 4 i + m % 4 of 64, so that lane (n, g) holds the scores of query row n and of
// all 16 tokens of block g: one pair of scales per lane, and its weights are, as they
// stand, the B operand of the value product, whose A operand is 16 bytes of a V block.
// Nothing of K, V or P passes through LDS.
//
// Bound: HBM, 2 d + 1/2 bytes per token and kv head.  A wave has a step's K and V (16 KiB at
// d = 128) in flight while it works on the step before; four waves a CU keep 64 KiB.
// Measured, a call among others with its join: 32 x 8192 tokens, 32 / 8 heads, d = 128, bf16:
// 86 us, 6.3 TB/s (a read-only probe over as many bytes: 7.0); 131,072 tokens of one request
// 50 us (5.4 TB/s); 40 requests up to 9001 tokens, d = 96, e4m3: 33 us (4.1 TB/s).  One VALU
// kernel with a wave per query and head took 1791 us for the first.
// Small calls are the chain lengths - page - bytes - merge: 7 us (16 x 2048 tokens, 2 kv
// heads, d = 64), and the launches.
#include "qkv_kv8_attn.h"

namespace {

using namespace qkv_kv8;

// d index of the first of the 8 coordinates that lane group g holds in product step ks
__host__ __device__ constexpr int dcol(int D, int ks, int g) {
  return D == 96 && ks == 2 ? 64 + 8 * g : 64 * (ks >> 1) + 16 * g + 8 * (ks & 1);
}

// A workgroup per (piece, kv head): its waves take every fourth step of 64 tokens and
// merge through LDS.
template <int D, bool FP8, bool QLO>
__global__ __launch_bounds__(kThr, 2) void decode8(Att A) {
  constexpr int KS = D / 32, NJ = D / 16, NK = (D + 63) / 64;
  __shared__ float red_o[kWaves][kRows][D + 4];
  __shared__ float red_ml[kWaves][kRows][2];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int h = blockIdx.x % A.H;
  Piece P;
  if (!locate<kRows>(A, blockIdx.x / A.H, P)) return;

  // ---- this lane's query row
  const int rr = P.rt * kRows + n, qi = rr / A.G, gq = rr - qi * A.G;
  const int64_t row = int64_t(P.r.q0) + qi;
  const bool live = qi < P.r.ql && row >= 0 && row < A.rows;
  const int hq = h * A.G + gq;
  // tokens below lim are seen; all live rows of the tile see those below lim_all (its first
  // row's: rows are query-major)
  const int lim = live ? limit(A, P.r, qi) : 0;
  const int lim_all = limit(A, P.r, P.rt * kRows / A.G);
  const int n_tok = P.r.kv;

  v4f o[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) o[j] = v4f{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;

  // K and V of the step that follows, in registers
  v4u kr[4][NK];
  v4u vr[NJ];
  float ks_r = 0.f, vs_r = 0.f;
  const int pg_sh = A.lg - 6;  // steps per page, log2
  const int32_t* const tab = A.table + int64_t(P.b) * A.width;
  int pages = 0;   // lane i: the page of this wave's i-th step from p_first on
  int p_first = 0;
  const int tok0 = 16 * (n >> 2) + (n & 3);
  const uint32_t k_off = static_cast<uint32_t>(tok0 * D + 16 * g);
  const uint32_t k_off2 = static_cast<uint32_t>(tok0 * D + 64 + 8 * g);  // D = 96: 8 bytes each
  const uint32_t v_off = static_cast<uint32_t>((g * D + n) * 16);
  auto page_of = [&](int i) {  // i: the wave's step count
    if (i - p_first >= 64 || i == 0) {
      p_first = i;
      const int st = P.s0 + wave + kWaves * (i + lane);
      pages = st < P.s1 ? tab[st >> pg_sh] : -1;
    }
    return __builtin_amdgcn_readlane(pages, i - p_first);
  };
  auto row_of = [&](int i, bool& ok) {
    const int pg = page_of(i);
    ok = pg >= 0 && pg < A.npages;
    const int st = P.s0 + wave + kWaves * i;
    const int64_t t = int64_t(st) * kStep & ((int64_t(1) << A.lg) - 1);
    return ((int64_t(ok ? pg : 0) * A.H + h) << A.lg) + t;
  };
  auto load_k = [&](int64_t row0) {
    ks_r = A.kscale[(row0 >> 4) + g];
    vs_r = A.vscale[(row0 >> 4) + g];
    const uint8_t* const p = A.kpool + row0 * D;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int x = 0; x < NK; ++x) {
        if (D == 96 && x == 1) {
          const v2u w = *reinterpret_cast<const v2u*>(p + k_off2 + 4 * i * D);
          kr[i][x] = v4u{w[0], w[1], 0, 0};
        } else {
          kr[i][x] = *reinterpret_cast<const v4u*>(p + k_off + 4 * i * D + 64 * x);
        }
      }
  };
  // (non-temporal: V passes once, and kept out of the caches' way 32 x 8192 tokens take 84 us
  // instead of 96.  K's lines are met by two loads each, half and half: 87 with both so.)
  auto load_v = [&](int64_t row0) {
    const uint8_t* const p = A.vpool + row0 * D;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
      vr[j] = __builtin_nontemporal_load(reinterpret_cast<const v4u*>(p + v_off + 256 * j));
  };

  const int steps = max(0, (P.s1 - P.s0 - wave + kWaves - 1) / kWaves);
  bool ok = false;
  int64_t row0 = 0;
  if (steps > 0) {
    row0 = row_of(0, ok);
    load_k(row0);
    load_v(row0);
  }
  v8h qh[KS], ql[QLO ? KS : 1];
  float c;  // scores to exponents, without the block's scale
  load_query<KS, QLO, kThr, 16>(A, row * A.q_ts + hq * A.q_hs, live,
                                [&](int k) { return dcol(D, k, g); }, &red_o[0][0][0], qh, ql, c);
#pragma unroll 1
  for (int it = 0; it < steps; ++it) {
    const int t0 = (P.s0 + wave + kWaves * it) * kStep;
    // ---- scores
    v4f s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[i] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const v4u w = kr[i][ks >> 1];
        const v8h a = ks & 1 ? widen8<FP8>(w[2], w[3]) : widen8<FP8>(w[0], w[1]);
        s[i] = mfma(a, qh[ks], s[i]);
        if constexpr (QLO) s[i] = mfma(a, ql[ks], s[i]);
      }
    }
    const float ck = c * ks_r, vs = vs_r;
    const bool pos = vs >= kLeast;
    float ref = m == -INFINITY ? 0.f : m - kUp;
    const float lv = (pos ? __builtin_amdgcn_logf(vs) : 0.f) - ref;
    float iv = pos ? __builtin_amdgcn_rcpf(vs) : 1.f;
    const bool was_ok = ok;
    const bool more = it + 1 < steps;
    if (more) {
      row0 = row_of(it + 1, ok);
      load_k(row0);
    }
    // ---- exponents of the weights, against the running maximum so far
    float y[16], top = -INFINITY;
    const bool edge = t0 + kStep > lim_all || !was_ok;
#pragma unroll
    for (int k = 0; k < 16; ++k) y[k] = fmaf(s[k >> 2][k & 3], ck, lv);
    if (edge) {
      asm volatile("");  // (a branch: as selects it would cost every step)
      const int left = was_ok ? lim - t0 - 16 * g : 0;  // of this lane's 16 tokens
#pragma unroll
      for (int k = 0; k < 16; ++k) y[k] = k < left ? y[k] : -INFINITY;
      // codes behind the cached tokens may be anything
      const int keep = was_ok ? n_tok - t0 - 16 * g : 0;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int k = keep - 4 * x;
        const uint32_t mask = k >= 4 ? ~0u : k <= 0 ? 0u : (1u << (8 * k)) - 1u;
#pragma unroll
        for (int j = 0; j < NJ; ++j) vr[j][x] &= mask;
      }
    }
    if (__any(!pos)) {  // a block of zeros
      asm volatile("");
      float big = -INFINITY;
#pragma unroll
      for (int k = 0; k < 16; ++k) big = fmaxf(big, y[k]);
      float others = pos ? big : -INFINITY;
      others = fmaxf(others, __shfl_xor(others, 16, 64));
      others = fmaxf(others, __shfl_xor(others, 32, 64));
      const float z = pos ? 0.f : stand_in(big + ref, fmaxf(m, others + ref));
#pragma unroll
      for (int k = 0; k < 16; ++k) y[k] += z;
      iv = pos ? iv : __builtin_amdgcn_exp2f(-z);
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int j = 0; j < NJ; ++j) vr[j][x] = pos ? vr[j][x] : 0;
    }
#pragma unroll
    for (int k = 0; k < 16; ++k) top = fmaxf(top, y[k]);
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    if (__any(top > kUp + kHead || m == -INFINITY)) {
      const float mn = fmaxf(m, top + ref);
      const float d = mn == -INFINITY ? 0.f : m - mn, f = __builtin_amdgcn_exp2f(d);
      const float by = mn == -INFINITY ? 0.f : mn - kUp - ref;
      m = mn;
      l = fall(l, d);
#pragma unroll
      for (int j = 0; j < NJ; ++j) o[j] *= f;
#pragma unroll
      for (int k = 0; k < 16; ++k) y[k] -= by;
    }
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      y[k] = __builtin_amdgcn_exp2f(y[k]);
      sum += y[k];
    }
    l = fmaf(sum * kSum, iv, l);
    v8h ph[2], pl[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      v4u hi, lo;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t a, b;
        split2(y[8 * u + 2 * j], y[8 * u + 2 * j + 1], a, b);
        hi[j] = a;
        lo[j] = b;
      }
      ph[u] = __builtin_bit_cast(v8h, hi);
      pl[u] = __builtin_bit_cast(v8h, lo);
    }
    // ---- values
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const v8h a = widen8<FP8>(vr[j][2 * u], vr[j][2 * u + 1]);
        o[j] = mfma(a, ph[u], o[j]);
        o[j] = mfma(a, pl[u], o[j]);
      }
    if (more) load_v(row0);
  }

  // ---- the waves' results to LDS: lane (n, g) has coordinates 16 j + 4 g + r of row n
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
#pragma unroll
  for (int j = 0; j < NJ; ++j)
    *reinterpret_cast<v4f*>(&red_o[wave][n][16 * j + 4 * g]) = o[j];
  if (g == 0) {
    red_ml[wave][n][0] = m;
    red_ml[wave][n][1] = l;
  }
  const int64_t slot = P.slot >= 0 ? place(A, P, h) : -1;
  __syncthreads();
  constexpr int PER = D / 8;  // threads of a row
  if (tid < kRows * PER) {
    const int r = tid / PER, d0 = 8 * (tid % PER);
    float M = -INFINITY, L = 0.f, x[8] = {};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) M = fmaxf(M, red_ml[w][r][0]);
    const float ref = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = __builtin_amdgcn_exp2f(red_ml[w][r][0] - ref);
      L += fall(red_ml[w][r][1], red_ml[w][r][0] - ref);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = fmaf(red_o[w][r][d0 + j], f, x[j]);
    }
    const int rr2 = P.rt * kRows + r, qi2 = rr2 / A.G;
    const int64_t row2 = int64_t(P.r.q0) + qi2;
    if (qi2 < P.r.ql && row2 >= 0 && row2 < A.rows) {
      if (P.slot < 0) {
        const float inv = inverse(L);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] *= inv;
        store8(A.out, (row2 * A.Hq + h * A.G + rr2 - qi2 * A.G) * D + d0, x, A.out_dtype, A.out_vec);
      } else if (slot >= 0) {
        const int64_t at = slot * kRows + r;
        store8(A.part_o, at * D + d0, x, QKV_F32, true);
        if (d0 == 0) {
          A.part_ml[2 * at] = M;
          A.part_ml[2 * at + 1] = L;
        }
      }
    }
  }
}

// Pieces that a launch aims at, per kv head: one workgroup per CU.  (decode8, 32 x 8192
// tokens, 8 kv heads, d = 128: 96 us; two per CU 105, three 104, four 118; 131,072 tokens:
// 48, 51, 54, 57.)
int32_t target_of(int32_t H) { return std::max(1, (qkv_num_cus() + H - 1) / H); }
// Cut tiles have more than C steps each and pieces of C, so they have fewer than
// 2 total / C <= 2 target pieces.
int64_t slots_of(int32_t H) { return int64_t(2 * target_of(H) + 1) * H; }
// Tiles of `rows` query rows, at most: a request's last one may be in part empty.
int64_t tiles_of(int64_t B, int64_t q_rows, int32_t G, int rows) {
  return q_rows * G / rows + std::min(B, q_rows);
}
// Bytes of a launch's partial results, and of its list of pieces.
int64_t part_bytes(int64_t B, int64_t q_rows, int32_t G, int32_t H, int rows, int32_t d) {
  const int64_t plan = B > 64 ? 16 * (tiles_of(B, q_rows, G, rows) + target_of(H)) : 0;
  return 256 + (slots_of(H) * (16 + rows * (d + 2) * 4) + plan) / 256 * 256 + 256;
}
// Lays them out at `at`.
void place_parts(Att& A, void* at, int rows, int32_t d) {
  A.used = static_cast<int32_t*>(at);
  A.desc = reinterpret_cast<int4*>(A.used + 64);
  A.part_o = reinterpret_cast<float*>(A.desc + A.nslots);
  A.part_ml = A.part_o + int64_t(A.nslots) * rows * d;
  // (nslots * rows * 8 bytes of part_ml: 16-byte aligned)
  A.plan = A.B > 64 ? reinterpret_cast<int4*>(A.part_ml + int64_t(A.nslots) * rows * 2) : nullptr;
}
// Requests of more rows than this go to prefill8.  us on decode8 / prefill8 at 64 rows a
// request, d = 128, 8 kv heads: 1 x 8000 tokens 18 / 28, 8 x 2000 21 / 27, 8 x 8000 61 / 49,
// 32 x 2000 57 / 46, 32 x 8000 195 / 146; at 32 rows decode8 has two tiles and is the
// faster one but for the last (109 / 116).
constexpr int kFew = 32;
// A cache of up to this many tokens a request is not cut: the join's launch costs more than
// the steps that it saves (one fp32 query over 512 tokens, 8 heads: 14 us against 17).  The
// host knows the table's width for it, not the lengths: under a wide table short requests
// have the join's launch, too.
constexpr int64_t kWhole = 1024;
constexpr int32_t kNever = INT32_MAX / 2;

// Whether prefill8 runs, and the workspace: decode8's part, then prefill8's where it runs.  The
// one rule for both: `max_q`, which may be wrong, decides (too small: decode8, which takes
// requests of any rows).
struct Layout {
  bool pre;
  int64_t at_pre, bytes;
};
Layout layout(int64_t B, int64_t rows, int32_t G, int32_t H, int32_t d, int64_t max_q) {
  Layout L;
  L.pre = std::min(max_q, rows) * G > kFew;
  L.at_pre = part_bytes(B, rows, G, H, kRows, d);
  L.bytes = L.at_pre + (L.pre ? part_bytes(B, rows, G, H, kPreRows, d) : 0);
  return L;
}

template <int D, bool FP8>
void launch(const Att& A, uint32_t pieces, hipStream_t s) {
  const uint32_t grid = pieces * A.H;
  if (A.plan) plan8<kRows><<<1, kPlanThr, (A.B + 1) * sizeof(int32_t), s>>>(A, pieces);
  if (A.q_dtype == QKV_F32) decode8<D, FP8, true><<<grid, kThr, 0, s>>>(A);
  else decode8<D, FP8, false><<<grid, kThr, 0, s>>>(A);
}

// The joins of what decode8 (A) and prefill8 (P) have cut; null: nothing.
template <int D>
void join(const Att* A, const Att* P, hipStream_t s) {
  const uint32_t a = A ? join_grid(*A, kRows) : 0, p = P ? join_grid(*P, kPreRows) : 0;
  if (A && P) join_both8<D><<<a + p, kThr, 0, s>>>(*A, *P, static_cast<int>(a));
  else if (A) join8<D, kRows><<<a, kThr, 0, s>>>(*A);
  else if (P) join8<D, kPreRows><<<p, kThr, 0, s>>>(*P);
}

}  // namespace

extern "C" int64_t qkv_kv8_attention_workspace_bytes(int32_t B, int64_t rows, int32_t Hq,
                                                     int32_t Hkv, int32_t d, int64_t max_q) {
  if (Hkv < 1 || d < 1) return 0;
  if (B < 1 || rows < 1) return 256;
  return layout(B, rows, Hq / Hkv, Hkv, d, max_q).bytes;
}

extern "C" int qkv_kv8_attention(const void* q, int32_t q_dtype, int64_t q_row_stride,
                                 int64_t q_head_stride, int64_t rows, const void* kpool,
                                 const float* kscale, const void* vpool, const float* vscale,
                                 int32_t fmt, int32_t num_pages, int32_t page_tokens,
                                 const int32_t* table, int32_t pages_per_seq,
                                 const int32_t* q_start, const int32_t* q_lens,
                                 const int32_t* kv_lens, int32_t B, int32_t Hq, int32_t Hkv,
                                 int32_t d, int64_t max_q, float scale, int32_t causal, void* out,
                                 int32_t out_dtype, void* workspace, int64_t ws_bytes,
                                 void* stream) {
  const int st = qkv_kv8_check(fmt, num_pages, page_tokens, Hkv, d);
  if (st != QKV_OK) return st;
  QKV_REQUIRE(qkv_dtype_ok(q_dtype) && qkv_dtype_ok(out_dtype), "unknown element type %d / %d",
              q_dtype, out_dtype);
  QKV_REQUIRE(Hq >= 1 && Hq % Hkv == 0, "query heads (%d) must be a multiple of kv heads (%d)", Hq,
              Hkv);
  QKV_REQUIRE(B >= 0 && B <= kMaxB && pages_per_seq >= 1,
              "batch %d must lie in [0, %d], pages_per_seq %d be positive", B, kMaxB, pages_per_seq);
  const int32_t G = Hq / Hkv;
  QKV_REQUIRE(rows >= 0 && rows * G < INT32_MAX / 2 && rows * Hq / kRows < (1 << 28),
              "rows must lie in [0, 2^30 / heads per kv head); got %lld",
              static_cast<long long>(rows));
  if (rows == 0 || B == 0) return QKV_OK;
  QKV_REQUIRE(q_start || !q_lens, "q_lens needs q_start");
  QKV_REQUIRE(q_start || rows % B == 0, "without q_start the rows (%lld) must be B (%d) times one "
              "length", static_cast<long long>(rows), B);
  QKV_REQUIRE(q && kpool && kscale && vpool && vscale && table && kv_lens && out,
              "qkv_kv8_attention: null pointer");
  QKV_REQUIRE(qkv_aligned(kpool, 16) && qkv_aligned(vpool, 16),
              "the pools must be 16-byte aligned");
  const Layout L = layout(B, rows, G, Hkv, d, max_q);
  QKV_REQUIRE(workspace && qkv_aligned(workspace, 256) && ws_bytes >= L.bytes,
              "qkv_kv8_attention: workspace too small or not 256-byte aligned");
  const int qb = q_dtype == QKV_F32 ? 4 : 2, ob = out_dtype == QKV_F32 ? 4 : 2;
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
  A.nslots = static_cast<int32_t>(slots_of(Hkv));
  place_parts(A, workspace, kRows, d);
  const int64_t longest = std::min<int64_t>(max_q, q_start ? rows : A.uniform_q);
  const bool pre = L.pre && longest * G > kFew;
  // decode8 runs too where, as far as the rows tell, a request may be short.  (Where one is
  // against that, prefill8 takes it: slower, the same result.)
  const bool dec = !pre || (q_start && rows <= (B - 1) * longest + kFew / G);
  QKV_REQUIRE((tiles_of(B, rows, G, kRows) + A.target) * Hkv <= INT32_MAX, "batch of %d requests "
              "and %lld rows is too large for one call", B, static_cast<long long>(rows));
  // without q_start the tiles are known
  auto tiles = [&](int r) {
    return q_start ? tiles_of(B, rows, G, r)
                   : int64_t(B) * ((int64_t(A.uniform_q) * G + r - 1) / r);
  };
  const bool cut = (int64_t(pages_per_seq) << A.lg) > kWhole;
  A.few = !pre ? INT32_MAX : dec ? kFew : 0;
  A.least = cut ? 4 : kNever;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dec) {
    // beside prefill8 this launch has only requests of up to kFew rows
    const uint32_t t = static_cast<uint32_t>(
        (pre ? std::min<int64_t>(tiles(kRows), int64_t(B) * (kFew / kRows)) : tiles(kRows)) +
        (cut ? A.target : 0));
    if (fmt == QKV_CODES_I8) {
      if (d == 128) launch<128, false>(A, t, s);
      else if (d == 96) launch<96, false>(A, t, s);
      else launch<64, false>(A, t, s);
    } else {
      if (d == 128) launch<128, true>(A, t, s);
      else if (d == 96) launch<96, true>(A, t, s);
      else launch<64, true>(A, t, s);
    }
    QKV_LAUNCHED();
  }
  Att P = A;
  bool cut8 = false;
  if (pre) {
    place_parts(P, static_cast<uint8_t*>(workspace) + L.at_pre, kPreRows, d);
    // cut only where the tiles, as far as the rows tell, do not fill the card
    const int64_t t = tiles(kPreRows);
    cut8 = cut && rows * G / kPreRows < P.target;
    P.least = cut8 ? 4 : kNever;
    // (pieces of cut tiles are within the target where the kernel counts them itself)
    const int64_t pieces = !cut8 ? t : P.plan ? t + P.target : std::max<int64_t>(t, P.target);
    qkv_kv8_prefill(P, d, fmt == QKV_CODES_E4M3, static_cast<uint32_t>(pieces), s);
    QKV_LAUNCHED();
  }
  const Att *const ja = dec && cut ? &A : nullptr, *const jp = cut8 ? &P : nullptr;
  if (d == 128) join<128>(ja, jp, s);
  else if (d == 96) join<96>(ja, jp, s);
  else join<64>(ja, jp, s);
  QKV_LAUNCHED();
  return QKV_OK;
}
