// A piece of 16 query rows over the 8-bit paged cache (qkv_kv8.h): decode8 (qkv_kv8_attn.hip)
// and the short tiles of share8 (qkv_kv8_shared.hip).
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
#pragma once

#include "qkv_kv8_attn.h"

namespace qkv_kv8 {

// d index of the first of the 8 coordinates that lane group g holds in product step ks
__host__ __device__ constexpr int dcol(int D, int ks, int g) {
  return D == 96 && ks == 2 ? 64 + 8 * g : 64 * (ks >> 1) + 16 * g + 8 * (ks & 1);
}

// Waves' results (tid 0 .. 255: four of them) of 16 rows, over every `waves`-th step of 64 tokens
// from number `turn` on, to LDS (red_o, red_ml), relative to their own maxima.  meanwhile() is called
// while the first pages' numbers are on their way.
template <int D, bool FP8, bool QLO, typename W, typename F>
__device__ __forceinline__ void decode_steps(const Att& A, const Piece& P, int h, int tid, int turn,
                                             W waves, float (*red_o)[kRows][D + 4],
                                             float (*red_ml)[kRows][2], F meanwhile) {
  constexpr int KS = D / 32, NJ = D / 16, NK = (D + 63) / 64;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int pg_sh = A.lg - 6;  // steps per page, log2
  const int32_t* const tab = A.table + int64_t(P.b) * A.width;
  int p_first = 0;
  // lane i: the page of this wave's i-th step from p_first on
  auto pages_from = [&](int i) {
    const int st = P.s0 + turn + waves * (i + lane);
    return st < P.s1 ? tab[st >> pg_sh] : -1;
  };
  int pages = pages_from(0);

  // ---- this lane's query row
  const int rr = P.rt * kRows + n, qi = rr / A.G, gq = rr - qi * A.G;
  const int64_t row = int64_t(P.r.q0) + qi;
  const bool live = qi < P.r.ql && row >= 0 && row < A.rows;
  const int hq = h * A.G + gq;
  // tokens below lim are seen; all live rows of the tile see those below lim_all (its first
  // row's: rows are query-major)
  const int lim = live ? limit(P, qi) : 0;
  const int lim_all = limit(P, P.rt * kRows / A.G);
  const int n_tok = P.r.kv;

  v4f o[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) o[j] = v4f{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;

  // K and V of the step that follows, in registers
  v4u kr[4][NK];
  v4u vr[NJ];
  float ks_r = 0.f, vs_r = 0.f;
  const int tok0 = 16 * (n >> 2) + (n & 3);
  const uint32_t k_off = static_cast<uint32_t>(tok0 * D + 16 * g);
  const uint32_t k_off2 = static_cast<uint32_t>(tok0 * D + 64 + 8 * g);  // D = 96: 8 bytes each
  const uint32_t v_off = static_cast<uint32_t>((g * D + n) * 16);
  auto page_of = [&](int i) {  // i: the wave's step count
    if (i - p_first >= 64) {
      p_first = i;
      pages = pages_from(i);
    }
    return __builtin_amdgcn_readlane(pages, i - p_first);
  };
  auto row_of = [&](int i, bool& ok) {
    const int pg = page_of(i);
    ok = pg >= 0 && pg < A.npages;
    const int st = P.s0 + turn + waves * i;
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

  const int steps = max(0, (P.s1 - P.s0 - turn + waves - 1) / waves);
  auto q_col = [&](int k) { return dcol(D, k, g); };
  const int64_t q_at = row * A.q_ts + hq * A.q_hs;
  const RawQuery<KS, QLO> raw = fetch_query<KS, QLO>(A, q_at, live, q_col);
  meanwhile();
  bool ok = false;
  int64_t row0 = 0;
  if (steps > 0) {
    row0 = row_of(0, ok);
    load_k(row0);
    load_v(row0);
  }
  v8h qh[KS], ql[QLO ? KS : 1];
  float c;  // scores to exponents, without the block's scale
  load_query<KS, QLO, kThr, 16>(A, raw, q_at, live, tid, q_col, &red_o[0][0][0], qh, ql, c);
#pragma unroll 1
  for (int it = 0; it < steps; ++it) {
    const int t0 = (P.s0 + turn + waves * it) * kStep;
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
}

// Four waves take every fourth step of a piece and merge.  ROWS: partial results are a row each,
// [kv head][row of the workspace], P.slot the one of the request's row 0; else tiles (place).
template <int D, bool FP8, bool QLO, bool ROWS>
__device__ __forceinline__ void decode_piece(const Att& A, const Piece& P, int h, int tid,
                                             float (*red_o)[kRows][D + 4],
                                             float (*red_ml)[kRows][2]) {
  decode_steps<D, FP8, QLO>(A, P, h, tid, __builtin_amdgcn_readfirstlane(tid >> 6),
                            std::integral_constant<int, kWaves>{}, red_o, red_ml, [] {});
  int64_t at = -1;  // where the partial result's row 0 goes
  if constexpr (ROWS) {
    if (P.slot >= 0) at = int64_t(h) * A.nslots + P.slot + P.rt * kRows;
  } else if (P.slot >= 0) {
    const int64_t slot = place(A, P, h);
    if (slot >= 0) at = slot * kRows;
  }
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
      } else if (at >= 0) {
        store8(A.part_o, (at + r) * D + d0, x, QKV_F32, true);
        if (d0 == 0) {
          A.part_ml[2 * (at + r)] = M;
          A.part_ml[2 * (at + r) + 1] = L;
        }
      }
    }
  }
}

}  // namespace qkv_kv8
