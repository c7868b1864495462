// A piece of 128 query rows over the 8-bit paged cache: decode8's mathematics
// (qkv_kv8_decode.h) on large tiles, for prefill8 (many rows of a request: a prompt, a chunk of
// one; qkv_kv8_prefill.hip) and the tall tiles of share8 (qkv_kv8_shared.hip).
//
// A workgroup of 8 waves takes 128 rows (query-major): wave w the rows 32 (w % 4) .. of
// every step of 64 tokens that is even (waves 0-3) or odd (4-7), so that a SIMD always has
// two waves and the longest tile, which a causal launch waits for, takes half as long.
// A step's codes become f16 in LDS once, in the order in which the matrix instruction
// takes them (images of 64 lanes x 16 bytes), double buffered with one barrier a round;
// the next round's bytes are in flight meanwhile.  Scores S^T = K Q^T and values
// O^T = V^T P^T run on v_mfma_f32_32x32x16_f16: a lane owns one query row, score register
// 8 b + j of a 32-token tile belongs to its block b, and the weights of a block are, as
// they stand, the B operand of the value product if the A operand takes the V block's
// dwords h and 2 + h.  The halves' sums meet in LDS at the end.
//
// Weights are f16 pairs, as decode8's, but for bf16 results of 16-bit queries, which keep
// 2^-8: there they are one f16 (half a step of 2^-11; their sum is of the unrounded ones).
// Against 64 bits both are 1.7e-3 off, the result's rounding, and the pair takes 17 % longer
// (2048 causal queries: 64.8 us against 55.3).
//
// Bound: the SIMDs' issue.  A round (128 tokens, 128 rows) is 2048 clocks of products and
// ~2700 of VALU work per SIMD (exponents 160 instructions a wave, widening 100), of which a
// third cannot overlap (two waves of one SIMD, one with products and one with multiply-adds
// alone: 527 and 506 us, together 693); LDS takes 2100 (reads 214 B a clock and CU, writes
// 76).  Measured 2.2 us a round, 12 us of set-up and end; 2048 causal queries, 32 / 8 heads,
// d = 128, bf16: 56 us a call (decode8 alone 245, four waves a workgroup and no order 74).
// No gain from: a wave's priority raised over its products, the scores of the next tile
// among the values of this one (86 against 82 us at 1024 queries over 4096 tokens), the
// weights' sum by a product with ones (84), rounds without masks as straight code (spills:
// 109).
#pragma once

#include "qkv_kv8_attn.h"

namespace qkv_kv8 {

constexpr int kPreThr = 512;

typedef float v16f __attribute__((ext_vector_type(16)));

__device__ __forceinline__ v16f mfma32(v4u a, v8h b, v16f c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), b, c, 0, 0, 0);
}

// Dynamic LDS: two buffers of both halves; at the end D / 32 coordinate tiles, m and l.
template <int D>
constexpr int kPreLds = std::max(4 * (2 * (D / 16) + 4 * (D / 32)) * 1024,
                                 (4 * (D / 32) * 16 + 16) * 256);

// sbuf: a block's ks, log2 vs, 1 / vs, and the step's blocks of zeros, a bit each.  ROWS: as
// decode_piece's.
template <int D, bool FP8, bool QLO, bool PLO, bool ROWS>
__device__ __forceinline__ void prefill_piece(const Att& A, const Piece& P, int h, int thread,
                                              uint8_t* lds, v4f (*sbuf)[2][4]) {
  constexpr int KK = D / 16;                     // 16-wide product steps of a score
  constexpr int DT = D / 32;                     // 32-wide coordinate tiles
  constexpr int CH = 4 * D;                      // 16-byte chunks of K and of V in a step
  constexpr int NC = (CH + 255) / 256;           // of them, per thread of a half
  constexpr int KB = 2 * KK * 1024, VB = 4 * DT * 1024;
  const int tid = thread & 255, lane = tid & 63;
  const int wave8 = __builtin_amdgcn_readfirstlane(thread >> 6);
  const int wave = wave8 & 3, th = wave8 >> 2;
  // the half's buffer i: K's images (32-token tile, product step), V's (coordinate tile, block)
  auto kbuf = [&](int i) { return lds + (2 * i + th) * (KB + VB); };
  auto vbuf = [&](int i) { return kbuf(i) + KB; };
  const int n = lane & 31, hf = lane >> 5;

  // ---- this lane's query row
  const int rr = P.rt * kPreRows + 32 * wave + n, qi = rr / A.G, gq = rr - qi * A.G;
  const int64_t row = int64_t(P.r.q0) + qi;
  const bool live = qi < P.r.ql && row >= 0 && row < A.rows;
  const int hq = h * A.G + gq;
  // tokens below lim are seen; all of the wave's live rows see those below lim_all (its
  // first row's: rows are query-major), and none those from lim_any on
  const int lim = live ? limit(P, qi) : 0;
  const int q_first = (P.rt * kPreRows + 32 * wave) / A.G;
  const int q_last = min(P.r.ql - 1, (P.rt * kPreRows + 32 * wave + 31) / A.G);
  const int lim_all = limit(P, q_first);
  const int lim_any = q_first < P.r.ql ? limit(P, q_last) : 0;
  // the workgroup's last token: its last live query's
  const int qlast = min(P.r.ql - 1, (P.rt * kPreRows + kPreRows - 1) / A.G);
  const int last = limit(P, qlast);
  const int s1 = min(P.s1, (max(last, 0) + kStep - 1) / kStep);

  v16f o[DT];
#pragma unroll
  for (int j = 0; j < DT; ++j)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[j][i] = 0.f;
  float m = -INFINITY, l = 0.f;

  // ---- a step's bytes: 16-byte chunks, a token's K row in turn, and V as it lies
  v4u kr[NC], vr[NC];
  float ks_r = 0.f, vs_r = 0.f;
  const int pg_sh = A.lg - 6;
  const int32_t* const tab = A.table + int64_t(P.b) * A.width;
  int pages = 0, p_first = 0;
  bool ok_r = false;  // of the step in flight
  auto fetch = [&](int st) {
    if (st == P.s0 + th || st - p_first >= 128) {
      p_first = st;
      pages = st + 2 * lane < P.s1 ? tab[(st + 2 * lane) >> pg_sh] : -1;
    }
    const int pg = __builtin_amdgcn_readlane(pages, (st - p_first) >> 1);
    ok_r = pg >= 0 && pg < A.npages;
    const int64_t row0 = ((int64_t(ok_r ? pg : 0) * A.H + h) << A.lg) +
                         (int64_t(st) * kStep & ((int64_t(1) << A.lg) - 1));
    if (tid < 4) {
      ks_r = A.kscale[(row0 >> 4) + tid];
      vs_r = A.vscale[(row0 >> 4) + tid];
    }
    const v4u* const kp = reinterpret_cast<const v4u*>(A.kpool + row0 * D);
    const v4u* const vp = reinterpret_cast<const v4u*>(A.vpool + row0 * D);
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int ch = tid + 256 * i;
      if (CH % 256 == 0 || ch < CH) {
        kr[i] = kp[ch];
        vr[i] = vp[ch];
      }
    }
  };
  // widened into buffer `to`
  auto put = [&](int st, int to) {
    const int keep = ok_r ? P.r.kv - st * kStep : 0;  // tokens of the step
    if (tid < 4) {
      const bool pos = vs_r >= kLeast;
      const uint32_t zeros = static_cast<uint32_t>(__ballot(!pos && keep > kBlk * tid));
      sbuf[to][th][tid] = v4f{ks_r, pos ? __builtin_amdgcn_logf(vs_r) : 0.f,
                          pos ? __builtin_amdgcn_rcpf(vs_r) : 1.f, __uint_as_float(zeros)};
    }
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int ch = tid + 256 * i;
      if (CH % 256 != 0 && ch >= CH) continue;
      {  // token ch / KK, coordinates 16 (ch % KK) ..: the places are swizzled by the product
         // step so that a row's chunks meet different banks
        const int t = ch / KK, k = ch % KK;
        uint8_t* const at = kbuf(to) + ((t >> 5) * KK + k) * 1024 + (((t & 31) ^ (k & 7)) << 4);
        *reinterpret_cast<v8h*>(at) = widen8<FP8>(kr[i][0], kr[i][1]);
        *reinterpret_cast<v8h*>(at + 512) = widen8<FP8>(kr[i][2], kr[i][3]);
      }
      {  // block ch / D, coordinate ch % D
        const int blk = ch / D, dd = ch % D;
        v4u w = vr[i];
        if (keep < kStep) {  // codes behind the cached tokens may be anything
          asm volatile("");  // (a branch: as selects it would cost every step)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int k = keep - 16 * blk - 4 * x;
            w[x] &= k >= 4 ? ~0u : k <= 0 ? 0u : (1u << (8 * k)) - 1u;
          }
        }
        uint8_t* const at = vbuf(to) + ((dd >> 5) * 4 + blk) * 1024 + ((dd & 31) << 4);
        *reinterpret_cast<v8h*>(at) = widen8<FP8>(w[0], w[2]);
        *reinterpret_cast<v8h*>(at + 512) = widen8<FP8>(w[1], w[3]);
      }
    }
  };

  const int mine = P.s0 + th;  // this half's first step
  auto q_col = [&](int k) { return 16 * k + 8 * hf; };
  const int64_t q_at = row * A.q_ts + hq * A.q_hs;
  const RawQuery<KK, QLO> raw = fetch_query<KK, QLO>(A, q_at, live, q_col);
  if (mine < s1) fetch(mine);
  v8h qh[KK], ql[QLO ? KK : 1];
  float c;  // scores to exponents, without the block's scale
  load_query<KK, QLO, kPreThr, 32>(A, raw, q_at, live, thread, q_col,
                                   reinterpret_cast<float*>(lds), qh, ql, c);
  if (mine < s1) put(mine, 0);
  bool ok = ok_r;  // of the step to come
  if (th == 1 && mine + 2 < s1) fetch(mine + 2);
  __syncthreads();
#pragma unroll 1
  for (int s0 = P.s0; s0 < s1; s0 += 2) {
    const int st = s0 + th, buf = ((s0 - P.s0) >> 1) & 1, t0 = st * kStep;
    const bool more = st + 2 < s1, was_ok = ok;
    // the second half widens its next step before the products, the first one behind them,
    // so that products meet the other wave's VALU work (1.5 %)
    if (th == 0) {
      if (more) fetch(st + 2);
      ok = ok_r;
    } else if (more) {
      ok = ok_r;
      put(st + 2, buf ^ 1);
      if (st + 4 < s1) fetch(st + 4);
    }
    if (st < s1 && t0 < lim_any) {
      // ---- scores: register 8 b + j of tile i is token 32 i + 16 b + (j & 3) + 8 (j >> 2) + 4 hf
      v16f s[2];
      constexpr int AHEAD = 4;  // operands read ahead of their product
      v4u a[AHEAD];
      auto k_at = [&](int x) {
        return *reinterpret_cast<const v4u*>(kbuf(buf) + x * 1024 + hf * 512 +
                                             ((n ^ (x % KK & 7)) << 4));
      };
#pragma unroll
      for (int x = 0; x < AHEAD; ++x) a[x] = k_at(x);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int j = 0; j < 16; ++j) s[i][j] = 0.f;
#pragma unroll
        for (int k = 0; k < KK; ++k) {
          const int x = i * KK + k;
          s[i] = mfma32(a[x % AHEAD], qh[k], s[i]);
          if constexpr (QLO) s[i] = mfma32(a[x % AHEAD], ql[k], s[i]);
          if (x + AHEAD < 2 * KK) a[x % AHEAD] = k_at(x + AHEAD);
        }
      }
      // ---- exponents of the weights, against the running maximum so far
      float iv[4];
      const int zeros = __builtin_amdgcn_readfirstlane(__float_as_int(sbuf[buf][th][0][3]));
      float top = -INFINITY, ref = m == -INFINITY ? 0.f : m - kUp;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const v4f sc = sbuf[buf][th][b];
        const float ck = c * sc[0], lv = sc[1] - ref;
        iv[b] = sc[2];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int e = 8 * (b & 1) + j;
          s[b >> 1][e] = fmaf(s[b >> 1][e], ck, lv);
        }
      }
      if (t0 + kStep > lim_all || !was_ok) {
        asm volatile("");
        const int left = (was_ok ? lim : 0) - t0 - 4 * hf;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 16; ++j)
            s[i][j] = 32 * i + (j & 3) + 8 * (j >> 2) < left ? s[i][j] : -INFINITY;
      }
      if (zeros != 0) {
        asm volatile("");
        float big[4], others = -INFINITY;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          big[b] = -INFINITY;
#pragma unroll
          for (int j = 0; j < 8; ++j) big[b] = fmaxf(big[b], s[b >> 1][8 * (b & 1) + j]);
          if (!(zeros >> b & 1)) others = fmaxf(others, big[b]);
        }
        others = fmaxf(others, __shfl_xor(others, 32, 64));
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          if (!(zeros >> b & 1)) continue;
          const float z = stand_in(big[b] + ref, fmaxf(m, others + ref));
#pragma unroll
          for (int j = 0; j < 8; ++j) s[b >> 1][8 * (b & 1) + j] += z;
          iv[b] = __builtin_amdgcn_exp2f(-z);
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) top = fmaxf(top, s[i][j]);
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      if (__any(top > kUp + kHead || m == -INFINITY)) {
        const float mn = fmaxf(m, top + ref);
        const float d = mn == -INFINITY ? 0.f : m - mn, f = __builtin_amdgcn_exp2f(d);
        const float by = mn == -INFINITY ? 0.f : mn - kUp - ref;
        m = mn;
        l = fall(l, d);
#pragma unroll
        for (int j = 0; j < DT; ++j)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[j][i] *= f;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 16; ++j) s[i][j] -= by;
      }
      if (zeros != 0) {  // their weights join l here (asked among the weights below: 1 % slower)
        asm volatile("");
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          if (!(zeros >> b & 1)) continue;
          float sum = 0.f;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            sum += __builtin_amdgcn_exp2f(s[b >> 1][8 * (b & 1) + j]);
            s[b >> 1][8 * (b & 1) + j] = -INFINITY;
          }
          l = fmaf(sum * kSum, iv[b], l);
        }
      }
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        float sum = 0.f;
        v4u hi, lo, v[DT];
#pragma unroll
        for (int j = 0; j < DT; ++j)
          v[j] = *reinterpret_cast<const v4u*>(vbuf(buf) + (j * 4 + b) * 1024 + lane * 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float p0 = __builtin_amdgcn_exp2f(s[b >> 1][8 * (b & 1) + 2 * j]);
          const float p1 = __builtin_amdgcn_exp2f(s[b >> 1][8 * (b & 1) + 2 * j + 1]);
          sum += p0 + p1;
          uint32_t x, y = 0;
          if constexpr (PLO) split2(p0, p1, x, y);
          else x = pk(p0, p1);
          hi[j] = x;
          lo[j] = y;
        }
        l = fmaf(sum * kSum, iv[b], l);
        // ---- values
#pragma unroll
        for (int j = 0; j < DT; ++j) {
          o[j] = mfma32(v[j], __builtin_bit_cast(v8h, hi), o[j]);
          if constexpr (PLO) o[j] = mfma32(v[j], __builtin_bit_cast(v8h, lo), o[j]);
        }
      }
    }
    if (th == 0 && more) put(st + 2, buf ^ 1);
    __syncthreads();
  }

  // ---- the halves join: the first takes over the first coordinate tiles, the second the
  // others (the loop's last barrier is behind the buffers' last readers)
  constexpr int KEEP = (DT + 1) / 2;
  l += __shfl_xor(l, 32, 64);
  float* const box = reinterpret_cast<float*>(lds) + lane;
  auto at_box = [&](int j, int i) { return box + ((wave * DT + j) * 16 + i) * 64; };
  float* const ml = reinterpret_cast<float*>(lds) + 4 * DT * 16 * 64 + lane;  // [half][wave][2]
#pragma unroll
  for (int j = 0; j < DT; ++j)
    if ((j < KEEP) == (th == 1))
#pragma unroll
      for (int i = 0; i < 16; ++i) *at_box(j, i) = o[j][i];
  ml[(2 * wave8) * 64] = m;
  ml[(2 * wave8 + 1) * 64] = l;
  const int64_t slot = ROWS || P.slot < 0 ? P.slot : place(A, P, h);
  __syncthreads();
  if (!live) return;
  const float m2 = ml[(2 * (wave8 ^ 4)) * 64], l2 = ml[(2 * (wave8 ^ 4) + 1) * 64];
  const float M = fmaxf(m, m2), base = M == -INFINITY ? 0.f : M;
  float e1 = __builtin_amdgcn_exp2f(m - base), e2 = __builtin_amdgcn_exp2f(m2 - base);
  const float L = fall(l, m - base) + fall(l2, m2 - base);
  // lane (n, hf) has coordinates 32 j + 8 q + 4 hf + 0 .. 3 of row n
  if (P.slot < 0) {
    const float inv = inverse(L);
    e1 *= inv;
    e2 *= inv;
  }
  const int64_t at = P.slot < 0 ? row * A.Hq + hq
                     : ROWS     ? int64_t(h) * A.nslots + slot + rr
                                : slot * kPreRows + 32 * wave + n;
  if (P.slot >= 0 && slot < 0) return;
#pragma unroll
  for (int j = 0; j < DT; ++j)
    if ((j < KEEP) == (th == 0))
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          x[i] = o[j][4 * q + i] * e1 + *at_box(j, 4 * q + i) * e2;
        const int64_t to = at * D + 32 * j + 8 * q + 4 * hf;
        if (P.slot < 0) store4(A.out, to, x, A.out_dtype, A.out_vec);
        else *reinterpret_cast<v4f*>(A.part_o + to) = v4f{x[0], x[1], x[2], x[3]};
      }
  if (P.slot >= 0 && hf == 0 && th == 0) {
    A.part_ml[2 * at] = M;
    A.part_ml[2 * at + 1] = L;
  }
}

}  // namespace qkv_kv8
