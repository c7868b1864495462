// Attention of many query rows of a request (a prompt, a chunk of one) over the 8-bit
// paged cache: decode8's mathematics (qkv_kv8_attn.hip) on tiles of 128 query rows.
//
// A workgroup of 4 waves takes 128 rows (query-major), a wave 32 of them, and steps through
// 64 tokens: the step's codes become f16 in LDS once, in the order in which the matrix
// instruction takes them (images of 64 lanes x 16 bytes), double buffered with one
// barrier a step; the next step's bytes are in flight meanwhile.  Scores S^T = K Q^T and
// values O^T = V^T P^T run on v_mfma_f32_32x32x16_f16: a lane owns one query row, score
// register 8 b + j of a 32-token tile belongs to its block b, and the weights of a block
// are, as they stand, the B operand of the value product if the A operand takes the V
// block's dwords h and 2 + h.
#include "qkv_kv8_attn.h"

namespace {

using namespace qkv_kv8;

typedef float v16f __attribute__((ext_vector_type(16)));

__device__ __forceinline__ v16f mfma32(v4u a, v8h b, v16f c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), b, c, 0, 0, 0);
}

template <int D, bool FP8, bool QLO, bool PLO>
__global__ __launch_bounds__(kThr, 2) void prefill8(Att A) {
  constexpr int KK = D / 16;                     // 16-wide product steps of a score
  constexpr int DT = D / 32;                     // 32-wide coordinate tiles
  constexpr int CH = 4 * D;                      // 16-byte chunks of K and of V in a step
  constexpr int NC = (CH + kThr - 1) / kThr;     // of them, per thread
  constexpr int KB = 2 * KK * 1024, VB = 4 * DT * 1024;
  __shared__ Shared sh;
  __shared__ v4f sbuf[2][4];                     // a block's ks, log2 vs, 1 / vs
  extern __shared__ __align__(16) uint8_t lds[];
  // of buffer i: K's images (32-token tile, product step), V's (coordinate tile, block)
  auto kbuf = [&](int i) { return lds + i * (KB + VB); };
  auto vbuf = [&](int i) { return lds + i * (KB + VB) + KB; };
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 31, hf = lane >> 5;
  const int h = blockIdx.x % A.H;
  Piece P;
  if (!locate<kPreRows>(A, blockIdx.x / A.H, sh, P)) return;

  // ---- this lane's query row
  const int rr = P.rt * kPreRows + 32 * wave + n, qi = rr / A.G, gq = rr - qi * A.G;
  const int64_t row = int64_t(P.r.q0) + qi;
  const bool live = qi < P.r.ql && row >= 0 && row < A.rows;
  const int hq = h * A.G + gq;
  v8h qh[KK], ql[QLO ? KK : 1];
  float c;
  {
    float x[KK][8];
    float amax = 0.f;
#pragma unroll
    for (int k = 0; k < KK; ++k) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[k][j] = 0.f;
      if (live) load8(A, row * A.q_ts + hq * A.q_hs + 16 * k + 8 * hf, x[k]);
#pragma unroll
      for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(x[k][j]));
    }
    amax = fmaxf(amax, __shfl_xor(amax, 32, 64));
    int ex = 0;
    if (amax > 0.f && amax < INFINITY) frexpf(amax, &ex);
    ex = max(ex, -110);
    const float up = ldexpf(1.f, 10 - ex);
    c = ldexpf(A.scale * kLog2e, ex - 10);
#pragma unroll
    for (int k = 0; k < KK; ++k) {
      v4u hi, lo;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t a, b;
        split2(x[k][2 * j] * up, x[k][2 * j + 1] * up, a, b);
        hi[j] = a;
        lo[j] = b;
      }
      qh[k] = __builtin_bit_cast(v8h, hi);
      if constexpr (QLO) ql[k] = __builtin_bit_cast(v8h, lo);
    }
  }
  const int lim = !live ? 0 : A.causal ? min(P.r.kv, P.r.kv - P.r.ql + qi + 1) : P.r.kv;
  int lim_all = live ? lim : INT32_MAX, lim_any = lim;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    lim_all = min(lim_all, __shfl_xor(lim_all, o, 64));
    lim_any = max(lim_any, __shfl_xor(lim_any, o, 64));
  }
  lim_all = __builtin_amdgcn_readfirstlane(lim_all);
  lim_any = __builtin_amdgcn_readfirstlane(lim_any);
  // the workgroup's last token: its last live query's
  const int qlast = min(P.r.ql - 1, (P.rt * kPreRows + kPreRows - 1) / A.G);
  const int last = A.causal ? min(P.r.kv, P.r.kv - P.r.ql + qlast + 1) : P.r.kv;
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
    if (st == P.s0 || st - p_first >= 64) {
      p_first = st;
      pages = st + lane < P.s1 ? tab[(st + lane) >> pg_sh] : -1;
    }
    const int pg = __builtin_amdgcn_readlane(pages, st - p_first);
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
      const int ch = tid + kThr * i;
      if (CH % kThr == 0 || ch < CH) {
        kr[i] = kp[ch];
        vr[i] = vp[ch];
      }
    }
  };
  // widened into buffer `to`
  auto put = [&](int st, int to) {
    const int keep = ok_r ? P.r.kv - st * kStep : 0;  // tokens of the step
    if (tid < 4) {
      const bool pos = vs_r > 0.f;
      sbuf[to][tid] = v4f{ks_r, pos ? __builtin_amdgcn_logf(vs_r) : 0.f,
                          pos ? __builtin_amdgcn_rcpf(vs_r) : 1.f, 0.f};
    }
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int ch = tid + kThr * i;
      if (CH % kThr != 0 && ch >= CH) continue;
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

  if (P.s0 < s1) {
    fetch(P.s0);
    put(P.s0, 0);
  }
  bool ok = ok_r;
  __syncthreads();
#pragma unroll 1
  for (int st = P.s0; st < s1; ++st) {
    const int buf = (st - P.s0) & 1, t0 = st * kStep;
    const bool more = st + 1 < s1, was_ok = ok;
    if (more) {
      fetch(st + 1);
      ok = ok_r;
    }
    if (t0 < lim_any) {
      // ---- scores: register 8 b + j of tile i is token 32 i + 16 b + (j & 3) + 8 (j >> 2) + 4 hf
      v16f s[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int j = 0; j < 16; ++j) s[i][j] = 0.f;
#pragma unroll
        for (int k = 0; k < KK; ++k) {
          const v4u a = *reinterpret_cast<const v4u*>(kbuf(buf) + (i * KK + k) * 1024 + hf * 512 +
                                                      ((n ^ (k & 7)) << 4));
          s[i] = mfma32(a, qh[k], s[i]);
          if constexpr (QLO) s[i] = mfma32(a, ql[k], s[i]);
        }
      }
      // ---- weights
      float iv[4];
      float top = -INFINITY;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const v4f sc = sbuf[buf][b];
        const float ck = c * sc[0];
        iv[b] = sc[2];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int e = 8 * (b & 1) + j;
          s[b >> 1][e] = fmaf(s[b >> 1][e], ck, sc[1]);
        }
      }
      if (t0 + kStep > lim_all || !was_ok) {
        const int left = (was_ok ? lim : 0) - t0 - 4 * hf;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 16; ++j)
            s[i][j] = 32 * i + (j & 3) + 8 * (j >> 2) < left ? s[i][j] : -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) top = fmaxf(top, s[i][j]);
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      if (__any(top > m + kHead || m == -INFINITY)) {
        const float mn = fmaxf(m, top);
        const float f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        l *= f;
#pragma unroll
        for (int j = 0; j < DT; ++j)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[j][i] *= f;
      }
      const float ref = m == -INFINITY ? 0.f : m - kUp;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        float sum = 0.f;
        v4u hi, lo;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float p0 = __builtin_amdgcn_exp2f(s[b >> 1][8 * (b & 1) + 2 * j] - ref);
          const float p1 = __builtin_amdgcn_exp2f(s[b >> 1][8 * (b & 1) + 2 * j + 1] - ref);
          sum += p0 + p1;
          uint32_t x, y = 0;
          if constexpr (PLO) split2(p0, p1, x, y);
          else x = pk(p0, p1);
          hi[j] = x;
          lo[j] = y;
        }
        l = fmaf(sum, iv[b], l);
        // ---- values
#pragma unroll
        for (int j = 0; j < DT; ++j) {
          const v4u a = *reinterpret_cast<const v4u*>(vbuf(buf) + (j * 4 + b) * 1024 + lane * 16);
          o[j] = mfma32(a, __builtin_bit_cast(v8h, hi), o[j]);
          if constexpr (PLO) o[j] = mfma32(a, __builtin_bit_cast(v8h, lo), o[j]);
        }
      }
    }
    if (more) put(st + 1, buf ^ 1);
    __syncthreads();
  }

  // ---- lane (n, hf) has coordinates 32 j + 8 q + 4 hf + 0 .. 3 of row n
  l += __shfl_xor(l, 32, 64);
  const int64_t slot = P.slot >= 0 ? place(A, P, h) : -1;
  if (!live) return;
  if (P.slot < 0) {
    const float inv = l > 0.f ? 1.f / l : 0.f;
    const int64_t at = (row * A.Hq + hq) * D + 4 * hf;
#pragma unroll
    for (int j = 0; j < DT; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float x[4] = {o[j][4 * q] * inv, o[j][4 * q + 1] * inv, o[j][4 * q + 2] * inv,
                            o[j][4 * q + 3] * inv};
        store4(A.out, at + 32 * j + 8 * q, x, A.out_dtype, A.out_vec);
      }
  } else if (slot >= 0) {
    const int64_t at = slot * kPreRows + 32 * wave + n;
#pragma unroll
    for (int j = 0; j < DT; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<v4f*>(A.part_o + at * D + 32 * j + 8 * q + 4 * hf) =
            v4f{o[j][4 * q], o[j][4 * q + 1], o[j][4 * q + 2], o[j][4 * q + 3]};
    if (hf == 0) {
      A.part_ml[2 * at] = m;
      A.part_ml[2 * at + 1] = l;
    }
  }
}

template <int D, bool FP8, bool QLO, bool PLO>
void start(const Att& A, uint32_t tiles, hipStream_t s) {
  constexpr int smem = 2 * (2 * (D / 16) + 4 * (D / 32)) * 1024;
  // (a failure is the launch's, which the caller reports)
  static const hipError_t attr [[maybe_unused]] = hipFuncSetAttribute(
      reinterpret_cast<const void*>(&prefill8<D, FP8, QLO, PLO>),
      hipFuncAttributeMaxDynamicSharedMemorySize, smem);
  prefill8<D, FP8, QLO, PLO><<<(tiles + A.target) * A.H, kThr, smem, s>>>(A);
}

template <int D, bool FP8>
void launch(const Att& A, uint32_t tiles, bool cut, hipStream_t s) {
  const bool qlo = A.q_dtype == QKV_F32, plo = A.out_dtype != QKV_BF16;
  if (qlo) {
    if (plo) start<D, FP8, true, true>(A, tiles, s);
    else start<D, FP8, true, false>(A, tiles, s);
  } else {
    if (plo) start<D, FP8, false, true>(A, tiles, s);
    else start<D, FP8, false, false>(A, tiles, s);
  }
  if (cut) join8<D, kPreRows><<<join_grid(A, kPreRows), kThr, 0, s>>>(A);
}

}  // namespace

void qkv_kv8_prefill(const Att& A, int32_t d, bool fp8, uint32_t tiles, bool cut, hipStream_t s) {
  if (fp8) {
    if (d == 128) launch<128, true>(A, tiles, cut, s);
    else if (d == 96) launch<96, true>(A, tiles, cut, s);
    else launch<64, true>(A, tiles, cut, s);
  } else {
    if (d == 128) launch<128, false>(A, tiles, cut, s);
    else if (d == 96) launch<96, false>(A, tiles, cut, s);
    else launch<64, false>(A, tiles, cut, s);
  }
}
