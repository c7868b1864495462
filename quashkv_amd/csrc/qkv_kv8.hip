// Append to, and reads from, the 8-bit paged cache (qkv_kv8.h).
//
// Quantising a block, whose definition the codes meet exactly:
//   a = max |x| over the finite new values;  s = 0 if a = 0, else max(a / Z, 2^-100)
//   with the product rounded to fp32 (Z = 127 for int8, 448 for e4m3);
//   code = the one nearest to x * fp32(1 / s), ties to even, at most Z; NaN gives 0.
// A block that holds earlier tokens keeps its scale unless the new one is larger; then
// their values, fp32(code * scale), are quantised anew.
// x * (1 / s) rounded to fp32 is off by half an ulp, which at a border between two codes
// would decide for the wrong one.  So the product is never rounded by itself:
// fma(x, 1 / s, M) with M = 1.5 * 2^23 times the spacing of the codes around it rounds the
// exact product once, to a multiple of that spacing, ties to even -- one instruction a
// value for int8, whose code then is the sum's low byte.
//
// Bytes bound it: 2 H d (in + 1) a row, and a decode step's token reads and writes its
// V block (16 tokens) beside that.  Measured, 24,000 bf16 rows of 8 heads, d = 128, cold:
// append 43 us (3.4 TB/s), read to bf16 35 us (4.2 TB/s); 64 rows, one per request: 5.7 and
// 6.2 us a kernel.  Rows in the caches take 32 and 29 us: the rest is a wave's chain, one
// block's loads (four a lane), the reduction over them, the stores, then the next block's.
#include "qkv_kv8.h"

namespace {

// The code of x at inverse scale inv, |x| at most what the largest code stands for (but for
// rounding): int8 in the low byte, e4m3 as a value that its conversion leaves as it is.
template <bool FP8>
__device__ __forceinline__ float near(float x, float inv) {
  if constexpr (FP8) {
    // the spacing is 2^-3 of the product's power of two, 2^-9 at least
    const uint32_t e = max(__float_as_uint(x * inv) & 0x7f800000u, 121u << 23);
    const float M = __uint_as_float(e + (20u << 23) + 0x400000u);
    return fmaf(x, inv, M) - M;
  } else {
    return fmaf(x, inv, 12582912.f);
  }
}

// Four codes of near() as bytes.
template <bool FP8>
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
  if constexpr (FP8) {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true));
  } else {
    const uint32_t ab = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x0c0c0400u);
    const uint32_t cd = __builtin_amdgcn_perm(__float_as_uint(d), __float_as_uint(c), 0x04000c0cu);
    return ab | cd;
  }
}

template <bool FP8>
__device__ __forceinline__ float value_of(uint32_t code) {
  if constexpr (FP8)
    return __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(code & 0xffu), 0);
  else
    return static_cast<float>(static_cast<int8_t>(code));
}

typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;  // of a workgroup, each with a unit of its own

// Eight consecutive elements from element `at` of x; vec: their address is 16-byte aligned.
template <int DT>
__device__ __forceinline__ void load8(const void* x, int64_t at, bool vec, float* to) {
  if (!vec) {
#pragma unroll
    for (int i = 0; i < 8; ++i) to[i] = qkv_load(x, at + i, DT);
  } else if constexpr (DT == QKV_F32) {
    const v4f* const p = reinterpret_cast<const v4f*>(static_cast<const float*>(x) + at);
    const v4f a = p[0], b = p[1];
#pragma unroll
    for (int i = 0; i < 8; ++i) to[i] = i < 4 ? a[i & 3] : b[i & 3];
  } else {
    const v4u w = *reinterpret_cast<const v4u*>(static_cast<const uint16_t*>(x) + at);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint16_t u = static_cast<uint16_t>(w[i >> 1] >> (16 * (i & 1)));
      to[i] = DT == QKV_BF16 ? qkv_bf16_to_f32(u)
                             : static_cast<float>(__builtin_bit_cast(_Float16, u));
    }
  }
}

// Eight consecutive elements to element `at` of a dense output.
template <int DT>
__device__ __forceinline__ void store8(void* x, int64_t at, bool vec, const float* v) {
  if (!vec) {
#pragma unroll
    for (int i = 0; i < 8; ++i) qkv_store(x, at + i, v[i], DT);
  } else if constexpr (DT == QKV_F32) {
    v4f* const p = reinterpret_cast<v4f*>(static_cast<float*>(x) + at);
    p[0] = v4f{v[0], v[1], v[2], v[3]};
    p[1] = v4f{v[4], v[5], v[6], v[7]};
  } else {
    v4u w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == QKV_BF16)
        w[i] = qkv_f32_to_bf16(v[2 * i]) | uint32_t(qkv_f32_to_bf16(v[2 * i + 1])) << 16;
      else
        w[i] = uint32_t(__builtin_bit_cast(uint16_t, static_cast<_Float16>(v[2 * i]))) |
               uint32_t(__builtin_bit_cast(uint16_t, static_cast<_Float16>(v[2 * i + 1]))) << 16;
    }
    *reinterpret_cast<v4u*>(static_cast<uint16_t*>(x) + at) = w;
  }
}

// A block's scale: of the largest of a wave's values, or the old one where that is larger.
// Values that are not finite do not count; they become what their codes stand for (the
// largest value, NaN 0).
template <bool FP8, int N>
__device__ __forceinline__ float scale_of(float* x, float old, bool& grew, float& inv) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
  auto wave_max = [](uint32_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = max(v, static_cast<uint32_t>(__shfl_xor(int(v), o, 64)));
    return v;
  };
  m = wave_max(m);
  const bool odd = m >= 0x7f800000u;
  if (odd) {
    m = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t u = __float_as_uint(x[i]) & 0x7fffffffu;
      m = max(m, u < 0x7f800000u ? u : 0u);
    }
    m = wave_max(m);
  }
  const float a = __uint_as_float(m);
  float sc = a > 0.f ? fmaxf(a * (1.f / kTop<FP8>), kScaleFloor) : 0.f;
  grew = sc > old;
  sc = grew ? sc : old;
  inv = sc > 0.f ? 1.f / sc : 0.f;
  if (odd) {
    const float top = kTop<FP8> * sc;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (x[i] != x[i]) x[i] = 0.f;
      x[i] = __builtin_amdgcn_fmed3f(x[i], -top, top);
    }
  }
  return sc;
}

struct App {
  const void* x[2];       // keys, values
  int64_t ts[2], hs[2];   // their row and head strides (elements)
  int32_t vec[2];         // whether 16-byte loads are aligned
  const int64_t* slots;
  int64_t rows;
  uint8_t* pool[2];
  float* scale[2];
  int64_t tokens;         // slots of the pool
  int32_t lg, H, chunk;
  int64_t units;          // chunks x heads
};

// A wave per (chunk of rows, head), a launch row each for keys and values.  A run: rows at
// consecutive slots of one block; the wave in whose chunk it begins does all of it, so that
// a block's largest value is a wave's reduction.  The chunk's slots and those that its
// last run may reach are read at once, a lane each.  Lane l has 8 coordinates of every
// (512 / D)-th token: whole rows in 16-byte loads, a key's codes in 8-byte stores.  A value
// block's codes turn through LDS, so that a lane stores the 16 tokens of a coordinate.
// (Loads of a pair of coordinates per token straight into that order, 4 bytes a lane: 41 us
// for the values of 24,000 rows, 8 heads, d = 128, the keys 23.)
template <int D, bool FP8, int DT>
__global__ __launch_bounds__(64 * kWaves) void append_runs(App A) {
  constexpr int LPR = D / 8, RPI = 64 / LPR, NI = (kBlk + RPI - 1) / RPI;
  __shared__ __align__(16) uint8_t turn[kWaves][kBlk * D];
  const int lane = threadIdx.x & 63, half = blockIdx.y;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t u = int64_t(blockIdx.x) * kWaves + wave;
  if (u >= A.units) return;
  const int64_t r0 = u / A.H * A.chunk;
  const int h = static_cast<int>(u % A.H);
  // lane i: row r0 - 1 + i
  const int64_t at = r0 - 1 + lane;
  int64_t sl = at >= 0 && at < A.rows ? A.slots[at] : -1;
  if (sl >= A.tokens) sl = -1;
  const int64_t prev = __shfl_up(static_cast<long long>(sl), 1, 64);
  const bool cont = lane > 0 && sl >= 0 && prev >= 0 && sl == prev + 1 && (sl & 15) != 0;
  const uint64_t conts = __ballot(cont);
  uint64_t heads = __ballot(sl >= 0 && !cont) & ((uint64_t(2) << A.chunk) - 2);
  const int64_t n = int64_t(1) << A.lg;
  const int sub = lane / LPR, c = 8 * (lane % LPR);
  while (heads) {
    const int i0 = __builtin_ctzll(heads);
    heads &= heads - 1;
    const int len = 1 + __builtin_ctzll(~(conts >> (i0 + 1)));
    const int64_t s = __shfl(static_cast<long long>(sl), i0, 64), r = r0 - 1 + i0;
    const int j0 = static_cast<int>(s & 15), j1 = j0 + len;  // the run's places in the block
    const int64_t row = ((s >> A.lg) * A.H + h) * n + (s & (n - 16));  // the block's first row
    float* const sp = A.scale[half] + (row >> 4);
    uint8_t* const base = A.pool[half] + row * D;
    const int64_t src = (r - j0) * A.ts[half] + h * A.hs[half];  // of place 0
    const float old = j0 > 0 ? *sp : 0.f;
    bool grew;
    float inv, x[NI][8];
#pragma unroll
    for (int t = 0; t < NI; ++t) {
      const int j = RPI * t + sub;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[t][i] = 0.f;
      if (sub < RPI && j >= j0 && j < j1)
        load8<DT>(A.x[half], src + j * A.ts[half] + c, A.vec[half], x[t]);
    }
    const float sc = scale_of<FP8, 8 * NI>(&x[0][0], old, grew, inv);
#pragma unroll
    for (int t = 0; t < NI; ++t) {
      const int j = RPI * t + sub;
      const bool in = sub < RPI && j < kBlk;
      v2u* const k = reinterpret_cast<v2u*>((half == 0 ? base : turn[wave]) + j * D + c);
      bool put = in && (half != 0 || (j >= j0 && j < j1));
      if (half == 0 && in && j < j0 && grew) {  // an earlier key at the new scale
        const v2u w = *k;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[t][i] = value_of<FP8>(w[i >> 2] >> (8 * (i & 3))) * old;
        put = true;
      }
      if (put) {
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = near<FP8>(x[t][i], inv);
        *k = v2u{pack4<FP8>(y[0], y[1], y[2], y[3]), pack4<FP8>(y[4], y[5], y[6], y[7])};
      }
    }
    if (half != 0) {
      // (a wave's LDS operations keep their order)
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
      for (int d0 = 0; d0 < D; d0 += 64) {
        const int dd = d0 + lane;
        if (dd >= D) continue;
        v4u* const v = reinterpret_cast<v4u*>(base + dd * kBlk);
        uint32_t w[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint8_t* const p = turn[wave] + 4 * q * D + dd;
          w[q] = p[0] | uint32_t(p[D]) << 8 | uint32_t(p[2 * D]) << 16 | uint32_t(p[3 * D]) << 24;
        }
        if (j0 > 0) {  // earlier tokens: their codes, or those at the new scale
          const v4u was = *v;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t e = was[q];
            if (grew) {
              float y[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) y[i] = near<FP8>(value_of<FP8>(e >> (8 * i)) * old, inv);
              e = pack4<FP8>(y[0], y[1], y[2], y[3]);
            }
            const int m = j0 - 4 * q;
            const uint32_t keep = m >= 4 ? ~0u : m <= 0 ? 0u : (1u << (8 * m)) - 1u;
            w[q] = (e & keep) | (w[q] & ~keep);
          }
        }
        *v = v4u{w[0], w[1], w[2], w[3]};
      }
      __builtin_amdgcn_wave_barrier();
    }
    if (lane == 0) *sp = sc;
  }
}

struct Rd {
  const int64_t* slots;
  int64_t rows;
  const uint8_t* pool[2];
  const float* scale[2];
  int64_t tokens;
  int32_t lg, H, chunk;
  int64_t units;
  void* out[2];
  int32_t vec[2];
};

// A wave per (chunk of up to 16 rows, head), lanes as in append_runs; a V block is read once
// for a run of consecutive slots in it, and turns through LDS too.
template <int D, bool FP8, int DT>
__global__ __launch_bounds__(64 * kWaves) void read_rows(Rd A) {
  constexpr int LPR = D / 8, RPI = 64 / LPR, NI = (kBlk + RPI - 1) / RPI;
  __shared__ __align__(16) uint8_t turn[kWaves][kBlk * D];
  const int lane = threadIdx.x & 63, half = blockIdx.y;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t u = int64_t(blockIdx.x) * kWaves + wave;
  if (u >= A.units) return;
  const int64_t r0 = u / A.H * A.chunk, n = int64_t(1) << A.lg;
  const int h = static_cast<int>(u % A.H);
  // lane i: row r0 + i
  const bool mine = lane < A.chunk && r0 + lane < A.rows;
  int64_t sl = mine ? A.slots[r0 + lane] : -1;
  if (sl >= A.tokens) sl = -1;
  const uint64_t rows = __ballot(mine);
  auto row_of = [&](int64_t s) { return ((s >> A.lg) * A.H + h) * n + (s & (n - 1)); };
  const int sub = lane / LPR, c = 8 * (lane % LPR);
  // eight codes to the chunk's row i
  auto put = [&](v2u w, float sc, int i) {
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = value_of<FP8>(w[j >> 2] >> (8 * (j & 3))) * sc;
    store8<DT>(A.out[half], ((r0 + i) * A.H + h) * D + c, A.vec[half], x);
  };
  if (half == 0) {
    v2u w[NI];
    float sc[NI];
#pragma unroll
    for (int t = 0; t < NI; ++t) {
      const int i = RPI * t + sub;
      const int64_t s = __shfl(static_cast<long long>(sl), i & 63, 64);
      w[t] = v2u{0, 0};
      sc[t] = 0.f;
      if (sub < RPI && i < A.chunk && s >= 0) {
        const int64_t row = row_of(s);
        w[t] = *reinterpret_cast<const v2u*>(A.pool[0] + row * D + c);
        sc[t] = A.scale[0][row >> 4];
      }
    }
#pragma unroll
    for (int t = 0; t < NI; ++t) {
      const int i = RPI * t + sub;
      if (sub < RPI && i < kBlk && (rows >> i & 1)) put(w[t], sc[t], i);
    }
  } else {
    const int64_t prev = __shfl_up(static_cast<long long>(sl), 1, 64);
    const bool cont = lane > 0 && sl >= 0 && sl == prev + 1 && (sl & 15) != 0;
    const uint64_t conts = __ballot(cont && mine);
    uint64_t heads = __ballot(mine && !cont);
    while (heads) {
      const int i0 = __builtin_ctzll(heads);
      heads &= heads - 1;
      const int64_t s = __shfl(static_cast<long long>(sl), i0, 64);
      const int len = s < 0 ? 1 : 1 + __builtin_ctzll(~(conts >> (i0 + 1)));
      const int j0 = s < 0 ? 0 : static_cast<int>(s & 15), j1 = j0 + len;
      float sc = 0.f;
      if (s >= 0) {
        const int64_t row = row_of(s) & ~int64_t(15);
        sc = A.scale[1][row >> 4];
#pragma unroll
        for (int e = 0; e < D; e += 64) {
          const int dd = e + lane;
          if (dd >= D) continue;
          const v4u w = *reinterpret_cast<const v4u*>(A.pool[1] + row * D + dd * kBlk);
#pragma unroll
          for (int j = 0; j < kBlk; ++j)
            turn[wave][j * D + dd] = static_cast<uint8_t>(w[j >> 2] >> (8 * (j & 3)));
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
      for (int t = 0; t < NI; ++t) {
        const int j = RPI * t + sub;
        if (sub >= RPI || j < j0 || j >= j1) continue;
        v2u w = {0, 0};
        if (s >= 0) w = *reinterpret_cast<const v2u*>(turn[wave] + j * D + c);
        put(w, sc, i0 + j - j0);
      }
      __builtin_amdgcn_wave_barrier();
    }
  }
}

// Rows of a wave's unit, by the rows alone.  Many rows are mostly prompts, whose runs fill a
// block: one wave a block.  Few are mostly a decode step's, each a run of its own, which would
// queue in one wave.  us of an append / a read with 16, 4 and 1 rows a unit (bf16, d = 128,
// cached):
//   24,000 rows of 24 requests, 8 heads    32 / 29     60 / 40    321 / 119
//   2000 rows of 5 requests, 8 heads        5 / 5      11 / 6      33 / 13
//   1496 rows of 8 requests, 8 heads      6.8 / 6.3   5.8 / 5.8   9.3 / 10.2
//   600 requests of a row, 8 heads         29 / 18     12 / 6      10 / 6
//   64 requests of a row, 8 heads          28 / 16    8.7 / 5.6   3.9 / 2.9
//   600 requests of a row, one head        28 / 16    8.9 / 5.6   4.1 / 3.1
//   2000 rows of 5 requests, 32 heads      13 / 12     35 / 15     49 / 43
// (So 600 decoding requests with one head, and 2000 rows of prompts with 8 heads or more, are not
// best served.)
int32_t chunk_of(int64_t rows) { return rows > 4096 ? 16 : rows > 512 ? 4 : 1; }

}  // namespace

int qkv_kv8_check(int32_t fmt, int32_t num_pages, int32_t page_tokens, int32_t H, int32_t d) {
  QKV_REQUIRE(fmt == QKV_CODES_I8 || fmt == QKV_CODES_E4M3, "unknown code format %d", fmt);
  QKV_REQUIRE(num_pages >= 1, "num_pages must be positive; got %d", num_pages);
  QKV_REQUIRE(qkv_page_lg(page_tokens) >= 0,
              "page_tokens must be 64 << k, k = 0 .. 5; got %d", page_tokens);
  QKV_REQUIRE(H >= 1 && H <= 65535, "kv heads must lie in [1, 65535]; got %d", H);
  if (!qkv_d_ok(d)) {
    qkv_set_error("the 8-bit cache runs head_dim 64, 96 or 128; got %d", d);
    return QKV_E_UNSUPPORTED;
  }
  return QKV_OK;
}

// F(D, FP8, DT) for the runtime d, format and element type
#define QKV_KV8_DT(F, D, FP8, dt)              \
  switch (dt) {                                \
    case QKV_F32: F(D, FP8, QKV_F32); break;   \
    case QKV_F16: F(D, FP8, QKV_F16); break;   \
    default: F(D, FP8, QKV_BF16); break;       \
  }
#define QKV_KV8_FMT(F, D, fmt, dt)                                          \
  if ((fmt) == QKV_CODES_I8) { QKV_KV8_DT(F, D, false, dt) } else { QKV_KV8_DT(F, D, true, dt) }
#define QKV_KV8_DISPATCH(F, d, fmt, dt)               \
  if ((d) == 128) { QKV_KV8_FMT(F, 128, fmt, dt) }    \
  else if ((d) == 96) { QKV_KV8_FMT(F, 96, fmt, dt) } \
  else { QKV_KV8_FMT(F, 64, fmt, dt) }

extern "C" int qkv_kv8_append(int32_t in_dtype, const void* keys, int64_t k_row_stride,
                              int64_t k_head_stride, const void* values, int64_t v_row_stride,
                              int64_t v_head_stride, const int64_t* slots, int64_t rows, int32_t H,
                              int32_t d, int32_t fmt, void* kpool, float* kscale, void* vpool,
                              float* vscale, int32_t num_pages, int32_t page_tokens,
                              void* stream) {
  const int st = qkv_kv8_check(fmt, num_pages, page_tokens, H, d);
  if (st != QKV_OK) return st;
  QKV_REQUIRE(qkv_dtype_ok(in_dtype), "unknown input dtype %d", in_dtype);
  QKV_REQUIRE(rows >= 0 && rows < INT32_MAX, "rows must lie in [0, 2^31 - 1); got %lld",
              static_cast<long long>(rows));
  if (rows == 0) return QKV_OK;
  QKV_REQUIRE(keys && values && slots && kpool && kscale && vpool && vscale,
              "qkv_kv8_append: null pointer");
  QKV_REQUIRE(qkv_aligned(kpool, 16) && qkv_aligned(vpool, 16),
              "the pools must be 16-byte aligned");
  const int es = in_dtype == QKV_F32 ? 4 : 2;
  auto aligned = [&](const void* p, int64_t rs, int64_t hs) {
    return int32_t(qkv_aligned(p, 16) && rs * es % 16 == 0 && hs * es % 16 == 0);
  };
  const int32_t chunk = chunk_of(rows);
  const int64_t units = (rows + chunk - 1) / chunk * H;
  App A{{keys, values},
        {k_row_stride, v_row_stride},
        {k_head_stride, v_head_stride},
        {aligned(keys, k_row_stride, k_head_stride), aligned(values, v_row_stride, v_head_stride)},
        slots,
        rows,
        {static_cast<uint8_t*>(kpool), static_cast<uint8_t*>(vpool)},
        {kscale, vscale},
        int64_t(num_pages) * page_tokens,
        qkv_page_lg(page_tokens),
        H,
        chunk,
        units};
  QKV_REQUIRE(units / kWaves < INT32_MAX, "too many rows (%lld) for one call",
              static_cast<long long>(rows));
  const dim3 grid(static_cast<uint32_t>((units + kWaves - 1) / kWaves), 2);
  hipStream_t s = static_cast<hipStream_t>(stream);
#define RUN(D, FP8, DT) append_runs<D, FP8, DT><<<grid, 64 * kWaves, 0, s>>>(A)
  QKV_KV8_DISPATCH(RUN, d, fmt, in_dtype)
#undef RUN
  QKV_LAUNCHED();
  return QKV_OK;
}

extern "C" int qkv_kv8_read(const int64_t* slots, int64_t rows, int32_t H, int32_t d, int32_t fmt,
                            const void* kpool, const float* kscale, const void* vpool,
                            const float* vscale, int32_t num_pages, int32_t page_tokens,
                            void* keys, void* values, int32_t out_dtype, void* stream) {
  const int st = qkv_kv8_check(fmt, num_pages, page_tokens, H, d);
  if (st != QKV_OK) return st;
  QKV_REQUIRE(qkv_dtype_ok(out_dtype), "unknown output dtype %d", out_dtype);
  QKV_REQUIRE(rows >= 0 && rows < INT32_MAX, "rows must lie in [0, 2^31 - 1); got %lld",
              static_cast<long long>(rows));
  if (rows == 0) return QKV_OK;
  QKV_REQUIRE(keys && values && slots && kpool && kscale && vpool && vscale,
              "qkv_kv8_read: null pointer");
  QKV_REQUIRE(qkv_aligned(kpool, 16) && qkv_aligned(vpool, 16),
              "the pools must be 16-byte aligned");
  const int32_t chunk = chunk_of(rows);
  const int64_t units = (rows + chunk - 1) / chunk * H;
  Rd A{slots,
       rows,
       {static_cast<const uint8_t*>(kpool), static_cast<const uint8_t*>(vpool)},
       {kscale, vscale},
       int64_t(num_pages) * page_tokens,
       qkv_page_lg(page_tokens),
       H,
       chunk,
       units,
       {keys, values},
       {qkv_aligned(keys, 16), qkv_aligned(values, 16)}};
  QKV_REQUIRE(units / kWaves < INT32_MAX, "too many rows (%lld) for one call",
              static_cast<long long>(rows));
  const dim3 grid(static_cast<uint32_t>((units + kWaves - 1) / kWaves), 2);
  hipStream_t s = static_cast<hipStream_t>(stream);
#define RUN(D, FP8, DT) read_rows<D, FP8, DT><<<grid, 64 * kWaves, 0, s>>>(A)
  QKV_KV8_DISPATCH(RUN, d, fmt, out_dtype)
#undef RUN
  QKV_LAUNCHED();
  return QKV_OK;
}
