// Append to, and reads from, the 8-bit paged cache (qkv_kv8.h).
//
// Quantising a block, whose definition the codes meet exactly:
//   a = max |x| over the finite new values;  s = 0 if a = 0, else max(a / Z, 2^-100)
//   with the product rounded to fp32 (Z = 127 for int8, 448 for e4m3);
//   code = the one nearest to x * fp32(1 / s), ties to even, at most Z; NaN gives 0.
// A block that holds earlier tokens keeps its scale unless the new one is larger; then
// their values, fp32(code * scale), are quantised anew.
// x * (1 / s) in fp32 is off by half an ulp, which at a border between two codes would
// decide for the wrong one: sticky_mul keeps what the rounding dropped in the last bit
// (round to odd), so that rounding to a code afterwards is rounding once.
//
// Bytes bound it: 2 H d (in + 1) a row, and a decode step's token reads and writes its
// V block (16 tokens) beside that.
#include "qkv_kv8.h"

namespace {

// x * m with the last bit set where the product is not exact (towards zero).
__device__ __forceinline__ float sticky_mul(float x, float m) {
  const float p = x * m, e = fmaf(x, m, -p);
  uint32_t u = __float_as_uint(p);
  if (e != 0.f) u = (u - ((e < 0.f) != (p < 0.f) ? 1u : 0u)) | 1u;
  return __uint_as_float(u);
}

// The code of x at inverse scale inv, one byte.
template <bool FP8>
__device__ __forceinline__ uint32_t code_of(float x, float inv) {
  constexpr float Z = kTop<FP8>;
  float p = x * inv;
  if (fabsf(p) >= Z) p = copysignf(Z, p);
  else p = sticky_mul(x, inv);
  if (p != p) p = 0.f;  // (NaN, or an infinity in a block of zeros)
  if constexpr (FP8)
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(p, p, 0, false)) & 0xffu;
  else
    return static_cast<uint32_t>(__float2int_rn(p)) & 0xffu;
}

template <bool FP8>
__device__ __forceinline__ float value_of(uint32_t code) {
  if constexpr (FP8)
    return __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(code & 0xffu), 0);
  else
    return static_cast<float>(static_cast<int8_t>(code));
}

struct App {
  const void* x[2];       // keys, values
  int64_t ts[2], hs[2];   // their token and head strides (elements)
  const int64_t* slots;
  int64_t rows;
  uint8_t* pool[2];
  float* scale[2];
  int64_t tokens;         // slots of the pool
  int32_t lg, H, chunk;
};

// A wave per (chunk of rows, head, half).  A run: rows whose slots ascend within one
// block.  The wave that holds a run's first row does all of it: lane l has the
// coordinates 2 l and 2 l + 1 of all 16 tokens.
template <int D, bool FP8, int DT>
__global__ __launch_bounds__(64) void append_runs(App A) {
  const int lane = threadIdx.x, h = blockIdx.y, half = blockIdx.z;
  const bool on = 2 * lane < D;
  const int c = on ? 2 * lane : 0;
  const int64_t r0 = int64_t(blockIdx.x) * A.chunk;
  const int64_t r1 = r0 + A.chunk < A.rows ? r0 + A.chunk : A.rows;
  const int64_t n = int64_t(1) << A.lg;
  for (int64_t r = r0; r < r1; ++r) {
    const int64_t s = A.slots[r];
    if (s < 0 || s >= A.tokens) continue;
    if (r > 0) {
      const int64_t prev = A.slots[r - 1];
      if (prev >= 0 && (prev >> 4) == (s >> 4) && prev < s) continue;  // inside a run
    }
    const int j0 = static_cast<int>(s & 15);
    float x[kBlk][2];
    uint32_t have = 0;  // tokens of the block that the run brings
#pragma unroll
    for (int j = 0; j < kBlk; ++j) x[j][0] = x[j][1] = 0.f;
    {
      int64_t rr = r, cur = s, last = -1;
#pragma unroll
      for (int j = 0; j < kBlk; ++j) {
        if (cur >= 0 && (cur >> 4) == (s >> 4) && cur > last && (cur & 15) == j) {
          const int64_t at = rr * A.ts[half] + h * A.hs[half] + c;
          if (on) {
            x[j][0] = qkv_load(A.x[half], at, DT);
            x[j][1] = qkv_load(A.x[half], at + 1, DT);
          }
          have |= 1u << j;
          last = cur;
          ++rr;
          cur = rr < A.rows ? A.slots[rr] : -1;
        }
      }
    }
    float a = 0.f;
#pragma unroll
    for (int j = 0; j < kBlk; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float m = fabsf(x[j][i]);
        if (m < INFINITY) a = fmaxf(a, m);
      }
    a = qkv_wave_max(a);
    const int64_t page = s >> A.lg, o = s & (n - 1);
    const int64_t row = (page * A.H + h) * n + (o & ~int64_t(15));  // block's first K row
    float* const sp = A.scale[half] + (row >> 4);
    const float old = j0 > 0 ? *sp : 0.f;
    float sc = a > 0.f ? fmaxf(a * (1.f / kTop<FP8>), kScaleFloor) : 0.f;
    const bool grew = sc > old;
    sc = grew ? sc : old;
    const float inv = sc > 0.f ? 1.f / sc : 0.f;
    uint8_t* const base = A.pool[half] + row * D;
    if (half == 0) {
      uint16_t* const k = reinterpret_cast<uint16_t*>(base + c);
#pragma unroll
      for (int j = 0; j < kBlk; ++j) {
        if (have >> j & 1) {
          if (on)
            k[j * (D / 2)] = static_cast<uint16_t>(code_of<FP8>(x[j][0], inv) |
                                                   code_of<FP8>(x[j][1], inv) << 8);
        } else if (j < j0 && grew && on) {
          const uint32_t u = k[j * (D / 2)];
          k[j * (D / 2)] =
              static_cast<uint16_t>(code_of<FP8>(value_of<FP8>(u) * old, inv) |
                                    code_of<FP8>(value_of<FP8>(u >> 8) * old, inv) << 8);
        }
      }
    } else if (on) {
      uint4* const v = reinterpret_cast<uint4*>(base + c * kBlk);
      uint32_t w[2][4] = {};
      if (j0 > 0) {
        *reinterpret_cast<uint4*>(w[0]) = v[0];
        *reinterpret_cast<uint4*>(w[1]) = v[1];
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t u = 0;
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const int j = 4 * q + b;
            uint32_t code = 0;
            if (have >> j & 1) {
              code = code_of<FP8>(x[j][i], inv);
            } else if (j < j0) {
              code = w[i][q] >> (8 * b) & 0xffu;
              if (grew) code = code_of<FP8>(value_of<FP8>(code) * old, inv);
            }
            u |= code << (8 * b);
          }
          w[i][q] = u;
        }
      v[0] = *reinterpret_cast<uint4*>(w[0]);
      v[1] = *reinterpret_cast<uint4*>(w[1]);
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
  int32_t lg, H;
  void* out[2];
};

// A wave per (row, head, half): lane l has the coordinates 2 l and 2 l + 1.
template <int D, bool FP8, int DT>
__global__ __launch_bounds__(256) void read_rows(Rd A) {
  const int lane = threadIdx.x & 63, h = blockIdx.y, half = blockIdx.z;
  const int64_t r = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (r >= A.rows || 2 * lane >= D) return;
  const int c = 2 * lane;
  const int64_t s = A.slots[r], n = int64_t(1) << A.lg;
  float v0 = 0.f, v1 = 0.f;
  if (s >= 0 && s < A.tokens) {
    const int64_t o = s & (n - 1), row = ((s >> A.lg) * A.H + h) * n + o;
    const float sc = A.scale[half][row >> 4];
    uint32_t a, b;
    if (half == 0) {
      const uint8_t* p = A.pool[0] + row * D + c;
      a = p[0];
      b = p[1];
    } else {
      const uint8_t* p = A.pool[1] + (row & ~int64_t(15)) * D + c * kBlk + (o & 15);
      a = p[0];
      b = p[kBlk];
    }
    v0 = value_of<FP8>(a) * sc;
    v1 = value_of<FP8>(b) * sc;
  }
  const int64_t at = (r * A.H + h) * D + c;
  qkv_store(A.out[half], at, v0, DT);
  qkv_store(A.out[half], at + 1, v1, DT);
}

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
  App A{{keys, values},
        {k_row_stride, v_row_stride},
        {k_head_stride, v_head_stride},
        slots,
        rows,
        {static_cast<uint8_t*>(kpool), static_cast<uint8_t*>(vpool)},
        {kscale, vscale},
        int64_t(num_pages) * page_tokens,
        qkv_page_lg(page_tokens),
        H,
        1};
  const dim3 grid(static_cast<uint32_t>((rows + A.chunk - 1) / A.chunk), H, 2);
  hipStream_t s = static_cast<hipStream_t>(stream);
#define RUN(D, FP8, DT) append_runs<D, FP8, DT><<<grid, 64, 0, s>>>(A)
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
  Rd A{slots,
       rows,
       {static_cast<const uint8_t*>(kpool), static_cast<const uint8_t*>(vpool)},
       {kscale, vscale},
       int64_t(num_pages) * page_tokens,
       qkv_page_lg(page_tokens),
       H,
       {keys, values}};
  const dim3 grid(static_cast<uint32_t>((rows + 3) / 4), H, 2);
  hipStream_t s = static_cast<hipStream_t>(stream);
#define RUN(D, FP8, DT) read_rows<D, FP8, DT><<<grid, 256, 0, s>>>(A)
  QKV_KV8_DISPATCH(RUN, d, fmt, out_dtype)
#undef RUN
  QKV_LAUNCHED();
  return QKV_OK;
}
