// Rotary positions of query and key rows (C ABI: qkv_rotary).
//
// The pair i of a head's first R coordinates -- (i, i + R / 2), or (2 i, 2 i + 1) where they are
// interleaved -- turns by the angle 2 pi p f_i at position p:
//   y1 = c (x1 cos - x2 sin),  y2 = c (x2 cos + x1 sin);
// coordinates behind R stay as they are.  f_i comes as turns in units of 2^-64, so that p f_i
// modulo a turn is an integer product modulo 2^64: exact but for the rounding of f_i itself,
// |p| 2^-65 turns, at any position.  Sine and cosine are fp32's of the nearest fp32 to the
// remainder in [-1/2, 1/2) (off by 2^-26 turns at most, 2^-25 half turns, and less the smaller it
// is); products and sums are fp32, rounded once to the rows' type.
//
// Bytes bound it, each row in and out: a workgroup has the angles of its rows in LDS, one sine
// and cosine for all heads, and then goes over the rows' pairs with 16-byte loads.
#include <algorithm>

#include "qkv_common.h"

namespace {

typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));

constexpr int kThr = 256;
constexpr int kMaxRows = 8;     // of a workgroup
constexpr int kMaxPairs = 256;  // R / 2

struct Rot {
  const void* x[2];           // queries, keys
  void* y[2];
  int64_t ts[2], hs[2];       // row and head strides (elements) in,
  int64_t to[2], ho[2];       // and out
  int32_t heads[2];
  int64_t rows;
  int32_t d, R, wg_rows;
  int32_t copy;               // whether the coordinates behind R are written
  const int32_t* pos;
  const int64_t* turns;
  float factor, sign;
};

// Eight consecutive elements, 16-byte aligned.
template <int DT>
__device__ __forceinline__ void load8(const void* x, int64_t at, float* to) {
  if constexpr (DT == QKV_F32) {
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

template <int DT>
__device__ __forceinline__ void store8(void* x, int64_t at, const float* v) {
  if constexpr (DT == QKV_F32) {
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

// VEC: pairs eight (half) or four (interleaved) at a time in 16-byte accesses; else one at a time.
template <int DT, bool PAIRS, bool VEC>
__global__ __launch_bounds__(kThr) void rotate(Rot A) {
  extern __shared__ float2 cs[];  // [row][pair] c cos, c sin
  const int tid = threadIdx.x;
  const int half = A.R / 2;
  const int64_t r0 = int64_t(blockIdx.x) * A.wg_rows;
  const int nr = static_cast<int>(min(int64_t(A.wg_rows), A.rows - r0));
  for (int i = tid; i < nr * half; i += kThr) {
    const int r = i / half, k = i - r * half;
    // (two's complement: the product modulo 2^64 is right for negative positions, too)
    const int64_t turn = static_cast<int64_t>(static_cast<uint64_t>(A.turns[k]) *
                                              static_cast<uint64_t>(int64_t(A.pos[r0 + r])));
    float s, c;
    sincospif(static_cast<float>(turn) * 0x1p-63f, &s, &c);
    cs[i] = float2{c * A.factor, s * A.factor * A.sign};
  }
  __syncthreads();
  constexpr int PER = VEC ? (PAIRS ? 4 : 8) : 1;  // pairs of a unit
  const int turned = (half + PER - 1) / PER;
  const int rest = A.copy ? (VEC ? (A.d - A.R) / 8 : A.d - A.R) : 0;
  const int units = turned + rest, heads = A.heads[0] + A.heads[1];
  for (int i = tid; i < nr * heads * units; i += kThr) {
    const int u = i % units, j = i / units, r = j / heads;
    int h = j - r * heads;
    const int w = h >= A.heads[0];
    h -= w ? A.heads[0] : 0;
    const int64_t x = (r0 + r) * A.ts[w] + h * A.hs[w], y = (r0 + r) * A.to[w] + h * A.ho[w];
    if (u >= turned) {  // behind R
      const int c = A.R + (u - turned) * (VEC ? 8 : 1);
      if constexpr (VEC) {
        float a[8];
        load8<DT>(A.x[w], x + c, a);
        store8<DT>(A.y[w], y + c, a);
      } else {
        qkv_store(A.y[w], y + c, qkv_load(A.x[w], x + c, DT), DT);
      }
      continue;
    }
    const int k0 = u * PER;
    const float2* const t = cs + r * half + k0;
    if constexpr (!VEC) {
      const int a = PAIRS ? 2 * k0 : k0, b = PAIRS ? a + 1 : a + half;
      const float p = qkv_load(A.x[w], x + a, DT), q = qkv_load(A.x[w], x + b, DT);
      qkv_store(A.y[w], y + a, p * t[0].x - q * t[0].y, DT);
      qkv_store(A.y[w], y + b, q * t[0].x + p * t[0].y, DT);
    } else if constexpr (PAIRS) {
      float a[8], b[8];
      load8<DT>(A.x[w], x + 2 * k0, a);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        b[2 * e] = a[2 * e] * t[e].x - a[2 * e + 1] * t[e].y;
        b[2 * e + 1] = a[2 * e + 1] * t[e].x + a[2 * e] * t[e].y;
      }
      store8<DT>(A.y[w], y + 2 * k0, b);
    } else {
      float a[8], b[8], p[8], q[8];
      load8<DT>(A.x[w], x + k0, a);
      load8<DT>(A.x[w], x + k0 + half, b);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[e] = a[e] * t[e].x - b[e] * t[e].y;
        q[e] = b[e] * t[e].x + a[e] * t[e].y;
      }
      store8<DT>(A.y[w], y + k0, p);
      store8<DT>(A.y[w], y + k0 + half, q);
    }
  }
}

template <int DT>
void launch(const Rot& A, bool pairs, bool vec, uint32_t grid, uint32_t lds, hipStream_t s) {
  if (pairs && vec) rotate<DT, true, true><<<grid, kThr, lds, s>>>(A);
  else if (pairs) rotate<DT, true, false><<<grid, kThr, lds, s>>>(A);
  else if (vec) rotate<DT, false, true><<<grid, kThr, lds, s>>>(A);
  else rotate<DT, false, false><<<grid, kThr, lds, s>>>(A);
}

}  // namespace

extern "C" int qkv_rotary(int32_t dtype, const void* q, int64_t q_row_stride,
                          int64_t q_head_stride, int32_t Hq, const void* k, int64_t k_row_stride,
                          int64_t k_head_stride, int32_t Hk, int64_t rows, int32_t d, int32_t R,
                          const int32_t* positions, const int64_t* turns, float factor,
                          int32_t interleaved, int32_t inverse, void* q_out, int64_t qo_row_stride,
                          int64_t qo_head_stride, void* k_out, int64_t ko_row_stride,
                          int64_t ko_head_stride, void* stream) {
  QKV_REQUIRE(qkv_dtype_ok(dtype), "unknown element type %d", dtype);
  QKV_REQUIRE(d >= 1 && R >= 2 && R % 2 == 0 && R <= d && R / 2 <= kMaxPairs,
              "the rotated part must be an even number of the head's %d coordinates, %d at most; "
              "got %d", d, 2 * kMaxPairs, R);
  QKV_REQUIRE(Hq >= 0 && Hk >= 0 && (int64_t(Hq) + Hk) * d <= (1 << 27),
              "%d and %d heads of %d are no row of up to 2^27 values", Hq, Hk, d);
  QKV_REQUIRE(rows >= 0 && rows < INT32_MAX, "rows must lie in [0, 2^31 - 1); got %lld",
              static_cast<long long>(rows));
  if (rows == 0 || Hq + Hk == 0) return QKV_OK;
  QKV_REQUIRE(positions && turns && (Hq == 0 || (q && q_out)) && (Hk == 0 || (k && k_out)),
              "qkv_rotary: null pointer");
  const int es = dtype == QKV_F32 ? 4 : 2;
  auto aligned = [&](const void* p, int64_t rs, int64_t hs) {
    return qkv_aligned(p, 16) && rs * es % 16 == 0 && hs * es % 16 == 0;
  };
  bool vec = d % 8 == 0 && R % (interleaved ? 8 : 16) == 0;
  if (Hq > 0) vec = vec && aligned(q, q_row_stride, q_head_stride) &&
                    aligned(q_out, qo_row_stride, qo_head_stride);
  if (Hk > 0) vec = vec && aligned(k, k_row_stride, k_head_stride) &&
                    aligned(k_out, ko_row_stride, ko_head_stride);
  const bool place = (Hq == 0 || (q == q_out && q_row_stride == qo_row_stride &&
                                  q_head_stride == qo_head_stride)) &&
                     (Hk == 0 || (k == k_out && k_row_stride == ko_row_stride &&
                                  k_head_stride == ko_head_stride));
  // rows of a workgroup: one until the card is full
  const int64_t many = rows / (4 * qkv_num_cus());
  const int32_t wg_rows = static_cast<int32_t>(std::max<int64_t>(1, std::min<int64_t>(kMaxRows, many)));
  Rot A{{q, k}, {q_out, k_out}, {q_row_stride, k_row_stride}, {q_head_stride, k_head_stride},
        {qo_row_stride, ko_row_stride}, {qo_head_stride, ko_head_stride}, {Hq, Hk}, rows, d, R,
        wg_rows, place ? 0 : 1, positions, turns, factor, inverse ? -1.f : 1.f};
  const uint32_t grid = static_cast<uint32_t>((rows + wg_rows - 1) / wg_rows);
  const uint32_t lds = wg_rows * (R / 2) * sizeof(float2);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == QKV_F32) launch<QKV_F32>(A, interleaved != 0, vec, grid, lds, s);
  else if (dtype == QKV_F16) launch<QKV_F16>(A, interleaved != 0, vec, grid, lds, s);
  else launch<QKV_BF16>(A, interleaved != 0, vec, grid, lds, s);
  QKV_LAUNCHED();
  return QKV_OK;
}
