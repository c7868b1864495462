// Rotary positions of query and key rows (C ABI: qkv_rotary).
//
// The pair i of a head's first R coordinates -- (i, i + R / 2), or (2 i, 2 i + 1) where they are
// interleaved -- turns by the angle 2 pi p f_i at position p:
//   y1 = c (x1 cos - x2 sin),  y2 = c (x2 cos + x1 sin);
// coordinates behind R stay as they are.  f_i comes as turns in units of 2^-64, so that p f_i
// modulo a turn is an integer product modulo 2^64: exact but for the rounding of f_i itself,
// |p| 2^-65 turns, at any position.  Sine and cosine are fp32's of the nearest fp32 to what is left
// beside the nearest quarter turn (within 1/8, so off by 2^-28 turns at most: a quarter of what
// the whole remainder's fp32 would be off); products and sums are fp32, rounded once to the rows' type.
//
// Bytes bound it, each row in and out: a workgroup has the angles of its rows in LDS, one sine
// and cosine for all heads, and then goes over the rows' pairs with 16-byte loads.  8192 bf16 rows
// of 40 heads, d = 128 (168 MB): 29 us over and over the same rows (5.8 TB/s; interleaved 31, 100 of
// the 128 coordinates 39), 36 over others each time (4.7; a 1 GiB copy reaches 5.0).  64 rows 4 us
// of kernel: a launch, the angles, a row.  Rows that 16-byte accesses do not fit go an element at
// a time, a load and a store each: the 8192 at an odd offset 111 us where aligned ones take 39
// (interleaved 117 / 47; fp32 130 / 72), heads of 70 coordinates 63.
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
  int32_t pairs;              // (kOne)
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

// i / n with inv = 1 / n, for i < 2^20: the product is off by i / n 2^-22 at most, and (i + 1/2) / n
// is 1 / 2 n or more from a whole number.  (Integer divisions: 8192 rows of 40 heads, d = 128,
// interleaved, bf16, 36 us, so 31.)
__device__ __forceinline__ int div_by(int i, float inv) {
  return static_cast<int>((static_cast<float>(i) + 0.5f) * inv);
}
constexpr int kMostUnits = 1 << 20;  // of a workgroup

__host__ __device__ __forceinline__ int div8(int n) { return (n + 7) / 8; }

// How a head is gone over: an element at a time (any alignment), eight neighbours in 16-byte
// accesses that hold their pairs (interleaved), that do with eight more half the part away (the
// part a multiple of 16), or that find the other halves in LDS (any part).
enum How { kOne, kPairs, kHalves, kTurned };

template <int DT, int HOW>
__global__ __launch_bounds__(kThr) void rotate(Rot A) {
  extern __shared__ float2 cs[];  // [row][pair] c cos, c sin; kTurned: heads behind them
  const int tid = threadIdx.x;
  const int half = A.R / 2;
  const int64_t r0 = int64_t(blockIdx.x) * A.wg_rows;
  const int nr = static_cast<int>(min(int64_t(A.wg_rows), A.rows - r0));
  for (int i = tid; i < nr * half; i += kThr) {
    const int r = i / half, k = i - r * half;
    // (two's complement: the product modulo 2^64 is right for negative positions, too)
    const uint64_t turn = static_cast<uint64_t>(A.turns[k]) *
                          static_cast<uint64_t>(int64_t(A.pos[r0 + r]));
    const uint32_t quarter = static_cast<uint32_t>((turn + (uint64_t(1) << 61)) >> 62);
    const int64_t rest = static_cast<int64_t>(turn - (uint64_t(quarter) << 62));
    float s, c;
    sincospif(static_cast<float>(rest) * 0x1p-63f, &s, &c);
    if (quarter & 1) {
      const float t = s;
      s = c;
      c = -t;
    }
    if (quarter & 2) {
      s = -s;
      c = -c;
    }
    cs[HOW == kTurned ? (r * 8 + (k & 7)) * div8(half) + (k >> 3) : i] =
        float2{c * A.factor, s * A.factor * A.sign};
  }
  __syncthreads();
  const int heads = A.heads[0] + A.heads[1];
  const float per_head = 1.f / static_cast<float>(heads);
  // row r and head j of both: which tensor, and its head's first elements there and in the output
  auto place = [&](int r, int j, int& w, int64_t& x, int64_t& y) {
    w = j >= A.heads[0];
    const int h = j - (w ? A.heads[0] : 0);
    x = (r0 + r) * A.ts[w] + h * A.hs[w];
    y = (r0 + r) * A.to[w] + h * A.ho[w];
  };
  if constexpr (HOW == kTurned) {
    // In LDS the k-th of a head lies at (k % 8) chunks + k / 8, so that lanes of neighbouring eights
    // meet neighbouring banks, wherever the other half begins; the angles likewise.
    const int chunks = A.d / 8, batch = kThr / chunks, many = div8(half);
    float* const box = reinterpret_cast<float*>(cs + A.wg_rows * 8 * many);
    const int v = tid / chunks, u = tid - v * chunks, c = 8 * u;
    float* const mine = box + v * A.d;
    for (int i0 = 0; i0 < nr * heads; i0 += batch) {
      const int i = i0 + v, r = div_by(i, per_head);
      const bool on = v < batch && i < nr * heads;
      int w = 0;
      int64_t x = 0, y = 0;
      float a[8];
      if (on) {
        place(r, i - r * heads, w, x, y);
        load8<DT>(A.x[w], x + c, a);
#pragma unroll
        for (int e = 0; e < 8; ++e) mine[e * chunks + u] = a[e];
      }
      __syncthreads();
      if (on) {
        const float2* const t = cs + r * 8 * many;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int k = c + e;
          if (k >= A.R) break;
          const bool low = k < half;
          const int o = low ? k + half : k - half, q = low ? k : o;  // the other one; the pair
          const float2 f = t[(q & 7) * many + (q >> 3)];
          const float other = mine[(o & 7) * chunks + (o >> 3)];
          a[e] = a[e] * f.x + (low ? -other : other) * f.y;
        }
        store8<DT>(A.y[w], y + c, a);
      }
      __syncthreads();
    }
    return;
  }
  constexpr int PER = HOW == kOne ? 1 : HOW == kPairs ? 4 : 8;  // pairs of a unit
  const int turned = (half + PER - 1) / PER;
  const int rest = !A.copy ? 0 : HOW == kOne ? A.d - A.R : A.d / 8 - (HOW == kPairs ? turned : A.R / 8);
  const float per_turned = 1.f / static_cast<float>(turned);
  for (int i = tid; i < nr * heads * turned; i += kThr) {
    const int j = div_by(i, per_turned), u = i - j * turned, r = div_by(j, per_head);
    int w;
    int64_t x, y;
    place(r, j - r * heads, w, x, y);
    const int k0 = u * PER;
    const float2* const t = cs + r * half + k0;
    if constexpr (HOW == kOne) {
      const int a = A.pairs ? 2 * k0 : k0, b = A.pairs ? a + 1 : a + half;
      const float p = qkv_load(A.x[w], x + a, DT), q = qkv_load(A.x[w], x + b, DT);
      qkv_store(A.y[w], y + a, p * t[0].x - q * t[0].y, DT);
      qkv_store(A.y[w], y + b, q * t[0].x + p * t[0].y, DT);
    } else if constexpr (HOW == kPairs) {
      float a[8], b[8];
      load8<DT>(A.x[w], x + 2 * k0, a);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool in = k0 + e < half;  // (R may end within the eight)
        const float2 f = in ? t[e] : float2{1.f, 0.f};
        b[2 * e] = in ? a[2 * e] * f.x - a[2 * e + 1] * f.y : a[2 * e];
        b[2 * e + 1] = in ? a[2 * e + 1] * f.x + a[2 * e] * f.y : a[2 * e + 1];
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
  // behind R (in a loop of its own: beside turned units in a wave it costs them, too)
  const float per_rest = 1.f / static_cast<float>(rest);
  for (int i = tid; i < nr * heads * rest; i += kThr) {
    const int j = div_by(i, per_rest), u = i - j * rest, r = div_by(j, per_head);
    int w;
    int64_t x, y;
    place(r, j - r * heads, w, x, y);
    if constexpr (HOW == kOne) {
      const int c = A.R + u;
      qkv_store(A.y[w], y + c, qkv_load(A.x[w], x + c, DT), DT);
    } else {
      const int c = HOW == kPairs ? 8 * (turned + u) : A.R + 8 * u;
      float a[8];
      load8<DT>(A.x[w], x + c, a);
      store8<DT>(A.y[w], y + c, a);
    }
  }
}

template <int DT>
void launch(const Rot& A, int how, uint32_t grid, uint32_t lds, hipStream_t s) {
  if (how == kOne) rotate<DT, kOne><<<grid, kThr, lds, s>>>(A);
  else if (how == kPairs) rotate<DT, kPairs><<<grid, kThr, lds, s>>>(A);
  else if (how == kHalves) rotate<DT, kHalves><<<grid, kThr, lds, s>>>(A);
  else rotate<DT, kTurned><<<grid, kThr, lds, s>>>(A);
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
  QKV_REQUIRE(Hq >= 0 && Hk >= 0 && (int64_t(Hq) + Hk) * d <= kMostUnits,
              "%d and %d heads of %d are no row of up to 2^20 values", Hq, Hk, d);
  QKV_REQUIRE(rows >= 0 && rows < INT32_MAX, "rows must lie in [0, 2^31 - 1); got %lld",
              static_cast<long long>(rows));
  if (rows == 0 || Hq + Hk == 0) return QKV_OK;
  QKV_REQUIRE(positions && turns && (Hq == 0 || (q && q_out)) && (Hk == 0 || (k && k_out)),
              "qkv_rotary: null pointer");
  const int es = dtype == QKV_F32 ? 4 : 2;
  auto aligned = [&](const void* p, int64_t rs, int64_t hs) {
    return qkv_aligned(p, 16) && rs * es % 16 == 0 && hs * es % 16 == 0;
  };
  bool vec = d % 8 == 0 && d <= 8 * kThr;
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
  const int64_t most = std::min<int64_t>(kMaxRows, kMostUnits / ((int64_t(Hq) + Hk) * d));
  const int32_t wg_rows = static_cast<int32_t>(std::max<int64_t>(1, std::min(most, many)));
  const int how = !vec ? kOne : interleaved ? kPairs : R % 16 == 0 ? kHalves : kTurned;
  // (kTurned: angles by eights, and the heads of a pass)
  const uint32_t lds = how == kTurned ? wg_rows * 8 * div8(R / 2) * sizeof(float2) +
                                            kThr / (d / 8) * d * sizeof(float)
                                      : wg_rows * (R / 2) * sizeof(float2);
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto from = [&](const void* p, int64_t stride, int64_t r) {
    return const_cast<char*>(static_cast<const char*>(p)) + r * stride * es;
  };
  const int64_t per = int64_t(wg_rows) << 23;  // a launch's rows: it has fewer than 2^32 threads
  for (int64_t r = 0; r < rows; r += per) {
    const int64_t n = std::min(per, rows - r);
    Rot A{{from(q, q_row_stride, r), from(k, k_row_stride, r)},
          {from(q_out, qo_row_stride, r), from(k_out, ko_row_stride, r)},
          {q_row_stride, k_row_stride}, {q_head_stride, k_head_stride},
          {qo_row_stride, ko_row_stride}, {qo_head_stride, ko_head_stride}, {Hq, Hk}, n, d, R,
          wg_rows, place ? 0 : 1, interleaved ? 1 : 0, positions + r, turns, factor,
          inverse ? -1.f : 1.f};
    const uint32_t grid = static_cast<uint32_t>((n + wg_rows - 1) / wg_rows);
    if (dtype == QKV_F32) launch<QKV_F32>(A, how, grid, lds, s);
    else if (dtype == QKV_F16) launch<QKV_F16>(A, how, grid, lds, s);
    else launch<QKV_BF16>(A, how, grid, lds, s);
    QKV_LAUNCHED();
  }
  return QKV_OK;
}
