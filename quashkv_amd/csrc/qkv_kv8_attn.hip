// Attention of a ragged batch of queries over the 8-bit paged cache (qkv_kv8.h).
#include <algorithm>

#include "qkv_kv8.h"

namespace {

struct Att {
  const void* q;
  int64_t q_ts, q_hs;
  int32_t q_dtype;
  int64_t rows;
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
  int32_t B, Hq, H, uniform_q;
  float scale;
  int32_t causal;
  void* out;
  int32_t out_dtype;
};

template <bool FP8>
__device__ __forceinline__ float value_of(uint32_t code) {
  if constexpr (FP8)
    return __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(code & 0xffu), 0);
  else
    return static_cast<float>(static_cast<int8_t>(code));
}

// A wave per (request, query, query head).
template <int D, bool FP8>
__global__ __launch_bounds__(64) void attend_rows(Att A) {
  __shared__ float qs[D], ps[64];
  const int lane = threadIdx.x, hq = blockIdx.y, h = hq / (A.Hq / A.H);
  const int64_t r = blockIdx.x;
  int b;
  int64_t i, qlen;
  if (A.q_start == nullptr) {
    b = static_cast<int>(r / A.uniform_q);
    i = r - int64_t(b) * A.uniform_q;
    qlen = A.uniform_q;
  } else {
    if (r < A.q_start[0] || r >= A.q_start[A.B]) return;
    int lo = 0, hi = A.B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (A.q_start[mid] <= r) lo = mid;
      else hi = mid;
    }
    b = lo;
    i = r - A.q_start[b];
    qlen = A.q_lens ? A.q_lens[b] : A.q_start[b + 1] - A.q_start[b];
    if (i >= qlen) return;
  }
  const int64_t n = int64_t(1) << A.lg;
  int64_t kv = A.kv_lens[b];
  if (kv > int64_t(A.width) * n) kv = int64_t(A.width) * n;
  const int64_t end = A.causal ? kv - qlen + i + 1 : kv;
  for (int c = lane; c < D; c += 64)
    qs[c] = qkv_load(A.q, r * A.q_ts + hq * A.q_hs + c, A.q_dtype);
  __syncthreads();
  float m = -INFINITY, l = 0.f, o[2] = {0.f, 0.f};
  for (int64_t t0 = 0; t0 < end; t0 += 64) {
    const int64_t t = t0 + lane;
    float x = -INFINITY, vs = 0.f;
    int64_t page = -1;
    if (t < end) page = A.table[int64_t(b) * A.width + (t >> A.lg)];
    const bool ok = page >= 0 && page < A.npages;
    const int64_t row = ok ? (page * A.H + h) * n + (t & (n - 1)) : 0;
    if (ok) {
      float s = 0.f;
      const uint8_t* k = A.kpool + row * D;
      for (int c = 0; c < D; ++c) s = fmaf(qs[c], value_of<FP8>(k[c]), s);
      x = s * A.kscale[row >> 4] * A.scale;
      vs = A.vscale[row >> 4];
    }
    const float mn = fmaxf(m, qkv_wave_max(x));
    if (mn == -INFINITY) continue;
    const float p = ok ? expf(x - mn) : 0.f, f = expf(m - mn);
    l = l * f + qkv_wave_sum(p);
    m = mn;
    __syncthreads();
    ps[lane] = ok ? p * vs : 0.f;
    __syncthreads();
    o[0] *= f;
    o[1] *= f;
    for (int j = 0; j < 64; ++j) {
      const float pj = ps[j];
      const int64_t rj = __shfl(static_cast<long long>(row), j, 64);
      if (!__shfl(ok ? 1 : 0, j, 64)) continue;
      const uint8_t* v = A.vpool + (rj & ~int64_t(15)) * D + (rj & 15);
      for (int y = 0; y < 2; ++y)
        if (lane + 64 * y < D)
          o[y] = fmaf(pj, value_of<FP8>(v[(lane + 64 * y) * kBlk]), o[y]);
    }
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  for (int y = 0; y < 2; ++y)
    if (lane + 64 * y < D)
      qkv_store(A.out, (r * A.Hq + hq) * D + lane + 64 * y, o[y] * inv, A.out_dtype);
}

}  // namespace

extern "C" int64_t qkv_kv8_attention_workspace_bytes(int32_t B, int64_t rows, int32_t Hq,
                                                     int32_t Hkv, int32_t d, int64_t max_q) {
  return 256;
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
  QKV_REQUIRE(Hq >= 1 && Hq <= 65535 && Hq % Hkv == 0,
              "query heads (%d) must be a multiple of kv heads (%d)", Hq, Hkv);
  QKV_REQUIRE(B >= 0 && pages_per_seq >= 1, "bad batch %d or pages_per_seq %d", B, pages_per_seq);
  QKV_REQUIRE(rows >= 0 && rows < INT32_MAX, "rows must lie in [0, 2^31 - 1); got %lld",
              static_cast<long long>(rows));
  if (rows == 0 || B == 0) return QKV_OK;
  QKV_REQUIRE(q_start || !q_lens, "q_lens needs q_start");
  QKV_REQUIRE(q_start || rows % B == 0, "without q_start the rows (%lld) must be B (%d) times one "
              "length", static_cast<long long>(rows), B);
  QKV_REQUIRE(q && kpool && kscale && vpool && vscale && table && kv_lens && out,
              "qkv_kv8_attention: null pointer");
  QKV_REQUIRE(qkv_aligned(kpool, 16) && qkv_aligned(vpool, 16),
              "the pools must be 16-byte aligned");
  QKV_REQUIRE(workspace && qkv_aligned(workspace, 256) &&
                  ws_bytes >= qkv_kv8_attention_workspace_bytes(B, rows, Hq, Hkv, d, max_q),
              "qkv_kv8_attention: workspace too small or not 256-byte aligned");
  Att A{q, q_row_stride, q_head_stride, q_dtype, rows, static_cast<const uint8_t*>(kpool), kscale,
        static_cast<const uint8_t*>(vpool), vscale, num_pages, qkv_page_lg(page_tokens), table,
        pages_per_seq, q_start, q_lens, kv_lens, B, Hq, Hkv, static_cast<int32_t>(rows / B), scale,
        causal, out, out_dtype};
  const dim3 grid(static_cast<uint32_t>(rows), Hq);
  hipStream_t s = static_cast<hipStream_t>(stream);
#define RUN(D)                                                              \
  if (fmt == QKV_CODES_I8) attend_rows<D, false><<<grid, 64, 0, s>>>(A);    \
  else attend_rows<D, true><<<grid, 64, 0, s>>>(A);
  if (d == 128) { RUN(128) } else if (d == 96) { RUN(96) } else { RUN(64) }
#undef RUN
  QKV_LAUNCHED();
  return QKV_OK;
}
