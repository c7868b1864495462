// Prefix sums and searches of the kernels that keep page tables (qkv_pages.hip,
// qkv_page_share.hip), and the checks that their entry points share.
#pragma once

#include "qkv_common.h"

namespace qkv_pages {

constexpr int kThr = 1024;      // of a kernel of one workgroup
constexpr int kMaxB = 16000;    // requests of a call (an int32 of each fits 64 KiB of LDS)

// (the HIP headers' min / max of 64-bit integers go through double)
__device__ __forceinline__ int64_t imin(int64_t a, int64_t b) { return a < b ? a : b; }
__device__ __forceinline__ int64_t imax(int64_t a, int64_t b) { return a > b ? a : b; }

template <int CTRL, int ROWS>
__device__ __forceinline__ int64_t dpp(int64_t v) {
  const int lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xf, false);
  const int hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(v >> 32), CTRL, ROWS, 0xf, false);
  return (static_cast<int64_t>(hi) << 32) | static_cast<uint32_t>(lo);
}

// Inclusive sum over the workgroup's threads; `total` gets the sum of all.
// part: one value per wave.
template <int THR>
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* part, int64_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  v += dpp<0x111, 0xf>(v);  // row_shr 1, 2, 4, 8
  v += dpp<0x112, 0xf>(v);
  v += dpp<0x114, 0xf>(v);
  v += dpp<0x118, 0xf>(v);
  v += dpp<0x142, 0xa>(v);  // row_bcast 15, 31
  v += dpp<0x143, 0xc>(v);
  __syncthreads();  // (part may still be read from the last call)
  if (lane == 63) part[wave] = v;
  __syncthreads();
  int64_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < THR / 64; ++w) {
    const int64_t u = part[w];
    if (w < wave) before += u;
    total += u;
  }
  return before + v;
}

// The request whose rows hold row r: the last b with start[b] <= r, -1 past the
// last row.  start: B + 1 first rows, ascending (equal where a request has none).
__device__ __forceinline__ int find_row(const int32_t* start, int B, int64_t r) {
  if (r >= start[B]) return -1;
  int lo = 0, hi = B;  // start[lo] <= r < start[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= r) lo = mid;
    else hi = mid;
  }
  return lo;
}

inline int check_table(const char* what, int32_t B, int32_t width, int32_t pool, int32_t page_tokens) {
  QKV_REQUIRE(B >= 0 && B <= kMaxB, "%s takes up to %d requests; got %d", what, kMaxB, B);
  QKV_REQUIRE(width >= 1, "pages_per_seq must be positive; got %d", width);
  QKV_REQUIRE(pool >= 1, "num_pages must be positive; got %d", pool);
  QKV_REQUIRE(qkv_page_lg(page_tokens) >= 0,
              "page_tokens must be 64 << k, k = 0 .. 5; got %d", page_tokens);
  return QKV_OK;
}

}  // namespace qkv_pages
