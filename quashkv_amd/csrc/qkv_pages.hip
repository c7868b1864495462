// Page tables and slot maps of a batch of requests, built on the device from
// their lengths (C ABI: qkv_page_plan, qkv_page_release).
//
// A request of `len` cached tokens holds ceil(len / n) pages of n tokens; with
// `add` new tokens it wants ceil((len + add) / n).  Two prefix sums over the
// requests -- of the new tokens (each request's first row) and of the pages
// asked for (each request's place in the free list) -- decide everything:
//   request b is served if its rows end within `rows`, its pages within the
//   table's width, its tokens within QKV_PAGED_TOKENS, and, where it asks for pages, the sum of the pages asked for
//   up to and including it within the free ones;
//   its k-th new page is free[count - 1 - (sum before b) - k];
//   its i-th row is token t = len + i at slot page(t / n) * n + t % n.
//
// Bytes are few (12 out per row), so latency bounds it: lengths are read once, a
// workgroup scans them 1024 at a time, and while the batch is small the same
// workgroup fills the rows from LDS.  64 requests of one token: 2.8 us (scans by LDS
// shuffles in 1024 threads: 6.4); 384 requests, 32,768 rows: 3.8 + 4.4 us.  Pages given back:
// 8 of 64 requests, 32 pages each, 2.8 us; 384 requests, 8 each, 5.2.
#include <algorithm>

#include "qkv_pages_dev.h"

namespace {

using namespace qkv_pages;

constexpr int kThrOne = 256;    // of a small batch's scan
constexpr int kFill = 256;      // of the fill
constexpr int kOneB = 2048;     // requests and rows that one workgroup does alone
constexpr int64_t kOneRows = 4096;

struct Plan {
  const int32_t* lens;
  const int32_t* add;
  int32_t B;
  int32_t* table;
  int32_t width;
  const int32_t* free_list;
  int32_t pool;
  const int32_t* free_count;
  int32_t lg;
  int64_t rows;
  int32_t* q_start;
  int32_t* q_lens;
  int32_t* kv_lens;
  int64_t* slots;
  int32_t* pos;
  int32_t* free_out;
  int32_t* first;  // [B] free-list place of a request's first new page
};

// Row r of request b: its slot and position, and the table entry of a page it opens.
__device__ __forceinline__ void fill_row(const Plan& P, int64_t r, int b, int64_t i, int64_t t0,
                                         int32_t qlen, int32_t first) {
  int64_t slot = -1, t = 0;
  if (i < qlen) {
    t = t0 + i;
    const int64_t n = int64_t(1) << P.lg, p = t >> P.lg, held = (t0 + n - 1) >> P.lg;
    int32_t page;
    if (p < held) {
      page = P.table[int64_t(b) * P.width + p];
    } else {
      page = P.free_list[first - (p - held)];
      if ((t & (n - 1)) == 0) P.table[int64_t(b) * P.width + p] = page;
    }
    slot = page < 0 ? -1 : (int64_t(page) << P.lg) + (t & (n - 1));
  }
  P.slots[r] = slot;
  P.pos[r] = static_cast<int32_t>(t);
}

template <int THR, bool ONE>
__global__ __launch_bounds__(THR) void plan_scan(Plan P) {
  extern __shared__ int32_t sh[];  // ONE: start[B + 1], t0[B], q_len[B], first[B]
  __shared__ int64_t part[THR / 64];
  const int tid = threadIdx.x, B = P.B;
  const int64_t n = int64_t(1) << P.lg;
  const int64_t count = imin(imax(*P.free_count, 0), P.pool);
  int64_t rows0 = 0, ask0 = 0, taken = 0;
  if (tid == 0) {
    P.q_start[0] = 0;
    if (ONE) sh[0] = 0;
  }
  for (int b0 = 0; b0 < B; b0 += THR) {
    const int b = b0 + tid;
    int64_t len = 0, add = 0, total;
    if (b < B) {
      len = imax(P.lens[b], 0);
      add = imax(P.add[b], 0);
    }
    const int64_t end = rows0 + block_scan<THR>(add, part, total);
    rows0 += total;
    const int64_t held = (len + n - 1) >> P.lg, want = (len + add + n - 1) >> P.lg;
    const bool fits = end <= P.rows && want <= P.width && len + add <= QKV_PAGED_TOKENS;
    const int64_t ask = fits ? want - held : 0;
    const int64_t top = ask0 + block_scan<THR>(ask, part, total);
    ask0 += total;
    const bool ok = fits && (ask == 0 || top <= count);
    if (b < B) {
      const int32_t start1 = static_cast<int32_t>(imin(end, INT32_MAX));
      const int32_t ql = ok ? static_cast<int32_t>(add) : 0;
      const int32_t first = static_cast<int32_t>(count - 1 - (top - ask));
      P.q_start[b + 1] = start1;
      P.q_lens[b] = ql;
      P.kv_lens[b] = static_cast<int32_t>(len + ql);
      if (ONE) {
        sh[b + 1] = start1;
        sh[B + 1 + b] = static_cast<int32_t>(len);
        sh[2 * B + 1 + b] = ql;
        sh[3 * B + 1 + b] = first;
      } else {
        P.first[b] = first;
      }
    }
    block_scan<THR>(ok ? ask : 0, part, total);
    taken += total;
  }
  if (tid == 0) *P.free_out = static_cast<int32_t>(count - taken);
  if (ONE) {
    __syncthreads();
    for (int64_t r = tid; r < P.rows; r += THR) {
      const int b = find_row(sh, B, r);
      if (b < 0) fill_row(P, r, 0, 0, 0, 0, 0);
      else fill_row(P, r, b, r - sh[b], sh[B + 1 + b], sh[2 * B + 1 + b], sh[3 * B + 1 + b]);
    }
  }
}

__global__ __launch_bounds__(kFill) void plan_fill(Plan P) {
  extern __shared__ int32_t sh[];
  for (int i = threadIdx.x; i <= P.B; i += kFill) sh[i] = P.q_start[i];
  __syncthreads();
  const int64_t r = int64_t(blockIdx.x) * kFill + threadIdx.x;
  if (r >= P.rows) return;
  const int b = find_row(sh, P.B, r);
  if (b < 0) {
    fill_row(P, r, 0, 0, 0, 0, 0);
    return;
  }
  const int32_t ql = P.q_lens[b];
  fill_row(P, r, b, r - sh[b], int64_t(P.kv_lens[b]) - ql, ql, P.first[b]);
}

__global__ __launch_bounds__(kThr) void release_pages(int32_t* lens, const uint8_t* done, int32_t B,
                                                      const int32_t* table, int32_t width, int32_t lg,
                                                      int32_t* free_list, int32_t pool,
                                                      int32_t* free_count) {
  extern __shared__ int32_t sh[];  // start[B + 1]: pages of the done requests before b
  __shared__ int64_t part[kThr / 64];
  const int tid = threadIdx.x;
  const int64_t n = int64_t(1) << lg;
  const int64_t count = imin(imax(*free_count, 0), pool);
  int64_t base = 0;
  if (tid == 0) sh[0] = 0;
  for (int b0 = 0; b0 < B; b0 += kThr) {
    const int b = b0 + tid;
    int64_t held = 0, total;
    if (b < B && done[b]) {
      held = imin((imax(lens[b], 0) + n - 1) >> lg, width);
      lens[b] = 0;
    }
    const int64_t end = base + block_scan<kThr>(held, part, total);
    base += total;
    if (b < B) sh[b + 1] = static_cast<int32_t>(imin(end, INT32_MAX));
  }
  __syncthreads();
  const int64_t put = imin(base, pool - count);  // (a page given back twice must not overflow)
  for (int64_t i = tid; i < put; i += kThr) {
    const int b = find_row(sh, B, i);
    free_list[count + i] = table[int64_t(b) * width + (i - sh[b])];
  }
  if (tid == 0) *free_count = static_cast<int32_t>(count + put);
}

}  // namespace

extern "C" int qkv_page_plan(const int32_t* lens, const int32_t* new_lens, int32_t B, int32_t* table,
                             int32_t pages_per_seq, const int32_t* free_list, int32_t num_pages,
                             const int32_t* free_count, int32_t page_tokens, int64_t rows,
                             int32_t* q_start, int32_t* q_lens, int32_t* kv_lens, int64_t* slots,
                             int32_t* positions, int32_t* free_count_out, int32_t* scratch,
                             void* stream) {
  const int st = check_table("qkv_page_plan", B, pages_per_seq, num_pages, page_tokens);
  if (st != QKV_OK) return st;
  QKV_REQUIRE(rows >= 0 && rows < INT32_MAX, "rows must lie in [0, 2^31 - 1); got %lld",
              static_cast<long long>(rows));
  QKV_REQUIRE(q_start && free_count && free_count_out && free_list &&
                  (B == 0 || (lens && new_lens && table && q_lens && kv_lens && scratch)) &&
                  (rows == 0 || (slots && positions)),
              "qkv_page_plan: null pointer");
  hipStream_t s = static_cast<hipStream_t>(stream);
  Plan P{lens,    new_lens, B,     table, pages_per_seq, free_list,      num_pages, free_count,
         qkv_page_lg(page_tokens), rows,  q_start,       q_lens,         kv_lens,   slots,
         positions, free_count_out, scratch};
  if (B <= kOneB && rows <= kOneRows) {
    const uint32_t lds = (4 * B + 1) * sizeof(int32_t);
    if (B <= kThrOne && rows <= kThrOne) plan_scan<kThrOne, true><<<1, kThrOne, lds, s>>>(P);
    else plan_scan<kThr, true><<<1, kThr, lds, s>>>(P);
  } else {
    plan_scan<kThr, false><<<1, kThr, 0, s>>>(P);
    QKV_LAUNCHED();
    if (rows > 0)
      plan_fill<<<static_cast<uint32_t>((rows + kFill - 1) / kFill), kFill,
                  (B + 1) * sizeof(int32_t), s>>>(P);
  }
  QKV_LAUNCHED();
  return QKV_OK;
}

extern "C" int qkv_page_release(int32_t* lens, const uint8_t* done, int32_t B, const int32_t* table,
                                int32_t pages_per_seq, int32_t* free_list, int32_t num_pages,
                                int32_t* free_count, int32_t page_tokens, void* stream) {
  const int st = check_table("qkv_page_release", B, pages_per_seq, num_pages, page_tokens);
  if (st != QKV_OK) return st;
  if (B == 0) return QKV_OK;
  QKV_REQUIRE(lens && done && table && free_list && free_count, "qkv_page_release: null pointer");
  release_pages<<<1, kThr, (B + 1) * sizeof(int32_t), static_cast<hipStream_t>(stream)>>>(
      lens, done, B, table, pages_per_seq, qkv_page_lg(page_tokens), free_list, num_pages,
      free_count);
  QKV_LAUNCHED();
  return QKV_OK;
}
