// Pages that several requests hold: forks, releases by the last holder, compaction
// (C ABI: qkv_page_fork, qkv_page_release_shared, qkv_page_compact).
//
// shares[p] counts the holders of page p beyond the first, so that pages which nobody
// shares (all that qkv_page_plan hands out) have 0 and need no care.  Requests share whole
// pages alone: a page in part filled is copied for the fork, so appends never meet a shared
// one.
//
// Only integers are added or compared, so that no order of atomics shows in a result.
//
// Few bytes, so latency bounds all of it.  Kernels alone: 4 forks of a 3001-token request (pages of
// 256) 3.1 us, 384 forks of 16 (pages of 128) 4.5 + 4.0 us, and released 4.1 and 14; 1200 pages
// compacted 8 us (their tables in the same workgroup, up to 4096 entries, where a launch of its
// own takes 4 us more).
#include <algorithm>

#include "qkv_pages_dev.h"

namespace {

using namespace qkv_pages;

struct Fork {
  int32_t* table;
  int32_t* lens;
  int32_t B, width;
  const int32_t* src;
  const int32_t* dst;
  const int32_t* tokens;
  int32_t F;
  const int32_t* free_list;
  int32_t pool;
  int32_t* free_count;
  int32_t* shares;
  int32_t lg;
  int32_t* granted;
  int32_t* src_pages;
  int32_t* dst_pages;
  int32_t* copy_tokens;
};

// Fork i's whole pages: table entries and holders, by the threads first, first + step, ...
__device__ __forceinline__ void share_row(const Fork& A, int i, int first, int step) {
  const int32_t got = A.granted[i];
  if (got <= 0) return;
  const int32_t* const from = A.table + int64_t(A.src[i]) * A.width;
  int32_t* const to = A.table + int64_t(A.dst[i]) * A.width;
  for (int c = first; c < got >> A.lg; c += step) {
    const int32_t page = from[c];
    to[c] = page;
    if (page >= 0 && page < A.pool) atomicAdd(&A.shares[page], 1);
  }
}

// Who is granted, from the lengths before the call: a pass over the forks for what each asks
// and which fork names a request first (LDS), then one with the prefix sum of the pages
// asked for.  Few forks: their table rows, too (a wave each).
template <int THR, bool ROWS>
__global__ __launch_bounds__(THR) void fork_plan(Fork A) {
  extern __shared__ int32_t named[];  // [B]: the first fork that names a request
  __shared__ int64_t part[THR / 64];
  const int tid = threadIdx.x;
  const int64_t n = int64_t(1) << A.lg;
  const int64_t room = int64_t(A.width) << A.lg;
  const int64_t count = imin(imax(*A.free_count, 0), A.pool);
  for (int b = tid; b < A.B; b += THR) named[b] = INT32_MAX;
  __syncthreads();
  for (int i = tid; i < A.F; i += THR) {
    const int32_t s = A.src[i], t = A.dst[i];
    int32_t got = -1;
    if (s >= 0 && s < A.B && t >= 0 && t < A.B && s != t) {
      const int64_t has = imin(imax(A.lens[s], 0), room);
      if (A.lens[t] <= 0)
        got = static_cast<int32_t>(A.tokens ? imin(imax(A.tokens[i], 0), has) : has);
      atomicMin(&named[t], i);
    }
    A.granted[i] = got;
  }
  __syncthreads();
  int64_t asked = 0, taken = 0;
  for (int i0 = 0; i0 < A.F; i0 += THR) {
    const int i = i0 + tid;
    int32_t got = -1, s = 0, t = 0;
    if (i < A.F) {
      got = A.granted[i];
      s = A.src[i];
      t = A.dst[i];
      if (got >= 0 && named[t] != i) got = -1;
    }
    const int32_t rest = got > 0 ? got & static_cast<int32_t>(n - 1) : 0;
    int64_t total;
    const int64_t top = asked + block_scan<THR>(rest != 0, part, total);
    asked += total;
    if (rest != 0 && top > count) got = -1;
    if (i < A.F) {
      const bool fresh = got > 0 && rest != 0;
      const int32_t whole = got > 0 ? got >> A.lg : 0;
      const int32_t page = fresh ? A.free_list[count - top] : -1;
      A.granted[i] = got;
      A.src_pages[i] = fresh ? A.table[int64_t(s) * A.width + whole] : -1;
      A.dst_pages[i] = page;
      A.copy_tokens[i] = fresh ? rest : 0;
      if (got >= 0) A.lens[t] = got;
      if (fresh) A.table[int64_t(t) * A.width + whole] = page;
    }
  }
  taken = imin(asked, count);  // (those behind the last free page are refused, and only they)
  if (tid == 0) *A.free_count = static_cast<int32_t>(count - taken);
  if (ROWS) {
    __syncthreads();
    for (int i = tid >> 6; i < A.F; i += THR / 64) share_row(A, i, tid & 63, 64);
  }
}

constexpr int kRowThr = 128;
__global__ __launch_bounds__(kRowThr) void fork_rows(Fork A) {
  share_row(A, blockIdx.x, threadIdx.x, kRowThr);
}

struct Release {
  int32_t* lens;
  const uint8_t* done;
  int32_t B;
  const int32_t* table;
  int32_t width, lg;
  int32_t* free_list;
  int32_t pool;
  int32_t* free_count;
  int32_t* shares;
};

// (One workgroup does all of it, so its own scope is enough: through device-wide fences between
// the passes, and a binary search for each entry in each of them, 384 requests of ~30 pages took
// 40 us instead of 14, 4 requests 11 instead of 4.)
__device__ __forceinline__ int32_t peek(const int32_t* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
}

constexpr int kOwn = 8;  // entries of a thread that are in flight at once

// Entries e (request order, page order) of the done requests, a run of them a thread, three
// passes: each takes a holder away; a page left below 0 has lost its last one, and the largest
// e among its entries is kept in its count, as INT32_MIN + (entries - 1 - e), below any
// count; that entry puts the page on the free list, at the place that a prefix sum over them gives.
template <int THR>
__global__ __launch_bounds__(THR) void release_shared(Release A) {
  extern __shared__ int32_t sh[];  // start[B + 1]: entries of the done requests before b
  __shared__ int64_t part[THR / 64];
  const int tid = threadIdx.x;
  const int64_t n = int64_t(1) << A.lg;
  const int64_t count = imin(imax(*A.free_count, 0), A.pool);
  int64_t base = 0;
  if (tid == 0) sh[0] = 0;
  for (int b0 = 0; b0 < A.B; b0 += THR) {
    const int b = b0 + tid;
    int64_t held = 0, total;
    if (b < A.B && A.done[b]) {
      held = imin((imax(A.lens[b], 0) + n - 1) >> A.lg, A.width);
      A.lens[b] = 0;
    }
    const int64_t end = base + block_scan<THR>(held, part, total);
    base += total;
    if (b < A.B) sh[b + 1] = static_cast<int32_t>(imin(end, 1 << 30));
  }
  __syncthreads();
  const int32_t E = sh[A.B], per = (E + THR - 1) / THR;
  const int32_t e0 = min(tid * per, E), e1 = min(e0 + per, E);
  const int b0 = e0 < E ? find_row(sh, A.B, e0) : 0;
  int32_t p[kOwn];
  // the pages (-1: none) of up to kOwn entries from e on; b: e's request, moved on
  auto pages = [&](int32_t e, int& b) {
#pragma unroll
    for (int k = 0; k < kOwn; ++k) {
      p[k] = -1;
      if (e + k < e1) {
        while (e + k >= sh[b + 1]) ++b;
        p[k] = A.table[int64_t(b) * A.width + (e + k - sh[b])];
      }
    }
#pragma unroll
    for (int k = 0; k < kOwn; ++k) p[k] = p[k] < A.pool ? p[k] : -1;
  };
  const bool once = per <= kOwn;  // a thread's pages stay in registers
  int b = b0;
  for (int32_t e = e0; e < e1; e += kOwn) {
    pages(e, b);
#pragma unroll
    for (int k = 0; k < kOwn; ++k)
      if (p[k] >= 0)
        __hip_atomic_fetch_add(&A.shares[p[k]], -1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
  }
  __syncthreads();
  b = b0;
  for (int32_t e = e0; e < e1; e += kOwn) {
    if (!once) pages(e, b);
    int32_t v[kOwn];
#pragma unroll
    for (int k = 0; k < kOwn; ++k) v[k] = p[k] >= 0 ? peek(&A.shares[p[k]]) : 0;
#pragma unroll
    for (int k = 0; k < kOwn; ++k)
      if (v[k] < 0)
        __hip_atomic_fetch_min(&A.shares[p[k]], INT32_MIN + (E - 1 - e - k), __ATOMIC_RELAXED,
                               __HIP_MEMORY_SCOPE_WORKGROUP);
  }
  __syncthreads();
  // (a page's count is read by all of its entries before its last one, which alone has that number,
  // sets it to 0: the others differ from either)
  int64_t mine = 0, total;
  auto last = [&](int32_t e, uint32_t& bits) {
    int32_t v[kOwn];
    bits = 0;
#pragma unroll
    for (int k = 0; k < kOwn; ++k) v[k] = p[k] >= 0 ? peek(&A.shares[p[k]]) : 0;
#pragma unroll
    for (int k = 0; k < kOwn; ++k)
      bits |= static_cast<uint32_t>(p[k] >= 0 && v[k] == INT32_MIN + (E - 1 - e - k)) << k;
  };
  uint32_t bits = 0;
  b = b0;
  for (int32_t e = e0; e < e1; e += kOwn) {
    if (!once) pages(e, b);
    last(e, bits);
    mine += __popc(bits);
  }
  int64_t at = count + block_scan<THR>(mine, part, total) - mine;
  const int64_t end = count + total;
  b = b0;
  for (int32_t e = e0; e < e1; e += kOwn) {
    if (!once) {
      pages(e, b);
      last(e, bits);
    }
#pragma unroll
    for (int k = 0; k < kOwn; ++k)
      if (bits >> k & 1) {
        __hip_atomic_store(&A.shares[p[k]], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        if (at < A.pool) A.free_list[at] = p[k];
        ++at;
      }
  }
  if (tid == 0) *A.free_count = static_cast<int32_t>(imin(end, A.pool));
}

struct Compact {
  int32_t* table;
  const int32_t* lens;
  int32_t B, width;
  int32_t* free_list;
  int32_t pool;
  int32_t* free_count;
  int32_t* shares;
  int32_t lg;
  int32_t* src_pages;
  int32_t* dst_pages;
  int32_t* moves;
  int32_t* remap;
  int32_t tables;     // whether compact_plan maps the tables, too
};

// Entries of the tables up to which it does.
constexpr int kFewEntries = 4096;

constexpr int kMaxPool = 1 << 20;  // pages of a compaction: a bit each in 128 KiB of LDS

// One workgroup: the pages in use as bits in LDS, U of them; the i-th in use at U or above goes
// to the i-th free one below U.
__global__ __launch_bounds__(kThr) void compact_plan(Compact A) {
  extern __shared__ uint32_t used[];  // [words]
  __shared__ int64_t part[kThr / 64];
  const int tid = threadIdx.x;
  const int words = (A.pool + 31) / 32, per = (words + kThr - 1) / kThr;
  const int32_t count = static_cast<int32_t>(imin(imax(*A.free_count, 0), A.pool));
  for (int w = tid; w < words; w += kThr)
    used[w] = A.pool - 32 * w >= 32 ? ~0u : (1u << (A.pool - 32 * w)) - 1u;
  for (int p = tid; p < A.pool; p += kThr) A.remap[p] = p;
  __syncthreads();
  for (int i = tid; i < count; i += kThr) {
    const int32_t p = A.free_list[i];
    if (p >= 0 && p < A.pool) atomicAnd(&used[p >> 5], ~(1u << (p & 31)));
  }
  __syncthreads();
  const int w0 = min(tid * per, words), w1 = min(w0 + per, words);
  int64_t mine = 0, U;
  for (int w = w0; w < w1; ++w) mine += __popc(used[w]);
  block_scan<kThr>(mine, part, U);
  // bits of word w that stand for pages below U
  auto low = [&](int w) {
    const int64_t k = U - 32 * int64_t(w);
    return k >= 32 ? ~0u : k <= 0 ? 0u : (1u << k) - 1u;
  };
  int64_t mv = 0, hl = 0, movers, holes;
  for (int w = w0; w < w1; ++w) {
    mv += __popc(used[w] & ~low(w));
    hl += __popc(~used[w] & low(w));
  }
  int64_t at = block_scan<kThr>(mv, part, movers) - mv;
  int64_t to = block_scan<kThr>(hl, part, holes) - hl;
  for (int w = w0; w < w1; ++w) {
    for (uint32_t m = used[w] & ~low(w); m != 0; m &= m - 1)
      A.src_pages[at++] = 32 * w + __ffs(m) - 1;
    for (uint32_t m = ~used[w] & low(w); m != 0; m &= m - 1)
      A.dst_pages[to++] = 32 * w + __ffs(m) - 1;
  }
  // (U pages in use, U places below U: as many movers as holes, half the pool at most)
  for (int64_t i = movers + tid; i < A.pool / 2; i += kThr) A.src_pages[i] = A.dst_pages[i] = -1;
  const int32_t left = A.pool - static_cast<int32_t>(U);
  for (int i = tid; i < left; i += kThr) A.free_list[i] = A.pool - 1 - i;
  if (tid == 0) {
    *A.moves = static_cast<int32_t>(movers);
    *A.free_count = left;
  }
  __syncthreads();
  for (int64_t i = tid; i < movers; i += kThr) {
    const int32_t s = A.src_pages[i], t = A.dst_pages[i];
    A.remap[s] = t;
    if (A.shares) {
      A.shares[t] = A.shares[s];
      A.shares[s] = 0;
    }
  }
  if (!A.tables) return;
  __syncthreads();
  for (int i = tid; i < A.B * A.width; i += kThr) {
    const int b = i / A.width, c = i - b * A.width;
    const int64_t n = int64_t(1) << A.lg;
    const int32_t p = A.table[i];
    if (c < (imax(A.lens[b], 0) + n - 1) >> A.lg && p >= 0 && p < A.pool) A.table[i] = A.remap[p];
  }
}

constexpr int kTabThr = 256;
__global__ __launch_bounds__(kTabThr) void compact_tables(Compact A) {
  const int b = blockIdx.x;
  const int64_t n = int64_t(1) << A.lg;
  const int64_t held = imin((imax(A.lens[b], 0) + n - 1) >> A.lg, A.width);
  int32_t* const row = A.table + int64_t(b) * A.width;
  for (int64_t c = threadIdx.x; c < held; c += kTabThr) {
    const int32_t p = row[c];
    if (p >= 0 && p < A.pool) row[c] = A.remap[p];
  }
}

}  // namespace

extern "C" int qkv_page_fork(int32_t* table, int32_t* lens, int32_t B, int32_t pages_per_seq,
                             const int32_t* src, const int32_t* dst, const int32_t* tokens,
                             int32_t forks, const int32_t* free_list, int32_t num_pages,
                             int32_t* free_count, int32_t* shares, int32_t page_tokens,
                             int32_t* granted, int32_t* src_pages, int32_t* dst_pages,
                             int32_t* copy_tokens, void* stream) {
  const int st = check_table("qkv_page_fork", B, pages_per_seq, num_pages, page_tokens);
  if (st != QKV_OK) return st;
  QKV_REQUIRE(forks >= 0 && forks <= kMaxB, "qkv_page_fork takes up to %d forks; got %d", kMaxB,
              forks);
  if (forks == 0) return QKV_OK;
  QKV_REQUIRE(src && dst && free_list && free_count && shares && granted && src_pages &&
                  dst_pages && copy_tokens && (B == 0 || (table && lens)),
              "qkv_page_fork: null pointer");
  Fork A{table,      lens,   B,  pages_per_seq,          src,     dst,       tokens,    forks,
         free_list,  num_pages, free_count, shares, qkv_page_lg(page_tokens), granted, src_pages,
         dst_pages, copy_tokens};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const uint32_t lds = B * sizeof(int32_t);
  if (forks <= 8) {
    fork_plan<512, true><<<1, 512, lds, s>>>(A);
  } else {
    fork_plan<kThr, false><<<1, kThr, lds, s>>>(A);
    QKV_LAUNCHED();
    fork_rows<<<forks, kRowThr, 0, s>>>(A);
  }
  QKV_LAUNCHED();
  return QKV_OK;
}

extern "C" int qkv_page_release_shared(int32_t* lens, const uint8_t* done, int32_t B,
                                       const int32_t* table, int32_t pages_per_seq,
                                       int32_t* free_list, int32_t num_pages, int32_t* free_count,
                                       int32_t* shares, int32_t page_tokens, void* stream) {
  const int st = check_table("qkv_page_release_shared", B, pages_per_seq, num_pages, page_tokens);
  if (st != QKV_OK) return st;
  if (B == 0) return QKV_OK;
  QKV_REQUIRE(lens && done && table && free_list && free_count && shares,
              "qkv_page_release_shared: null pointer");
  Release A{lens, done, B, table, pages_per_seq, qkv_page_lg(page_tokens), free_list, num_pages,
            free_count, shares};
  const uint32_t lds = (B + 1) * sizeof(int32_t);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (int64_t(B) * pages_per_seq <= 256 * kOwn && B <= 256) release_shared<256><<<1, 256, lds, s>>>(A);
  else release_shared<kThr><<<1, kThr, lds, s>>>(A);
  QKV_LAUNCHED();
  return QKV_OK;
}

extern "C" int qkv_page_compact(int32_t* table, const int32_t* lens, int32_t B,
                                int32_t pages_per_seq, int32_t* free_list, int32_t num_pages,
                                int32_t* free_count, int32_t* shares, int32_t page_tokens,
                                int32_t* src_pages, int32_t* dst_pages, int32_t* moves,
                                int32_t* remap, void* stream) {
  const int st = check_table("qkv_page_compact", B, pages_per_seq, num_pages, page_tokens);
  if (st != QKV_OK) return st;
  QKV_REQUIRE(num_pages <= kMaxPool, "qkv_page_compact takes pools of up to %d pages; got %d",
              kMaxPool, num_pages);
  QKV_REQUIRE(free_list && free_count && moves && remap && (num_pages < 2 || (src_pages && dst_pages)) &&
                  (B == 0 || (table && lens)),
              "qkv_page_compact: null pointer");
  Compact A{table,      lens,   B,  pages_per_seq,          free_list, num_pages, free_count,
            shares, qkv_page_lg(page_tokens), src_pages, dst_pages, moves, remap,
            int64_t(B) * pages_per_seq <= kFewEntries};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const uint32_t lds = (num_pages + 31) / 32 * sizeof(uint32_t);
  if (lds > (48 << 10))  // more LDS than a kernel has by default
    QKV_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&compact_plan),
                                hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds)));
  compact_plan<<<1, kThr, lds, s>>>(A);
  QKV_LAUNCHED();
  if (!A.tables) compact_tables<<<B, kTabThr, 0, s>>>(A);
  QKV_LAUNCHED();
  return QKV_OK;
}
