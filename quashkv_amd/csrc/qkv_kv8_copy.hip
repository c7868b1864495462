// Copies of pages inside the 8-bit paged cache (C ABI: qkv_kv8_copy_pages): what a fork needs
// of a page in part filled, and what a compaction moves.
//
// A (page, head) of K, and of V, is n d bytes in a row, its first b blocks of 16 tokens the
// first 16 b d of them in both pools: plain copies, whose bytes bound them.  A workgroup takes
// 16 KiB, four 16-byte loads a lane; how many pages there are is known on the device alone
// (a compaction's moves), so the workgroups go over the pieces in strides of the grid.  351 MB in
// and out (pages of 256 tokens, 8 heads, d = 128): 66 us, 5.3 TB/s, as a 1 GiB copy; 4 pages in part
// filled 3.7 us.
#include <algorithm>

#include "qkv_kv8.h"

namespace {

typedef uint32_t v4u __attribute__((ext_vector_type(4)));

constexpr int kThr = 256;
constexpr int kLoads = 4;                      // of 16 bytes, a lane's
constexpr int kPiece = kThr * kLoads * 16;     // bytes of a piece

struct Copy {
  const int32_t* src;
  const int32_t* dst;
  const int32_t* tokens;
  int32_t n;
  const int32_t* count;
  int32_t H, lg, npages;
  int32_t row;        // bytes of a block's tokens: 16 d
  int32_t pieces;     // of a (page, head, half)
  uint8_t* pool[2];
  float* scale[2];
};

__global__ __launch_bounds__(kThr) void copy_pages(Copy A) {
  const int tid = threadIdx.x;
  const int64_t n = A.count ? min(max(*A.count, 0), A.n) : A.n;
  const int64_t units = n * A.H * 2 * A.pieces;
  const int nb = 1 << (A.lg - 4);
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int piece = static_cast<int>(u % A.pieces);
    const int64_t v = u / A.pieces;
    const int half = static_cast<int>(v & 1);
    const int h = static_cast<int>((v >> 1) % A.H);
    const int64_t i = (v >> 1) / A.H;
    const int32_t from = A.src[i], to = A.dst[i];
    if (from < 0 || from >= A.npages || to < 0 || to >= A.npages || from == to) continue;
    const int blocks = A.tokens ? (min(max(A.tokens[i], 0), 1 << A.lg) + kBlk - 1) >> 4 : nb;
    const int64_t a = (int64_t(from) * A.H + h) * nb, b = (int64_t(to) * A.H + h) * nb;
    const int bytes = blocks * A.row - piece * kPiece;
    const v4u* const x = reinterpret_cast<const v4u*>(A.pool[half] + a * A.row + piece * kPiece);
    v4u* const y = reinterpret_cast<v4u*>(A.pool[half] + b * A.row + piece * kPiece);
    v4u w[kLoads];
#pragma unroll
    for (int k = 0; k < kLoads; ++k)
      if (16 * (tid + kThr * k) < bytes) w[k] = x[tid + kThr * k];
    if (piece == 0 && tid < blocks) A.scale[half][b + tid] = A.scale[half][a + tid];
#pragma unroll
    for (int k = 0; k < kLoads; ++k)
      if (16 * (tid + kThr * k) < bytes) y[tid + kThr * k] = w[k];
  }
}

}  // namespace

extern "C" int qkv_kv8_copy_pages(const int32_t* src, const int32_t* dst, const int32_t* tokens,
                                  int32_t n, const int32_t* count, int32_t H, int32_t d,
                                  int32_t fmt, void* kpool, float* kscale, void* vpool,
                                  float* vscale, int32_t num_pages, int32_t page_tokens,
                                  void* stream) {
  const int st = qkv_kv8_check(fmt, num_pages, page_tokens, H, d);
  if (st != QKV_OK) return st;
  QKV_REQUIRE(n >= 0, "the number of pages must not be negative; got %d", n);
  if (n == 0) return QKV_OK;
  QKV_REQUIRE(src && dst && kpool && kscale && vpool && vscale,
              "qkv_kv8_copy_pages: null pointer");
  QKV_REQUIRE(qkv_aligned(kpool, 16) && qkv_aligned(vpool, 16),
              "the pools must be 16-byte aligned");
  const int32_t row = kBlk * d, pieces = (page_tokens * d + kPiece - 1) / kPiece;
  Copy A{src, dst, tokens, n, count, H, qkv_page_lg(page_tokens), num_pages, row, pieces,
         {static_cast<uint8_t*>(kpool), static_cast<uint8_t*>(vpool)}, {kscale, vscale}};
  const int64_t units = int64_t(n) * H * 2 * pieces;
  const uint32_t grid = static_cast<uint32_t>(std::min<int64_t>(units, 8 * qkv_num_cus()));
  copy_pages<<<grid, kThr, 0, static_cast<hipStream_t>(stream)>>>(A);
  QKV_LAUNCHED();
  return QKV_OK;
}
