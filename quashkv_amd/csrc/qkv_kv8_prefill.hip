// Attention of many query rows of a request (a prompt, a chunk of one) over the 8-bit paged
// cache: pieces of 128 rows (qkv_kv8_prefill.h).
#include <atomic>

#include "qkv_kv8_prefill.h"

namespace {

using namespace qkv_kv8;

template <int D, bool FP8, bool QLO, bool PLO>
__global__ __launch_bounds__(kPreThr, 2) void prefill8(Att A) {
  __shared__ v4f sbuf[2][2][4];
  extern __shared__ __align__(16) uint8_t lds[];
  Piece P;
  if (!locate<kPreRows>(A, blockIdx.x / A.H, P)) return;
  prefill_piece<D, FP8, QLO, PLO, false>(A, P, blockIdx.x % A.H, threadIdx.x, lds, sbuf);
}

template <int D, bool FP8, bool QLO, bool PLO>
void start(const Att& A, uint32_t pieces, hipStream_t s) {
  constexpr int smem = kPreLds<D>;
  // more LDS than a kernel has by default, asked for once per device (a failure is the
  // launch's, which the caller reports)
  static std::atomic<uint64_t> asked{0};
  int dev = 0;
  (void)hipGetDevice(&dev);
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (!(asked.load(std::memory_order_relaxed) & bit)) {
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(&prefill8<D, FP8, QLO, PLO>),
                              hipFuncAttributeMaxDynamicSharedMemorySize, smem);
    asked.fetch_or(bit, std::memory_order_relaxed);
  }
  prefill8<D, FP8, QLO, PLO><<<pieces * A.H, kPreThr, smem, s>>>(A);
}

template <int D, bool FP8>
void launch(const Att& A, uint32_t pieces, hipStream_t s) {
  if (A.plan) plan8<kPreRows><<<1, kPlanThr, (A.B + 1) * sizeof(int32_t), s>>>(A, pieces);
  if (A.q_dtype == QKV_F32) start<D, FP8, true, true>(A, pieces, s);
  else if (A.out_dtype != QKV_BF16) start<D, FP8, false, true>(A, pieces, s);
  else start<D, FP8, false, false>(A, pieces, s);
}

}  // namespace

void qkv_kv8_prefill(const Att& A, int32_t d, bool fp8, uint32_t pieces, hipStream_t s) {
  if (fp8) {
    if (d == 128) launch<128, true>(A, pieces, s);
    else if (d == 96) launch<96, true>(A, pieces, s);
    else launch<64, true>(A, pieces, s);
  } else {
    if (d == 128) launch<128, false>(A, pieces, s);
    else if (d == 96) launch<96, false>(A, pieces, s);
    else launch<64, false>(A, pieces, s);
  }
}
