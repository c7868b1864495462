// Attention of a ragged batch of queries over the 8-bit paged cache (qkv_kv8.h).
//
// The kernel of short requests is in qkv_kv8_decode.h, with its mathematics and figures.
#include "qkv_kv8_decode.h"

namespace {

using namespace qkv_kv8;

// A workgroup per (piece, kv head).
template <int D, bool FP8, bool QLO>
__global__ __launch_bounds__(kThr, 2) void decode8(Att A) {
  __shared__ float red_o[kWaves][kRows][D + 4];
  __shared__ float red_ml[kWaves][kRows][2];
  Piece P;
  if (!locate<kRows>(A, blockIdx.x / A.H, P)) return;
  decode_piece<D, FP8, QLO, false>(A, P, blockIdx.x % A.H, threadIdx.x, red_o, red_ml);
}

// Pieces that a launch aims at, per kv head: one workgroup per CU.  (decode8, 32 x 8192
// tokens, 8 kv heads, d = 128: 96 us; two per CU 105, three 104, four 118; 131,072 tokens:
// 48, 51, 54, 57.)
int32_t target_of(int32_t H) { return std::max(1, (qkv_num_cus() + H - 1) / H); }
// Cut tiles have more than C steps each and pieces of C, so they have fewer than
// 2 total / C <= 2 target pieces.
int64_t slots_of(int32_t H) { return int64_t(2 * target_of(H) + 1) * H; }
// Tiles of `rows` query rows, at most: a request's last one may be in part empty.
int64_t tiles_of(int64_t B, int64_t q_rows, int32_t G, int rows) {
  return q_rows * G / rows + std::min(B, q_rows);
}
// Bytes of a launch's partial results, and of its list of pieces.
int64_t part_bytes(int64_t B, int64_t q_rows, int32_t G, int32_t H, int rows, int32_t d) {
  const int64_t plan = B > 64 ? 16 * (tiles_of(B, q_rows, G, rows) + target_of(H)) : 0;
  return 256 + (slots_of(H) * (16 + rows * (d + 2) * 4) + plan) / 256 * 256 + 256;
}
// Lays them out at `at`.
void place_parts(Att& A, void* at, int rows, int32_t d) {
  A.used = static_cast<int32_t*>(at);
  A.desc = reinterpret_cast<int4*>(A.used + 64);
  A.part_o = reinterpret_cast<float*>(A.desc + A.nslots);
  A.part_ml = A.part_o + int64_t(A.nslots) * rows * d;
  // (nslots * rows * 8 bytes of part_ml: 16-byte aligned)
  A.plan = A.B > 64 ? reinterpret_cast<int4*>(A.part_ml + int64_t(A.nslots) * rows * 2) : nullptr;
}
// Requests of more rows than this go to prefill8.  us on decode8 / prefill8 at 64 rows a
// request, d = 128, 8 kv heads: 1 x 8000 tokens 18 / 28, 8 x 2000 21 / 27, 8 x 8000 61 / 49,
// 32 x 2000 57 / 46, 32 x 8000 195 / 146; at 32 rows decode8 has two tiles and is the
// faster one but for the last (109 / 116).
constexpr int kFew = 32;
// A cache of up to this many tokens a request is not cut: the join's launch costs more than
// the steps that it saves (one fp32 query over 512 tokens, 8 heads: 14 us against 17).  The
// host knows the table's width for it, not the lengths: under a wide table short requests
// have the join's launch, too.
constexpr int64_t kWhole = 1024;
constexpr int32_t kNever = INT32_MAX / 2;

// Whether prefill8 runs, and the workspace: decode8's part, then prefill8's where it runs.  The
// one rule for both: `max_q`, which may be wrong, decides (too small: decode8, which takes
// requests of any rows).
struct Layout {
  bool pre;
  int64_t at_pre, bytes;
};
Layout layout(int64_t B, int64_t rows, int32_t G, int32_t H, int32_t d, int64_t max_q) {
  Layout L;
  L.pre = std::min(max_q, rows) * G > kFew;
  L.at_pre = part_bytes(B, rows, G, H, kRows, d);
  L.bytes = L.at_pre + (L.pre ? part_bytes(B, rows, G, H, kPreRows, d) : 0);
  return L;
}

template <int D, bool FP8>
void launch(const Att& A, uint32_t pieces, hipStream_t s) {
  const uint32_t grid = pieces * A.H;
  if (A.plan) plan8<kRows><<<1, kPlanThr, (A.B + 1) * sizeof(int32_t), s>>>(A, pieces);
  if (A.q_dtype == QKV_F32) decode8<D, FP8, true><<<grid, kThr, 0, s>>>(A);
  else decode8<D, FP8, false><<<grid, kThr, 0, s>>>(A);
}

// The joins of what decode8 (A) and prefill8 (P) have cut; null: nothing.
template <int D>
void join(const Att* A, const Att* P, hipStream_t s) {
  const uint32_t a = A ? join_grid(*A, kRows) : 0, p = P ? join_grid(*P, kPreRows) : 0;
  if (A && P) join_both8<D><<<a + p, kThr, 0, s>>>(*A, *P, static_cast<int>(a));
  else if (A) join8<D, kRows><<<a, kThr, 0, s>>>(*A);
  else if (P) join8<D, kPreRows><<<p, kThr, 0, s>>>(*P);
}

}  // namespace

extern "C" int64_t qkv_kv8_attention_workspace_bytes(int32_t B, int64_t rows, int32_t Hq,
                                                     int32_t Hkv, int32_t d, int64_t max_q) {
  if (Hkv < 1 || d < 1) return 0;
  if (B < 1 || rows < 1) return 256;
  return layout(B, rows, Hq / Hkv, Hkv, d, max_q).bytes;
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
  QKV_REQUIRE(Hq >= 1 && Hq % Hkv == 0, "query heads (%d) must be a multiple of kv heads (%d)", Hq,
              Hkv);
  QKV_REQUIRE(B >= 0 && B <= kMaxB && pages_per_seq >= 1,
              "batch %d must lie in [0, %d], pages_per_seq %d be positive", B, kMaxB, pages_per_seq);
  const int32_t G = Hq / Hkv;
  QKV_REQUIRE(rows >= 0 && rows * G < INT32_MAX / 2 && rows * Hq / kRows < (1 << 28),
              "rows must lie in [0, 2^30 / heads per kv head); got %lld",
              static_cast<long long>(rows));
  if (rows == 0 || B == 0) return QKV_OK;
  QKV_REQUIRE(q_start || !q_lens, "q_lens needs q_start");
  QKV_REQUIRE(q_start || rows % B == 0, "without q_start the rows (%lld) must be B (%d) times one "
              "length", static_cast<long long>(rows), B);
  QKV_REQUIRE(q && kpool && kscale && vpool && vscale && table && kv_lens && out,
              "qkv_kv8_attention: null pointer");
  QKV_REQUIRE(qkv_aligned(kpool, 16) && qkv_aligned(vpool, 16),
              "the pools must be 16-byte aligned");
  const Layout L = layout(B, rows, G, Hkv, d, max_q);
  QKV_REQUIRE(workspace && qkv_aligned(workspace, 256) && ws_bytes >= L.bytes,
              "qkv_kv8_attention: workspace too small or not 256-byte aligned");
  const int qb = q_dtype == QKV_F32 ? 4 : 2, ob = out_dtype == QKV_F32 ? 4 : 2;
  Att A{};
  A.q = q;
  A.q_ts = q_row_stride;
  A.q_hs = q_head_stride;
  A.q_dtype = q_dtype;
  A.q_vec = qkv_aligned(q, 16) && q_row_stride * qb % 16 == 0 && q_head_stride * qb % 16 == 0;
  A.rows = static_cast<int32_t>(rows);
  A.kpool = static_cast<const uint8_t*>(kpool);
  A.kscale = kscale;
  A.vpool = static_cast<const uint8_t*>(vpool);
  A.vscale = vscale;
  A.npages = num_pages;
  A.lg = qkv_page_lg(page_tokens);
  A.table = table;
  A.width = pages_per_seq;
  A.q_start = q_start;
  A.q_lens = q_lens;
  A.kv_lens = kv_lens;
  A.B = B;
  A.Hq = Hq;
  A.H = Hkv;
  A.G = G;
  A.uniform_q = static_cast<int32_t>(rows / B);
  A.scale = scale;
  A.causal = causal;
  A.out = out;
  A.out_dtype = out_dtype;
  A.out_vec = qkv_aligned(out, 16) && d * ob % 16 == 0;
  A.target = target_of(Hkv);
  A.per_target = 1.f / A.target;
  A.nslots = static_cast<int32_t>(slots_of(Hkv));
  place_parts(A, workspace, kRows, d);
  const int64_t longest = std::min<int64_t>(max_q, q_start ? rows : A.uniform_q);
  const bool pre = L.pre && longest * G > kFew;
  // decode8 runs too where, as far as the rows tell, a request may be short.  (Where one is
  // against that, prefill8 takes it: slower, the same result.)
  const bool dec = !pre || (q_start && rows <= (B - 1) * longest + kFew / G);
  QKV_REQUIRE((tiles_of(B, rows, G, kRows) + A.target) * Hkv <= INT32_MAX, "batch of %d requests "
              "and %lld rows is too large for one call", B, static_cast<long long>(rows));
  // without q_start the tiles are known
  auto tiles = [&](int r) {
    return q_start ? tiles_of(B, rows, G, r)
                   : int64_t(B) * ((int64_t(A.uniform_q) * G + r - 1) / r);
  };
  const bool cut = (int64_t(pages_per_seq) << A.lg) > kWhole;
  A.few = !pre ? INT32_MAX : dec ? kFew : 0;
  A.least = cut ? 4 : kNever;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dec) {
    // beside prefill8 this launch has only requests of up to kFew rows
    const uint32_t t = static_cast<uint32_t>(
        (pre ? std::min<int64_t>(tiles(kRows), int64_t(B) * (kFew / kRows)) : tiles(kRows)) +
        (cut ? A.target : 0));
    if (fmt == QKV_CODES_I8) {
      if (d == 128) launch<128, false>(A, t, s);
      else if (d == 96) launch<96, false>(A, t, s);
      else launch<64, false>(A, t, s);
    } else {
      if (d == 128) launch<128, true>(A, t, s);
      else if (d == 96) launch<96, true>(A, t, s);
      else launch<64, true>(A, t, s);
    }
    QKV_LAUNCHED();
  }
  Att P = A;
  bool cut8 = false;
  if (pre) {
    place_parts(P, static_cast<uint8_t*>(workspace) + L.at_pre, kPreRows, d);
    // cut only where the tiles, as far as the rows tell, do not fill the card
    const int64_t t = tiles(kPreRows);
    cut8 = cut && rows * G / kPreRows < P.target;
    P.least = cut8 ? 4 : kNever;
    // (pieces of cut tiles are within the target where the kernel counts them itself)
    const int64_t pieces = !cut8 ? t : P.plan ? t + P.target : std::max<int64_t>(t, P.target);
    qkv_kv8_prefill(P, d, fmt == QKV_CODES_E4M3, static_cast<uint32_t>(pieces), s);
    QKV_LAUNCHED();
  }
  const Att *const ja = dec && cut ? &A : nullptr, *const jp = cut8 ? &P : nullptr;
  if (d == 128) join<128>(ja, jp, s);
  else if (d == 96) join<96>(ja, jp, s);
  else join<64>(ja, jp, s);
  QKV_LAUNCHED();
  return QKV_OK;
}
