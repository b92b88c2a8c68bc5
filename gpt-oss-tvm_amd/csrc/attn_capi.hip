// C ABI of the attention-block entry points: argument validation, then the
// launchers of attn_kernels.hip.  Declarations and reference citations:
// include/attn_gfx950.h.
#include <float.h>
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/attn_gfx950.h"

extern "C" {
int attn_launch_rms_norm(const void* x, int n, int H, const void* w, float eps, void* out,
                         hipStream_t s);
int attn_launch_qkv_rope_append(const void* qkv, const void* bias, int n, const int* positions,
                                const int* slots, const float* inv_freq, float conc, void* cache,
                                int num_pages, void* q_out, bool fp8, hipStream_t s);
int attn_launch_decode(const void* q, int batch, const void* cache, const int* page_indptr,
                       const int* page_indices, int num_pages, const int* kv_len, int window,
                       float sm_scale, const void* sinks, int splits, int cps, float* part_o,
                       float* part_ml, int* arrive, void* out, hipStream_t s);
int attn_launch_prefill(const void* q, const int* q_indptr, int batch, int max_q_len,
                        const void* cache, const int* page_indptr, const int* page_indices,
                        int num_pages, const int* kv_len, int window, float sm_scale,
                        const void* sinks, void* out, int splits, int rows, float* part_o,
                        float* part_ml, hipStream_t s);
int attn_launch_bias_residual(const void* x, const void* y, const void* bias, int64_t n, int H,
                              void* out, hipStream_t s);
int attn_launch_embedding(const int* ids, int n, const void* table, int vocab, int H, void* out,
                          hipStream_t s);
size_t attn_sample_state_bytes();
int attn_launch_gemv(const void* x, int K, const void* W, int N, void* out,
                     const void* norm_w, float eps, const void* bias, const void* res,
                     hipStream_t s);
int attn_launch_qkv_gemv(const void* x, int K, const void* W, const void* norm_w,
                         float eps, const void* bias, const int* positions, const int* slots,
                         const float* inv_freq, float conc, void* cache, int num_pages,
                         void* q_out, hipStream_t s);
int attn_launch_rows_plain(const void* x, int M, int K, const void* W, int N, const void* norm_w,
                           float eps, void* out, hipStream_t s);
int attn_launch_rows_bias_residual(const void* x, int M, int K, const void* W, int N,
                                   const void* bias, const void* res, void* out, hipStream_t s);
int attn_launch_rows_qkv(const void* x, int M, int K, const void* W, const void* norm_w, float eps,
                         const void* bias, const int* positions, const int* slots,
                         const float* inv_freq, float conc, void* cache, int num_pages,
                         void* q_out, hipStream_t s);
int attn_launch_sample(const void* logits, int batch, int V, float temperature, float top_p,
                       float uniform, int* out, void* state, hipStream_t s);
int attn_launch_fp8_quantize(const void* src, int src_pages, const int* src_slots, int n,
                             void* cache, int num_pages, const int* slots, hipStream_t s);
int attn_launch_fp8_read(const void* cache, int num_pages, const int* slots, int n, void* k_out,
                         void* v_out, hipStream_t s);
int attn_launch_fp8_decode(const void* q, int batch, const void* cache, const int* page_indptr,
                           const int* page_indices, int num_pages, const int* kv_len,
                           int64_t max_span, int window, float sm_scale, const void* sinks,
                           int splits, int least, float* part_o, float* part_ml, int* arrive,
                           void* out, hipStream_t s);
int attn_launch_fp8_chunk(const void* q, const int* q_indptr, int batch, int max_q_len,
                          const void* cache, const int* page_indptr, const int* page_indices,
                          int num_pages, const int* kv_len, int window, float sm_scale,
                          const void* sinks, void* out, int tokens, int splits, int halves,
                          int rows, float* part_o, float* part_ml, hipStream_t s);
}

namespace {

constexpr int64_t kHeadDim = 64, kQHeads = 64, kKvHeads = 8, kPage = 16;
constexpr int64_t kDecChunk = 128;     // keys per chunk of a decode workgroup
constexpr int64_t kMaxTokens = 1 << 24;
constexpr int64_t kMaxPages = ((int64_t)1 << 31) / kPage;

inline bool a16(const void* p) { return ((uintptr_t)p & 15u) == 0; }
inline bool a4(const void* p) { return ((uintptr_t)p & 3u) == 0; }
inline hipStream_t as_stream(moe_stream_t s) { return (hipStream_t)s; }
inline int status(int launch_rc) { return launch_rc == 0 ? MOE_OK : MOE_ERR_LAUNCH; }

// Chunks of 128 keys per decode workgroup: more with larger batches, where
// there are workgroups enough (a workgroup's fixed costs, the page-table
// reads before its first loads and the published partial after its last
// chunk, then spread over more keys).  It depends on the batch only (the
// kernel makes a span of at most two chunks one split), so a call's results
// do not depend on the span bound (a captured graph fixes the
// bound at the pool's capacity).
int64_t decode_cps(int64_t batch) { return batch >= 32 ? 8 : batch >= 8 ? 4 : batch >= 2 ? 2 : 1; }
int64_t decode_splits(int64_t batch, int64_t max_span) {
  const int64_t keys = kDecChunk * decode_cps(batch);
  return (max_span + keys - 1) / keys;
}

// Workgroups that a tile's keys are shared out over in prefill attention: as many
// as fit the chip at once (a tile has 16 workgroups, a CU holds two), each with
// about 192 keys or more (a causal tile sees half of the new ones), at most 16.
// Measured, us without and with (new tokens + cached): 9 + 1500 60.6 and 18.3, 64 +
// 8000 296 and 37.7, 300 + 600 43.3 and 31.4, 300 + 6000 238 and 86, 1024 + 0 46.3 and
// 45.2.  One round more than fits cost more than the shares gained (300 + 6000 in
// 560 workgroups 104 us); 700 + 0 in two shares took 35.3 against 33.3.  The shares
// follow from the whole call, so a sequence's last bits depend on what else is in
// it (decode's do not); merged in fp32, they are no further off than the plain
// form (against 64 bits, plain and shared: 9 + 1500 1.35e-4 and 1.11e-4, 300 + 6000
// 1.35e-4 and 1.28e-4, 1024 + 0 1.14e-4 and 1.08e-4).
constexpr int64_t kPfSplitKeys = 192, kPfMaxSplits = 16, kPfWorkgroups = 512;
int64_t prefill_splits(int64_t batch, int64_t max_q_len, int64_t max_kv_len, int64_t window) {
  if (batch <= 0 || batch > kPfWorkgroups) return 1;  // (and no overflow below)
  const int64_t wgs = (max_q_len + 63) / 64 * batch * 16;
  const int64_t keys = (window > 0 ? std::min(max_kv_len, window + 64) : max_kv_len) - max_q_len / 2;
  if (wgs <= 0) return 1;
  const int64_t s = std::min(kPfWorkgroups / wgs, keys / kPfSplitKeys);
  return std::max<int64_t>(1, std::min(s, kPfMaxSplits));
}

}  // namespace

extern "C" {

int attn_rms_norm(const uint16_t* x, int64_t n, int64_t H, const uint16_t* w, float eps,
                  uint16_t* out, moe_stream_t stream) {
  if (n < 0 || n > kMaxTokens || H <= 0 || H % 8 || H > 65536) return MOE_ERR_SHAPE;
  if (n == 0) return MOE_OK;
  if (!x || !w || !out) return MOE_ERR_NULL;
  if (!a16(x) || !a16(w) || !a16(out)) return MOE_ERR_ALIGN;
  return status(attn_launch_rms_norm(x, (int)n, (int)H, w, eps, out, as_stream(stream)));
}

static int rope_append(const uint16_t* qkv, const uint16_t* qkv_bias, int64_t n,
                       const int32_t* positions, const int32_t* slots, const float* inv_freq,
                       float concentration, void* kv_cache, int64_t num_pages, uint16_t* q_out,
                       bool fp8, moe_stream_t stream) {
  if (n < 0 || n > kMaxTokens || num_pages <= 0 || num_pages > kMaxPages) return MOE_ERR_SHAPE;
  if (n == 0) return MOE_OK;
  if (!qkv || !qkv_bias || !positions || !slots || !inv_freq || !kv_cache || !q_out)
    return MOE_ERR_NULL;
  if (!a16(qkv) || !a16(qkv_bias) || !a16(kv_cache) || !a16(q_out) || !a4(positions) ||
      !a4(slots) || !a4(inv_freq))
    return MOE_ERR_ALIGN;
  return status(attn_launch_qkv_rope_append(qkv, qkv_bias, (int)n, positions, slots, inv_freq,
                                            concentration, kv_cache, (int)num_pages, q_out, fp8,
                                            as_stream(stream)));
}

int attn_qkv_rope_append(const uint16_t* qkv, const uint16_t* qkv_bias, int64_t n,
                         const int32_t* positions, const int32_t* slots, const float* inv_freq,
                         float concentration, void* kv_cache, int64_t num_pages, uint16_t* q_out,
                         moe_stream_t stream) {
  return rope_append(qkv, qkv_bias, n, positions, slots, inv_freq, concentration, kv_cache,
                     num_pages, q_out, false, stream);
}

// Workspace of attn_decode: the arrival counts [65536][8] (int32; zero before the
// first call, left zero by every call), then the split partials o
// [batch][64][splits][64] and (m, l) [batch][64][splits][2].  The counts' place
// does not depend on the batch: a call's partials never lie where a call of more
// sequences on the same workspace counts.
constexpr size_t kDecodeCounts = (size_t)65536 * kKvHeads * 4;

size_t attn_decode_workspace_bytes(int64_t batch, int64_t max_span) {
  if (batch <= 0 || max_span <= 0) return 0;
  const size_t parts = (size_t)batch * kQHeads * (size_t)decode_splits(batch, max_span);
  return kDecodeCounts + parts * (kHeadDim + 2) * sizeof(float) + 256;
}

int attn_decode(const uint16_t* q, int64_t batch, const void* kv_cache, int64_t num_pages,
                const int32_t* page_indptr, const int32_t* page_indices, const int32_t* kv_len,
                int64_t max_span, int32_t window, float sm_scale, const uint16_t* sinks,
                uint16_t* out, void* workspace, size_t workspace_bytes, moe_stream_t stream) {
  if (batch < 0 || batch > 65535 || num_pages <= 0 || num_pages > kMaxPages) return MOE_ERR_SHAPE;
  if (batch == 0) return MOE_OK;
  if (max_span <= 0 || max_span > kMaxPages * kPage) return MOE_ERR_SHAPE;
  if (!q || !kv_cache || !page_indptr || !page_indices || !kv_len || !sinks || !out || !workspace)
    return MOE_ERR_NULL;
  if (!a16(q) || !a16(kv_cache) || !a16(out) || !a16(workspace) || !a4(page_indptr) ||
      !a4(page_indices) || !a4(kv_len) || ((uintptr_t)sinks & 1u))
    return MOE_ERR_ALIGN;
  if (workspace_bytes < attn_decode_workspace_bytes(batch, max_span)) return MOE_ERR_WORKSPACE;
  const int64_t splits = decode_splits(batch, max_span);
  if (splits > 65535) return MOE_ERR_SHAPE;
  int* arrive = (int*)workspace;
  float* part_o = (float*)((char*)workspace + kDecodeCounts);
  float* part_ml = part_o + (size_t)batch * kQHeads * splits * kHeadDim;
  return status(attn_launch_decode(q, (int)batch, kv_cache, page_indptr, page_indices,
                                   (int)num_pages, kv_len, window, sm_scale, sinks, (int)splits,
                                   (int)decode_cps(batch), part_o, part_ml, arrive, out,
                                   as_stream(stream)));
}

static int prefill(const uint16_t* q, int64_t rows, const int32_t* q_indptr, int64_t batch,
                   int64_t max_q_len, const void* kv_cache, int64_t num_pages,
                   const int32_t* page_indptr, const int32_t* page_indices, const int32_t* kv_len,
                   int64_t splits, int32_t window, float sm_scale, const uint16_t* sinks,
                   uint16_t* out, float* part_o, float* part_ml, moe_stream_t stream) {
  if (batch < 0 || max_q_len < 0 || max_q_len > kMaxTokens || num_pages <= 0 ||
      num_pages > kMaxPages)
    return MOE_ERR_SHAPE;
  if (batch == 0 || max_q_len == 0) return MOE_OK;
  const int64_t tiles = (max_q_len + 63) / 64;
  if (tiles * batch >= ((int64_t)1 << 31)) return MOE_ERR_SHAPE;
  if (!q || !q_indptr || !kv_cache || !page_indptr || !page_indices || !kv_len || !sinks || !out)
    return MOE_ERR_NULL;
  if (!a16(q) || !a16(kv_cache) || !a16(out) || !a4(q_indptr) || !a4(page_indptr) ||
      !a4(page_indices) || !a4(kv_len) || ((uintptr_t)sinks & 1u))
    return MOE_ERR_ALIGN;
  return status(attn_launch_prefill(q, q_indptr, (int)batch, (int)max_q_len, kv_cache,
                                    page_indptr, page_indices, (int)num_pages, kv_len, window,
                                    sm_scale, sinks, out, (int)splits, (int)rows, part_o, part_ml,
                                    as_stream(stream)));
}

int attn_prefill(const uint16_t* q, const int32_t* q_indptr, int64_t batch, int64_t max_q_len,
                 const void* kv_cache, int64_t num_pages, const int32_t* page_indptr,
                 const int32_t* page_indices, const int32_t* kv_len, int32_t window,
                 float sm_scale, const uint16_t* sinks, uint16_t* out, moe_stream_t stream) {
  return prefill(q, 0, q_indptr, batch, max_q_len, kv_cache, num_pages, page_indptr, page_indices,
                 kv_len, 1, window, sm_scale, sinks, out, nullptr, nullptr, stream);
}

// Workspace: the shares' o [splits][rows][64][64], then (m, l) [splits][rows][64][2]
size_t attn_prefill_workspace_bytes(int64_t rows, int64_t batch, int64_t max_q_len,
                                    int64_t max_kv_len, int32_t window) {
  if (rows <= 0 || rows > kMaxTokens || batch <= 0 || max_q_len <= 0 || max_q_len > kMaxTokens)
    return 0;
  const int64_t splits = prefill_splits(batch, max_q_len, max_kv_len, window);
  return splits <= 1 ? 0 : (size_t)(splits * rows * kQHeads * (kHeadDim + 2)) * sizeof(float);
}

int attn_prefill_split(const uint16_t* q, int64_t rows, const int32_t* q_indptr, int64_t batch,
                       int64_t max_q_len, const void* kv_cache, int64_t num_pages,
                       const int32_t* page_indptr, const int32_t* page_indices,
                       const int32_t* kv_len, int64_t max_kv_len, int32_t window, float sm_scale,
                       const uint16_t* sinks, uint16_t* out, void* workspace,
                       size_t workspace_bytes, moe_stream_t stream) {
  if (rows < 0 || rows > kMaxTokens) return MOE_ERR_SHAPE;
  const size_t need = attn_prefill_workspace_bytes(rows, batch, max_q_len, max_kv_len, window);
  if (need == 0)
    return prefill(q, rows, q_indptr, batch, max_q_len, kv_cache, num_pages, page_indptr,
                   page_indices, kv_len, 1, window, sm_scale, sinks, out, nullptr, nullptr, stream);
  if (!workspace) return MOE_ERR_NULL;
  if (!a16(workspace)) return MOE_ERR_ALIGN;
  if (workspace_bytes < need) return MOE_ERR_WORKSPACE;
  const int64_t splits = prefill_splits(batch, max_q_len, max_kv_len, window);
  float* part_o = (float*)workspace;
  return prefill(q, rows, q_indptr, batch, max_q_len, kv_cache, num_pages, page_indptr,
                 page_indices, kv_len, splits, window, sm_scale, sinks, out, part_o,
                 part_o + splits * rows * kQHeads * kHeadDim, stream);
}

int attn_bias_residual(const uint16_t* x, const uint16_t* y, const uint16_t* bias, int64_t n,
                       int64_t H, uint16_t* out, moe_stream_t stream) {
  if (n < 0 || n > kMaxTokens || H <= 0 || H % 4 || H > 65536) return MOE_ERR_SHAPE;
  if (n == 0) return MOE_OK;
  if (!x || !y || !bias || !out) return MOE_ERR_NULL;
  if (((uintptr_t)x & 7u) || ((uintptr_t)y & 7u) || ((uintptr_t)bias & 7u) || ((uintptr_t)out & 7u))
    return MOE_ERR_ALIGN;
  return status(attn_launch_bias_residual(x, y, bias, n, (int)H, out, as_stream(stream)));
}

int attn_embedding(const int32_t* ids, int64_t n, const uint16_t* table, int64_t vocab, int64_t H,
                   uint16_t* out, moe_stream_t stream) {
  if (n < 0 || n > kMaxTokens || vocab <= 0 || vocab >= ((int64_t)1 << 31) || H <= 0 || H % 8 ||
      H > 65536)
    return MOE_ERR_SHAPE;
  if (n == 0) return MOE_OK;
  if (!ids || !table || !out) return MOE_ERR_NULL;
  if (!a4(ids) || !a16(table) || !a16(out)) return MOE_ERR_ALIGN;
  return status(attn_launch_embedding(ids, (int)n, table, (int)vocab, (int)H, out,
                                      as_stream(stream)));
}

size_t attn_sample_workspace_bytes(int64_t batch) {
  return batch > 0 ? (size_t)batch * attn_sample_state_bytes() : 0;
}

int attn_sample_top_p(const uint16_t* logits, int64_t batch, int64_t vocab, float temperature,
                      float top_p, float uniform, int32_t* out_ids, void* workspace,
                      size_t workspace_bytes, moe_stream_t stream) {
  if (batch < 0 || batch > 65535 || vocab <= 0 || vocab >= ((int64_t)1 << 30)) return MOE_ERR_SHAPE;
  if (batch == 0) return MOE_OK;
  if (!(temperature >= 0.0f) || !(top_p > 0.0f) || !(uniform >= 0.0f)) return MOE_ERR_UNSUPPORTED;
  if (!logits || !out_ids || !workspace) return MOE_ERR_NULL;
  if (!a16(logits) || !a4(out_ids) || !a16(workspace)) return MOE_ERR_ALIGN;
  if (workspace_bytes < attn_sample_workspace_bytes(batch)) return MOE_ERR_WORKSPACE;
  return status(attn_launch_sample(logits, (int)batch, (int)vocab, temperature, top_p, uniform,
                                   out_ids, workspace, as_stream(stream)));
}

namespace {
// Tokens of the fused dense projections: the GEMV entry points, the rows ones of
// QKV and of the output.  QKV above kRowsNormTokens tokens takes them normed, and
// rows of at most kWideQkvK.
constexpr int64_t kGemvTokens = 8, kRowsQkvTokens = 64, kRowsOutTokens = 48;
constexpr int64_t kRowsNormTokens = 16, kWideQkvK = 3072;

int check_gemv(const void* x, int64_t M, int64_t most, int64_t K, const void* W, int64_t N,
               const void* out) {
  if (M < 1 || M > most || K <= 0 || K % 8 || K > 4096 || N <= 0 || N >= ((int64_t)1 << 31))
    return MOE_ERR_SHAPE;
  if (!x || !W || !out) return MOE_ERR_NULL;
  if (!a16(x) || !a16(W) || ((uintptr_t)out & 1u)) return MOE_ERR_ALIGN;
  return MOE_OK;
}

// One token takes the vector-ALU GEMV (it streams W at the HBM's rate and its
// sums need no second operand tile); from two tokens on its dot products bind
// it (the unembedding at 5 tokens: 750 us against 188 at one), and the matrix
// core form takes the call.
int bias_residual(int64_t most, const uint16_t* x, int64_t M, int64_t K, const uint16_t* W,
                  int64_t N, const uint16_t* bias, const uint16_t* residual, uint16_t* out,
                  moe_stream_t stream) {
  int rc = check_gemv(x, M, most, K, W, N, out);
  if (rc) return rc;
  if (!bias || !residual) return MOE_ERR_NULL;
  if (((uintptr_t)bias & 1u) || ((uintptr_t)residual & 1u)) return MOE_ERR_ALIGN;
  if (M > 1)
    return status(attn_launch_rows_bias_residual(x, (int)M, (int)K, W, (int)N, bias, residual,
                                                 out, as_stream(stream)));
  return status(attn_launch_gemv(x, (int)K, W, (int)N, out, nullptr, 0.0f, bias, residual,
                                 as_stream(stream)));
}

int qkv_rope_append(int64_t most, const uint16_t* x, int64_t M, int64_t K, const uint16_t* W,
                    const uint16_t* norm_w, float eps, const uint16_t* qkv_bias,
                    const int32_t* positions, const int32_t* slots, const float* inv_freq,
                    float concentration, void* kv_cache, int64_t num_pages, uint16_t* q_out,
                    moe_stream_t stream) {
  int rc = check_gemv(x, M, most, K, W, kHeadDim * (kQHeads + 2 * kKvHeads), q_out);
  if (rc) return rc;
  if (num_pages <= 0 || num_pages > kMaxPages) return MOE_ERR_SHAPE;
  if (M > kRowsNormTokens && (norm_w || K > kWideQkvK)) return MOE_ERR_SHAPE;
  if (!qkv_bias || !positions || !slots || !inv_freq || !kv_cache) return MOE_ERR_NULL;
  if (!a16(kv_cache) || !a4(positions) || !a4(slots) || !a4(inv_freq) ||
      ((uintptr_t)qkv_bias & 1u) || (norm_w && ((uintptr_t)norm_w & 1u)))
    return MOE_ERR_ALIGN;
  if (M > 1)
    return status(attn_launch_rows_qkv(x, (int)M, (int)K, W, norm_w, eps, qkv_bias, positions,
                                       slots, inv_freq, concentration, kv_cache, (int)num_pages,
                                       q_out, as_stream(stream)));
  return status(attn_launch_qkv_gemv(x, (int)K, W, norm_w, eps, qkv_bias, positions, slots,
                                     inv_freq, concentration, kv_cache, (int)num_pages, q_out,
                                     as_stream(stream)));
}
}  // namespace

int attn_gemv(const uint16_t* x, int64_t M, int64_t K, const uint16_t* W, int64_t N,
              const uint16_t* norm_w, float eps, uint16_t* out, moe_stream_t stream) {
  int rc = check_gemv(x, M, kGemvTokens, K, W, N, out);
  if (rc) return rc;
  if (norm_w && ((uintptr_t)norm_w & 1u)) return MOE_ERR_ALIGN;
  if (M > 1)
    return status(attn_launch_rows_plain(x, (int)M, (int)K, W, (int)N, norm_w, eps, out,
                                         as_stream(stream)));
  return status(attn_launch_gemv(x, (int)K, W, (int)N, out, norm_w, eps, nullptr, nullptr,
                                 as_stream(stream)));
}

int attn_gemv_bias_residual(const uint16_t* x, int64_t M, int64_t K, const uint16_t* W, int64_t N,
                            const uint16_t* bias, const uint16_t* residual, uint16_t* out,
                            moe_stream_t stream) {
  return bias_residual(kGemvTokens, x, M, K, W, N, bias, residual, out, stream);
}

int attn_rows_bias_residual(const uint16_t* x, int64_t M, int64_t K, const uint16_t* W, int64_t N,
                            const uint16_t* bias, const uint16_t* residual, uint16_t* out,
                            moe_stream_t stream) {
  return bias_residual(kRowsOutTokens, x, M, K, W, N, bias, residual, out, stream);
}

int attn_qkv_gemv_rope_append(const uint16_t* x, int64_t M, int64_t K, const uint16_t* W,
                              const uint16_t* norm_w, float eps, const uint16_t* qkv_bias,
                              const int32_t* positions, const int32_t* slots,
                              const float* inv_freq, float concentration, void* kv_cache,
                              int64_t num_pages, uint16_t* q_out, moe_stream_t stream) {
  return qkv_rope_append(kGemvTokens, x, M, K, W, norm_w, eps, qkv_bias, positions, slots,
                         inv_freq, concentration, kv_cache, num_pages, q_out, stream);
}

int attn_rows_qkv_rope_append(const uint16_t* x, int64_t M, int64_t K, const uint16_t* W,
                              const uint16_t* norm_w, float eps, const uint16_t* qkv_bias,
                              const int32_t* positions, const int32_t* slots,
                              const float* inv_freq, float concentration, void* kv_cache,
                              int64_t num_pages, uint16_t* q_out, moe_stream_t stream) {
  return qkv_rope_append(kRowsQkvTokens, x, M, K, W, norm_w, eps, qkv_bias, positions, slots,
                         inv_freq, concentration, kv_cache, num_pages, q_out, stream);
}

// ---------------------------------------------------------------------------
// The 8-bit cache

int attn_qkv_rope_append_fp8(const uint16_t* qkv, const uint16_t* qkv_bias, int64_t n,
                             const int32_t* positions, const int32_t* slots, const float* inv_freq,
                             float concentration, void* kv_cache, int64_t num_pages,
                             uint16_t* q_out, moe_stream_t stream) {
  if (num_pages >= kMaxPages) return MOE_ERR_SHAPE;
  return rope_append(qkv, qkv_bias, n, positions, slots, inv_freq, concentration, kv_cache,
                     num_pages, q_out, true, stream);
}

int attn_kv_quantize_fp8(const void* src, int64_t src_pages, const int32_t* src_slots, int64_t n,
                         void* kv_cache, int64_t num_pages, const int32_t* slots,
                         moe_stream_t stream) {
  if (n < 0 || n > kMaxTokens || src_pages <= 0 || src_pages >= kMaxPages || num_pages <= 0 ||
      num_pages >= kMaxPages)
    return MOE_ERR_SHAPE;
  if (n == 0) return MOE_OK;
  if (!src || !src_slots || !kv_cache || !slots) return MOE_ERR_NULL;
  if (!a16(src) || !a16(kv_cache) || !a4(src_slots) || !a4(slots)) return MOE_ERR_ALIGN;
  return status(attn_launch_fp8_quantize(src, (int)src_pages, src_slots, (int)n, kv_cache,
                                         (int)num_pages, slots, as_stream(stream)));
}

int attn_kv_read_fp8(const void* kv_cache, int64_t num_pages, const int32_t* slots, int64_t n,
                     uint16_t* k_out, uint16_t* v_out, moe_stream_t stream) {
  if (n < 0 || n > kMaxTokens || num_pages <= 0 || num_pages >= kMaxPages) return MOE_ERR_SHAPE;
  if (n == 0) return MOE_OK;
  if (!kv_cache || !slots || !k_out || !v_out) return MOE_ERR_NULL;
  if (!a16(kv_cache) || !a4(slots) || !a16(k_out) || !a16(v_out)) return MOE_ERR_ALIGN;
  return status(attn_launch_fp8_read(kv_cache, (int)num_pages, slots, (int)n, k_out, v_out,
                                     as_stream(stream)));
}

namespace {
constexpr int64_t kFp8Block = 64;  // keys of a block of the 8-bit attention kernels
// 64-key blocks that a span of keys can touch
int64_t fp8_blocks(int64_t span) { return (span + 2 * (kFp8Block - 1)) / kFp8Block; }
// Blocks that a split has at least (a wave of the workgroup takes one), splits at most.
constexpr int64_t kFp8SplitBlocks = 4, kFp8MaxSplits = 64;

// Decode: blocks that a split has at least, and splits at most.  A split costs its start
// and its part of the merge, so a batch that fills the chip with a workgroup a head
// (64 sequences) is split only where sequences are longer than 64 blocks (64 of 1024 to
// 4096 keys: 38.7 us, in halves 41.0; 16 of up to 2000: 13.7 in halves, 12.2 in
// quarters).  One sequence alone takes more than 32 where they have 16 blocks each (131072
// keys: 37.3 us in 32, 34.8 in 64; 20000 keys: 15.3 in 32, 18.9 in 64).
int64_t fp8_decode_least(int64_t batch) {
  return batch >= 64 ? 64 : std::max(kFp8SplitBlocks, batch / 2);
}
int64_t fp8_decode_splits(int64_t batch, int64_t max_span) {
  const int64_t least = fp8_decode_least(batch), most = batch == 1 ? kFp8MaxSplits : 32;
  return std::min(most, (fp8_blocks(max_span) + least - 1) / least);
}

// Tokens of a chunk's query tile, and how many splits its keys are shared out over: as
// many as let its workgroups fit the chip at once (two a CU; three of several tiles of 2).
//  * 64 of more than 32 tokens, without a window, where they are two rounds of the chip.
//  * 4 tokens up to 20 tokens, where their tiles are two rounds of the chip or less, and
//    for longer chunks where there are few of these tiles over few keys; us in tiles of
//    4 and of 32, (sequences of) tokens over (up to) cached: 16 of 20 over 2000 29.0 and
//    33.1, of 24 over 2000 37.0 and 34.9, 32 of 16 over 4000 74.2 and 75.2, of 20 over 1000
//    33.6 and 26.8, 64 of 16 over 1000 53.3 and 41.3; 8 of 24 over 1000 15.8 and 23.1, 24 over
//    8000 22.0 and 25.5, 64 over 6000 27.9 and 25.7, 128 over 3000 28.2 and 30.2, 200 over 500
//    14.2 and 21.7, 100 over 6000 42.3 and 35.5.
//  * 2 tokens of up to 2 and of 5 to 12: a wave's blocks take half as long, and three
//    workgroups share a CU; us in tiles of 4 and of 2, sequences of tokens over up to
//    cached: 16 of 5 over 4000 31.8 and 27.1, 128 of 5 over 1000 56.1 and 39.6, one of 9
//    over 8000 18.7 and 16.7, 16 of 12 over 4000 44.0 and 40.4; but 16 of 3 over 4000
//    22.2 and 23.8, 16 of 16 over 4000 37.2 and 47.1.
//  * Two splits of 32 tokens make the halves of one workgroup, joined in LDS: half the parts
//    to be written and merged, none for two; us without and with: 1000 over 1000 59.9
//    and 45.2, 700 29.5 and 21.8, 300 over 6000 59.3 and 56.7, 128 over 16000 62.7 and 57.2.
//    Of an odd number one is given up, which pays from seven on (280 over 4000 45.7 and
//    43.8) or over few keys: three, 550 over 1000 39.2 and 35.9, over 1500 44.5 and 43.6,
//    over 2500 55.5 and 59.1, over 6000 93 and 114; five, 380 over 3000 47.2 and 48.2.
constexpr int64_t kFp8OddSplits = 7, kFp8OddKeys = 600;
constexpr int64_t kFp8ChunkWgs = 512, kFp8PairWgs = 768, kFp8PairTokens = 12, kFp8FewTokens = 20,
                  kFp8FewTiles = 64, kFp8FewKeys = 130000;
struct Fp8Chunk {
  int64_t tokens, splits, tiles;  // tiles of the longest sequence
  int64_t halves = 1;             // of a split, one workgroup's
};
Fp8Chunk fp8_chunk(int64_t batch, int64_t max_q_len, int64_t max_kv_len, int64_t window) {
  auto tiles_of = [&](int64_t tokens) { return (max_q_len + tokens - 1) / tokens; };
  max_kv_len = std::min(max_kv_len, kMaxPages * kPage);  // (and no overflow below)
  if (window <= 0 && max_q_len > 32 && tiles_of(64) * kKvHeads >= (512 + batch - 1) / batch)
    return Fp8Chunk{64, 1, tiles_of(64)};
  const int64_t reach = window > 0 ? std::min(max_kv_len, window + max_q_len) : max_kv_len;
  const int64_t small = tiles_of(4) <= kFp8FewTiles  // tiles of 4, or too many
                            ? tiles_of(4) * std::min(batch, kFp8FewTiles + 1)
                            : kFp8FewTiles + 1;
  const bool rounds = tiles_of(4) == 1 || tiles_of(4) * batch <= 2 * kFp8FewTiles;
  const bool few = (max_q_len <= kFp8FewTokens && rounds) ||
                   (small <= kFp8FewTiles && reach > 0 && small * reach <= kFp8FewKeys);
  const bool pairs = max_q_len <= 2 || (max_q_len > 4 && max_q_len <= kFp8PairTokens);
  const int64_t tokens = pairs ? 2 : few ? 4 : 32;
  const int64_t wgs = pairs && max_q_len > 2 ? kFp8PairWgs : kFp8ChunkWgs;
  const int64_t keys = window > 0 ? std::min(max_kv_len, window + tokens) : max_kv_len;
  if (keys <= 0 || batch > kFp8ChunkWgs) return Fp8Chunk{tokens, 1, tiles_of(tokens)};
  const int64_t most = std::min(kFp8MaxSplits, wgs / (tiles_of(tokens) * batch * kKvHeads));
  const int64_t splits = std::max<int64_t>(1, std::min(most, fp8_blocks(keys) / kFp8SplitBlocks));
  const bool pays = splits % 2 == 0 || splits >= kFp8OddSplits || keys <= kFp8OddKeys * splits;
  if (tokens == 32 && splits > 1 && pays)
    return Fp8Chunk{tokens, splits / 2, tiles_of(tokens), 2};
  return Fp8Chunk{tokens, splits, tiles_of(tokens)};
}
}  // namespace

// Workspace of attn_decode_fp8: arrival counts as attn_decode's, then the splits'
// o [splits][batch][64][64] and (m, l) [splits][batch][64][2].
size_t attn_decode_fp8_workspace_bytes(int64_t batch, int64_t max_span) {
  if (batch <= 0 || batch > 65535 || max_span <= 0 || max_span > kMaxPages * kPage) return 0;
  const size_t parts = (size_t)batch * kQHeads * (size_t)fp8_decode_splits(batch, max_span);
  return kDecodeCounts + parts * (kHeadDim + 2) * sizeof(float);
}

int attn_decode_fp8(const uint16_t* q, int64_t batch, const void* kv_cache, int64_t num_pages,
                    const int32_t* page_indptr, const int32_t* page_indices, const int32_t* kv_len,
                    int64_t max_span, int32_t window, float sm_scale, const uint16_t* sinks,
                    uint16_t* out, void* workspace, size_t workspace_bytes, moe_stream_t stream) {
  if (batch < 0 || batch > 65535 || num_pages <= 0 || num_pages >= kMaxPages) return MOE_ERR_SHAPE;
  if (batch == 0) return MOE_OK;
  if (max_span <= 0 || max_span > kMaxPages * kPage) return MOE_ERR_SHAPE;
  if (!(sm_scale > 0.0f && sm_scale <= FLT_MAX)) return MOE_ERR_UNSUPPORTED;
  if (!q || !kv_cache || !page_indptr || !page_indices || !kv_len || !sinks || !out || !workspace)
    return MOE_ERR_NULL;
  if (!a16(q) || !a16(kv_cache) || !a16(out) || !a16(workspace) || !a4(page_indptr) ||
      !a4(page_indices) || !a4(kv_len) || ((uintptr_t)sinks & 1u))
    return MOE_ERR_ALIGN;
  if (workspace_bytes < attn_decode_fp8_workspace_bytes(batch, max_span)) return MOE_ERR_WORKSPACE;
  const int64_t splits = fp8_decode_splits(batch, max_span);
  float* part_o = (float*)((char*)workspace + kDecodeCounts);
  return status(attn_launch_fp8_decode(q, (int)batch, kv_cache, page_indptr, page_indices,
                                       (int)num_pages, kv_len, max_span, window, sm_scale, sinks,
                                       (int)splits, (int)fp8_decode_least(batch), part_o,
                                       part_o + (size_t)splits * batch * kQHeads * kHeadDim,
                                       (int*)workspace, out, as_stream(stream)));
}

// Workspace: the splits' o [splits][rows][64][64], then (m, l) [splits][rows][64][2], rows
// the tokens of the sequences' tiles, whatever rows q has beside them (a split call's
// workgroups are few, so at most 35 MB).
int64_t fp8_chunk_rows(const Fp8Chunk& chunk, int64_t batch) {
  return chunk.tokens * chunk.tiles * batch;
}

size_t attn_prefill_fp8_workspace_bytes(int64_t rows, int64_t batch, int64_t max_q_len,
                                        int64_t max_kv_len, int32_t window) {
  if (rows <= 0 || rows > kMaxTokens || batch <= 0 || batch > kMaxTokens || max_q_len <= 0 ||
      max_q_len > kMaxTokens)
    return 0;
  const Fp8Chunk chunk = fp8_chunk(batch, max_q_len, max_kv_len, window);
  if (chunk.splits <= 1) return 0;
  return (size_t)(chunk.splits * fp8_chunk_rows(chunk, batch) * kQHeads * (kHeadDim + 2)) *
         sizeof(float);
}

int attn_prefill_fp8(const uint16_t* q, int64_t rows, const int32_t* q_indptr, int64_t batch,
                     int64_t max_q_len, const void* kv_cache, int64_t num_pages,
                     const int32_t* page_indptr, const int32_t* page_indices,
                     const int32_t* kv_len, int64_t max_kv_len, int32_t window, float sm_scale,
                     const uint16_t* sinks, uint16_t* out, void* workspace, size_t workspace_bytes,
                     moe_stream_t stream) {
  if (rows < 0 || rows > kMaxTokens || batch < 0 || max_q_len < 0 || max_q_len > kMaxTokens ||
      num_pages <= 0 || num_pages >= kMaxPages)
    return MOE_ERR_SHAPE;
  if (rows == 0 || batch == 0 || max_q_len == 0) return MOE_OK;
  if (batch > kMaxTokens) return MOE_ERR_SHAPE;  // (and no overflow below)
  // as many tiles of 64 tokens as a launch of attn_prefill holds
  if ((max_q_len + 63) / 64 * batch >= ((int64_t)1 << 24)) return MOE_ERR_SHAPE;
  const Fp8Chunk chunk = fp8_chunk(batch, max_q_len, max_kv_len, window);
  if (!(sm_scale > 0.0f && sm_scale <= FLT_MAX)) return MOE_ERR_UNSUPPORTED;
  if (!q || !q_indptr || !kv_cache || !page_indptr || !page_indices || !kv_len || !sinks || !out)
    return MOE_ERR_NULL;
  if (!a16(q) || !a16(kv_cache) || !a16(out) || !a4(q_indptr) || !a4(page_indptr) ||
      !a4(page_indices) || !a4(kv_len) || ((uintptr_t)sinks & 1u))
    return MOE_ERR_ALIGN;
  const size_t need = attn_prefill_fp8_workspace_bytes(rows, batch, max_q_len, max_kv_len, window);
  if (need && !workspace) return MOE_ERR_NULL;
  if (need && !a16(workspace)) return MOE_ERR_ALIGN;
  if (workspace_bytes < need) return MOE_ERR_WORKSPACE;
  float* part_o = (float*)workspace;
  const int64_t part_rows = need ? fp8_chunk_rows(chunk, batch) : 0;
  return status(attn_launch_fp8_chunk(
      q, q_indptr, (int)batch, (int)max_q_len, kv_cache, page_indptr, page_indices, (int)num_pages,
      kv_len, window, sm_scale, sinks, out, (int)chunk.tokens, (int)chunk.splits,
      (int)chunk.halves, (int)part_rows, part_o,
      need ? part_o + chunk.splits * part_rows * kQHeads * kHeadDim : nullptr,
      as_stream(stream)));
}

}  // extern "C"
