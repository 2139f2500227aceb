// extern "C" entry points of the KV cache in pages: every argument is checked before the first launch, nothing is allocated, nothing
// synchronises.
#include "common.h"
#include "cache.h"

using namespace bsattn;

static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

static int check_cache(const bsattn_cache* c) {
  if (c == nullptr || c->k_codes == nullptr || c->v_codes == nullptr || c->k_scales == nullptr || c->v_scales == nullptr ||
      c->page_table == nullptr || c->lengths == nullptr || c->refs == nullptr || c->free_from == nullptr) return BSATTN_ERR_NULL;
  if (c->pages <= 0 || c->heads <= 0 || c->sequences <= 0 || c->max_pages <= 0) return BSATTN_ERR_SHAPE;
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return BSATTN_ERR_HEAD_DIM;
  if (c->dtype != BSATTN_F16 && c->dtype != BSATTN_BF16) return BSATTN_ERR_DTYPE;
  // pages and tokens of a sequence are counted in 32 bits
  if (c->max_pages > 0x7fffffff / PAGE - 1 || c->pages > 0x3fffffff || c->heads > 65535) return BSATTN_ERR_RANGE;
  if (!aligned16(c->k_codes) || !aligned16(c->v_codes) || !aligned16(c->k_scales) || !aligned16(c->v_scales)) return BSATTN_ERR_STRIDE;
  return BSATTN_OK;
}

// rows of 16-bit values (or fp32 ones) of `elem` bytes
static int check_rows(const void* p, const int64_t* s, int elem) {
  if (p == nullptr || s == nullptr) return BSATTN_ERR_NULL;
  if (s[3] != 1 || !aligned16(p)) return BSATTN_ERR_STRIDE;
  for (int i = 0; i < 3; ++i)
    if ((s[i] * elem) % 16 != 0) return BSATTN_ERR_STRIDE;
  return BSATTN_OK;
}

static int check_workspace(const void* ws, size_t bytes, size_t need) {
  if (ws == nullptr || bytes < need) return BSATTN_ERR_WORKSPACE;
  return aligned16(ws) ? BSATTN_OK : BSATTN_ERR_STRIDE;
}

extern "C" {

int bsattn_cache_append_workspace(const bsattn_cache* cache, int B, int N, size_t* bytes) {
  if (const int rc = check_cache(cache); rc != BSATTN_OK) return rc;
  if (bytes == nullptr) return BSATTN_ERR_NULL;
  if (B <= 0 || N < 0) return BSATTN_ERR_SHAPE;
  if (B > CACHE_ROWS_MAX || N > cache->max_pages * PAGE || (int64_t)B * (N / PAGE + 2) > 0x7fffffffLL ||
      (int64_t)N * (cache->head_dim / 8) > 0x7fffffffLL) return BSATTN_ERR_RANGE;
  *bytes = cache_append_workspace_bytes(B, N);
  return BSATTN_OK;
}

int bsattn_cache_append(const bsattn_cache* cache, const void* k, const void* v, const int64_t* k_strides, const int64_t* v_strides,
                        const int32_t* sequences, const int32_t* at, const int32_t* counts, int B, int N, void* workspace,
                        size_t workspace_bytes, void* stream) {
  size_t need = 0;
  if (const int rc = bsattn_cache_append_workspace(cache, B, N, &need); rc != BSATTN_OK) return rc;
  if (sequences == nullptr && B > cache->sequences) return BSATTN_ERR_SHAPE;
  CacheAppend a = {};
  if (N > 0) {
    if (const int rc = check_rows(k, k_strides, 2); rc != BSATTN_OK) return rc;
    if (const int rc = check_rows(v, v_strides, 2); rc != BSATTN_OK) return rc;
    for (int i = 0; i < 3; ++i) { a.ks[i] = k_strides[i]; a.vs[i] = v_strides[i]; }
  }
  if (const int rc = check_workspace(workspace, workspace_bytes, need); rc != BSATTN_OK) return rc;
  a.k = k; a.v = v;
  a.sequences = sequences; a.at = at; a.counts = counts;
  a.B = B; a.N = N;
  return launch_cache_append(*cache, a, workspace, (hipStream_t)stream);
}

int bsattn_cache_read(const bsattn_cache* cache, void* k, void* v, const int64_t* k_strides, const int64_t* v_strides,
                      const int32_t* sequences, const int32_t* start, int B, int N, void* stream) {
  if (const int rc = check_cache(cache); rc != BSATTN_OK) return rc;
  if (B <= 0 || N <= 0 || (sequences == nullptr && B > cache->sequences)) return BSATTN_ERR_SHAPE;
  if ((int64_t)N * (cache->head_dim / 8) > 0x7fffffffLL) return BSATTN_ERR_RANGE;
  if (const int rc = check_rows(k, k_strides, 2); rc != BSATTN_OK) return rc;
  if (const int rc = check_rows(v, v_strides, 2); rc != BSATTN_OK) return rc;
  return launch_cache_read(*cache, k, v, k_strides, v_strides, sequences, start, B, N, (hipStream_t)stream);
}

int bsattn_cache_attn_workspace(const bsattn_cache* cache, int B, int H, int N, size_t* bytes) {
  if (const int rc = check_cache(cache); rc != BSATTN_OK) return rc;
  if (bytes == nullptr) return BSATTN_ERR_NULL;
  if (B <= 0 || H <= 0 || N <= 0 || H % cache->heads != 0) return BSATTN_ERR_SHAPE;
  // rows of a tile are told apart with products of 32 bits
  const int64_t group = H / cache->heads;
  if (N * group > 0x3fffffffLL || N * group > 0xffffffffLL / group || (int64_t)B * H * N > 0x7fffffffLL || N * group / 16 + 1 > 0xffffffffLL / B / B) return BSATTN_ERR_RANGE;
  *bytes = cache_attn_workspace_bytes(*cache, B, H, N);
  return BSATTN_OK;
}

int bsattn_cache_attn(const bsattn_cache* cache, const void* q, void* o, float* lse, const uint8_t* mask, const int64_t* mask_strides,
                      int Bm, int Hm, int Nm, const int32_t* sequences, const int32_t* counts, int B, int H, int N, int out_dtype,
                      float sm_scale, const int64_t* q_strides, const int64_t* o_strides, void* workspace, size_t workspace_bytes,
                      void* stream) {
  size_t need = 0;
  if (const int rc = bsattn_cache_attn_workspace(cache, B, H, N, &need); rc != BSATTN_OK) return rc;
  if (sequences == nullptr && B > cache->sequences) return BSATTN_ERR_SHAPE;
  if (out_dtype != cache->dtype && out_dtype != BSATTN_F32) return BSATTN_ERR_DTYPE;
  if (const int rc = check_rows(q, q_strides, 2); rc != BSATTN_OK) return rc;
  if (const int rc = check_rows(o, o_strides, out_dtype == BSATTN_F32 ? 4 : 2); rc != BSATTN_OK) return rc;
  CacheAttn a = {};
  if (mask != nullptr) {
    if (mask_strides == nullptr) return BSATTN_ERR_NULL;
    if ((Bm != 1 && Bm != B) || (Hm != 1 && Hm != cache->heads && Hm != H) || (Nm != 1 && Nm != pages_of(N))) return BSATTN_ERR_SHAPE;
    a.mask = mask;
    a.mask_heads = Hm == 1 ? 0 : (Hm == cache->heads ? 1 : 2);
    a.ms[0] = Bm == 1 ? 0 : mask_strides[0];
    a.ms[1] = Hm == 1 ? 0 : mask_strides[1];
    a.ms[2] = Nm == 1 ? 0 : mask_strides[2];
    a.ms[3] = mask_strides[3];
  }
  if (const int rc = check_workspace(workspace, workspace_bytes, need); rc != BSATTN_OK) return rc;
  a.q = q; a.o = o; a.lse = lse;
  a.sequences = sequences; a.counts = counts;
  a.B = B; a.H = H; a.N = N;
  a.out_f32 = out_dtype == BSATTN_F32;
  a.sm_scale = sm_scale;
  for (int i = 0; i < 3; ++i) { a.qs[i] = q_strides[i]; a.os[i] = o_strides[i]; }
  return launch_cache_attn(*cache, a, workspace, (hipStream_t)stream);
}

int bsattn_cache_fork(const bsattn_cache* cache, const int32_t* parents, const int32_t* children, int n, void* stream) {
  if (const int rc = check_cache(cache); rc != BSATTN_OK) return rc;
  if (parents == nullptr || children == nullptr) return BSATTN_ERR_NULL;
  if (n <= 0) return BSATTN_ERR_SHAPE;
  if (n > cache->sequences) return BSATTN_ERR_RANGE;
  return launch_cache_fork(*cache, parents, children, n, (hipStream_t)stream);
}

int bsattn_cache_free(const bsattn_cache* cache, const int32_t* sequences, const int32_t* keep, int n, void* stream) {
  if (const int rc = check_cache(cache); rc != BSATTN_OK) return rc;
  if (n <= 0) return BSATTN_ERR_SHAPE;
  if (n > cache->sequences) return BSATTN_ERR_RANGE;
  return launch_cache_free(*cache, sequences, keep, n, (hipStream_t)stream);
}

int bsattn_cache_compact_workspace(const bsattn_cache* cache, size_t* bytes) {
  if (const int rc = check_cache(cache); rc != BSATTN_OK) return rc;
  if (bytes == nullptr) return BSATTN_ERR_NULL;
  *bytes = cache_compact_workspace_bytes(*cache);
  return BSATTN_OK;
}

int bsattn_cache_compact(const bsattn_cache* cache, void* workspace, size_t workspace_bytes, void* stream) {
  size_t need = 0;
  if (const int rc = bsattn_cache_compact_workspace(cache, &need); rc != BSATTN_OK) return rc;
  if (const int rc = check_workspace(workspace, workspace_bytes, need); rc != BSATTN_OK) return rc;
  return launch_cache_compact(*cache, workspace, (hipStream_t)stream);
}

}  // extern "C"
