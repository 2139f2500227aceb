// Drives the argument validation of the cache's C entry points in a build whose host code carries the address and undefined-behaviour
// sanitizers: every call below must be refused before any device work, so the program needs no GPU.  Pointers that are never
// dereferenced point at a small real buffer, so that a validation path that did read them would be caught.
#include <climits>
#include <cstdint>
#include <cstdio>
#include <initializer_list>
#include "bsattn.h"

static int failures = 0;
#define EXPECT(call, want) do { const int rc_ = (call); if (rc_ != (want)) { \
  std::printf("line %d: %s returned %d, expected %d\n", __LINE__, #call, rc_, (int)(want)); ++failures; } } while (0)

int main() {
  alignas(16) static unsigned char buf[64];
  uint8_t* const B8 = buf;
  int32_t* const I = (int32_t*)buf;
  const int64_t ok[4] = {2 * 64 * 64, 64 * 64, 64, 1}, inner[4] = {2 * 64 * 64, 64 * 64, 64, 2}, odd[4] = {2 * 64 * 68, 64 * 68, 68, 1};
  const size_t big = (size_t)1 << 40;
  size_t n = 0;
  const bsattn_cache good = {B8, B8, B8, B8, I, I, I, I, nullptr, 8, 2, 64, 3, 4, BSATTN_F16};
  auto append = [&](const bsattn_cache* c, const void* k, const int64_t* ks, const int32_t* seq, int B, int N, void* ws, size_t wsb) {
    return bsattn_cache_append(c, k, buf, ks, ok, seq, nullptr, nullptr, B, N, ws, wsb, nullptr);
  };
  auto attn = [&](const bsattn_cache* c, const void* q, const uint8_t* mask, const int64_t* ms, int Bm, int Hm, int Nm, const int32_t* seq, int B, int H, int N,
                  int odt, const int64_t* qs, void* ws, size_t wsb) {
    return bsattn_cache_attn(c, q, buf, nullptr, mask, ms, Bm, Hm, Nm, seq, nullptr, B, H, N, odt, 0.1f, qs, ok, ws, wsb, nullptr);
  };
  // the cache itself
  EXPECT(append(nullptr, buf, ok, nullptr, 2, 5, buf, big), BSATTN_ERR_NULL);
  for (int i = 0; i < 8; ++i) {
    bsattn_cache c = good;
    uint8_t** const b[4] = {&c.k_codes, &c.v_codes, &c.k_scales, &c.v_scales};
    int32_t** const w[4] = {&c.page_table, &c.lengths, &c.refs, &c.free_from};
    if (i < 4) *b[i] = nullptr; else *w[i - 4] = nullptr;
    EXPECT(append(&c, buf, ok, nullptr, 2, 5, buf, big), BSATTN_ERR_NULL);
    EXPECT(attn(&c, buf, nullptr, nullptr, 1, 1, 1, nullptr, 2, 4, 5, 0, ok, buf, big), BSATTN_ERR_NULL);
    EXPECT(bsattn_cache_read(&c, buf, buf, ok, ok, nullptr, nullptr, 2, 5, nullptr), BSATTN_ERR_NULL);
    EXPECT(bsattn_cache_fork(&c, I, I, 1, nullptr), BSATTN_ERR_NULL);
    EXPECT(bsattn_cache_free(&c, nullptr, nullptr, 1, nullptr), BSATTN_ERR_NULL);
    EXPECT(bsattn_cache_compact(&c, buf, big, nullptr), BSATTN_ERR_NULL);
  }
  for (int i = 0; i < 4; ++i)
    for (int v : {0, -1, INT_MIN}) {
      bsattn_cache c = good;
      int32_t* const f[4] = {&c.pages, &c.heads, &c.sequences, &c.max_pages};
      *f[i] = v;
      EXPECT(append(&c, buf, ok, nullptr, 2, 5, buf, big), BSATTN_ERR_SHAPE);
    }
  for (int i = 0; i < 4; ++i) {
    bsattn_cache c = good;
    int32_t* const f[4] = {&c.pages, &c.heads, &c.max_pages, &c.max_pages};
    *f[i] = i == 3 ? INT_MAX / 64 : INT_MAX;
    EXPECT(attn(&c, buf, nullptr, nullptr, 1, 1, 1, nullptr, 2, 4, 5, 0, ok, buf, big), BSATTN_ERR_RANGE);
  }
  { bsattn_cache c = good; c.head_dim = 32; EXPECT(append(&c, buf, ok, nullptr, 2, 5, buf, big), BSATTN_ERR_HEAD_DIM); }
  { bsattn_cache c = good; c.dtype = BSATTN_F32; EXPECT(append(&c, buf, ok, nullptr, 2, 5, buf, big), BSATTN_ERR_DTYPE); }
  { bsattn_cache c = good; c.v_scales = buf + 4; EXPECT(append(&c, buf, ok, nullptr, 2, 5, buf, big), BSATTN_ERR_STRIDE); }
  // append
  EXPECT(append(&good, nullptr, ok, nullptr, 2, 5, buf, big), BSATTN_ERR_NULL);
  EXPECT(append(&good, buf, nullptr, nullptr, 2, 5, buf, big), BSATTN_ERR_NULL);
  EXPECT(append(&good, buf, inner, nullptr, 2, 5, buf, big), BSATTN_ERR_STRIDE);
  EXPECT(append(&good, buf, odd, nullptr, 2, 5, buf, big), BSATTN_ERR_STRIDE);
  EXPECT(append(&good, buf + 2, ok, nullptr, 2, 5, buf, big), BSATTN_ERR_STRIDE);
  EXPECT(append(&good, buf, ok, nullptr, 0, 5, buf, big), BSATTN_ERR_SHAPE);
  EXPECT(append(&good, buf, ok, nullptr, 4, 5, buf, big), BSATTN_ERR_SHAPE);
  EXPECT(append(&good, buf, ok, nullptr, 2, -1, buf, big), BSATTN_ERR_SHAPE);
  EXPECT(append(&good, buf, ok, I, 1025, 5, buf, big), BSATTN_ERR_RANGE);
  EXPECT(append(&good, buf, ok, nullptr, 2, 257, buf, big), BSATTN_ERR_RANGE);
  EXPECT(append(&good, buf, ok, nullptr, 2, INT_MAX, buf, big), BSATTN_ERR_RANGE);
  { bsattn_cache c = good; c.max_pages = 1 << 24; EXPECT(append(&c, buf, ok, nullptr, 2, 1 << 29, buf, big), BSATTN_ERR_RANGE); }
  EXPECT(append(&good, buf, ok, nullptr, 2, 5, nullptr, big), BSATTN_ERR_WORKSPACE);
  EXPECT(append(&good, buf, ok, nullptr, 2, 5, buf, 16), BSATTN_ERR_WORKSPACE);
  EXPECT(append(&good, buf, ok, nullptr, 2, 5, buf + 8, big), BSATTN_ERR_STRIDE);
  EXPECT(bsattn_cache_append_workspace(&good, 2, 5, nullptr), BSATTN_ERR_NULL);
  EXPECT(bsattn_cache_append_workspace(&good, 2, 5, &n), BSATTN_OK);
  // read
  EXPECT(bsattn_cache_read(&good, nullptr, buf, ok, ok, nullptr, nullptr, 2, 5, nullptr), BSATTN_ERR_NULL);
  EXPECT(bsattn_cache_read(&good, buf, buf, ok, inner, nullptr, nullptr, 2, 5, nullptr), BSATTN_ERR_STRIDE);
  EXPECT(bsattn_cache_read(&good, buf, buf, ok, ok, nullptr, nullptr, 4, 5, nullptr), BSATTN_ERR_SHAPE);
  EXPECT(bsattn_cache_read(&good, buf, buf, ok, ok, I, nullptr, 2, 0, nullptr), BSATTN_ERR_SHAPE);
  EXPECT(bsattn_cache_read(&good, buf, buf, ok, ok, I, nullptr, 2, INT_MAX, nullptr), BSATTN_ERR_RANGE);
  // attention
  EXPECT(attn(&good, nullptr, nullptr, nullptr, 1, 1, 1, nullptr, 2, 4, 5, 0, ok, buf, big), BSATTN_ERR_NULL);
  EXPECT(attn(&good, buf, buf, nullptr, 1, 1, 1, nullptr, 2, 4, 5, 0, ok, buf, big), BSATTN_ERR_NULL);
  EXPECT(attn(&good, buf, nullptr, nullptr, 1, 1, 1, nullptr, 2, 3, 5, 0, ok, buf, big), BSATTN_ERR_SHAPE);
  EXPECT(attn(&good, buf, nullptr, nullptr, 1, 1, 1, nullptr, 2, 4, 0, 0, ok, buf, big), BSATTN_ERR_SHAPE);
  EXPECT(attn(&good, buf, nullptr, nullptr, 1, 1, 1, nullptr, 4, 4, 5, 0, ok, buf, big), BSATTN_ERR_SHAPE);
  EXPECT(attn(&good, buf, buf, ok, 3, 1, 1, nullptr, 2, 4, 5, 0, ok, buf, big), BSATTN_ERR_SHAPE);
  EXPECT(attn(&good, buf, buf, ok, 1, 3, 1, nullptr, 2, 4, 5, 0, ok, buf, big), BSATTN_ERR_SHAPE);
  EXPECT(attn(&good, buf, buf, ok, 1, 1, 2, nullptr, 2, 4, 64, 0, ok, buf, big), BSATTN_ERR_SHAPE);
  EXPECT(attn(&good, buf, nullptr, nullptr, 1, 1, 1, nullptr, 2, 4, 5, BSATTN_BF16, ok, buf, big), BSATTN_ERR_DTYPE);
  EXPECT(attn(&good, buf, nullptr, nullptr, 1, 1, 1, nullptr, 2, 4, 5, 0, odd, buf, big), BSATTN_ERR_STRIDE);
  EXPECT(attn(&good, buf, nullptr, nullptr, 1, 1, 1, I, 2, 4, INT_MAX, 0, ok, buf, big), BSATTN_ERR_RANGE);
  EXPECT(attn(&good, buf, nullptr, nullptr, 1, 1, 1, I, INT_MAX, 4, 5, 0, ok, buf, big), BSATTN_ERR_RANGE);
  EXPECT(attn(&good, buf, nullptr, nullptr, 1, 1, 1, I, 1, INT_MAX - 1, 5, 0, ok, buf, big), BSATTN_ERR_RANGE);
  EXPECT(attn(&good, buf, nullptr, nullptr, 1, 1, 1, nullptr, 2, 4, 5, 0, ok, nullptr, big), BSATTN_ERR_WORKSPACE);
  EXPECT(attn(&good, buf, nullptr, nullptr, 1, 1, 1, nullptr, 2, 4, 5, 0, ok, buf, 16), BSATTN_ERR_WORKSPACE);
  EXPECT(bsattn_cache_attn_workspace(&good, 2, 4, 5, &n), BSATTN_OK);
  // fork, free, compact
  EXPECT(bsattn_cache_fork(&good, nullptr, I, 1, nullptr), BSATTN_ERR_NULL);
  EXPECT(bsattn_cache_fork(&good, I, I, 0, nullptr), BSATTN_ERR_SHAPE);
  EXPECT(bsattn_cache_fork(&good, I, I, 4, nullptr), BSATTN_ERR_RANGE);
  EXPECT(bsattn_cache_free(&good, I, I, -1, nullptr), BSATTN_ERR_SHAPE);
  EXPECT(bsattn_cache_free(&good, I, I, 4, nullptr), BSATTN_ERR_RANGE);
  EXPECT(bsattn_cache_compact_workspace(&good, nullptr), BSATTN_ERR_NULL);
  EXPECT(bsattn_cache_compact_workspace(&good, &n), BSATTN_OK);
  EXPECT(bsattn_cache_compact(&good, nullptr, big, nullptr), BSATTN_ERR_WORKSPACE);
  EXPECT(bsattn_cache_compact(&good, buf, 16, nullptr), BSATTN_ERR_WORKSPACE);
  EXPECT(bsattn_cache_compact(&good, buf + 4, big, nullptr), BSATTN_ERR_STRIDE);
  if (failures == 0) std::printf("ok\n");
  return failures != 0;
}
