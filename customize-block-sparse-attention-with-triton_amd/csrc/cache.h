// A KV cache held in 4 bits, in pages of 64 tokens (bsattn_cache of the C ABI): what its kernels share.
//
// A page of a head holds, for keys and for values, 64 rows of D / 2 bytes (two values a byte, the lower four bits first) and D / 32 x 64
// scale bytes.  A value is (-1)^sign * {0, .5, 1, 1.5, 2, 3, 4, 6}[code] * 2^(byte - 127); 32 values of a token share a byte.  The scale
// of token t lies at byte (t % 4) * 16 + (t / 4 % 4) * 4 + t / 16 of its 64: the order in which the lanes of cache_attn_kernel take them,
// one 4-byte load of a lane for its keys and one 16-byte load for its values.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "bsattn.h"

namespace bsattn {

constexpr int PAGE = BSATTN_PAGE;
constexpr int CACHE_ROWS_MAX = BSATTN_CACHE_ROWS_MAX;
constexpr int NOT_FINITE = 255;                                    // scale byte of values that are not a number
__host__ __device__ constexpr int scale_at(int t) { return (t & 3) * 16 + (t >> 2 & 3) * 4 + (t >> 4); }
// Largest scale byte that is written: 6 times the scale is finite in the type of the cache.
template <bool BF16> __host__ __device__ constexpr int scale_cap() { return BF16 ? 252 : 140; }
__host__ __device__ constexpr int page_codes(int D) { return PAGE * D / 2; }          // bytes of a head's page
__host__ __device__ constexpr int page_scales(int D) { return PAGE * (D / 32); }
__host__ __device__ inline int pages_of(int tokens) { return (tokens + PAGE - 1) / PAGE; }

// Words of bsattn_cache.status
enum { STATUS_ROW = BSATTN_CACHE_BAD_ROW, STATUS_FULL = BSATTN_CACHE_FULL, STATUS_PAGE = BSATTN_CACHE_BAD_PAGE };
__device__ __forceinline__ void report(int32_t* status, int what) {
  if (status != nullptr) __hip_atomic_store(status + what, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
}

// Row of a call -> sequence of the cache (-1: there is none of that number)
__device__ __forceinline__ int sequence_of(const int32_t* sequences, int b, int count) {
  const int s = sequences != nullptr ? sequences[b] : b;
  return s >= 0 && s < count ? s : -1;
}
// Tokens of a sequence, at most what its row of the page table has room for (whatever stands in memory)
__device__ __forceinline__ int length_of(const bsattn_cache& c, int s) {
  const int n = c.lengths[s];
  const int64_t most = (int64_t)c.max_pages * PAGE;
  return n < 0 ? 0 : (n > most ? (int)most : n);
}
// Where a head's page begins, in heads' pages
__device__ __forceinline__ int64_t page_of_head(const bsattn_cache& c, int page, int h) { return (int64_t)page * c.heads + h; }

// Sum over the lanes up to this one
__device__ __forceinline__ int wave_upto(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);       // lanes 1, 2, 4, 8 further down in a row of 16
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);       // a row's last lane to the next row
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);       // lane 31 to the upper rows
  return x;
}

// The largest of the wavefront's, none of them negative
__device__ __forceinline__ int wave_most(int x) {
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));
  return __builtin_amdgcn_readlane(x, 63);
}

struct CacheAttn {
  const void* q; void* o; float* lse;
  const uint8_t* mask; int64_t ms[4];                // strides of the mask's batch, heads, blocks of 64 queries, pages (0: one for all)
  int mask_heads;                                    // 0: one for all heads, 1: one per head of the cache, 2: one per head of q
  const int32_t *sequences, *counts;
  int B, H, N, out_f32;
  float sm_scale;
  int64_t qs[3], os[3];
};
size_t cache_attn_workspace_bytes(const bsattn_cache& c, int B, int H, int N);
int launch_cache_attn(const bsattn_cache& c, const CacheAttn& a, void* ws, hipStream_t st);

struct CacheAppend {
  const void *k, *v;
  int64_t ks[3], vs[3];
  const int32_t *sequences, *at, *counts;
  int B, N;
};
size_t cache_append_workspace_bytes(int B, int N);
int launch_cache_append(const bsattn_cache& c, const CacheAppend& a, void* ws, hipStream_t st);
int launch_cache_read(const bsattn_cache& c, void* k, void* v, const int64_t* ks, const int64_t* vs, const int32_t* sequences,
                      const int32_t* start, int B, int N, hipStream_t st);
int launch_cache_fork(const bsattn_cache& c, const int32_t* parents, const int32_t* children, int n, hipStream_t st);
int launch_cache_free(const bsattn_cache& c, const int32_t* sequences, const int32_t* keep, int n, hipStream_t st);
size_t cache_compact_workspace_bytes(const bsattn_cache& c);
int launch_cache_compact(const bsattn_cache& c, void* ws, hipStream_t st);

}  // namespace bsattn
