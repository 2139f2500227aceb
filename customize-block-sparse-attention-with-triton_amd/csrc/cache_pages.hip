// What a KV cache in pages needs around its attention: appending (into 4 bits), reading back, forking, freeing, compacting.
//
// Which page is whose is decided by one workgroup where an order matters (append: free pages go by number, in the order of rows and
// tokens; compact: holes to movers), on the device, so that a captured step works on as the sequences grow; the data moves in a second
// launch over the whole GPU.  No result depends on the pace of anything: the counters are sums, and what free pages there are is read
// from the numbers of holders, not from a list.
#include <hip/hip_runtime.h>
#include <algorithm>
#include "common.h"
#include "kernel_util.h"
#include "cache.h"

namespace bsattn {

constexpr int PLAN = 1024;            // threads of a workgroup that decides, at most

// All T threads have come here, and what they wrote into LDS is there.  (One wavefront's accesses to LDS keep their order, and its loads from
// memory go on.)
template <int T>
__device__ __forceinline__ void meet() {
  if constexpr (T == 64) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  } else {
    __syncthreads();
  }
}

// Exclusive sum over the workgroup's T threads; total: of all.  scratch: T / 64 words of LDS.
template <int T>
__device__ __forceinline__ int block_scan(int x, int* scratch, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, upto = wave_upto(x);
  if constexpr (T == 64) {
    total = __builtin_amdgcn_readlane(upto, 63);
    return upto - x;
  }
  __syncthreads();                    // (the scratch of the scan before has been read)
  if (lane == 63) scratch[wave] = upto;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < T / 64; ++w) {
    const int z = scratch[w];
    before += w < wave ? z : 0;
    total += z;
  }
  return before + upto - x;
}

// A page loses a holder; whether it was the last one.  A page that nobody holds stays as it is, which is reported (a subtraction that finds no
// holder left is taken back: until then there is none to be had either, so that as many succeed as there were holders).
__device__ __forceinline__ bool last_leaves(const bsattn_cache& c, int page) {
  const int holders = atomicSub(&c.refs[page], 1);
  if (holders > 0) return holders == 1;
  atomicAdd(&c.refs[page], 1);
  report(c.status, STATUS_PAGE);
  return false;
}

// An entry of the page table gives its page up
__device__ __forceinline__ void give_up(const bsattn_cache& c, int32_t* entry) {
  const int page = *entry;
  *entry = -1;
  if (page < 0 || page >= c.pages) report(c.status, STATUS_PAGE);
  else if (last_leaves(c, page)) atomicMin(c.free_from, page);
}

// ---- append ----
struct AppendPlan {                   // what the deciding workgroup leaves for the launch that writes
  // [B]: sequence and tokens to write, as the call's numbers had them before it changed anything (they may be the cache's own lengths);
  // position of the first token (-1: nothing to write); page whose first tokens are copied or -1
  int32_t *sequence, *count, *begin, *source;
  int32_t *give_from, *give_to;       // [B]: places in the sequence's row of the table whose pages are given up
  int32_t *entry, *fresh;             // pages written to: held page + 1 | TAKE; free pages taken
};
constexpr unsigned TAKE = 0x80000000u;

// Pages that an append of B rows of N tokens may write to
static int64_t append_pages(int B, int N) { return (int64_t)B * (N / PAGE + 2); }

// T threads: as many as the call has rows, at least, and half the pages that it may write to, up to 1024 (one wavefront, which needs no barriers,
// for the steps of up to 64 sequences: 4.0 us where 1024 threads took 9.4).  All of its time is loads that wait for each other (row, length, table,
// holders): the first free pages are looked for beside them, and what it notes for itself stays in LDS where there is room for it.
template <int T>
__global__ __launch_bounds__(T) void append_plan_kernel(const bsattn_cache c, const CacheAppend a, const AppendPlan plan) {
  __shared__ int scratch[T / 64];
  __shared__ __align__(16) int seq[T];
  constexpr int OWNERS = 4096;
  __shared__ short owner[OWNERS];
  __shared__ int clash;
  __shared__ int first[T], off[T + 1], taken[T], bad_row[T];
  __shared__ int lowest;
  constexpr bool NOTES = T < PLAN;     // at most 2 T pages to write to (launch_cache_append)
  __shared__ int lds_entry[NOTES ? 2 * T : 1], lds_fresh[NOTES ? 2 * T : 1];
  int* const entry = NOTES ? lds_entry : plan.entry;
  int* const fresh = NOTES ? lds_fresh : plan.fresh;
  const int b = threadIdx.x;
  // how many hold the pages from the first one that may be free on, 4 VECS a thread (the last vector ends with the last page)
  constexpr int VECS = T == 64 ? 4 : 2, EACH = 4 * VECS;
  typedef int int4v __attribute__((ext_vector_type(4), aligned(4)));
  const int from = min(max(0, *c.free_from), c.pages);
  int4v holders[VECS];
  auto vec_of = [&](int p0, int x) { return p0 + EACH * (int)threadIdx.x + 4 * x; };
  auto look = [&](int p0) {
    if (c.pages >= 4) {
#pragma unroll
      for (int x = 0; x < VECS; ++x) holders[x] = *reinterpret_cast<const int4v*>(c.refs + min(vec_of(p0, x), c.pages - 4));
    } else {
#pragma unroll
      for (int x = 0; x < VECS; ++x) holders[x] = int4v{c.refs[0], c.pages > 1 ? c.refs[1] : 1, c.pages > 2 ? c.refs[2] : 1, 1};
    }
  };
  int at = 0, count = 0, old = 0, s = -1, last = 0, held = 0, entries = 0;
  if (b < a.B) {
    s = sequence_of(a.sequences, b, c.sequences);
    count = a.counts != nullptr ? a.counts[b] : a.N;
    if (s >= 0) old = length_of(c, s);
    at = a.at != nullptr ? a.at[b] : old;
  }
  look(from);
  seq[b] = s;
  if (s >= 0) owner[s % (unsigned)OWNERS] = (short)b;
  taken[b] = 0; bad_row[b] = 0;
  if (b == 0) clash = 0;
  meet<T>();
  // a row finds another one's number where it has put its own: a sequence named twice, or numbers that share the place
  if (s >= 0 && owner[s % (unsigned)OWNERS] != b) clash = 1;
  meet<T>();
  bool refused = false;
  if (b < a.B) {
    refused = s < 0 || count < 0 || count > a.N || at < 0 || at > old || (int64_t)at + count > (int64_t)c.max_pages * PAGE;
    if (clash != 0)
      for (int x = 0; x < a.B; x += 4) {              // (T is a multiple of 4)
        const uintx4 y = *reinterpret_cast<const uintx4*>(seq + x);
#pragma unroll
        for (int i = 0; i < 4; ++i) refused |= x + i < b && (int)y[i] == s;
      }
    if (refused) report(c.status, STATUS_ROW);
    else {
      last = pages_of(at + count); held = pages_of(old);
      entries = count > 0 ? last - at / PAGE : 0;
    }
  }
  first[b] = at / PAGE;
  int total_entries;
  off[b] = block_scan<T>(refused ? 0 : entries, scratch, total_entries);
  if (b == T - 1) off[T] = total_entries;
  meet<T>();
  // row of an entry: the last one that begins at or in front of it (rows without entries begin where the next one does)
  auto row_of = [&](int e) {
    int lo = 0, hi = T;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (off[mid] <= e) lo = mid; else hi = mid;
    }
    return lo;
  };
  // what each row needs is kept in its thread's registers: others ask for it through LDS
  __shared__ int r_at[T], r_held[T];
  r_at[b] = at; r_held[b] = held;
  meet<T>();
  // 1. the pages that the rows write to, and which of them need another
  for (int e = threadIdx.x; e < total_entries; e += T) {
    const int r = row_of(e), j = first[r] + e - off[r];
    int page = -1;
    if (j < r_held[r]) {
      page = c.page_table[(int64_t)seq[r] * c.max_pages + j];
      if (page < 0 || page >= c.pages) { bad_row[r] = 1; page = -1; }
    }
    const bool take = page < 0 || c.refs[page] > 1;
    if (take) atomicAdd(&taken[r], 1);
    entry[e] = (int)((unsigned)(page + 1) | (take ? TAKE : 0u));
  }
  meet<T>();
  if (bad_row[b]) {
    if (!refused) report(c.status, STATUS_PAGE);
    refused = true;
    taken[b] = 0;
  }
  int needed;
  const int rank = block_scan<T>(taken[b], scratch, needed);
  // 2. free pages, from the lowest number on; from page 0 on where there are too few (free_from is a note that may be too high, say of a handle
  // that has not seen what another one freed: no row is refused for it)
  int found = 0, start = from;
  for (bool again = false;; again = true) {
    for (int p0 = start; p0 < c.pages && found < needed; p0 += EACH * T) {
      if (again || p0 > from) look(p0);
      unsigned free = 0;
#pragma unroll
      for (int x = 0; x < VECS; ++x) {
        const int at = vec_of(p0, x);
        const unsigned four = (holders[x][0] <= 0 ? 1 : 0) | (holders[x][1] <= 0 ? 2 : 0) | (holders[x][2] <= 0 ? 4 : 0) | (holders[x][3] <= 0 ? 8 : 0);
        free |= (four >> min(at - min(at, max(0, c.pages - 4)), 4)) << 4 * x;
      }
      int here;
      int at_rank = found + block_scan<T>(__popc(free), scratch, here);
      for (; free != 0 && at_rank < needed; free &= free - 1) fresh[at_rank++] = vec_of(p0, 0) + __builtin_ctz(free);
      found += here;
    }
    if (found >= needed || start == 0) break;
    found = 0; start = 0;
  }
  meet<T>();
  if (!refused && taken[b] > 0 && rank + taken[b] > found) {
    report(c.status, STATUS_FULL);
    refused = true;
  }
  __shared__ int go[T], source[T];
  go[b] = b < a.B && !refused;
  source[b] = -1;
  int granted;
  (void)block_scan<T>(go[b] ? taken[b] : 0, scratch, granted);
  if (threadIdx.x == 0) {
    // pages below the first free one stay used: all free ones in front of the last that is taken are taken
    lowest = granted > 0 ? fresh[granted - 1] + 1 : start;
  }
  meet<T>();
  // 3. the tables
  int done = 0;
  for (int e0 = 0; e0 < total_entries; e0 += T) {
    const int e = e0 + threadIdx.x;
    int r = -1, page = -1, j = 0;
    bool take = false;
    if (e < total_entries) {
      r = row_of(e);
      j = first[r] + e - off[r];
      const unsigned x = (unsigned)entry[e];
      page = (int)(x & ~TAKE) - 1;
      take = (x & TAKE) != 0 && !bad_row[r];
    }
    int here;
    const int k = done + block_scan<T>(take, scratch, here);
    done += here;
    if (r >= 0 && go[r]) {
      if (take) {
        const int taken_page = fresh[k];
        c.page_table[(int64_t)seq[r] * c.max_pages + j] = taken_page;
        c.refs[taken_page] = 1;
        if (page >= 0 && j == first[r] && r_at[r] % PAGE != 0) source[r] = page;
        if (page >= 0 && last_leaves(c, page)) atomicMin(&lowest, page);
      }
    }
  }
  meet<T>();
  if (b < a.B) {
    plan.sequence[b] = s;
    plan.count[b] = count;
    plan.begin[b] = go[b] && count > 0 ? at : -1;
    plan.source[b] = source[b];
    plan.give_from[b] = go[b] ? last : 0;
    plan.give_to[b] = go[b] ? held : 0;
    if (go[b]) c.lengths[s] = at + count;
  }
  if (threadIdx.x == 0) *c.free_from = lowest;
}

// Eight values of a lane and their scale, shared by four lanes
template <bool BF16>
__device__ __forceinline__ unsigned quantise8(uintx4 x, int& byte) {
  float v[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (BF16) {
      v[2 * i] = __builtin_bit_cast(float, x[i] << 16);
      v[2 * i + 1] = __builtin_bit_cast(float, x[i] & 0xffff0000u);
    } else {
      const unsigned pair = x[i];                      // (a bit cast of a vector's element takes the vector's first one)
      const half2v h = __builtin_bit_cast(half2v, pair);
      v[2 * i] = (float)h[0]; v[2 * i + 1] = (float)h[1];
    }
  }
  // the bits of magnitudes are in the order of the magnitudes, infinity and what is not a number behind all others
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __builtin_bit_cast(unsigned, v[i]) & 0x7fffffffu);
  top = max(top, (unsigned)__shfl_xor((int)top, 1));
  top = max(top, (unsigned)__shfl_xor((int)top, 2));
  if (top >= 0x7f800000u) { byte = NOT_FINITE; return 0u; }
  byte = (int)(top >> 23) - 2 + ((top & 0x7fffffu) >= 0x600000u ? 1 : 0);
  byte = min(max(byte, 0), scale_cap<BF16>());
  // (the instruction divides by the scale exactly, rounds to the nearest, of two the even one, and stops at 6)
  const float scale = __builtin_bit_cast(float, (unsigned)byte << 23);
  unsigned w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], scale, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], scale, 3);
  return w;
}

// What a thread has under way: the data of a page are three loads behind each other (sequence, table, page), 3 us that one 16-byte piece
// a thread left half of the bandwidth unused for (8 000 tokens of four prompts read back: 40 us, 1 050 MB 397).
constexpr int AT_ONCE = 4;

// Grid: (rows x heads x stretches of a row's tokens, keys and values).  A lane takes 8 values: 16 bytes in, 4 out.
template <int D, bool BF16>
__global__ __launch_bounds__(256) void append_kernel(const bsattn_cache c, const CacheAppend a, const AppendPlan plan, unsigned stretches) {
  constexpr int PER = D / 8;
  const unsigned bh = blockIdx.x / stretches, stretch = blockIdx.x % stretches;
  const int b = bh / (unsigned)c.heads, h = bh % (unsigned)c.heads;
  const int begin = plan.begin[b];
  const int s = plan.sequence[b], count = plan.count[b];
  const bool values = blockIdx.y != 0;
  if (stretch == 0 && h == 0 && !values) {
    // pages behind the new end
    const int to = plan.give_to[b];
    for (int j = plan.give_from[b] + threadIdx.x; j < to; j += blockDim.x) give_up(c, c.page_table + (int64_t)s * c.max_pages + j);
  }
  if (begin < 0) return;
  const int32_t* table = c.page_table + (int64_t)s * c.max_pages;
  uint8_t* const codes = values ? c.v_codes : c.k_codes;
  uint8_t* const scales = values ? c.v_scales : c.k_scales;
  if (stretch == 0) {
    const int source = plan.source[b], tokens = begin % PAGE;
    if (source >= 0) {
      // the tokens in front of the first new one come along from the page that others keep
      const int64_t from = page_of_head(c, source, h), to = page_of_head(c, table[begin / PAGE], h);
      for (int i = threadIdx.x; i < tokens * (D / 32); i += blockDim.x) {
        *reinterpret_cast<uintx4*>(codes + to * page_codes(D) + 16 * i) = *reinterpret_cast<const uintx4*>(codes + from * page_codes(D) + 16 * i);
        const int at = (i % (D / 32)) * PAGE + scale_at(i / (D / 32));
        scales[to * page_scales(D) + at] = scales[from * page_scales(D) + at];
      }
    }
  }
  const unsigned short* x = (const unsigned short*)(values ? a.v : a.k);
  const int64_t* xs = values ? a.vs : a.ks;
  x += b * xs[0] + h * xs[1];
  uintx4 in[AT_ONCE];
  int pages[AT_ONCE];
#pragma unroll
  for (int y = 0; y < AT_ONCE; ++y) {
    const unsigned i = (stretch * AT_ONCE + y) * blockDim.x + threadIdx.x;
    const int token = min((int)(i / PER), count - 1), d = (int)(i % PER);
    in[y] = *reinterpret_cast<const uintx4*>(x + token * xs[2] + 8 * d);
    pages[y] = table[(begin + token) / PAGE];
  }
#pragma unroll
  for (int y = 0; y < AT_ONCE; ++y) {
    const unsigned i = (stretch * AT_ONCE + y) * blockDim.x + threadIdx.x;
    const int token = (int)(i / PER), d = (int)(i % PER);
    if (token >= count) break;                         // (whole groups of four lanes: PER is a multiple of 4)
    int byte;
    const unsigned w = quantise8<BF16>(in[y], byte);
    const int slot = (begin + token) % PAGE;
    const int64_t page = page_of_head(c, pages[y], h);
    *reinterpret_cast<unsigned*>(codes + page * page_codes(D) + slot * (D / 2) + 4 * d) = w;
    if ((d & 3) == 0) scales[page * page_scales(D) + (d >> 2) * PAGE + scale_at(slot)] = (uint8_t)byte;
  }
}

// ---- read ----
template <bool BF16>
__device__ __forceinline__ uintx4 values8(unsigned w, float scale) {
  if constexpr (BF16)
    return uintx4{__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0)),
                  __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1)),
                  __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2)),
                  __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3))};
  else
    return uintx4{__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 0)),
                  __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 1)),
                  __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 2)),
                  __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 3))};
}
struct CacheRead {
  void *k, *v;
  int64_t ks[3], vs[3];
  const int32_t *sequences, *start;
  int B, N;
};
template <int D, bool BF16>
__global__ __launch_bounds__(256) void read_kernel(const bsattn_cache c, const CacheRead a, unsigned stretches) {
  constexpr int PER = D / 8;
  const unsigned bh = blockIdx.x / stretches, stretch = blockIdx.x % stretches;
  const int b = bh / (unsigned)c.heads, h = bh % (unsigned)c.heads;
  const bool values = blockIdx.y != 0;
  const int s = sequence_of(a.sequences, b, c.sequences), length = s >= 0 ? length_of(c, s) : 0;
  if (s < 0) report(c.status, STATUS_ROW);
  const int64_t start = a.start != nullptr ? a.start[b] : 0;
  const uint8_t* const codes = values ? c.v_codes : c.k_codes;
  const uint8_t* const scales = values ? c.v_scales : c.k_scales;
  int pages[AT_ONCE];
#pragma unroll
  for (int y = 0; y < AT_ONCE; ++y) {
    const int64_t at = start + (int)(((stretch * AT_ONCE + y) * blockDim.x + threadIdx.x) / PER);
    pages[y] = -1;
    if (at >= 0 && at < length) {
      pages[y] = c.page_table[(int64_t)s * c.max_pages + at / PAGE];
      if (pages[y] < 0 || pages[y] >= c.pages) { report(c.status, STATUS_PAGE); pages[y] = -1; }
    }
  }
  unsigned w[AT_ONCE], byte[AT_ONCE];
#pragma unroll
  for (int y = 0; y < AT_ONCE; ++y) {
    const unsigned i = (stretch * AT_ONCE + y) * blockDim.x + threadIdx.x;
    const int slot = (int)((start + i / PER) % PAGE), d = (int)(i % PER);
    w[y] = byte[y] = 0;
    if (pages[y] >= 0) {
      const int64_t head = page_of_head(c, pages[y], h);
      w[y] = *reinterpret_cast<const unsigned*>(codes + head * page_codes(D) + slot * (D / 2) + 4 * d);
      byte[y] = scales[head * page_scales(D) + (d >> 2) * PAGE + scale_at(slot)];
    }
  }
  unsigned short* x = (unsigned short*)(values ? a.v : a.k);
  const int64_t* xs = values ? a.vs : a.ks;
  x += b * xs[0] + h * xs[1];
#pragma unroll
  for (int y = 0; y < AT_ONCE; ++y) {
    const unsigned i = (stretch * AT_ONCE + y) * blockDim.x + threadIdx.x;
    const int token = (int)(i / PER), d = (int)(i % PER);
    if (token >= a.N) break;
    // (past the L2: 26 -> 24 us, 314 -> 289)
    __builtin_nontemporal_store(values8<BF16>(w[y], __builtin_bit_cast(float, byte[y] << 23)), reinterpret_cast<uintx4*>(x + token * xs[2] + 8 * d));
  }
}

// ---- fork ----
// A workgroup a pair.  Nothing that one pair reads is written by another: a parent is nobody's child, a child has one pair.
__global__ __launch_bounds__(256) void fork_kernel(const bsattn_cache c, const int32_t* parents, const int32_t* children, int n) {
  __shared__ int wrong, no_page;
  const int i = blockIdx.x, parent = sequence_of(parents, i, c.sequences), child = sequence_of(children, i, c.sequences);
  if (threadIdx.x == 0) { wrong = parent < 0 || child < 0; no_page = 0; }
  __syncthreads();
  for (int x = threadIdx.x; x < n; x += 256) {
    const int y = children[x];
    if (y == parent || (x < i && y == child)) wrong = 1;
  }
  __syncthreads();
  const bool refused = wrong != 0 || c.lengths[child] != 0;
  if (refused) {
    if (threadIdx.x == 0) report(c.status, STATUS_ROW);
    return;
  }
  const int length = length_of(c, parent), pages = pages_of(length);
  const int32_t* from = c.page_table + (int64_t)parent * c.max_pages;
  int32_t* to = c.page_table + (int64_t)child * c.max_pages;
  for (int j = threadIdx.x; j < pages; j += 256) {
    const int page = from[j];
    if (page < 0 || page >= c.pages) no_page = 1;
  }
  __syncthreads();
  if (no_page != 0) {
    if (threadIdx.x == 0) report(c.status, STATUS_PAGE);
    return;
  }
  for (int j = threadIdx.x; j < pages; j += 256) {
    const int page = from[j];
    to[j] = page;
    atomicAdd(&c.refs[page], 1);
  }
  __syncthreads();                     // (all threads have seen the child's length)
  if (threadIdx.x == 0) c.lengths[child] = length;
}

// ---- free ----
__global__ __launch_bounds__(256) void free_kernel(const bsattn_cache c, const int32_t* sequences, const int32_t* keep, int n) {
  __shared__ int wrong;
  const int i = blockIdx.x, s = sequence_of(sequences, i, c.sequences), kept = keep != nullptr ? keep[i] : 0;
  if (threadIdx.x == 0) wrong = s < 0 || kept < 0;
  __syncthreads();
  if (sequences != nullptr)
    for (int x = threadIdx.x; x < i; x += 256)
      if (sequences[x] == s) wrong = 1;
  __syncthreads();
  if (wrong != 0) {
    if (threadIdx.x == 0) report(c.status, STATUS_ROW);
    return;
  }
  const int length = length_of(c, s);
  if (kept >= length) return;
  int32_t* table = c.page_table + (int64_t)s * c.max_pages;
  for (int j = pages_of(kept) + threadIdx.x; j < pages_of(length); j += 256) give_up(c, table + j);
  __syncthreads();                     // (all threads have seen the length)
  if (threadIdx.x == 0) c.lengths[s] = kept;
}

// ---- compact ----
struct CompactPlan { int32_t *count, *used, *holes, *movers, *to; };      // moves; pages in use; targets and sources; new number of a page from `used` on

// A page is in use or free, whatever number stands there: so there are as many free ones below `used` as used ones behind, a target for each move.
__device__ __forceinline__ bool in_use(int refs) { return refs > 0; }

__global__ __launch_bounds__(PLAN) void compact_plan_kernel(const bsattn_cache c, const CompactPlan plan) {
  __shared__ int scratch[PLAN / 64];
  int used = 0, mine = 0;
  for (int p = threadIdx.x; p < c.pages; p += PLAN) mine += in_use(c.refs[p]);
  (void)block_scan<PLAN>(mine, scratch, used);
  int holes = 0, movers = 0;
  for (int p0 = 0; p0 < c.pages; p0 += 4 * PLAN) {
    int refs[4], x_holes = 0, x_movers = 0;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int p = p0 + 4 * (int)threadIdx.x + x;
      refs[x] = p < c.pages ? c.refs[p] : 0;
      x_holes += p < used && !in_use(refs[x]);              // (used <= pages)
      x_movers += p >= used && in_use(refs[x]);
    }
    int n_holes, n_movers;
    int at_hole = holes + block_scan<PLAN>(x_holes, scratch, n_holes), at_mover = movers + block_scan<PLAN>(x_movers, scratch, n_movers);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int p = p0 + 4 * (int)threadIdx.x + x;
      if (p < used && !in_use(refs[x])) plan.holes[at_hole++] = p;
      if (p >= used && in_use(refs[x])) plan.movers[at_mover++] = p;
      if (p >= used && p < c.pages && !in_use(refs[x])) plan.to[p] = p;
    }
    holes += n_holes; movers += n_movers;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < movers; i += PLAN) {
    const int from = plan.movers[i], to = plan.holes[i];
    plan.to[from] = to;
    c.refs[to] = c.refs[from];
    c.refs[from] = 0;
  }
  if (threadIdx.x == 0) { *plan.count = movers; *plan.used = used; *c.free_from = used; }
}

// Moves the pages, and renames them in the tables.  Grid-stride over stretches of a page's bytes (keys, values, their scales).
constexpr int MOVE_PIECES = 4;
__global__ __launch_bounds__(256) void compact_move_kernel(const bsattn_cache c, const CompactPlan plan) {
  const int moves = *plan.count, used = *plan.used;
  const unsigned codes = (unsigned)c.heads * page_codes(c.head_dim) / 16, scales = (unsigned)c.heads * page_scales(c.head_dim) / 16;
  const unsigned pieces = 2 * (codes + scales), stretches = (pieces + 256 * MOVE_PIECES - 1) / (256 * MOVE_PIECES);
  for (int64_t item = blockIdx.x; item < (int64_t)moves * stretches; item += gridDim.x) {
    const int m = (int)(item / stretches);
    const unsigned first = (unsigned)(item - (int64_t)m * stretches) * 256 * MOVE_PIECES + threadIdx.x;
    const int64_t from = plan.movers[m], to = plan.holes[m];
    uintx4 x[MOVE_PIECES];
    uintx4* target[MOVE_PIECES];
#pragma unroll
    for (int y = 0; y < MOVE_PIECES; ++y) {
      unsigned i = first + 256 * y;
      target[y] = nullptr;
      if (i >= pieces) continue;
      const bool values = i >= codes + scales;
      if (values) i -= codes + scales;
      const bool is_scale = i >= codes;
      if (is_scale) i -= codes;
      uint8_t* all = is_scale ? (values ? c.v_scales : c.k_scales) : (values ? c.v_codes : c.k_codes);
      const int64_t page = 16 * (int64_t)(is_scale ? scales : codes);
      target[y] = reinterpret_cast<uintx4*>(all + to * page) + i;
      x[y] = reinterpret_cast<const uintx4*>(all + from * page)[i];
    }
#pragma unroll
    for (int y = 0; y < MOVE_PIECES; ++y)
      if (target[y] != nullptr) *target[y] = x[y];
  }
  if (moves == 0) return;
  const int64_t entries = (int64_t)c.sequences * c.max_pages;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < entries; i += (int64_t)gridDim.x * 256) {
    const int page = c.page_table[i];
    if (page >= used && page < c.pages) c.page_table[i] = plan.to[page];
  }
}

// ---- host ----
static size_t rounded(size_t n) { return (n + 255) / 256 * 256; }

size_t cache_append_workspace_bytes(int B, int N) {
  return 6 * rounded((size_t)B * 4) + 2 * rounded((size_t)append_pages(B, N) * 4);
}

int launch_cache_append(const bsattn_cache& c, const CacheAppend& a, void* ws, hipStream_t st) {
  AppendPlan plan;
  char* at = (char*)ws;
  plan.sequence = (int32_t*)at; at += rounded((size_t)a.B * 4);
  plan.count = (int32_t*)at; at += rounded((size_t)a.B * 4);
  plan.begin = (int32_t*)at; at += rounded((size_t)a.B * 4);
  plan.source = (int32_t*)at; at += rounded((size_t)a.B * 4);
  plan.give_from = (int32_t*)at; at += rounded((size_t)a.B * 4);
  plan.give_to = (int32_t*)at; at += rounded((size_t)a.B * 4);
  plan.entry = (int32_t*)at; at += rounded((size_t)append_pages(a.B, a.N) * 4);
  plan.fresh = (int32_t*)at;
  const int64_t lanes = (int64_t)a.N * (c.head_dim / 8);
  const int threads = lanes <= 64 ? 64 : 256;
  const int64_t stretches = std::max<int64_t>(1, (lanes + AT_ONCE * threads - 1) / (AT_ONCE * threads)), blocks = (int64_t)a.B * c.heads * stretches;
  if (blocks > 0x7fffffffLL) return BSATTN_ERR_RANGE;
  const int64_t take = append_pages(a.B, a.N);
  if (take <= 128 && a.B <= 64) hipLaunchKernelGGL(append_plan_kernel<64>, dim3(1), dim3(64), 0, st, c, a, plan);
  else if (take <= 512 && a.B <= 256) hipLaunchKernelGGL(append_plan_kernel<256>, dim3(1), dim3(256), 0, st, c, a, plan);
  else hipLaunchKernelGGL(append_plan_kernel<PLAN>, dim3(1), dim3(PLAN), 0, st, c, a, plan);
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)blocks, 2), dim3(threads), 0, st, c, a, plan, (unsigned)stretches); };
  const bool bf16 = c.dtype == BSATTN_BF16;
  if (c.head_dim == 64) bf16 ? go(append_kernel<64, true>) : go(append_kernel<64, false>);
  else if (c.head_dim == 128) bf16 ? go(append_kernel<128, true>) : go(append_kernel<128, false>);
  else bf16 ? go(append_kernel<256, true>) : go(append_kernel<256, false>);
  return launch_status();
}

int launch_cache_read(const bsattn_cache& c, void* k, void* v, const int64_t* ks, const int64_t* vs, const int32_t* sequences,
                      const int32_t* start, int B, int N, hipStream_t st) {
  CacheRead a = {k, v, {ks[0], ks[1], ks[2]}, {vs[0], vs[1], vs[2]}, sequences, start, B, N};
  const int64_t lanes = (int64_t)N * (c.head_dim / 8);
  const int threads = lanes <= 64 ? 64 : 256;
  const int64_t stretches = (lanes + AT_ONCE * threads - 1) / (AT_ONCE * threads), blocks = (int64_t)B * c.heads * stretches;
  if (blocks > 0x7fffffffLL) return BSATTN_ERR_RANGE;
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)blocks, 2), dim3(threads), 0, st, c, a, (unsigned)stretches); };
  const bool bf16 = c.dtype == BSATTN_BF16;
  if (c.head_dim == 64) bf16 ? go(read_kernel<64, true>) : go(read_kernel<64, false>);
  else if (c.head_dim == 128) bf16 ? go(read_kernel<128, true>) : go(read_kernel<128, false>);
  else bf16 ? go(read_kernel<256, true>) : go(read_kernel<256, false>);
  return launch_status();
}

int launch_cache_fork(const bsattn_cache& c, const int32_t* parents, const int32_t* children, int n, hipStream_t st) {
  hipLaunchKernelGGL(fork_kernel, dim3(n), dim3(256), 0, st, c, parents, children, n);
  return launch_status();
}

int launch_cache_free(const bsattn_cache& c, const int32_t* sequences, const int32_t* keep, int n, hipStream_t st) {
  hipLaunchKernelGGL(free_kernel, dim3(n), dim3(256), 0, st, c, sequences, keep, n);
  return launch_status();
}

size_t cache_compact_workspace_bytes(const bsattn_cache& c) { return 256 + 3 * rounded((size_t)c.pages * 4); }

int launch_cache_compact(const bsattn_cache& c, void* ws, hipStream_t st) {
  CompactPlan plan;
  plan.count = (int32_t*)ws; plan.used = plan.count + 1;
  plan.holes = plan.count + 64;
  plan.movers = plan.holes + rounded((size_t)c.pages * 4) / 4;
  plan.to = plan.movers + rounded((size_t)c.pages * 4) / 4;
  hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(PLAN), 0, st, c, plan);
  hipLaunchKernelGGL(compact_move_kernel, dim3(8 * compute_units()), dim3(256), 0, st, c, plan);
  return launch_status();
}

}  // namespace bsattn
