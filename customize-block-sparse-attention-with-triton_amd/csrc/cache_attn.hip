// Attention of new tokens over a KV cache held in 4 bits: one pass over the kept pages with the running maximum and sum of a softmax.
//
// A tile is 16 QT rows (token, head) of the queries that share a head of the cache.  A wavefront takes a page at a time, keys and values
// straight from memory to registers, and both products on the matrix cores with 16-bit operands:
//   S^T = K Q^T   A = 16 tokens x 32 columns of K, converted from 4 bits with their scale (exact), B = Q^T
//   O^T = V^T P^T A = 16 columns x 32 tokens of V, B = P^T
// The lanes (n = l % 16, g = l / 16) of S^T hold query n and tokens 16 t + 4 i + g (t, i = 0..3: register i of tile t), which are the tokens
// that B of the second product takes from the same lane: P never leaves its registers.  Tokens and columns of a sum may go in any order,
// so the orders are those in which lanes read memory: of K, lane (n, g) reads for token 16 t + 4 (n % 4) + n / 4 its columns from g D / 4 on
// (D / 8 bytes in a row, 16 rows an instruction), of V for each of its 16 tokens the columns from n D / 16 on (four whole rows an
// instruction); column block s of the second product is column n D / 16 + s.  The scales lie as the lanes take them (cache.h).
//
// What bounds it: one token per sequence reads every kept page once: the cache's bytes.  Per page and wavefront (D = 128) there are 128
// conversions, 64 byte permutes for V and about 200 other vector instructions against 8.7 KB, 32 matrix instructions per 16 rows.
// Prompt pieces have 64 rows per tile: the conversions are shared by four times as many products and the matrix cores bound it.
//
// Who walks what.  The pages of a (sequence, tile) are dealt round robin to `splits` x 4 wavefronts (so that a mask's dense stretches, the
// last blocks for instance, go to all of them); splits in proportion to the pages, found on the device from the lengths: the host never
// knows them, and a captured launch follows sequences as they grow.  The four wavefronts of a workgroup meet in LDS, workgroups in the
// workspace: the last one in adds up all parts in their order (count_in in fwd_tile.h), so results do not depend on the pace.
#include <hip/hip_runtime.h>
#include <algorithm>
#include "common.h"
#include "kernel_util.h"
#include "cache.h"

namespace bsattn {

constexpr int WAVES = 4;
constexpr float LN2 = 0.6931471805599453f, LOG2E = 1.4426950408889634f;
// Numerators are 2^HEADROOM at most: in fp16, whose steps are equal below 2^-14, small ones keep their digits 15 powers of two further
// down (without it weights of 2^-16 beside one of 1 were 2^-9 off).
template <bool BF16> __device__ constexpr float HEADROOM = BF16 ? 0.f : 15.f;
constexpr float NO_MASS = -3.0e38f;           // reference exponent of a row that has seen tokens, all with scores of -inf

struct CacheAttnParams {
  bsattn_cache c;
  CacheAttn a;
  int group, rows, tiles, W, min_pages, max_splits;      // query heads per head of the cache; N * group; tiles of them; workgroups to share (0: a unit each)
  float scale; unsigned flip;                            // |sm_scale| log2 e; sign bits if sm_scale < 0
  float *part_o, *part_ml;
  unsigned long long *arrivals, epoch;
};

// Counts a part in, by one thread, once all accesses of its workgroup to it have been acknowledged; returns how many are in.  The counter
// holds (launch mark << 16 | parts); stale contents carry another mark.
__device__ __forceinline__ int count_part(unsigned long long* arrivals, unsigned long long epoch) {
  unsigned long long seen = __hip_atomic_load(arrivals, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  for (;;) {     // (ends: the counter only changes when another part is counted, at most as often as there are parts)
    const unsigned long long want = (seen >> 16) == epoch ? seen + 1 : ((epoch << 16) | 1ull);
    if (__hip_atomic_compare_exchange_strong(arrivals, &seen, want, __ATOMIC_RELAXED, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT))
      return (int)(want & 0xffffull);
  }
}

template <bool BF16>
__device__ __forceinline__ floatx4 mfma16(uintx4 a, uintx4 b, floatx4 c) {
  if constexpr (BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}

// Byte SEL of w: two values in 4 bits -> two packed 16-bit values times `scale`
template <bool BF16, int SEL>
__device__ __forceinline__ unsigned convert2(unsigned w, float scale) {
  if constexpr (BF16) return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, SEL));
  else return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, SEL));
}
template <bool BF16>
__device__ __forceinline__ uintx4 convert8(unsigned w, float scale) {
  return uintx4{convert2<BF16, 0>(w, scale), convert2<BF16, 1>(w, scale), convert2<BF16, 2>(w, scale), convert2<BF16, 3>(w, scale)};
}
// Scale byte `at` of w as a power of two (255: infinity, which the conversions take for "not a number")
__device__ __forceinline__ float scale_of(unsigned w, int at) { return __builtin_bit_cast(float, ((w >> (8 * at)) & 0xffu) << 23); }

// Over the four lanes of a query: x and the lane's of the other row of 16 in its pair of rows, then of the other pair.  (The parts of a
// swap are copied out of its result first: a bit cast of a vector's element takes the vector's first one.)
template <class F>
__device__ __forceinline__ float quad(float x, F&& f) {
  const unsigned u = __builtin_bit_cast(unsigned, x);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const unsigned a0 = a[0], a1 = a[1];
  const unsigned y = __builtin_bit_cast(unsigned, f(__builtin_bit_cast(float, a0), __builtin_bit_cast(float, a1)));
  const auto b = __builtin_amdgcn_permlane32_swap(y, y, false, false);
  const unsigned b0 = b[0], b1 = b[1];
  return f(__builtin_bit_cast(float, b0), __builtin_bit_cast(float, b1));
}
__device__ __forceinline__ float quad_max(float x) { return quad(x, [](float a, float b) { return fmaxf(a, b); }); }
__device__ __forceinline__ float quad_sum(float x) { return quad(x, [](float a, float b) { return a + b; }); }

// A lane's share of a head's page
template <int D>
struct PageRegs {
  static constexpr int KW = D / 32, VW = D >= 128 ? D / 128 : 1, KS = D == 256 ? 2 : 1;     // words of K per tile, of V per token, of K's scales
  unsigned k[4][KW], ks[KS], v[16][VW];
  uintx4 vs;
  unsigned char kept[4];                      // this page in the mask's rows of the lane's queries (where they differ)
};

template <int N> struct Words;
template <> struct Words<1> { typedef unsigned type; };
template <> struct Words<2> { typedef uintx2 type; };
template <> struct Words<4> { typedef uintx4 type; };

template <int D>
__device__ __forceinline__ void load_page(PageRegs<D>& r, const bsattn_cache& c, int64_t at, int n, int g) {
  constexpr int ROW = D / 2;
  const int krow = 4 * (n & 3) + (n >> 2);
  const uint8_t* kc = c.k_codes + at * page_codes(D) + krow * ROW + g * (D / 8);
  const uint8_t* ks = c.k_scales + at * page_scales(D) + (D == 64 ? g >> 1 : (D == 128 ? g : 2 * g)) * PAGE + n * 4;
  const uint8_t* vc = c.v_codes + at * page_codes(D) + g * ROW + n * (D / 32);
  const uint8_t* vs = c.v_scales + at * page_scales(D) + (D == 64 ? n >> 3 : (D == 128 ? n >> 2 : n >> 1)) * PAGE + g * 16;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    if constexpr (D == 256) {
      const uintx4 a = *reinterpret_cast<const uintx4*>(kc + t * 16 * ROW), b = *reinterpret_cast<const uintx4*>(kc + t * 16 * ROW + 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) { r.k[t][i] = a[i]; r.k[t][4 + i] = b[i]; }
    } else {
      const auto a = *reinterpret_cast<const typename Words<D / 32>::type*>(kc + t * 16 * ROW);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) r.k[t][i] = a[i];
    }
  }
#pragma unroll
  for (int i = 0; i < PageRegs<D>::KS; ++i) r.ks[i] = *reinterpret_cast<const unsigned*>(ks + i * PAGE);
#pragma unroll
  for (int j = 0; j < 16; ++j) {              // token 16 (j / 4) + 4 (j % 4) + g
    if constexpr (D == 64) r.v[j][0] = *reinterpret_cast<const unsigned short*>(vc + 4 * j * ROW);
    else if constexpr (D == 128) r.v[j][0] = *reinterpret_cast<const unsigned*>(vc + 4 * j * ROW);
    else {
      const uintx2 a = *reinterpret_cast<const uintx2*>(vc + 4 * j * ROW);
      r.v[j][0] = a[0]; r.v[j][1] = a[1];
    }
  }
  r.vs = *reinterpret_cast<const uintx4*>(vs);
}

// What tile `tile` of row b walks: its sequence, the position of the row's first query, and pages 0 .. pages - 1
struct Unit { int seq, first, count, pages; };
template <int ROWS>
__device__ __forceinline__ Unit unit_of(const CacheAttnParams& prm, int b, int tile) {
  Unit u = {sequence_of(prm.a.sequences, b, prm.c.sequences), 0, 0, 0};
  u.count = prm.a.counts != nullptr ? prm.a.counts[b] : prm.a.N;
  if (u.seq < 0 || u.count < 0 || u.count > prm.a.N) {
    report(prm.c.status, STATUS_ROW);
    u.seq = -1; u.count = 0;
    return u;
  }
  u.first = length_of(prm.c, u.seq) - u.count;
  const int t0 = tile * ROWS / prm.group, t1 = (min(prm.rows, (tile + 1) * ROWS) - 1) / prm.group;
  const int last = u.first + min(u.count - 1, t1);
  u.pages = t0 < u.count && last >= 0 ? last / PAGE + 1 : 0;
  return u;
}

template <int D, bool BF16, int QT>
__global__ __launch_bounds__(64 * WAVES, (D * QT >= 512 || QT == 4) ? 1 : 2) void cache_attn_kernel(const CacheAttnParams prm) {
  constexpr int ROWS = 16 * QT, PITCH = D + 4, KSTEPS = D / 32, DT = D / 16;
  extern __shared__ __align__(16) float lds[];           // [WAVES][ROWS][PITCH] parts of O | [WAVES][ROWS][2] (m, l) | [ROWS][2]
  float* const lds_ml = lds + WAVES * ROWS * PITCH;
  float* const lds_row = lds_ml + WAVES * ROWS * 2;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
  const bsattn_cache& c = prm.c;
  const int h = blockIdx.x % (unsigned)c.heads;
  const int units = prm.a.B * prm.tiles;
  int unit = blockIdx.x / (unsigned)c.heads, split = 0, splits = 1, first_wg = 0;
  // unit -> (row of the call, tile): the tiles with the most pages first
  auto row_of = [&](int u) { return u % prm.a.B; };
  auto tile_of = [&](int u) { return prm.tiles - 1 - u / prm.a.B; };
  if (prm.W > 0) {
    // the workgroups of a head, W + units of them, are given to the units in proportion to their pages (every wavefront finds out
    // by itself)
    const int w = unit;
    int64_t total = 0;
    for (int u0 = 0; u0 < units; u0 += 64) {
      int p = 0;
      if (u0 + lane < units) p = unit_of<ROWS>(prm, row_of(u0 + lane), tile_of(u0 + lane)).pages;
      for (int x = 32; x > 0; x >>= 1) p += __shfl_xor(p, x);
      total += p;
    }
    const int per = (int)max((int64_t)prm.min_pages, (total + prm.W - 1) / prm.W);
    int before = 0;
    unit = -1;
    for (int u0 = 0; u0 < units && unit < 0; u0 += 64) {
      int s = 0, pages = 0;
      if (u0 + lane < units) {
        pages = unit_of<ROWS>(prm, row_of(u0 + lane), tile_of(u0 + lane)).pages;
        s = min(prm.max_splits, max(1, (pages + per - 1) / per));
      }
      int upto = s;
      for (int x = 1; x < 64; x <<= 1) {
        const int y = __shfl_up(upto, x);
        if (lane >= x) upto += y;
      }
      const unsigned long long has = __ballot(before + upto > w);
      if (has != 0) {
        const int at = __builtin_ctzll(has);
        unit = u0 + at;
        splits = __builtin_amdgcn_readlane(s, at);
        first_wg = before + __builtin_amdgcn_readlane(upto, at) - splits;
        split = w - first_wg;
      }
      before += __builtin_amdgcn_readlane(upto, 63);
    }
    if (unit < 0) return;                     // (all wavefronts alike)
  }
  const int b = row_of(unit), tile = tile_of(unit);
  const Unit un = unit_of<ROWS>(prm, b, tile);
  const int pages = __builtin_amdgcn_readfirstlane(un.pages), stride = splits * WAVES, slot = split * WAVES + wave;

  // ---- queries: B operands, lane (n, g) has columns g D / 4 + 8 s .. + 7 of row n ----
  uintx4 qf[QT][KSTEPS];
  int limit[QT];                              // last token that the lane's query sees
  const uint8_t* mrow[QT];                    // its row of the mask
  const int block0 = prm.a.ms[2] != 0 ? (int)(tile * ROWS / prm.group) / PAGE : 0;        // rows of the mask that the tile's queries have
  const int block1 = prm.a.ms[2] != 0 ? min((min(prm.rows, (tile + 1) * ROWS) - 1) / prm.group, max(un.count - 1, 0)) / PAGE : 0;
  const bool rows_differ = prm.a.mask != nullptr && (prm.a.mask_heads == 2 || block0 < block1);
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const int r = tile * ROWS + 16 * qt + n;
    const int token = r / prm.group, head = h * prm.group + (r - token * prm.group);
    const bool real = r < prm.rows && token < un.count;
    limit[qt] = real ? un.first + token : 0x7fffffff;       // (rows that are not asked for: their results are not written)
    mrow[qt] = prm.a.mask;
    if (rows_differ && real)
      mrow[qt] += b * prm.a.ms[0] + (prm.a.mask_heads == 2 ? head : (prm.a.mask_heads == 1 ? h : 0)) * prm.a.ms[1] + (token / PAGE) * prm.a.ms[2];
    else if (prm.a.mask != nullptr)
      mrow[qt] += b * prm.a.ms[0] + (prm.a.mask_heads == 2 ? h * prm.group : (prm.a.mask_heads == 1 ? h : 0)) * prm.a.ms[1] +
                  block0 * prm.a.ms[2];
#pragma unroll
    for (int s = 0; s < KSTEPS; ++s) {
      qf[qt][s] = uintx4{0, 0, 0, 0};
      if (real) {
        qf[qt][s] = *reinterpret_cast<const uintx4*>((const unsigned short*)prm.a.q + b * prm.a.qs[0] + head * prm.a.qs[1] + token * prm.a.qs[2] + g * (D / 4) + 8 * s);
#pragma unroll
        for (int i = 0; i < 4; ++i) qf[qt][s][i] ^= prm.flip;
      }
    }
  }

  floatx4 o[QT][DT];
  float m[QT], l[QT];
  bool seen[QT];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    m[qt] = -INFINITY; l[qt] = 0.f; seen[qt] = false;
#pragma unroll
    for (int s = 0; s < DT; ++s) o[qt][s] = floatx4{0.f, 0.f, 0.f, 0.f};
  }

  // ---- the wavefront's pages: slot + i * stride, 64 of them looked up at a time ----
  const int mine = pages > slot ? (pages - slot + stride - 1) / stride : 0;
  int chunk = -64, table = -1;
  unsigned long long bits = 0;
  const int heads_kept = prm.a.mask_heads == 2 ? prm.group : 1;
  // next kept page: its number in the cache and in the sequence
  auto next = [&](int& page, int& index) -> bool {
    while (bits == 0) {
      chunk += 64;
      if (chunk >= mine) return false;
      const int i = chunk + lane, p = slot + i * stride;
      bool keep = i < mine;
      table = -1;
      if (keep) {
        table = c.page_table[(int64_t)un.seq * c.max_pages + p];
        if (table < 0 || table >= c.pages) { report(c.status, STATUS_PAGE); keep = false; }
      }
      if (prm.a.mask != nullptr && keep) {
        // kept by any of the tile's queries
        const uint8_t* row = prm.a.mask + b * prm.a.ms[0] + (prm.a.mask_heads == 2 ? h * prm.group : (prm.a.mask_heads == 1 ? h : 0)) * prm.a.ms[1] + p * prm.a.ms[3];
        keep = false;
        for (int q = block0; q <= block1; ++q)
          for (int x = 0; x < heads_kept; ++x) keep |= row[x * prm.a.ms[1] + q * prm.a.ms[2]] != 0;
      }
      bits = __ballot(keep);
    }
    const int j = __builtin_ctzll(bits);
    bits &= bits - 1;
    page = __builtin_amdgcn_readlane(table, j);
    index = slot + (chunk + j) * stride;
    return true;
  };
  auto load = [&](PageRegs<D>& r, int page, int index) {
    load_page<D>(r, c, page_of_head(c, page, h), n, g);
    if (rows_differ) {
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) r.kept[qt] = mrow[qt][index * prm.a.ms[3]];
    }
  };

  auto take = [&](const PageRegs<D>& r, int page, int index) {
    const int base = index * PAGE;
    floatx4 s[QT][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) s[qt][t] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < KSTEPS; ++k) {
        const uintx4 a = convert8<BF16>(r.k[t][k], scale_of(r.ks[D == 256 ? k >> 2 : 0], t));
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) s[qt][t] = mfma16<BF16>(a, qf[qt][k], s[qt][t]);
      }
    }
    // pages that some of the tile's queries do not see whole
    bool lacks = false;
    int see[QT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      see[qt] = rows_differ && limit[qt] != 0x7fffffff && r.kept[qt] == 0 ? -1 : limit[qt];
      lacks |= see[qt] < base + PAGE - 1;
    }
    const bool part = __ballot(lacks) != 0;
    uintx4 vs = r.vs;
    bool odd = false;                         // values that are not numbers in a page that not all queries see
    if (part) {
      int last = -1;                          // last token that any query sees
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        if (see[qt] != 0x7fffffff) last = max(last, see[qt]);
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (base + 16 * t + 4 * i + g > see[qt]) s[qt][t][i] = -INFINITY;
      }
      for (int x = 32; x > 0; x >>= 1) last = max(last, __shfl_xor(last, x));
      // what no query sees may hold anything: nothing of it may reach the sums (0 times what is not finite).  Values that are not
      // numbers and that some see are left out of the product and put where they belong below.
      bool bad = false;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const unsigned byte = 0xffu << (8 * t);
          const bool nobody = base + 16 * t + 4 * i + g > last;
          if (!nobody && (vs[i] & byte) == byte) bad = true;
          if (nobody || (vs[i] & byte) == byte) vs[i] &= ~byte;
        }
      odd = __ballot(bad) != 0;
    }
    uintx4 p[QT][2];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      float top = fmaxf(max3f(s[qt][0][0], s[qt][0][1], s[qt][0][2]), s[qt][0][3]);
#pragma unroll
      for (int t = 1; t < 4; ++t) top = max3f(max3f(top, s[qt][t][0], s[qt][t][1]), s[qt][t][2], s[qt][t][3]);
      top = fmaxf(m[qt], quad_max(top));
      if (__ballot(top > m[qt]) != 0) {
        const float fade = m[qt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m[qt] - top) * prm.scale);
        l[qt] *= fade;
#pragma unroll
        for (int x = 0; x < DT; ++x)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[qt][x][i] *= fade;
        m[qt] = top;
      }
      const float ref = m[qt] == -INFINITY ? 0.f : m[qt] * prm.scale - HEADROOM<BF16>;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[qt][t][i], prm.scale, -ref));
          if (part && base + 16 * t + 4 * i + g > see[qt]) e[i] = 0.f;
          l[qt] += e[i];
        }
        // P is rounded to the operands' type: half a step each, without a bias, against sums of the numerators as they are
        p[qt][t >> 1][2 * (t & 1)] = pack2<BF16>(e[0], e[1]);
        p[qt][t >> 1][2 * (t & 1) + 1] = pack2<BF16>(e[2], e[3]);
      }
      seen[qt] |= !part || see[qt] >= base;
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (int w = 0; w < PageRegs<D>::VW; ++w) {
        unsigned x[8][4];                     // of 8 tokens, 4 pairs of columns (2 at D = 64)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int t = 2 * half + (j >> 2), i = j & 3;
          const float sc = scale_of(vs[i], t);
          x[j][0] = convert2<BF16, 0>(r.v[8 * half + j][w], sc);
          x[j][1] = convert2<BF16, 1>(r.v[8 * half + j][w], sc);
          if constexpr (D > 64) {
            x[j][2] = convert2<BF16, 2>(r.v[8 * half + j][w], sc);
            x[j][3] = convert2<BF16, 3>(r.v[8 * half + j][w], sc);
          }
        }
#pragma unroll
        for (int e = 0; e < (D == 64 ? 2 : 4); ++e) {
          uintx4 lo, hi;
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            lo[y] = __builtin_amdgcn_perm(x[2 * y + 1][e], x[2 * y][e], 0x05040100u);
            hi[y] = __builtin_amdgcn_perm(x[2 * y + 1][e], x[2 * y][e], 0x07060302u);
          }
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) {
            o[qt][8 * w + 2 * e] = mfma16<BF16>(lo, p[qt][half], o[qt][8 * w + 2 * e]);
            o[qt][8 * w + 2 * e + 1] = mfma16<BF16>(hi, p[qt][half], o[qt][8 * w + 2 * e + 1]);
          }
        }
      }
    }
    if (odd) {
      // rare: values that are not numbers reach the queries that see their token, all others stay clear of them
      const uint8_t* bytes = c.v_scales + page_of_head(c, page, h) * page_scales(D);
      for (int t = 0; t < PAGE; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (bytes[((4 * g + i) * DT / 32) * PAGE + scale_at(t)] != NOT_FINITE) continue;
#pragma unroll
          for (int qt = 0; qt < QT; ++qt)
            if (base + t <= see[qt])
#pragma unroll
              for (int x = 0; x < DT; ++x) o[qt][x][i] = __builtin_nanf("");
        }
    }
  };

  {
    PageRegs<D> now, ahead;
    int page = 0, index = 0, page1 = 0, index1 = 0;
    bool more = next(page, index);
    if (more) load(now, page, index);
    while (more) {
      more = next(page1, index1);
      if (more) load(ahead, page1, index1);
      take(now, page, index);
      now = ahead;
      page = page1; index = index1;
    }
  }

  // ---- the wavefronts meet ----
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    l[qt] = quad_sum(l[qt]);
    m[qt] = m[qt] == -INFINITY ? (seen[qt] ? NO_MASS : -INFINITY) : m[qt] * prm.scale - HEADROOM<BF16>;
    if (g == 0) {
      lds_ml[(wave * ROWS + 16 * qt + n) * 2] = m[qt];
      lds_ml[(wave * ROWS + 16 * qt + n) * 2 + 1] = l[qt];
    }
  }
  __syncthreads();
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) top = fmaxf(top, lds_ml[(w * ROWS + 16 * qt + n) * 2]);
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float mw = lds_ml[(w * ROWS + 16 * qt + n) * 2];
      if (mw != -INFINITY) sum += lds_ml[(w * ROWS + 16 * qt + n) * 2 + 1] * __builtin_amdgcn_exp2f(mw - top);
    }
    if (wave == 0 && g == 0) { lds_row[(16 * qt + n) * 2] = top; lds_row[(16 * qt + n) * 2 + 1] = sum; }
    const float f = m[qt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[qt] - top);
    float* out = lds + (wave * ROWS + 16 * qt + n) * PITCH;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int x = 0; x < DT; x += 4)
        *reinterpret_cast<floatx4*>(out + (4 * g + i) * DT + x) = floatx4{o[qt][x][i] * f, o[qt][x + 1][i] * f, o[qt][x + 2][i] * f, o[qt][x + 3][i] * f};
  }
  __syncthreads();

  // result row r of the tile, columns d .. d + 3, not yet divided by the sum
  const int real_rows = min(ROWS, prm.rows - tile * ROWS);
  auto put = [&](int r, int d, floatx4 x, float top, float sum) {
    const int row = tile * ROWS + r, token = row / prm.group, head = h * prm.group + (row - token * prm.group);
    const bool none = token >= un.count || top == -INFINITY;
    const float f = none ? 0.f : 1.0f / sum;            // (a row that has seen tokens and has no mass: 0 times infinity, not a number)
    const int64_t at = b * prm.a.os[0] + head * prm.a.os[1] + token * prm.a.os[2] + d;
    store_out4<BF16>(prm.a.o, at, prm.a.out_f32 != 0, none ? 0.f : x[0] * f, none ? 0.f : x[1] * f, none ? 0.f : x[2] * f, none ? 0.f : x[3] * f);
    if (prm.a.lse != nullptr && d == 0)
      prm.a.lse[((int64_t)b * prm.a.H + head) * prm.a.N + token] = none || sum == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * LN2;
  };
  constexpr int QUADS = D / 4;
  float* slot_o = nullptr;
  if (splits > 1) slot_o = prm.part_o + ((int64_t)(first_wg + split) * c.heads + h) * (ROWS * D);
  for (int e = threadIdx.x; e < real_rows * QUADS; e += 64 * WAVES) {
    const int r = e / QUADS, d = 4 * (e % QUADS);
    floatx4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < WAVES; ++w) x += *reinterpret_cast<const floatx4*>(lds + (w * ROWS + r) * PITCH + d);
    if (splits == 1) put(r, d, x, lds_row[2 * r], lds_row[2 * r + 1]);
    else coherent_store4(slot_o + r * D + d, x[0], x[1], x[2], x[3]);
  }
  if (splits == 1) return;

  // ---- the workgroups meet ----
  if (threadIdx.x < 2 * real_rows)
    coherent_store(prm.part_ml + ((int64_t)(first_wg + split) * c.heads + h) * (ROWS * 2) + threadIdx.x, lds_row[threadIdx.x]);
  wait_vm<0>();
  __syncthreads();
  unsigned long long* arrivals = prm.arrivals + (int64_t)unit * c.heads + h;
  int* const count = reinterpret_cast<int*>(lds_ml);
  if (threadIdx.x == 0) *count = count_part(arrivals, prm.epoch);
  __syncthreads();
  if (*(volatile int*)count != splits) return;
  // weights of the parts: [split][row] in the room of the parts of O, found by 256 / ROWS threads a row
  {
    constexpr int PER = 64 * WAVES / ROWS;
    const int r = threadIdx.x / PER, x = threadIdx.x % PER;
    float top = -INFINITY, sum = 0.f;
    const float* ml = prm.part_ml + ((int64_t)first_wg * c.heads + h) * (ROWS * 2) + 2 * r;
    const int64_t step = (int64_t)c.heads * (ROWS * 2);
    if (r < real_rows) for (int s = x; s < splits; s += PER) top = fmaxf(top, coherent_load(ml + s * step));
#pragma unroll
    for (int y = PER / 2; y > 0; y >>= 1) top = fmaxf(top, __shfl_xor(top, y));
    if (r < real_rows) for (int s = x; s < splits; s += PER) {
      const float ms = coherent_load(ml + s * step), f = ms == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ms - top);
      lds[s * ROWS + r] = f;
      sum += f == 0.f ? 0.f : f * coherent_load(ml + s * step + 1);
    }
#pragma unroll
    for (int y = PER / 2; y > 0; y >>= 1) sum += __shfl_xor(sum, y);
    if (x == 0) { lds_row[2 * r] = top; lds_row[2 * r + 1] = sum; }
  }
  __syncthreads();
  {
    const float* part = prm.part_o + ((int64_t)first_wg * c.heads + h) * (ROWS * D);
    const int64_t step = (int64_t)c.heads * (ROWS * D);
    for (int e = threadIdx.x; e < real_rows * QUADS; e += 64 * WAVES) {
      const int r = e / QUADS, d = 4 * (e % QUADS);
      floatx4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
      for (int s = 0; s < splits; ++s) {
        const float f = lds[s * ROWS + r];
        const float* from = part + s * step + r * D + d;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] += f * coherent_load(from + i);
      }
      put(r, d, x, lds_row[2 * r], lds_row[2 * r + 1]);
    }
  }
  // back to zero, so that a replay of this launch (same mark) starts from a clean counter
  if (threadIdx.x == 0) __hip_atomic_store(arrivals, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// ---- host ----
struct CachePlan { int qt, tiles, W, max_splits; int64_t units; };      // W = 0: a workgroup per (unit, head)
static CachePlan cache_plan(const bsattn_cache& c, int B, int H, int N) {
  CachePlan p;
  const int64_t rows = (int64_t)N * (H / c.heads);
  p.qt = rows <= 16 ? 1 : (rows <= 32 || c.head_dim == 256 ? 2 : 4);
  p.tiles = (int)((rows + 16 * p.qt - 1) / (16 * p.qt));
  p.units = (int64_t)B * p.tiles;
  const int per_cu = p.qt == 1 && c.head_dim < 256 ? 2 : 1;
  const int64_t fill = (int64_t)compute_units() * per_cu;
  p.max_splits = 256 / p.qt;
  // shared where a workgroup a unit would leave compute units idle or wait for the longest sequence
  p.W = p.units * c.heads < 4 * fill && p.units <= 1024 ? (int)std::max<int64_t>(1, fill / c.heads) : 0;
  return p;
}

static size_t rounded(size_t n) { return (n + 255) / 256 * 256; }
size_t cache_attn_workspace_bytes(const bsattn_cache& c, int B, int H, int N) {
  const CachePlan p = cache_plan(c, B, H, N);
  if (p.W == 0) return 256;
  const size_t slots = ((size_t)p.W + p.units) * c.heads, rows = 16 * (size_t)p.qt;
  return rounded(slots * rows * c.head_dim * 4) + rounded(slots * rows * 8) + rounded((size_t)p.units * c.heads * 8);
}

template <int D, bool BF16, int QT>
static void launch_one(const CacheAttnParams& prm, unsigned blocks, hipStream_t st) {
  constexpr int LDS = (WAVES * 16 * QT * (D + 4) + WAVES * 16 * QT * 2 + 16 * QT * 2) * 4;
  static std::atomic<unsigned long long> configured{0};     // raising the dynamic LDS limit is idempotent
  once_per_device(configured, [] { (void)hipFuncSetAttribute((const void*)cache_attn_kernel<D, BF16, QT>, hipFuncAttributeMaxDynamicSharedMemorySize, LDS); });
  hipLaunchKernelGGL((cache_attn_kernel<D, BF16, QT>), dim3(blocks), dim3(64 * WAVES), LDS, st, prm);
}
template <int D, bool BF16>
static void launch_rows(const CacheAttnParams& prm, int qt, unsigned blocks, hipStream_t st) {
  if (qt == 1) launch_one<D, BF16, 1>(prm, blocks, st);
  else if (D == 256 || qt == 2) launch_one<D, BF16, 2>(prm, blocks, st);
  else if constexpr (D != 256) launch_one<D, BF16, 4>(prm, blocks, st);
}

int launch_cache_attn(const bsattn_cache& c, const CacheAttn& a, void* ws, hipStream_t st) {
  const CachePlan p = cache_plan(c, a.B, a.H, a.N);
  CacheAttnParams prm = {};
  prm.c = c; prm.a = a;
  prm.group = a.H / c.heads;
  prm.rows = a.N * prm.group;
  prm.tiles = p.tiles;
  prm.W = p.W; prm.max_splits = p.max_splits;
  prm.min_pages = WAVES;
  prm.scale = fabsf(a.sm_scale) * LOG2E;
  prm.flip = a.sm_scale < 0.f ? 0x80008000u : 0u;
  if (p.W > 0) {
    const size_t slots = ((size_t)p.W + p.units) * c.heads, rows = 16 * (size_t)p.qt;
    char* at = (char*)ws;
    prm.part_o = (float*)at; at += rounded(slots * rows * c.head_dim * 4);
    prm.part_ml = (float*)at; at += rounded(slots * rows * 8);
    prm.arrivals = (unsigned long long*)at;
    prm.epoch = next_epoch();
  }
  const int64_t blocks = (p.W + p.units) * c.heads;
  if (blocks > 0x7fffffffLL) return BSATTN_ERR_RANGE;
  const bool bf16 = c.dtype == BSATTN_BF16;
  if (c.head_dim == 64) bf16 ? launch_rows<64, true>(prm, p.qt, (unsigned)blocks, st) : launch_rows<64, false>(prm, p.qt, (unsigned)blocks, st);
  else if (c.head_dim == 128) bf16 ? launch_rows<128, true>(prm, p.qt, (unsigned)blocks, st) : launch_rows<128, false>(prm, p.qt, (unsigned)blocks, st);
  else bf16 ? launch_rows<256, true>(prm, p.qt, (unsigned)blocks, st) : launch_rows<256, false>(prm, p.qt, (unsigned)blocks, st);
  return launch_status();
}

}  // namespace bsattn
