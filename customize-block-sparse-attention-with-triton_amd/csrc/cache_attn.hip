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
// What bounds it: one token per sequence reads every kept page once: the cache's bytes (32 sequences of up to 64 000 tokens, 949 MB: 172 us,
// 5.5 of the 5.85 TB/s that plain reads of pages in any order reach), and below some 100 MB the steps that wait for each other (lengths, table,
// page, parts: 11 us of the 20 for 58 MB).  Prompt pieces have 32 rows a tile; a wavefront's page (D = 128) takes 128 conversions, 64 byte permutes
// and about 270 other vector instructions beside 64 matrix ones: the vector ALU bounds it (777 queries of 12 000 and of 6 000 tokens: it is active in 80 %
// of the cycles in which a SIMD has wavefronts, the matrix cores in 34 %; 757 TFLOP/s, 4 096 of 60 000 865; a large matrix product 1 200 to 1 390).
// Measured and not kept: tiles of 64 rows (one wavefront a SIMD, nothing beside its waits); pages converted once for four wavefronts of a workgroup,
// through LDS (8 % slower, and parts of four times the rows to merge); the matrix cores' own 4-bit operands for K with Q in two parts of
// 8 bits (products are added with 11 bits behind the largest one's first: not a sum in 32 bits).
//
// Who walks what.  The pages of all (sequence, tile) units of a head lie behind each other on an axis that is cut into equal ranges, one for
// each workgroup that the GPU holds at a time (a unit's end counts GAP pages: a workgroup that goes on into the next one has a merge to
// do; a cut next to a unit's begin or end goes there).  Where the cuts fall the device finds out from the lengths: the host never knows
// them, and a captured launch follows sequences as they grow.  A range's pages go round robin to the workgroup's four wavefronts, which meet in
// LDS.  With a mask the pages of a unit lie on the axis in columns of STEP (one of each 1 / STEP of the sequence): what a mask keeps next to
// each other, the last blocks for instance, goes to all of the unit's workgroups.
//
// Units of several workgroups meet in the workspace, without a counter (64 workgroups that count themselves in by compare-and-swap took
// 200 us).  Each stores its part, waits until the stores are acknowledged, stores the launch's mark into its flag, waits for that, and
// reads the flags of all: the last one to store its flag sees them all set, and adds up the parts in their order.  More than one may
// see that; they write the same bits.  Nobody waits for anybody.  Who sees all flags clears them, so that a replay of a captured launch,
// which carries the same mark, finds none set; what other launches have left carries another mark.
#include <hip/hip_runtime.h>
#include <algorithm>
#include <cfloat>
#include <type_traits>
#include "common.h"
#include "kernel_util.h"
#include "cache.h"

namespace bsattn {

constexpr int WAVES = 4;
constexpr int STEP = 16;                      // (see above)
constexpr int AT_ONCE = 4;                    // blocks of 64 units looked at at once
// Pages of the shortest range (parts cost more to merge than pages to walk), and how near to a unit's end a cut goes there.  (Two cuts
// are always more than NEAR positions apart: one at most is near an end.)  us with 8 and with 12 pages: 16 rows at D = 128, 3 000 tokens 11.7 and 13.4, at
// D = 64 11.8 and 13.3; 32 rows, two of 2 000 tokens 23.3 and 24.9, at D = 256 40 of 3 000 32.0 and 34.0 (with 6 all as with 8).  16 rows at D = 256, whose
// parts are the largest beside what they are made of: 8 sequences of 500 to 6 000, 15 rows each 29.4 and 23.2, two of 16 000, 8 rows 22.3 and 21.3, but single
// ones of a few thousand, a row each 15.8 and 17.2 to 18.8 (with 16 pages 25.6, 23.0, 18.8 to 21.0).
template <int D, int QT> constexpr int LEAST = QT == 1 && D < 256 ? 8 : (QT == 1 ? 12 : 8);
constexpr int NEAR = 6, GAP = 12;
constexpr float LN2 = 0.6931471805599453f, LOG2E = 1.4426950408889634f;
// Numerators are 2^HEADROOM at most: in fp16, whose steps are equal below 2^-14, small ones keep their digits 15 powers of two further
// down (without it weights of 2^-16 beside one of 1 were 2^-9 off).
template <bool BF16> __device__ constexpr float HEADROOM = BF16 ? 0.f : 15.f;
constexpr float NO_MASS = -3.0e38f;           // reference exponent of a row that has seen tokens, all with scores of -inf

struct CacheAttnParams {
  bsattn_cache c;
  CacheAttn a;
  int group, rows, tiles, W;      // query heads per head of the cache; N * group; tiles of them; workgroups of a head (0: one a unit)
  unsigned per_row;               // 2^32 / a.B rounded up (by_group)
  unsigned per_group;             // 2^32 / group rounded up (by_group)
  float scale; unsigned flip;                            // |sm_scale| log2 e; sign bits if sm_scale < 0
  float *part_o, *part_ml;
  unsigned long long *flags, mark;
};

typedef float floatx2 __attribute__((ext_vector_type(2)));
// Eight bytes that other workgroups have written (see coherent_load)
__device__ __forceinline__ floatx2 coherent_load2(const float* p) {
  return __builtin_bit_cast(floatx2, __hip_atomic_load((const unsigned long long*)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

// Sixteen, by a buffer's descriptor: of all loads that the compiler waits for by itself only these take 16 bytes past the caches (64 parts in
// two loads of 8 bytes each: 2.8 us more)
__device__ __forceinline__ __amdgpu_buffer_rsrc_t coherent_memory(float* p, int bytes) {
  constexpr int WORDS = 0x20000;              // data format: 32 bits
  return __builtin_amdgcn_make_buffer_rsrc(p, 0, bytes, WORDS);
}
__device__ __forceinline__ floatx4 coherent_load4(__amdgpu_buffer_rsrc_t r, int at) {
  constexpr int SC1 = 16;
  return __builtin_bit_cast(floatx4, __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, SC1));
}

// row / group, exact for row * group < 2^32
__device__ __forceinline__ int by_group(unsigned row, int group, unsigned per_group) { return group == 1 ? (int)row : (int)__umulhi(row, per_group); }

// The kernel's arguments, from memory
typedef const CacheAttnParams __attribute__((address_space(4)))* ParamsAgain;
__device__ __forceinline__ ParamsAgain params_again() {
  ParamsAgain p = (ParamsAgain)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return p;
}

__device__ __forceinline__ void coherent_store2(float* p, float a, float b) {
  const floatx2 x = {a, b};
  __hip_atomic_store((unsigned long long*)p, __builtin_bit_cast(unsigned long long, x), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
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
// Scale byte `at` of w where a conversion takes its power of two from: of the operand only the exponent counts (all codes and scales with 200
// other patterns in the other bits give the same; 255 is "not a number" whatever they are), so the other bytes may stay
__device__ __forceinline__ float scale_of(unsigned w, int at) { return __builtin_bit_cast(float, at < 3 ? w << (23 - 8 * at) : w >> 1); }

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
__device__ __forceinline__ void load_keys(PageRegs<D>& r, const bsattn_cache& c, int64_t at, int n, int g) {
  constexpr int ROW = D / 2;
  const uint8_t* codes = c.k_codes + at * page_codes(D);
  const uint8_t* scales = c.k_scales + at * page_scales(D);
  const unsigned lane_codes = (4 * (n & 3) + (n >> 2)) * ROW + g * (D / 8);
  const unsigned lane_scales = (D == 64 ? g >> 1 : (D == 128 ? g : 2 * g)) * PAGE + n * 4;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
#pragma unroll
    for (int x = 0; x < D / 32; x += 4) {
      const auto a = *reinterpret_cast<const typename Words<(D / 32 < 4 ? D / 32 : 4)>::type*>(codes + lane_codes + t * 16 * ROW + 4 * x);
#pragma unroll
      for (int i = 0; i < (D / 32 < 4 ? D / 32 : 4); ++i) r.k[t][x + i] = a[i];
    }
  }
#pragma unroll
  for (int i = 0; i < PageRegs<D>::KS; ++i) r.ks[i] = *reinterpret_cast<const unsigned*>(scales + lane_scales + i * PAGE);
}
template <int D>
__device__ __forceinline__ void load_values(PageRegs<D>& r, const bsattn_cache& c, int64_t at, int n, int g) {
  constexpr int ROW = D / 2;
  const uint8_t* codes = c.v_codes + at * page_codes(D);
  const uint8_t* scales = c.v_scales + at * page_scales(D);
  const unsigned lane_codes = g * ROW + n * (D / 32), lane_scales = (D == 64 ? n >> 3 : (D == 128 ? n >> 2 : n >> 1)) * PAGE + g * 16;
#pragma unroll
  for (int j = 0; j < 16; ++j) {              // token 16 (j / 4) + 4 (j % 4) + g
    if constexpr (D == 64) r.v[j][0] = *reinterpret_cast<const unsigned short*>(codes + lane_codes + 4 * j * ROW);
    else if constexpr (D == 128) r.v[j][0] = *reinterpret_cast<const unsigned*>(codes + lane_codes + 4 * j * ROW);
    else {
      const uintx2 a = *reinterpret_cast<const uintx2*>(codes + lane_codes + 4 * j * ROW);
      r.v[j][0] = a[0]; r.v[j][1] = a[1];
    }
  }
  r.vs = *reinterpret_cast<const uintx4*>(scales + lane_scales);
}

// What tile `tile` of row b walks: its sequence, the position of the row's first query, and pages 0 .. pages - 1
struct Unit { int seq, first, count, pages; };
template <int ROWS, bool REPORT>
__device__ __forceinline__ Unit unit_of(const CacheAttnParams& prm, int b, int tile) {
  Unit u = {sequence_of(prm.a.sequences, b, prm.c.sequences), 0, 0, 0};
  u.count = prm.a.counts != nullptr ? prm.a.counts[b] : prm.a.N;
  if (u.seq < 0 || u.count < 0 || u.count > prm.a.N) {
    if (REPORT) report(prm.c.status, STATUS_ROW);
    u.seq = -1; u.count = 0;
    if (REPORT) return u;
  }
  // (without reports there are no branches, so that the loads of several units go out together)
  u.first = length_of(prm.c, REPORT ? u.seq : max(u.seq, 0)) - u.count;
  int t0 = 0, t1 = prm.a.N - 1;
  if (prm.tiles > 1) {
    t0 = by_group(tile * ROWS, prm.group, prm.per_group);
    t1 = by_group(min(prm.rows, (tile + 1) * ROWS) - 1, prm.group, prm.per_group);
  }
  const int last = u.first + min(u.count - 1, t1);
  u.pages = t0 < u.count && last >= 0 ? last / PAGE + 1 : 0;
  return u;
}

// Floats of LDS for the (m, l) of parts that meet there: four wavefronts' for each row, or those of a thread each 4 columns
template <int D, int QT> constexpr int ML_FLOATS = WAVES * 16 * QT * 2 > 2 * (64 * WAVES / (D / 4)) ? WAVES * 16 * QT * 2 : 2 * (64 * WAVES / (D / 4));

// Adds a part of a row (its reference exponent m, its sum l, 4 columns y) to what (top, sum, x) have of it
__device__ __forceinline__ void merge(float& top, float& sum, floatx4& x, float m, float l, floatx4 y) {
  const float high = fmaxf(top, m);
  const float a = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - high), b = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - high);
  sum = sum * a + l * b;
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = x[i] * a + y[i] * b;
  top = high;
}

// Workgroups of a compute unit (and wavefronts of a SIMD): what the registers leave room for
template <int D, int QT> constexpr int PER_CU = D * QT >= 512 ? 1 : (QT == 1 && D < 128 ? 3 : 2);

// FINE: P goes into the second product as two bf16 parts, the rounded value and what it lacks (2^-17 together), for results in fp32 of a bf16 cache:
// one part alone leaves them 8 bits behind the point (2e-3 of a result), of which a caller that merges them would get no more than 16-bit results hold.
// (fp16, which the forward takes for P then, has no room for a cache's values.  An fp16 cache's P has 11 bits already.)  Twice the matrix
// instructions of the second product: one to five tokens, bound by other things, take 0 to 6 % longer (24 sequences 20.8 -> 21.2 us, 32 long ones 174 both),
// pieces of prompts up to a quarter (777 tokens of two prompts 228 -> 282, at D = 64 600 of 3 000 to 9 000 54 -> 62).
template <int D, bool BF16, int QT, bool MASK, bool FINE>
__global__ __launch_bounds__(64 * WAVES, (PER_CU<D, QT>)) void cache_attn_kernel(const CacheAttnParams prm) {
  constexpr int ROWS = 16 * QT, PITCH = D + 4, KSTEPS = D / 32, DT = D / 16;
  extern __shared__ __align__(16) float lds[];           // [WAVES][ROWS][PITCH] parts of O | their (m, l) | 1 word
  float* const lds_ml = lds + WAVES * ROWS * PITCH;
  volatile int* const lds_last = reinterpret_cast<int*>(lds_ml + ML_FLOATS<D, QT>);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
  const bsattn_cache& c = prm.c;
  const int w = blockIdx.x / (unsigned)c.heads;
  // (the ranges of a head go to all XCDs, which are not equally near to all memory; tiles of one sequence share an L2's copy of its pages)
  const int h = prm.W > 0 && prm.tiles == 1 ? (blockIdx.x + w) % (unsigned)c.heads : blockIdx.x - w * c.heads;
  const int units = prm.a.B * prm.tiles;
  // positions of a unit's pages on the axis
  auto positions = [&](int pages) { return MASK ? (pages + STEP - 1) / STEP * STEP : pages; };

  // ---- the range ----
  int lo = 0, hi = 0, each = 1, longer = 0;
  auto cut_at = [&](int x) { return each * x + min(x, longer); };            // begin of range x
  // the range that holds a position
  auto holder = [&](int x) {
    const int of_longer = (each + 1) * longer;
    return x < of_longer ? (int)((unsigned)x / (unsigned)(each + 1)) : longer + (int)((unsigned)(x - of_longer) / (unsigned)each);
  };
  // the workgroup's of an axis of `total` positions, of which one unit has `longest`; false: it has none.  What walks a range takes
  // total / ranges pages' time, what merges the longest unit's parts longest / total * ranges parts' of its rows: their sum is least at MOST ranges.
  auto cut = [&](int total, int longest) -> bool {
    hi = total;
    if (prm.W == 0) return true;
    constexpr float MOST = 4.8f;              // (of 2 to 9, over calls of 1 to 40 rows; 20 sequences of up to 114 000 tokens, 7 tokens of 4 heads on one: 76 us unbounded, so 30)
    const int most = (int)((float)total * MOST * __builtin_amdgcn_rsqf((float)longest * (float)min(ROWS, prm.rows)));
    const int ranges = min(prm.W, max(units, min(most, total / (LEAST<D, QT>))));
    if (w >= ranges) return false;
    // the first `longer` ranges are one position longer than `each`
    each = (unsigned)total / (unsigned)ranges; longer = total - each * ranges;
    lo = cut_at(w);
    hi = lo + each + (w < longer ? 1 : 0);
    return true;
  };
  // Units are looked at 64 at a time, a lane each.  Where there are more, every block's share of the axis is added up first, several blocks' loads
  // under way at once, and then only those that the range meets are looked at.
  int starts = 0;                             // where a lane's block begins on the axis
  unsigned long long blocks = 1;
  if (prm.W > 0 && units > 64) {
    int share = 0, longest = 0;
    for (int k = 0; 64 * k < units; k += AT_ONCE) {
      int length[AT_ONCE];
#pragma unroll
      for (int x = 0; x < AT_ONCE; ++x) {
        const int u = min(64 * (k + x) + lane, units - 1), tile_back = prm.tiles == 1 ? 0 : by_group(u, prm.a.B, prm.per_row);
        length[x] = positions(unit_of<ROWS, false>(prm, u - tile_back * prm.a.B, prm.tiles - 1 - tile_back).pages) + GAP;
      }
#pragma unroll
      for (int x = 0; x < AT_ONCE; ++x) {
        const int sum = __builtin_amdgcn_readlane(wave_upto(64 * (k + x) + lane < units ? length[x] : 0), 63);
        if (lane == k + x) share = sum;
        longest = max(longest, length[x]);
      }
    }
    const int upto = wave_upto(share);
    if (!cut(__builtin_amdgcn_readlane(upto, 63), wave_most(longest))) return;
    starts = upto - share;
    blocks = __ballot(starts < hi && upto > lo);
  }
  for (; blocks != 0; blocks &= blocks - 1) {
  const int block = __builtin_ctzll(blocks), base = prm.W > 0 ? 64 * block : w;
  Unit mine = {-1, 0, 0, 0};                  // a lane's unit, how much of the axis it has, and where it begins there
  int length = 0;
  if (prm.W > 0 ? base + lane < units : lane == 0) {
    const int tile_back = prm.tiles == 1 ? 0 : by_group(base + lane, prm.a.B, prm.per_row);
    mine = unit_of<ROWS, true>(prm, base + lane - tile_back * prm.a.B, prm.tiles - 1 - tile_back);
    length = positions(mine.pages) + GAP;
  }
  const int upto = wave_upto(length), begin = __builtin_amdgcn_readlane(starts, block) + upto - length;
  if (hi == 0 && !cut(__builtin_amdgcn_readlane(upto, 63), wave_most(length))) return;
  for (unsigned long long mates = __ballot(length > 0 && begin < hi && begin + length > lo); mates != 0; mates &= mates - 1) {
  const int at = __builtin_ctzll(mates), unit = base + at, unit_back = prm.tiles == 1 ? 0 : by_group(unit, prm.a.B, prm.per_row);
  const int b = unit - unit_back * prm.a.B, tile = prm.tiles - 1 - unit_back;
  const Unit un = {__builtin_amdgcn_readlane(mine.seq, at), __builtin_amdgcn_readlane(mine.first, at), __builtin_amdgcn_readlane(mine.count, at),
                   __builtin_amdgcn_readlane(mine.pages, at)};
  const int unit_begin = __builtin_amdgcn_readlane(begin, at), unit_positions = positions(un.pages);
  int first_wg = w, last_wg = w;              // workgroups of the unit
  if (prm.W > 0) {
    first_wg = holder(unit_begin);
    last_wg = unit_positions > 0 ? holder(unit_begin + unit_positions - 1) : first_wg;
    if (first_wg < last_wg && cut_at(first_wg + 1) - unit_begin <= NEAR) ++first_wg;
    if (first_wg < last_wg && unit_begin + unit_positions - cut_at(last_wg) <= NEAR) --last_wg;
    if (w < first_wg || w > last_wg) continue;
  }
  const int splits = last_wg - first_wg + 1, split = w - first_wg;
  const int from = split == 0 ? 0 : cut_at(w) - unit_begin, to = w == last_wg ? unit_positions : cut_at(w + 1) - unit_begin;      // its positions

  const bool by_head = MASK && prm.a.mask_heads == 2;
  int block0 = 0, block1 = 0;                 // rows of the mask that the tile's queries have
  const uint8_t* tile_mask = nullptr;         // the first of them, of the tile's first head
  if constexpr (MASK) {
    if (prm.a.ms[2] != 0) {
      block0 = by_group(tile * ROWS, prm.group, prm.per_group) / PAGE;
      block1 = max(block0, min(by_group(min(prm.rows, (tile + 1) * ROWS) - 1, prm.group, prm.per_group), un.count - 1) / PAGE);
    }
    tile_mask = prm.a.mask + b * prm.a.ms[0] + (by_head ? h * prm.group : (prm.a.mask_heads == 1 ? h : 0)) * prm.a.ms[1] + block0 * prm.a.ms[2];
  }
  const bool rows_differ = MASK && (by_head || block0 < block1);

  // ---- the wavefront's pages, 64 positions looked up at a time: every fourth position of the range, or with a mask every fourth kept page
  // of those that all four wavefronts look up (2 of 200 000 tokens of which a tenth is kept: 25.3 -> 24.4 us)
  const int own = MASK ? to - from : (to > from + wave ? (to - from - wave + WAVES - 1) / WAVES : 0), columns = unit_positions / STEP;
  auto page_at = [&](int i) {                 // page of the wavefront's position i
    if constexpr (!MASK) return from + wave + WAVES * i;
    const int x = from + i;
    return (x % STEP) * columns + x / STEP;
  };
  // the next 64 are asked for when the ones in front of them are taken up, the first ones in front of the queries
  int chunk = -64, table = -1, kept_before = 0, table_ahead = -1;
  unsigned char kept_ahead = 0;               // the first of the mask's rows
  unsigned long long bits = 0;
  auto ask = [&](int at) {
    const int p = page_at(at + lane);
    table_ahead = -1;
    if (at + lane < own && p < un.pages) {
      table_ahead = c.page_table[(int64_t)un.seq * c.max_pages + p];
      if constexpr (MASK) kept_ahead = tile_mask[p * prm.a.ms[3]];
    }
  };
  ask(0);

  // ---- queries: B operands, lane (n, g) has columns g D / 4 + 8 s .. + 7 of row n ----
  uintx4 qf[QT][KSTEPS];
  int limit[QT];                              // last token that the lane's query sees
  const uint8_t* mrow[QT];                    // its row of the mask
  // last token that any of the tile's queries sees
  const int last_token = un.first + min(un.count - 1, by_group(min(prm.rows, (tile + 1) * ROWS) - 1, prm.group, prm.per_group));
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const int r = tile * ROWS + 16 * qt + n;
    const bool asked = r < prm.rows && by_group(r, prm.group, prm.per_group) < un.count;
    const int row = asked ? r : tile * ROWS;                // (rows that are not asked for: any query will do, their results are not written)
    const int token = by_group(row, prm.group, prm.per_group), of_group = row - token * prm.group;
    limit[qt] = asked ? un.first + token : 0x7fffffff;
    mrow[qt] = tile_mask;
    if (rows_differ) mrow[qt] += (by_head ? of_group : 0) * prm.a.ms[1] + (block1 > block0 ? token / PAGE - block0 : 0) * prm.a.ms[2];
    const unsigned short* q = (const unsigned short*)prm.a.q + b * prm.a.qs[0] + (h * prm.group + of_group) * prm.a.qs[1] + token * prm.a.qs[2] + g * (D / 4);
#pragma unroll
    for (int s = 0; s < KSTEPS; ++s) qf[qt][s] = *reinterpret_cast<const uintx4*>(q + 8 * s);
  }
  if (prm.flip != 0)
#pragma unroll
    for (int qt = 0; qt < QT; ++qt)
#pragma unroll
      for (int s = 0; s < KSTEPS; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) qf[qt][s][i] ^= prm.flip;

  floatx4 o[QT][DT];
  float m[QT], l[QT];
  unsigned marks = 0;                         // bit 4 qt + i: columns (4 g + i) DT .. are not numbers; bit 16 + qt: the query has seen a token
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    m[qt] = -INFINITY; l[qt] = 0.f;
#pragma unroll
    for (int s = 0; s < DT; ++s) o[qt][s] = floatx4{0.f, 0.f, 0.f, 0.f};
  }

  // next kept page: its number in the cache and in the sequence
  auto next = [&](int& page, int& index) -> bool {
    while (bits == 0) {
      chunk += 64;
      if (chunk >= own) return false;
      const int p = page_at(chunk + lane);
      const bool there = chunk + lane < own && p < un.pages;
      table = table_ahead;
      bool keep = there;
      if constexpr (MASK) {                   // kept by any of the tile's queries
        keep = there && kept_ahead != 0;
        if (rows_differ && there)
          for (int q = 0; q <= block1 - block0; ++q)
            for (int x = 0; x < (by_head ? prm.group : 1); ++x) keep |= tile_mask[x * prm.a.ms[1] + q * prm.a.ms[2] + p * prm.a.ms[3]] != 0;
      }
      if (keep && (table < 0 || table >= c.pages)) { report(c.status, STATUS_PAGE); keep = false; }
      if (chunk + 64 < own) ask(chunk + 64);
      bits = __ballot(keep);
      if constexpr (MASK) {
        const int rank = kept_before + __builtin_popcountll(bits & ((1ull << lane) - 1));
        kept_before += __builtin_popcountll(bits);
        bits = __ballot(keep && rank % WAVES == wave);
      }
    }
    const int j = __builtin_ctzll(bits);
    bits &= bits - 1;
    page = __builtin_amdgcn_readlane(table, j);
    index = page_at(chunk + j);
    return true;
  };
  // One page at a time.  Its keys' registers are free for the next page's once the scores are there, its values' once they are in O: the
  // loads of a page are under way for most of the time that the page in front of it takes.
  PageRegs<D> r = {};                         // (not left open: the compiler would keep a unit's last page for the next one)
  int page = 0, index = 0;
  auto load_kept = [&] {
    if constexpr (MASK)
      if (rows_differ)
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) r.kept[qt] = mrow[qt][index * prm.a.ms[3]];
  };
  bool more = next(page, index);
  if (more) {
    load_keys<D>(r, c, page_of_head(c, page, h), n, g);
    load_values<D>(r, c, page_of_head(c, page, h), n, g);
    load_kept();
  }
  const int place = __builtin_amdgcn_s_getreg(4 | 3 << 11);    // the wavefront's on its SIMD (HW_ID, bits 0 .. 3)
  unsigned clock = 0;                         // in 10 ns, as it was at the page in front
  while (more) {
    // Of the wavefronts of a SIMD the one that came first would be served first, and end up to a fifth earlier: they take turns, 10 us each (by
    // the clock, which all see, not by their pages: 777 tokens of two prompts 234 -> 231 us)
    if constexpr (PER_CU<D, QT> > 1) {
      const int now = ((clock >> 10) + place) % PER_CU<D, QT>;
      clock = (unsigned)__builtin_amdgcn_s_memrealtime();
      if (now == 0) __builtin_amdgcn_s_setprio(0);
      else if (now == 1) __builtin_amdgcn_s_setprio(1);
      else __builtin_amdgcn_s_setprio(2);
    }
    const int token0 = index * PAGE, this_page = page;
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
      see[qt] = limit[qt];
      if constexpr (MASK) if (rows_differ && limit[qt] != 0x7fffffff && r.kept[qt] == 0) see[qt] = -1;
      lacks |= see[qt] < token0 + PAGE - 1;
    }
    const bool part = __ballot(lacks) != 0;
    more = next(page, index);
    __builtin_amdgcn_sched_barrier(0);
    if (more) {
      load_keys<D>(r, c, page_of_head(c, page, h), n, g);
      load_kept();
    }
    bool odd = false;                         // values that are not numbers in a page that not all queries see
    if (part) {
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        const int up_to = see[qt] - token0 - g;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (16 * t + 4 * i > up_to) s[qt][t][i] = -INFINITY;
      }
      // what no query sees may hold anything: nothing of it may reach the sums (0 times what is not finite).  Values that are not
      // numbers and that some see are left out of the product and put where they belong below.
      bool bad = false;
      const int up_to = last_token - token0 - g;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const unsigned byte = 0xffu << (8 * t);
          const bool nobody = 16 * t + 4 * i > up_to;
          if (!nobody && (r.vs[i] & byte) == byte) bad = true;
          if (nobody || (r.vs[i] & byte) == byte) r.vs[i] &= ~byte;
        }
      odd = __ballot(bad) != 0;
    }
    uintx4 p[QT][2], rest[QT][2];
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
          l[qt] += e[i];
        }
        // P is rounded to the operands' type: half a step each, without a bias, against sums of the numerators as they are
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const unsigned pair = pack2<BF16>(e[2 * i], e[2 * i + 1]);
          p[qt][t >> 1][2 * (t & 1) + i] = pair;
          if constexpr (FINE)
            rest[qt][t >> 1][2 * (t & 1) + i] = pack2<true>(e[2 * i] - __builtin_bit_cast(float, pair << 16), e[2 * i + 1] - __builtin_bit_cast(float, pair & 0xffff0000u));
        }
      }
      if (!part || see[qt] >= token0) marks |= 0x10000u << qt;
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (int w = 0; w < PageRegs<D>::VW; ++w) {
        unsigned x[8][4];                     // of 8 tokens, 4 pairs of columns (2 at D = 64)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float sc = scale_of(r.vs[j & 3], 2 * half + (j >> 2));
          x[j][0] = convert2<BF16, 0>(r.v[8 * half + j][w], sc);
          x[j][1] = convert2<BF16, 1>(r.v[8 * half + j][w], sc);
          if constexpr (D > 64) {
            x[j][2] = convert2<BF16, 2>(r.v[8 * half + j][w], sc);
            x[j][3] = convert2<BF16, 3>(r.v[8 * half + j][w], sc);
          }
        }
#pragma unroll
        for (int e = 0; e < (D == 64 ? 2 : 4); ++e) {
          uintx4 low, high;
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            low[y] = __builtin_amdgcn_perm(x[2 * y + 1][e], x[2 * y][e], 0x05040100u);
            high[y] = __builtin_amdgcn_perm(x[2 * y + 1][e], x[2 * y][e], 0x07060302u);
          }
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) {
            o[qt][8 * w + 2 * e] = mfma16<BF16>(low, p[qt][half], o[qt][8 * w + 2 * e]);
            o[qt][8 * w + 2 * e + 1] = mfma16<BF16>(high, p[qt][half], o[qt][8 * w + 2 * e + 1]);
            if constexpr (FINE) {
              o[qt][8 * w + 2 * e] = mfma16<BF16>(low, rest[qt][half], o[qt][8 * w + 2 * e]);
              o[qt][8 * w + 2 * e + 1] = mfma16<BF16>(high, rest[qt][half], o[qt][8 * w + 2 * e + 1]);
            }
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if (odd) {
      // rare: values that are not numbers reach the queries that see their token, all others stay clear of them
      const uint8_t* bytes = c.v_scales + page_of_head(c, this_page, h) * page_scales(D);
      for (int t = 0; t < PAGE; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (bytes[((4 * g + i) * DT / 32) * PAGE + scale_at(t)] != NOT_FINITE) continue;
#pragma unroll
          for (int qt = 0; qt < QT; ++qt)
            if (token0 + t <= see[qt]) marks |= 1u << (4 * qt + i);
        }
    }
    if (!more) break;
    load_values<D>(r, c, page_of_head(c, page, h), n, g);
  }

  // ---- the wavefronts meet ----
  const int tile_rows = min(ROWS, prm.rows - tile * ROWS);
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    l[qt] = quad_sum(l[qt]);
    m[qt] = m[qt] == -INFINITY ? ((marks >> (16 + qt) & 1) != 0 ? NO_MASS : -INFINITY) : m[qt] * prm.scale - HEADROOM<BF16>;
    if (g == 0) {
      if (16 * qt + n < tile_rows) {
        lds_ml[2 * (wave * tile_rows + 16 * qt + n)] = m[qt];
        lds_ml[2 * (wave * tile_rows + 16 * qt + n) + 1] = l[qt];
      }
    }
  }
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    float* out = lds + (wave * ROWS + 16 * qt + n) * PITCH;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool odd = (marks >> (4 * qt + i) & 1) != 0;
#pragma unroll
      for (int x = 0; x < DT; x += 4)
        *reinterpret_cast<floatx4*>(out + (4 * g + i) * DT + x) =
            odd ? floatx4{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")} : floatx4{o[qt][x][i], o[qt][x + 1][i], o[qt][x + 2][i], o[qt][x + 3][i]};
    }
  }
  __syncthreads();

  // (from here on the arguments are read again: kept over the pages they would crowd the scalar registers)
  const ParamsAgain late = params_again();
  constexpr int QUADS = D / 4;
  const int real_rows = min(ROWS, late->rows - tile * ROWS);
  const int cells = real_rows * QUADS;        // a cell: 4 columns of a row
  // what is added up for the result: parts `part_step` floats apart, rows `pitch` apart, their references and sums in lds_ml
  int parts_n = WAVES, part_step = ROWS * PITCH, pitch = PITCH;
  bool last_in = true;
  if (splits > 1) {
    // ---- the workgroups meet ----
    // A workgroup has two parts at most: of the unit that goes on from the range in front of it, and of the one that goes on behind it.  Those
    // of a head lie close together, rows that are not there take no room: what merges them asks many places at once (one sequence of 160 000
    // tokens, 64 parts a head: with the heads' parts in turn 8.5 us for it, so 5.4).
    auto slot_of = [&](int x) { return (int64_t)(h * late->W + first_wg + x) * 2 + (x == 0); };
    const int slot_rows = min(ROWS, late->rows);
    float* slot_o = late->part_o + slot_of(split) * (slot_rows * D);
    for (int e = threadIdx.x; e < cells; e += 64 * WAVES) {
      const int r = e / QUADS, d = 4 * (e % QUADS);
      floatx4 x = {0.f, 0.f, 0.f, 0.f};
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int y = 0; y < WAVES; ++y)
        merge(top, sum, x, lds_ml[2 * (y * real_rows + r)], lds_ml[2 * (y * real_rows + r) + 1], *reinterpret_cast<const floatx4*>(lds + (y * ROWS + r) * PITCH + d));
      coherent_store4(slot_o + 4 * e, x[0], x[1], x[2], x[3]);
      if (d == 0) coherent_store2(late->part_ml + slot_of(split) * (slot_rows * 2) + 2 * r, top, sum);
    }
    wait_vm<0>();
    __syncthreads();
    if (threadIdx.x < 64) {
      if (threadIdx.x == 0) __hip_atomic_store(late->flags + slot_of(split), late->mark, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      wait_vm<0>();
      bool all = true;
#pragma unroll 4
      for (int y = lane; y < splits; y += 64) all &= __hip_atomic_load(late->flags + slot_of(y), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == late->mark;
      all = __ballot(!all) == 0;
      if (threadIdx.x == 0) *lds_last = all;
    }
    __syncthreads();
    last_in = *lds_last != 0;
    if (last_in) {
      // The parts go to `teams` groups of threads, where there are few rows; the groups meet in LDS
      const int teams = max(1, 64 * WAVES / cells);
      const float* const parts_ml = late->part_ml + slot_of(0) * (slot_rows * 2);
      const auto parts_o = coherent_memory(late->part_o + slot_of(0) * (slot_rows * D), 4 * (2 * splits - 1) * (slot_rows * D));
      // CELLS cells of a thread at a time, and PARTS parts of each (more of either is more code and more places asked for in vain where there are few
      // parts, as is the rule: 24 sequences 20.6 us with 16 parts for 20.2, 100 000 tokens of 16 heads on one 36 with four cells for 27)
      auto add_up = [&](auto count) {
        constexpr int CELLS = decltype(count)::value, PARTS = CELLS == 1 ? 8 : 6;
        for (int e0 = threadIdx.x; e0 < cells * teams; e0 += 64 * WAVES * CELLS) {
          const int team = e0 / cells;          // (0 where there is more than one cell a thread)
          int cell[CELLS];
          floatx4 x[CELLS];
          float top[CELLS], sum[CELLS];
#pragma unroll
          for (int k = 0; k < CELLS; ++k) {
            cell[k] = min(e0 - team * cells + 64 * WAVES * k, cells - 1);
            x[k] = floatx4{0.f, 0.f, 0.f, 0.f};
            top[k] = -INFINITY; sum[k] = 0.f;
          }
          for (int y0 = team; y0 < splits; y0 += teams * PARTS) {
            floatx2 ml[PARTS][CELLS];
            floatx4 part[PARTS][CELLS];
#pragma unroll
            for (int j = 0; j < PARTS; ++j) {
              const int y = min(y0 + j * teams, splits - 1);
              const int slot = y == 0 ? 0 : 2 * y - 1;              // (behind the first part's)
              const float* at_ml = parts_ml + (int64_t)slot * (slot_rows * 2);
#pragma unroll
              for (int k = 0; k < CELLS; ++k) {
                ml[j][k] = coherent_load2(at_ml + 2 * (cell[k] / QUADS));
                part[j][k] = coherent_load4(parts_o, 4 * (slot * (slot_rows * D) + 4 * cell[k]));
              }
            }
#pragma unroll
            for (int j = 0; j < PARTS; ++j)
              if (y0 + j * teams < splits)
#pragma unroll
                for (int k = 0; k < CELLS; ++k)
                  merge(top[k], sum[k], x[k], ml[j][k][0], ml[j][k][1], part[j][k]);
          }
#pragma unroll
          for (int k = 0; k < CELLS; ++k) {
            if (e0 + 64 * WAVES * k >= cells * teams) break;
            *reinterpret_cast<floatx4*>(lds + 4 * (e0 + 64 * WAVES * k)) = x[k];
            if (cell[k] % QUADS == 0) {
              lds_ml[2 * (team * real_rows + cell[k] / QUADS)] = top[k];
              lds_ml[2 * (team * real_rows + cell[k] / QUADS) + 1] = sum[k];
            }
          }
        }
      };
      if (cells <= 64 * WAVES) add_up(std::integral_constant<int, 1>{});
      else add_up(std::integral_constant<int, 2>{});
      __syncthreads();
      parts_n = teams; part_step = 4 * cells; pitch = D;
      for (int y = threadIdx.x; y < splits; y += 64 * WAVES) __hip_atomic_store(late->flags + slot_of(y), 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  if (last_in)
    for (int e = threadIdx.x; e < cells; e += 64 * WAVES) {
      const int r = e / QUADS, d = 4 * (e % QUADS);
      const int row = tile * ROWS + r, token = by_group(row, late->group, late->per_group), head = h * late->group + (row - token * late->group);
      floatx4 x = {0.f, 0.f, 0.f, 0.f};
      float top = -INFINITY, sum = 0.f;
      for (int y = 0; y < parts_n; ++y)
        merge(top, sum, x, lds_ml[2 * (y * real_rows + r)], lds_ml[2 * (y * real_rows + r) + 1], *reinterpret_cast<const floatx4*>(lds + y * part_step + r * pitch + d));
      const bool none = token >= un.count || top == -INFINITY;
      const float f = 1.0f / sum;             // (a row that has seen tokens and has no mass: 0 times infinity, not a number)
      store_out4<BF16>(late->a.o, b * late->a.os[0] + head * late->a.os[1] + token * late->a.os[2] + d, late->a.out_f32 != 0, none ? 0.f : x[0] * f,
                       none ? 0.f : x[1] * f, none ? 0.f : x[2] * f, none ? 0.f : x[3] * f);
      if (late->a.lse != nullptr && d == 0)
        late->a.lse[((int64_t)b * late->a.H + head) * late->a.N + token] = none || sum == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * LN2;
    }
  __syncthreads();                            // (the next unit's parts go where these are)
  }
  }
}

// ---- host ----
// W = 0: a workgroup per (unit, head)
struct CachePlan { int qt, tiles, W; int64_t units; };
static CachePlan cache_plan(const bsattn_cache& c, int B, int H, int N) {
  CachePlan p;
  const int64_t rows = (int64_t)N * (H / c.heads);
  p.qt = rows <= 16 ? 1 : 2;
  p.tiles = (int)((rows + 16 * p.qt - 1) / (16 * p.qt));
  p.units = (int64_t)B * p.tiles;
  const int per_cu = p.qt == 1 ? (c.head_dim < 128 ? 3 : 2) : (p.qt == 2 && c.head_dim < 256 ? 2 : 1);
  const int64_t fill = (int64_t)compute_units() * per_cu;
  // Ranges wherever the device can find them, up to 2048 units of a head: the host does not know the lengths, and a workgroup a unit takes as long as
  // the longest one, 0.29 us a page (us in ranges and with a workgroup a unit): 513 sequences of one head, one of them of 200 000 tokens, 30 and 897;
  // 400 of 8 heads, 200 to 2 000 tokens and one of 100 000, 107 and 607, without that one 89 and 91, all of 1 000 tokens 101 and 103; 30 prompts, 300
  // queries, 400 to 9 000 tokens 604 and 653, all of 4 000 798 and 795, of 400 and one of 60 000 534 and 1 101.  Two kinds of calls are better off without:
  // - many units of one token that have a few pages each, through which every workgroup looks: 513 of 200 to 2 000 tokens 24 and 22, 2 000 of 50 to 500
  //   31 and 22, 700 of 50 to 100 11 and 7.  No more than 64 pages a sequence, which the cache's tables say, bound what a long one costs there.
  // - so many heads that few ranges are left for each, and a part of the GPU idle: 192 heads of 30 sequences 159 and 143, 300 heads 296 and 221 (100 heads
  //   74 and 79).  Of few units these are in ranges all the same (192 heads of 4 sequences 24 and 27).
  const bool pieces = p.tiles > 1, many_heads = c.heads > fill / 4;
  const bool ranges = p.units <= 2048 && p.units * ((int64_t)c.max_pages + STEP + GAP) < 0x7fffffffLL &&      // (the axis is counted in 32 bits)
                      (many_heads ? p.units * c.heads < (pieces ? 16 : 6) * fill : pieces || p.units <= 512 || c.max_pages > 64);
  p.W = ranges ? (int)std::max<int64_t>(1, fill / c.heads) : 0;
  return p;
}

static size_t rounded(size_t n) { return (n + 255) / 256 * 256; }
size_t cache_attn_workspace_bytes(const bsattn_cache& c, int B, int H, int N) {
  const CachePlan p = cache_plan(c, B, H, N);
  if (p.W == 0) return 256;
  const size_t slots = 2 * (size_t)p.W * c.heads, rows = 16 * (size_t)p.qt;
  return rounded(slots * rows * c.head_dim * 4) + rounded(slots * rows * 8) + rounded(slots * 8);
}

template <int D, bool BF16, int QT, bool MASK, bool FINE>
static void launch_one(const CacheAttnParams& prm, unsigned blocks, hipStream_t st) {
  constexpr int LDS = (WAVES * 16 * QT * (D + 4) + ML_FLOATS<D, QT> + 4) * 4;
  static std::atomic<unsigned long long> configured{0};     // raising the dynamic LDS limit is idempotent
  once_per_device(configured, [] { (void)hipFuncSetAttribute((const void*)cache_attn_kernel<D, BF16, QT, MASK, FINE>, hipFuncAttributeMaxDynamicSharedMemorySize, LDS); });
  hipLaunchKernelGGL((cache_attn_kernel<D, BF16, QT, MASK, FINE>), dim3(blocks), dim3(64 * WAVES), LDS, st, prm);
}
template <int D, bool BF16, int QT>
static void launch_rows(const CacheAttnParams& prm, unsigned blocks, hipStream_t st) {
  const bool fine = BF16 && prm.a.out_f32 != 0;
  if (prm.a.mask != nullptr) fine ? launch_one<D, BF16, QT, true, BF16>(prm, blocks, st) : launch_one<D, BF16, QT, true, false>(prm, blocks, st);
  else fine ? launch_one<D, BF16, QT, false, BF16>(prm, blocks, st) : launch_one<D, BF16, QT, false, false>(prm, blocks, st);
}
template <int D, bool BF16>
static void launch_tiles(const CacheAttnParams& prm, int qt, unsigned blocks, hipStream_t st) {
  if (qt == 1) launch_rows<D, BF16, 1>(prm, blocks, st);
  else launch_rows<D, BF16, 2>(prm, blocks, st);
}

int launch_cache_attn(const bsattn_cache& c, const CacheAttn& a, void* ws, hipStream_t st) {
  const CachePlan p = cache_plan(c, a.B, a.H, a.N);
  CacheAttnParams prm = {};
  prm.c = c; prm.a = a;
  prm.group = a.H / c.heads;
  prm.rows = a.N * prm.group;
  prm.per_row = a.B > 1 ? 0xffffffffu / a.B + 1u : 0u;
  prm.per_group = prm.group > 1 ? 0xffffffffu / prm.group + 1u : 0u;
  prm.tiles = p.tiles;
  prm.W = p.W;
  // (not 0: a score of -inf, which stands for a token that is not seen, stays one)
  prm.scale = std::max(fabsf(a.sm_scale) * LOG2E, FLT_MIN);
  prm.flip = a.sm_scale < 0.f ? 0x80008000u : 0u;
  if (p.W > 0) {
    const size_t slots = 2 * (size_t)p.W * c.heads, rows = 16 * (size_t)p.qt;
    char* at = (char*)ws;
    prm.part_o = (float*)at; at += rounded(slots * rows * c.head_dim * 4);
    prm.part_ml = (float*)at; at += rounded(slots * rows * 8);
    prm.flags = (unsigned long long*)at;
    prm.mark = next_epoch();
  }
  const int64_t blocks = (p.W > 0 ? p.W : p.units) * c.heads;
  if (blocks > 0x7fffffffLL) return BSATTN_ERR_RANGE;
  const bool bf16 = c.dtype == BSATTN_BF16;
  if (c.head_dim == 64) bf16 ? launch_tiles<64, true>(prm, p.qt, (unsigned)blocks, st) : launch_tiles<64, false>(prm, p.qt, (unsigned)blocks, st);
  else if (c.head_dim == 128) bf16 ? launch_tiles<128, true>(prm, p.qt, (unsigned)blocks, st) : launch_tiles<128, false>(prm, p.qt, (unsigned)blocks, st);
  else bf16 ? launch_tiles<256, true>(prm, p.qt, (unsigned)blocks, st) : launch_tiles<256, false>(prm, p.qt, (unsigned)blocks, st);
  return launch_status();
}

}  // namespace bsattn
