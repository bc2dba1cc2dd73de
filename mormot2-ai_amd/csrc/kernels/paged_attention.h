// paged_attention.h - attention of one new token of each sequence over its pages: the
// kernel that paged.hip, paged_q8.hip and paged_shared.hip (own tokens) instantiate.
#pragma once

#include <type_traits>

#include "common.h"
#include "../paged.h"

namespace ihip {

// --------------------------------------------------------- paged_attention
struct PagedAttnArgs {
  const float* q;
  const char *kc, *vc;
  const int *table, *lengths;
  const int* offsets;  // [seqs + 1]: a sequence's row of q and y is its last, offsets[s + 1] - 1; null: row s (both below rows)
  float* y;
  const float* sinks;
  float* part;  // [blocks][2][16 * hd + 32]: a block's pieces of sequences that other blocks share
  int* done;    // [blocks] counters, 32 ints apart, zero between launches
  int64_t q_stride, pages, page_stride, slot_stride, head_stride, window;
  float scale;  // of the scores, times log2 e
  int32_t seqs, heads, kvh, hd, page_size, max_pages;
  int32_t group, tiles;  // query heads of a KV head, in tiles of 16
  int32_t rows;          // of q and y
  int32_t cus;
};

// 8-bit pages: single scales beside the codes, of key `at` of page p at p * s_page + at *
// s_slot + (KV head) * s_head
struct PagedAttn8Args : PagedAttnArgs {
  const float *ks, *vs;
  int64_t s_page, s_slot, s_head;
};

// groups of sequences whose first tokens are the same (paged_shared.hip): the own tokens'
// attention joined with that of the prefix, which a launch before has left
struct PagedSharedArgs : PagedAttn8Args {
  const int *members, *shared;  // [groups + 1], [groups]: a group's sequences, their common tokens
  float* pieces;  // [blocks][2][16 CT (hd + 2)]: parts of a prefix that blocks share
  float* sums;    // [seqs][heads][2], the maximum (base 2) and sum of a prefix that is one block's, its values in y
  int* plan;      // SHARED_PLAN's numbers, then [groups][3]: tiles before the group's, keys' tiles, columns' tiles
  int32_t groups, pad;
};
constexpr int SHARED_PLAN = 4;  // all tiles, the blocks that share them

typedef _Float16 half2 __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));
typedef uint32_t uintx2 __attribute__((ext_vector_type(2)));

constexpr float LOG2E = 1.44269504088896340736f;
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ bool finite(float x) { return (float_bits(x) & 0x7f800000u) != 0x7f800000u; }

// a value of the cache; T: 0 float, 1 half, 2 bf16, 3 an 8-bit code (without its scale)
template <int T>
__device__ __forceinline__ float load1(const char* p)
{
  if constexpr (T == 0) return *(const float*)p;
  else if constexpr (T == 3) return (float)*(const int8_t*)p;
  else if constexpr (T == 1) return half_to_float(*(const uint16_t*)p);
  else return bits_float((uint32_t)*(const uint16_t*)p << 16);
}

template <int T>
__device__ __forceinline__ floatx4 mfma16(uintx4 a, uintx4 b, floatx4 c)
{
  if constexpr (T == 1 || T == 3)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// two 8-bit codes as halves: byte b of code + 128 behind 0x64 is the half 1152 + code,
// and the difference is exact
__device__ __forceinline__ uint32_t halves_of(uint32_t biased)
{
  const half2 h = __builtin_bit_cast(half2, biased) - half2{(_Float16)1152.f, (_Float16)1152.f};
  return __builtin_bit_cast(uint32_t, h);
}
// four codes (each + 128) of a word as halves, in their order
__device__ __forceinline__ uintx2 codes4(uint32_t w)
{
  return uintx2{halves_of(__builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)),
                halves_of(__builtin_amdgcn_perm(0x64646464u, w, 0x04030402u))};
}

// two singles as NP parts of the cache's type that add up to them: halves (the
// first towards zero, the second to nearest: 22 bits, of values scaled into a
// half's normal range) or bf16 (towards zero: all 24 bits)
template <int T>
__device__ __forceinline__ void split2(float x, float y, uint32_t* part)
{
  if constexpr (T == 1 || T == 3) {
    const auto hi = __builtin_amdgcn_cvt_pkrtz(x, y);
    part[0] = __builtin_bit_cast(uint32_t, hi);
    const _Float16 lx = (_Float16)(x - (float)hi[0]), ly = (_Float16)(y - (float)hi[1]);
    part[1] = (uint32_t)__builtin_bit_cast(uint16_t, lx) | (uint32_t)__builtin_bit_cast(uint16_t, ly) << 16;
  } else {
#pragma unroll
    for (int i = 0; i < 3; i++) {
      const uint32_t hx = float_bits(x), hy = float_bits(y);
      part[i] = __builtin_amdgcn_perm(hy, hx, 0x07060302u);
      x = x - bits_float(hx & 0xffff0000u);
      y = y - bits_float(hy & 0xffff0000u);
    }
  }
}

// At least 64 clocks: what reads the products before it may lie behind any branch, where
// the compiler counts the wait states (40 clocks at most) along one of the ways alone.
// (A sleep: an asm statement costs these kernels two registers, and bf16 heads of 128 the
// second block of a CU.)
__device__ __forceinline__ void products_done()
{
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_sleep(1);
  __builtin_amdgcn_sched_barrier(0);
}

// a block's barrier for what it has in LDS: loads and stores of memory stay on their way
// (__syncthreads waits for them)
__device__ __forceinline__ void lds_barrier()
{
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

__device__ __forceinline__ uint64_t lane_value(uint64_t v, int lane)
{
  return (uint64_t)__builtin_amdgcn_readlane((uint32_t)(v >> 32), lane) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((uint32_t)v, lane);
}

// the maximum and the sum over the four lanes of a head (lanes c, c + 16, c + 32,
// c + 48)
__device__ __forceinline__ float quad_max(float v)
{
  v = fmaxf(v, xpart<16>(v));
  return fmaxf(v, xpart<32>(v));
}
__device__ __forceinline__ float quad_sum(float v)
{
  v = v + xpart<16>(v);
  return v + xpart<32>(v);
}

template <typename A>
constexpr bool is_shared = false;
template <>
constexpr bool is_shared<PagedSharedArgs> = true;

// the last g of the n with first[g] <= i, first[0] <= i (first ascending; any other
// array ends within it too)
__device__ __forceinline__ int find_last(const int* first, int n, int i)
{
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= i) lo = mid;
    else hi = mid;
  }
  return lo;
}

// `all` tiles shared out evenly over B blocks: block i takes first(i) .. first(i + 1) - 1
struct PieceShare {
  uint32_t all, B, quot, rem;
  __device__ __forceinline__ PieceShare(uint32_t a, uint32_t b) : all(a), B(b), quot(a / b), rem(a % b) {}
  __device__ __forceinline__ uint32_t first(uint32_t i) const { return i * quot + i * rem / B; }
  __device__ __forceinline__ uint32_t block_of(uint32_t u) const
  {
    uint32_t k = (uint32_t)((double)u * B / all);
    while (k > 0 && first(k) > u) k--;
    while (first(k + 1) <= u) k++;
    return k;
  }
};

// what a block works on: a sequence, one of its KV heads, 16 of that one's query heads
struct AttnItem {
  int s, row, kv;   // sequence, its row of q and y, KV head
  int heads;        // query heads of the tile
  int head0;        // the first of them
};

template <int T, int D>
struct AttnShape {
  static constexpr int ES = T == 0 ? 4 : T == 3 ? 1 : 2;  // bytes of a value
  static constexpr int KS = T == 0 ? 16 : 32;          // keys of a wave's step
  static constexpr int DS = D == 512 ? 2 : 1;          // waves that share a head's dimensions (registers)
  static constexpr int DW = D / DS;                    // dimensions of a wave
  static constexpr int KG = 4 / DS;                    // groups of keys: the others' waves
  static constexpr int TK = KG * KS;                   // keys of a block's tile
  static constexpr int NT = KS / 16;                   // score tiles of a step
  static constexpr int QL = 16 / ES;                   // values of a key load
  static constexpr int NQ = DW / (4 * QL);             // key loads of a lane and key
  static constexpr int FL = T == 0 ? 4 : 8;            // values of a lane in a product's factor
  static constexpr int NF = DW / (4 * FL);             // factors of a lane and key
  static constexpr int NP = T == 0 ? 1 : T == 2 ? 3 : 2;  // parts of a single value
  static constexpr int VL = T == 3 ? DW / 16 : T != 0 && D > 64 ? 8 : 4;  // values of a value load
  static constexpr int NJ = DW / (16 * VL);            // value loads of a lane and key
  static constexpr int OS = D + 4;                     // a head's row in o_s
  // weights enter the product times this: into the halves' normal range. The two parts
  // hold 22 bits of those down to 2^-18 of the largest; smaller ones are off by 2^-40 of
  // the largest at most. (8-bit pages: of weights times their values' scales, off by 2^-39
  // of the largest scale that the wave has met, whatever that one's weight)
  static constexpr float PS = T == 1 || T == 3 ? 32768.f : 1.f;

  // the first of the FL values that lane group g has of factor f: 8-bit keys come in loads
  // of 16 values, two factors each
  static __device__ __forceinline__ int factor(int f, int g)
  {
    return T == 3 ? (f >> 1) * 64 + g * 16 + (f & 1) * 8 : f * 4 * FL + g * FL;
  }
};

template <int T>
struct AttnScales {};
template <>
struct AttnScales<3> {
  float sc[4][64];  // the steps' scales, a wave's 32 keys' and then its values'
};

template <int T, int D>
struct AttnLds : AttnScales<T> {
  using S = AttnShape<T, D>;
  uintx4 q[S::NP * S::DS * S::NF * 64];  // the query tile as the matrix cores take it, by lane
  float o[16 * S::OS];           // a piece's values
  float m[16], l[16];            // its maxima and sums
  float wm[4][16], wl[4][16];    // the waves'
  float qs[16];                  // powers of two that the queries were divided by
  int64_t off[4][2][S::KS];      // byte offsets of the steps' keys
  floatx4 x[S::DS > 1 ? 2 : 1][S::DS > 1 ? 4 : 1][S::NT][64];  // the waves' shares of the scores
};

// a tile's heads' part of a prefix (PagedSharedArgs), in LDS
struct AttnPrefix {
  float m[16], l[16];          // its maxima (base 2) and sums
  int first[16], count[16];    // the blocks of its pieces; count 0: in y and sums
  int col[16];                 // a head's column in the pieces
  int members[64], shared[64]; // the groups, of 3 to 63 (of fewer the search reads no more)
};

// a sequence's group, -1 where it has none, and how many of its tokens are read once for
// the group
__device__ __forceinline__ int64_t shared_tokens(const PagedSharedArgs& a, const AttnPrefix& px, int seq, int& g)
{
  g = -1;
  if (a.groups < 1) return 0;
  int at, m0, m1, n0;
  if (a.groups > 2 && a.groups < 64) {
    at = find_last(px.members, a.groups, seq);
    m0 = px.members[at], m1 = px.members[at + 1], n0 = px.shared[at];
  } else {
    at = find_last(a.members, a.groups, seq);
    m0 = a.members[at], m1 = a.members[at + 1], n0 = a.shared[at];
  }
  if (seq < m0 || seq >= m1) return 0;
  const int64_t n = paged_common(m0, m1, n0, a.seqs, a.max_pages, a.page_size);
  if (n > 0) g = at;
  return n;
}

// The heads of a piece whose sums are not all finite, again by the formula's own
// steps in single: the matrix cores' parts turn an infinity into NaN (0 times it
// is added), and a key of score -infinity has weight 0. Waves take keys in turn,
// lanes dimensions. Slow, and only for such data.
template <int T, int D, typename A>
__device__ __forceinline__ void paged_walk(const A& a, const AttnItem& it, int64_t j0, int64_t j1,
                                           AttnLds<T, D>& s)
{
  using S = AttnShape<T, D>;
  constexpr int NV = D / 64;
  float* const tmp = (float*)s.q;
  const int t = threadIdx.x, lane = t & 63, w = t >> 6;
  for (int h = 0; h < it.heads; h++) {
    float q[NV], acc[NV];
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const int d = lane + 64 * i;
      q[i] = d < a.hd ? a.q[it.row * a.q_stride + (int64_t)(it.head0 + h) * a.hd + d] * a.scale : 0.f;
      acc[i] = 0.f;
    }
    float m = -__builtin_inff(), l = 0.f;
    for (int64_t j = j0 + w; j < j1; j += 4) {
      const uint32_t pg = (uint32_t)j / (uint32_t)a.page_size;
      const int page = a.table[(int64_t)it.s * a.max_pages + pg];
      const int64_t at = paged_value(page, (int)((uint32_t)j % (uint32_t)a.page_size), a.pages, a.page_stride, a.slot_stride);
      if (at < 0) continue;
      const int64_t row = (at + it.kv * a.head_stride) * S::ES;
      float x = 0.f, vscale = 1.f, kscale = 1.f;
      if constexpr (T == 3) {
        const int64_t sc = page * a.s_page + (int64_t)((uint32_t)j % (uint32_t)a.page_size) * a.s_slot + it.kv * a.s_head;
        kscale = a.ks[sc];
        vscale = a.vs[sc];
      }
#pragma unroll
      for (int i = 0; i < NV; i++)
        if (lane + 64 * i < a.hd) x = __builtin_fmaf(q[i], load1<T>(a.kc + row + (lane + 64 * i) * S::ES), x);
      x = wave_sum(x, 64);
      if constexpr (T == 3) x *= kscale;
      if (x == -__builtin_inff()) continue;
      const float m2 = x > m || x != x ? x : m;
      const float f = m == -__builtin_inff() ? 0.f : exp2_fast(m - m2), p = exp2_fast(x - m2);
      l = l * f + p;
      m = m2;
#pragma unroll
      for (int i = 0; i < NV; i++)
        if (lane + 64 * i < a.hd)
          acc[i] = __builtin_fmaf(p, load1<T>(a.vc + row + (lane + 64 * i) * S::ES) * (T == 3 ? vscale : 1.f), acc[i] * f);
    }
#pragma unroll
    for (int i = 0; i < NV; i++) tmp[w * D + lane + 64 * i] = acc[i];
    if (lane == 0) {
      s.wm[w][0] = m;
      s.wl[w][0] = l;
    }
    __syncthreads();
    float M = -__builtin_inff(), L = 0.f, f[4];
    for (int i = 0; i < 4; i++) M = s.wm[i][0] > M || s.wm[i][0] != s.wm[i][0] ? s.wm[i][0] : M;
    for (int i = 0; i < 4; i++) {
      f[i] = s.wl[i][0] == 0.f ? 0.f : exp2_fast(s.wm[i][0] - M);
      L += f[i] * s.wl[i][0];
    }
    for (int d = t; d < a.hd; d += 256) {
      float v = 0.f;
      for (int i = 0; i < 4; i++)
        if (s.wl[i][0] != 0.f) v += f[i] * tmp[i * D + d];
      s.o[h * S::OS + d] = v;
    }
    if (t == 0) {
      s.m[h] = M;
      s.l[h] = L;
    }
    __syncthreads();
  }
}

// the query tile into LDS in the lanes' order: lane (c, g) = (l & 15, l >> 4) holds
// head c, values 4 QL i + QL g .. of load i; heads past the tile and values past
// head_dim are 0. Halves: a head's values times a power of two, so that the
// largest is below 2^14 and the second parts stay normal.
template <int T, int D>
__device__ __forceinline__ void stage_query(const PagedAttnArgs& a, const AttnItem& it, AttnLds<T, D>& s)
{
  using S = AttnShape<T, D>;
  const int t = threadIdx.x;
  const float* const q = a.q + it.row * a.q_stride + (int64_t)it.head0 * a.hd;
  if constexpr (T == 1) {
    const int c = t >> 4;
    float top = 0.f;
    if (c < it.heads)
      for (int d = t & 15; d < a.hd; d += 16) top = fmaxf(top, fabsf(q[c * a.hd + d] * a.scale));
    top = fmaxf(top, xpart<1>(top));
    top = fmaxf(top, xpart<2>(top));
    top = fmaxf(top, xpart<4>(top));
    top = fmaxf(top, xpart<8>(top));
    if ((t & 15) == 0) {
      int e = (int)(float_bits(top) >> 23) - 126;  // top < 2^e
      if (top == 0.f || !finite(top)) e = 14;
      s.qs[c] = ldexpf(1.f, max(e - 14, -120));
    }
    __syncthreads();
  }
  for (int i = t; i < S::DS * S::NF * 64; i += 256) {
    const int c = i & 15, d0 = S::factor(i >> 6, (i >> 4) & 3);
    float v[S::FL];
    const bool in = c < it.heads && d0 < a.hd;
    float f = a.scale;
    if constexpr (T == 1) f = 1.f / s.qs[c];
#pragma unroll
    for (int j = 0; j < S::FL; j++) {
      v[j] = in ? q[c * a.hd + d0 + j] : 0.f;
      v[j] = T == 1 ? v[j] * a.scale * f : v[j] * f;
    }
    if constexpr (T == 0) {
      s.q[i] = uintx4{float_bits(v[0]), float_bits(v[1]), float_bits(v[2]), float_bits(v[3])};
    } else {
      uint32_t part[4][S::NP];
#pragma unroll
      for (int j = 0; j < 4; j++) split2<T>(v[2 * j], v[2 * j + 1], part[j]);
#pragma unroll
      for (int n = 0; n < S::NP; n++) s.q[n * S::DS * S::NF * 64 + i] = uintx4{part[0][n], part[1][n], part[2][n], part[3][n]};
    }
  }
  __syncthreads();
}

// The same with all of a thread's factors on their way at once (8-bit pages and groups);
// gives the power of two of the lane's head
template <int T, int D>
__device__ __forceinline__ float stage_query_once(const PagedAttnArgs& a, const AttnItem& it, AttnLds<T, D>& s)
{
  using S = AttnShape<T, D>;
  constexpr int TILE = S::DS * S::NF * 64, R = (TILE + 255) / 256;
  const int t = threadIdx.x, c = t & 15;
  const float* const q = a.q + it.row * a.q_stride + (int64_t)(it.head0 + min(c, it.heads - 1)) * a.hd;
  float v[R][S::FL];
#pragma unroll
  for (int r = 0; r < R; r++) {
    const int i = t + 256 * r, d0 = S::factor(i >> 6, (i >> 4) & 3);
    const bool in = i < TILE && c < it.heads && d0 < a.hd;
#pragma unroll
    for (int j = 0; j < S::FL; j++) v[r][j] = in ? q[d0 + j] : 0.f;
  }
  float power = 1.f;
  if constexpr (T == 1 || T == 3) {
    float top = 0.f;
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
      for (int j = 0; j < S::FL; j++) top = fmaxf(top, fabsf(v[r][j] * a.scale));
    top = quad_max(top);
    if ((t & 63) < 16) s.wm[t >> 6][c] = top;
    lds_barrier();
    top = fmaxf(fmaxf(s.wm[0][c], s.wm[1][c]), fmaxf(s.wm[2][c], s.wm[3][c]));
    int e = (int)(float_bits(top) >> 23) - 126;  // top < 2^e
    if (top == 0.f || !finite(top)) e = 14;
    power = ldexpf(1.f, max(e - 14, -120));
  }
#pragma unroll
  for (int r = 0; r < R; r++) {
    const int i = t + 256 * r;
    if (i >= TILE) break;
    const float f = T == 1 || T == 3 ? 1.f / power : a.scale;
#pragma unroll
    for (int j = 0; j < S::FL; j++) v[r][j] = T == 1 || T == 3 ? v[r][j] * a.scale * f : v[r][j] * f;
    if constexpr (T == 0) {
      s.q[i] = uintx4{float_bits(v[r][0]), float_bits(v[r][1]), float_bits(v[r][2]), float_bits(v[r][3])};
    } else {
      uint32_t part[4][S::NP];
#pragma unroll
      for (int j = 0; j < 4; j++) split2<T>(v[r][2 * j], v[r][2 * j + 1], part[j]);
#pragma unroll
      for (int n = 0; n < S::NP; n++) s.q[n * TILE + i] = uintx4{part[0][n], part[1][n], part[2][n], part[3][n]};
    }
  }
  lds_barrier();
  return power;
}

// Attention of one token of each sequence. The work of all sequences and KV heads
// is one row of tiles of TK keys, shared out evenly over the grid's blocks
// (ragged lengths leave no block idle, and a captured grid fits the lengths of
// every replay); a block walks its tiles in pieces of one (sequence, KV head). A
// piece that is the whole of its item is written at once; the others go to
// `part`, and the last block of an item to arrive joins them in order.
//
// A wave takes KS keys a step. Scores are K q^T with the keys as the matrix
// cores' rows and the group's heads as columns (16 of them, zeros past the
// group), so that lane (c, g) holds head c's scores of keys 4 g .. 4 g + 3 of each
// 16 - which is how the value product takes its weights: values V^T with
// dimensions as rows, keys as the inner index, each lane loading 8 dimensions of
// the 8 keys that it has the weights of and turning them by byte permutes in its
// registers. No key, value or weight goes through LDS, and the running maximum, sum
// and rescale are a lane's own. Queries and weights enter as 2 half or 3 bf16
// parts (f32 caches: the f32 matrix cores), so the sums are those of single.
//
// HBM bound: the cache is read once (again for each 16 query heads of a KV head
// beyond 16). 64 sequences of 16384 keys, 8 KV heads of 128 in bf16 705 to 718 us, 6.0
// TB/s of the 6.2 that a streaming read takes; single 6.3, heads of 256 5.5, of 64 5.0 to
// 5.8; few long sequences lose the join (three of 110000: 136 us, 5.0), one short one
// is a chain of round trips (1152 keys 12.5 us). Pages of [kv_heads, page_size,
// head_dim] read up to 6% faster than [page_size, kv_heads, head_dim]. Heads
// beyond 256 give a wave half of the dimensions, two waves adding their shares of the
// scores in LDS, as the values of 512 do not fit the registers beside the keys (one
// wave each, spilling: 16 sequences of 8192, 2 KV heads 252 us, so 116).
template <int T, int D, bool FULL, typename A>
__device__ __forceinline__ void paged_attention_t(const A& a)
{
  using S = AttnShape<T, D>;
  __shared__ AttnLds<T, D> s;
  const int t = threadIdx.x, lane = t & 63, c = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const uint32_t grid = gridDim.x, b = blockIdx.x, per = a.kvh * a.tiles;
  const int hd = FULL ? D : a.hd, row_out = a.heads * a.hd;

  __shared__ typename std::conditional<is_shared<A>, AttnPrefix, int>::type px;
  if constexpr (is_shared<A>) {
    // the groups into LDS, where a sequence's is searched (each wave for itself, the same)
    if (a.groups > 2 && a.groups < 64) {
      px.members[lane] = lane <= a.groups ? a.members[lane] : 0;
      px.shared[lane] = lane < a.groups ? a.shared[lane] : 0;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
  }
  // a sequence's row, -1 where it has none in this step
  auto row_of = [&](int seq) {
    return a.offsets ? paged_row(a.offsets[seq], a.offsets[seq + 1], a.rows) : paged_row(seq, seq + 1, a.rows);
  };
  auto tiles_of = [&](int seq, int64_t& lo, int64_t& hi) {
    lo = hi = 0;
    if constexpr (is_shared<A>) {
      // (a sequence without a token of its own has a tile without keys, for its prefix)
      const int length = a.lengths[seq], row = row_of(seq);
      int grp;
      const int64_t common = shared_tokens(a, px, seq, grp);
      if (row < 0 || length < 0) return 0u;
      paged_range(length, a.window, a.max_pages, a.page_size, &lo, &hi);
      lo = min(hi, common);
      return max(1u, (uint32_t)((hi - lo + S::TK - 1) / S::TK));
    }
    if (row_of(seq) < 0) return 0u;
    paged_range(a.lengths[seq], a.window, a.max_pages, a.page_size, &lo, &hi);
    return (uint32_t)((hi - lo + S::TK - 1) / S::TK);
  };
  // the heads' part of their sequence's prefix; whether there is one
  auto prefix_of = [&](const AttnItem& it) {
    if constexpr (is_shared<A>) {
      int grp;
      if (shared_tokens(a, px, it.s, grp) == 0) return false;
      const int pall = a.plan[0], pb = a.plan[1], pct = a.plan[2] * 16;
      if (pall <= 0) return false;
      const uint32_t before = a.plan[SHARED_PLAN + 3 * grp], pn = a.plan[SHARED_PLAN + 3 * grp + 1];
      const int cts = a.plan[SHARED_PLAN + 3 * grp + 2];
      const int64_t size = (int64_t)pct * (a.hd + 2);
      const int h = t >> 4;
      lds_barrier();
      if (h < it.heads) {
        const int col = (it.s - a.members[grp]) * a.group + it.head0 - it.kv * a.group + h;
        const uint32_t u0 = before + (uint32_t)(it.kv * cts + col / pct) * pn;
        const PieceShare share(pall, pb);
        const int b0 = share.block_of(u0), b1 = share.block_of(u0 + pn - 1);
        const int c16 = col % pct;
        float m = -__builtin_inff(), l = 0.f;
        if (b0 == b1) {
          if ((t & 15) == 0) {
            const float* const e = a.sums + 2 * ((int64_t)it.s * a.heads + it.head0 + h);
            m = e[0];
            l = e[1];
          }
        } else {
          for (int i = t & 15; i <= b1 - b0; i += 16) {
            const float* const e = a.pieces + (2 * (int64_t)(b0 + i) + (i == 0)) * size + pct * a.hd + c16;
            const float pm = e[0], pl = e[pct];
            if (pl == 0.f) continue;
            const float m2 = pm > m || pm != pm ? pm : m;
            l = (m == -__builtin_inff() ? 0.f : l * exp2_fast(m - m2)) + pl * exp2_fast(pm - m2);
            m = m2;
          }
        }
        auto meet = [&](float om, float ol) {
          const float m2 = om > m || om != om ? om : m;
          l = (l == 0.f ? 0.f : l * exp2_fast(m - m2)) + (ol == 0.f ? 0.f : ol * exp2_fast(om - m2));
          m = m2;
        };
        meet(xpart<1>(m), xpart<1>(l));
        meet(xpart<2>(m), xpart<2>(l));
        meet(xpart<4>(m), xpart<4>(l));
        meet(xpart<8>(m), xpart<8>(l));
        if ((t & 15) == 0) {
          px.m[h] = m;
          px.l[h] = l;
          px.first[h] = b0;
          px.count[h] = b0 == b1 ? 0 : b1 - b0 + 1;
          px.col[h] = c16;
        }
      }
      lds_barrier();
      return true;
    } else {
      return false;
    }
  };
  // 4 values of a head, own ones over the maximum m with sum l, joined with the prefix's and
  // the sink's weight
  auto with_prefix = [&](const AttnItem& it, int h, int d, float m, float l, float (&v)[4]) {
    if constexpr (is_shared<A>) {
      const int pct = a.plan[2] * 16;
      const int64_t size = (int64_t)pct * (a.hd + 2);
      const float pm = px.m[h], pl = px.l[h];
      float M = -__builtin_inff();
      auto top = [&](float x) { M = x > M || x != x ? x : M; };
      if (l != 0.f) top(m);
      if (pl != 0.f) top(pm);
      // (a sink above all of them has weight 1, an infinite one too, as in finish)
      const float sk = a.sinks ? a.sinks[it.head0 + h] * LOG2E : -__builtin_inff();
      const bool sink = sk > M;
      if (sink) M = sk;
      const float fo = l != 0.f ? exp2_fast(m - M) : 0.f, fp = pl != 0.f ? exp2_fast(pm - M) : 0.f;
      const float L = l * fo + pl * fp + (sink ? 1.f : sk != -__builtin_inff() ? exp2_fast(sk - M) : 0.f);
      float p[4] = {0.f, 0.f, 0.f, 0.f};
      if (pl != 0.f) {
        if (px.count[h] == 0) {
          const float* const e = a.y + (int64_t)it.row * a.heads * a.hd + (int64_t)(it.head0 + h) * a.hd + d;
#pragma unroll
          for (int i = 0; i < 4; i++) p[i] = e[i];
        } else {
          const int np = px.count[h];
          // (4 pieces' loads on their way at once)
          for (int i0 = 0; i0 < np; i0 += 4) {
            float x[4];
            floatx4 o4[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
              const int i = min(i0 + k, np - 1);
              const float* const e = a.pieces + (2 * (int64_t)(px.first[h] + i) + (i == 0)) * size;
              x[k] = e[pct * a.hd + px.col[h]];
              o4[k] = *(const floatx4*)(e + (int64_t)px.col[h] * a.hd + d);
            }
#pragma unroll
            for (int k = 0; k < 4; k++) {
              const float w2 = i0 + k >= np || x[k] == -__builtin_inff() ? 0.f : exp2_fast(x[k] - pm);
#pragma unroll
              for (int j = 0; j < 4; j++) p[j] = __builtin_fmaf(w2, w2 != 0.f ? o4[k][j] : 0.f, p[j]);
            }
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float x = (fo != 0.f ? v[i] * fo : 0.f) + (fp != 0.f ? p[i] * fp : 0.f);
        v[i] = L != 0.f && (l != 0.f || pl != 0.f) ? x / L : 0.f;
      }
    }
  };
  // What an item (a sequence's KV head) costs beside its tiles of keys, in tiles: its query,
  // the waves' meeting, the prefix. The blocks share out tiles and these, so that one
  // with many short items has as much to do (three prompts' 480 items of 1 to 8 tiles, on
  // one block a CU: 140 us without, the others through at 50).
  constexpr uint32_t OV = T == 3 || is_shared<A> ? 3 : 0;
  // all tiles (each wave for itself); rows without a key are zeros
  uint32_t all = 0, n0 = 0, live = 0;  // tiles, those of the lane's first sequence; sequences with any
  uint32_t longest = 0;
  int64_t lo0 = 0, hi0 = 0;  // of the first 64 sequences, a lane each
  for (int s0 = 0; s0 < a.seqs; s0 += 64) {
    const int seq = s0 + lane;
    uint32_t n = 0;
    bool zero = false;
    if (seq < a.seqs) {
      int64_t lo, hi;
      n = tiles_of(seq, lo, hi);
      if (s0 == 0) n0 = n, lo0 = lo, hi0 = hi;
      zero = !is_shared<A> && n == 0 && a.lengths[seq] >= 0 && row_of(seq) >= 0 && (uint32_t)seq % grid == b;
    }
    if (n) all += (n + OV) * per;
    if (OV) longest = max(longest, n);
    live += __popcll(__ballot(n != 0));
    for (uint64_t z = __ballot(zero); z; z &= z - 1) {
      float* const y = a.y + (int64_t)row_of(s0 + __builtin_ctzll(z)) * row_out;
      for (int i = t; i < row_out; i += 256) y[i] = 0.f;
    }
  }
  all = __builtin_amdgcn_readfirstlane(wave_sum(all, 64));
  // Block i of B takes tiles first(i) .. first(i + 1) - 1. One block a CU where the
  // blocks have 32 tiles and more and the items 24 (their streams then cover each
  // other's latencies: 64 sequences of 8192, 8 KV heads of 64, two blocks a CU 222 us,
  // one 196; 16384 of 128 731, 718; of 200 sequences up to 4000, 16 tiles an item, the
  // starts and ends of pieces need the second block: 301, one 313), else all.
  // Many items of few tiles go to a block each and whole, in turn: what a block with two
  // parts of them spends is their starts and ends, not their tiles.
  const bool whole = OV && live * per * 4 >= grid && wave_max((int)longest) <= 8;
  const uint32_t B = whole ? min(grid, live * per) : T != 3 && all >= 32 * grid && all / 24 >= live * per ? min(grid, (uint32_t)a.cus) : min(grid, all);
  if (b >= B) return;
  const uint32_t quot = all / B, rem = all % B;
  auto first = [&](uint32_t i) { return i * quot + i * rem / B; };
  uint32_t u = first(b);
  uint32_t end = first(b + 1);
  for (uint32_t turn = b;; turn += B) {
  if (OV && whole) {
    if (turn >= live * per) return;
    u = turn;
  }
  // the sequence of tile u (or of item u of those that are whole)
  int seq = 0;
  uint32_t before = 0, n = 0;  // tiles before the sequence, tiles of a KV head's item
  int64_t lo = 0, hi = 0;
  for (int s0 = 0;; s0 += 64) {
    uint32_t m = s0 == 0 ? n0 : 0;
    if ((s0 > 0 || (OV && whole && turn != b && a.seqs > 64)) && s0 + lane < a.seqs) m = tiles_of(s0 + lane, lo0, hi0);
    const uint32_t items = m;
    if (OV && m) m = whole ? 1 : m + OV;
    m *= per;
    uint32_t upto = m;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const uint32_t o = __shfl_up(upto, d, 64);
      if (lane >= d) upto += o;
    }
    const uint64_t there = __ballot(before + upto > u);
    if (there) {
      const int f = __builtin_ctzll(there);
      seq = __builtin_amdgcn_readfirstlane(s0 + f);
      before += __builtin_amdgcn_readlane(upto - m, f);
      n = __builtin_amdgcn_readlane(items, f);
      lo = (int64_t)lane_value((uint64_t)lo0, f);
      hi = (int64_t)lane_value((uint64_t)hi0, f);
      break;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }

  if (OV && whole) {
    u = (u - before) * (n + OV);
    end = u + n + OV;
    before = 0;
  }

  for (;;) {
    // (of an item the first OV are nothing but its cost; its tiles lie behind them)
    const uint32_t item = (u - before) / (n + OV), at = (u - before) - item * (n + OV);
    const uint32_t tile0 = at > OV ? at - OV : 0, upto = min(n + OV, at + (end - u));
    const uint32_t tile1 = upto > OV ? upto - OV : 0;
    if (OV && tile1 == tile0) return;  // (the block's range ends before the item's first tile)
    AttnItem it;
    it.s = seq;
    it.row = row_of(seq);
    it.kv = item / a.tiles;
    const int tile16 = item - it.kv * a.tiles;
    it.heads = min(16, a.group - 16 * tile16);
    it.head0 = it.kv * a.group + 16 * tile16;
    const char* const kb = a.kc + (int64_t)it.kv * a.head_stride * S::ES;
    const char* const vb = a.vc + (int64_t)it.kv * a.head_stride * S::ES;
    const float* sb = nullptr;  // 8-bit pages: of the lane's half, keys' or values'
    float scale = 0.f;          // the next step's, of the lane's key
    if constexpr (T == 3) sb = (lane < S::KS ? a.ks : a.vs) + (int64_t)it.kv * a.s_head;
    const int* const table = a.table + (int64_t)seq * a.max_pages;
    const int kg = w / S::DS, dh = w % S::DS;  // the wave's keys of a tile, its dimensions
    const int64_t wlo = lo + kg * S::KS;
    const int64_t jend = min(hi, lo + (int64_t)tile1 * S::TK);  // the piece's keys end here
    // a step's key of this lane: its page's table entry
    auto entry = [&](uint32_t tile) {
      const int64_t j = wlo + (int64_t)tile * S::TK + (lane & (S::KS - 1));
      return j < jend ? table[(uint32_t)j / (uint32_t)a.page_size] : -1;
    };
    // the offsets of a step's keys into LDS, the keys that are there as bits
    auto locate = [&](uint32_t tile, int page) {
      const int64_t j = wlo + (int64_t)tile * S::TK + (lane & (S::KS - 1));
      const int64_t at = paged_value(page, (int)((uint32_t)j % (uint32_t)a.page_size), a.pages, a.page_stride, a.slot_stride);
      if (lane < S::KS) s.off[w][tile & 1][lane] = at < 0 ? 0 : at * S::ES;
      if constexpr (T == 3)
        scale = at < 0 ? 0.f : sb[page * a.s_page + (int64_t)((uint32_t)j % (uint32_t)a.page_size) * a.s_slot];
      // other lanes read it: no instruction, but no reordering or forwarding past here
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      return (uint32_t)__ballot(at >= 0) & (uint32_t)((1ull << S::KS) - 1);
    };
    uint32_t tile = tile0;
    const int page0 = entry(tile);
    int page = entry(tile + 1);
    float sscale = 1.f;
    if constexpr (OV != 0) {
      sscale = stage_query_once<T, D>(a, it, s);
    } else {
      stage_query<T, D>(a, it, s);
      if constexpr (T == 1) sscale = s.qs[c];
    }

    uintx4 kr[S::NT][S::NQ];
    auto load_keys = [&](uint32_t tile) {
#pragma unroll
      for (int i = 0; i < S::NT; i++) {
        const char* const p = kb + s.off[w][tile & 1][16 * i + c];
#pragma unroll
        for (int j = 0; j < S::NQ; j++) {
          const int d0 = dh * S::DW + j * 4 * S::QL + g * S::QL;
          const bool in = FULL || d0 < hd;
          kr[i][j] = *(const uintx4*)(p + (in ? d0 : 0) * S::ES);
          if (!in) kr[i][j] = uintx4{0, 0, 0, 0};
        }
      }
    };

    floatx4 o[S::NJ][S::VL];
#pragma unroll
    for (int i = 0; i < S::NJ; i++)
#pragma unroll
      for (int j = 0; j < S::VL; j++) o[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
    float m = -__builtin_inff(), l = 0.f;
    // 8-bit pages: weights enter the product times their value's scale over vtop, a power
    // of two above the largest of those that the wave has met, and the sums are over vtop
    float vtop = 0x1p-100f, vinv = 0x1p100f;
    uint32_t steps = 0;  // of this wave: up to the last tile with a key of its own
    if (S::DS > 1) {
      steps = tile1 - tile0;  // the waves meet in each step
    } else if (wlo + (int64_t)tile0 * S::TK < hi) {
      const uint32_t mine = (uint32_t)((hi - wlo + S::TK - 1) / S::TK);
      steps = min(tile1, mine) - tile0;
    }
    // The scores are read on both sides of branches, and the values' sums in a block that
    // few steps enter and behind the loop: products_done() stands before each. Keys are
    // located and loaded one step past the piece's last too, as a condition there would
    // keep the loads from covering the products: entry() has no page there and the loads
    // read the pool's first row.
    uint32_t there = locate(tile, page0);
    if (steps) load_keys(tile);
    // (what the item's heads have of a prefix, looked up while the first keys are on their way)
    bool pre = false;
    if constexpr (is_shared<A>) pre = prefix_of(it);
    for (uint32_t i = 0; i < steps; i++, tile++) {
      // the step's values, on their way while its scores are formed
      constexpr int NV = 4 * S::NT;  // keys of a lane: 16 q + 4 g + r
      uintx4 vr[NV][S::NJ];
#pragma unroll
      for (int k = 0; k < NV; k++) {
        const char* const p = vb + s.off[w][tile & 1][16 * (k >> 2) + 4 * g + (k & 3)];
#pragma unroll
        for (int j = 0; j < S::NJ; j++) {
          const int d0 = dh * S::DW + j * 16 * S::VL + c * S::VL;
          const char* const v = p + (FULL || d0 < hd ? d0 : 0) * S::ES;
          if constexpr (S::VL * S::ES == 4) {
            vr[k][j] = uintx4{*(const uint32_t*)v, 0, 0, 0};
          } else if constexpr (S::VL * S::ES == 16) {
            vr[k][j] = *(const uintx4*)v;
          } else {
            const uintx2 h = *(const uintx2*)v;
            vr[k][j] = uintx4{h[0], h[1], 0, 0};
          }
        }
      }
      const uint32_t now = there;
      floatx4 ksc[T == 3 ? S::NT : 1], vsc[T == 3 ? S::NT : 1];
      if constexpr (T == 3) {
        s.sc[w][lane] = scale;
        if (__any(lane >= 32 && fabsf(scale) >= vtop)) {
          const uint32_t top = __builtin_amdgcn_readfirstlane(float_bits(wave_max(lane >= 32 ? fabsf(scale) : 0.f)));
          const float v2 = bits_float(min((top & 0x7f800000u) + 0x00800000u, 0x7f000000u));
          const float f = vtop / v2;
          vtop = v2;
          vinv = 1.f / v2;
          products_done();
#pragma unroll
          for (int j = 0; j < S::NJ; j++)
#pragma unroll
            for (int e = 0; e < S::VL; e++) o[j][e] *= f;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int k = 0; k < S::NT; k++) {
          ksc[k] = *(const floatx4*)&s.sc[w][16 * k + 4 * g] * sscale;
          vsc[k] = *(const floatx4*)&s.sc[w][32 + 16 * k + 4 * g] * vinv;
        }
      }
      there = locate(tile + 1, page);
      page = entry(tile + 2);
      floatx4 x[S::NT];
#pragma unroll
      for (int k = 0; k < S::NT; k++) x[k] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < S::NF; j++) {
        uintx4 kf[T == 3 ? S::NT : 1];
        if constexpr (T == 3)
#pragma unroll
          for (int k = 0; k < S::NT; k++) {
            const uintx2 lo = codes4(kr[k][j / 2][2 * (j & 1)] ^ 0x80808080u), hi = codes4(kr[k][j / 2][2 * (j & 1) + 1] ^ 0x80808080u);
            kf[k] = uintx4{lo[0], lo[1], hi[0], hi[1]};
          }
#pragma unroll
        for (int n2 = 0; n2 < S::NP; n2++) {
          const uintx4 q = s.q[(n2 * S::DS * S::NF + dh * S::NF + j) * 64 + lane];
#pragma unroll
          for (int k = 0; k < S::NT; k++) {
            if constexpr (T == 0) {
#pragma unroll
              for (int e = 0; e < 4; e++)
                x[k] = __builtin_amdgcn_mfma_f32_16x16x4f32(bits_float(kr[k][j][e]), bits_float(q[e]), x[k], 0, 0, 0);
            } else if constexpr (T == 3) {
              x[k] = mfma16<T>(kf[k], q, x[k]);
            } else {
              x[k] = mfma16<T>(kr[k][j], q, x[k]);
            }
          }
        }
      }
      load_keys(tile + 1);
      products_done();
      if constexpr (S::DS > 1) {
        // the scores of all dimensions: two waves' shares added, the same sum in both
#pragma unroll
        for (int k = 0; k < S::NT; k++) s.x[tile & 1][w][k][lane] = x[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < S::NT; k++) x[k] += s.x[tile & 1][w ^ 1][k][lane];
      }
      // masked keys: no weight, and values of zero (0 times NaN is NaN)
      float top = -__builtin_inff();
      if (now == (uint32_t)((1ull << S::KS) - 1)) {
#pragma unroll
        for (int k = 0; k < S::NT; k++)
#pragma unroll
          for (int r = 0; r < 4; r++) {
            x[k][r] = x[k][r] * (T == 3 ? ksc[T == 3 ? k : 0][r] : sscale);
            top = fmaxf(top, x[k][r]);
          }
      } else {
#pragma unroll
        for (int k = 0; k < NV; k++) {
          const bool in = now >> (16 * (k >> 2) + 4 * g + (k & 3)) & 1;
          x[k >> 2][k & 3] = in ? x[k >> 2][k & 3] * (T == 3 ? ksc[T == 3 ? k >> 2 : 0][k & 3] : sscale) : -__builtin_inff();
          top = fmaxf(top, x[k >> 2][k & 3]);
          if constexpr (T != 3)  // (codes are finite)
#pragma unroll
            for (int j = 0; j < S::NJ; j++)
              if (!in) vr[k][j] = uintx4{0, 0, 0, 0};
        }
      }
      top = quad_max(top);
      if (__any(top > m)) {
        const float m2 = fmaxf(top, m), f = m == -__builtin_inff() ? 0.f : exp2_fast(m - m2);
        m = m2;
        l *= f;
#pragma unroll
        for (int j = 0; j < S::NJ; j++)
#pragma unroll
          for (int e = 0; e < S::VL; e++) o[j][e] *= f;
      }
      const float shift = m == -__builtin_inff() ? 0.f : m;
      float p[NV];
#pragma unroll
      for (int k = 0; k < NV; k++) {
        p[k] = exp2_fast(x[k >> 2][k & 3] - shift);
        l += p[k];
      }
      if constexpr (T == 0) {
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
          for (int j = 0; j < S::NJ; j++)
#pragma unroll
            for (int e = 0; e < 4; e++)
              o[j][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(bits_float(vr[k][j][e]), p[k], o[j][e], 0, 0, 0);
      } else {
        uint32_t part[4][S::NP];
#pragma unroll
        for (int k = 0; k < 4; k++) {
          if constexpr (T == 3) {
            const floatx4 sc = vsc[k >> 1] * S::PS;
            split2<T>(p[2 * k] * sc[2 * k & 3], p[2 * k + 1] * sc[2 * k + 1 & 3], part[k]);
          } else {
            split2<T>(p[2 * k] * S::PS, p[2 * k + 1] * S::PS, part[k]);
          }
        }
#pragma unroll
        for (int j = 0; j < S::NJ; j++)
#pragma unroll
          for (int e = 0; e < S::VL; e++) {
            uintx4 v;
#pragma unroll
            for (int k = 0; k < 4; k++)
              if constexpr (T == 3) {
                // code e of both keys: the two keys' codes of a pair of dimensions side by
                // side, then those of one of them behind 0x64
                const uint32_t pair = __builtin_amdgcn_perm(vr[2 * k + 1][j][e / 4], vr[2 * k][j][e / 4],
                                                            e & 2 ? 0x07030602u : 0x05010400u) ^ 0x80808080u;
                v[k] = halves_of(__builtin_amdgcn_perm(0x64646464u, pair, e & 1 ? 0x04030402u : 0x04010400u));
              } else
              v[k] = __builtin_amdgcn_perm(vr[2 * k + 1][j][e / 2], vr[2 * k][j][e / 2], e & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
            for (int n2 = 0; n2 < S::NP; n2++)
              o[j][e] = mfma16<T>(v, uintx4{part[0][n2], part[1][n2], part[2][n2], part[3][n2]}, o[j][e]);
          }
      }
    }

    // the waves' sums meet
    products_done();
    l = quad_sum(l);
    if (g == 0 && dh == 0) {
      s.wm[kg][c] = m;
      s.wl[kg][c] = l;
    }
    __syncthreads();
    float M = s.wm[0][c];
#pragma unroll
    for (int i = 1; i < S::KG; i++) M = fmaxf(M, s.wm[i][c]);
    const float Ms = M == -__builtin_inff() ? 0.f : M;
    const float f = exp2_fast(m - Ms) * (1.f / S::PS) * (T == 3 ? vtop : 1.f);
    bool odd = false;
    if (w == 0 && g == 0) {
      float L = 0.f;
#pragma unroll
      for (int i = 0; i < S::KG; i++) L += s.wl[i][c] * exp2_fast(s.wm[i][c] - Ms);
      s.m[c] = M;
      s.l[c] = L;
      odd = c < it.heads && !finite(L);
    }
    for (int r4 = 0; r4 < S::KG; r4++) {
      if (kg == r4) {
#pragma unroll
        for (int j = 0; j < S::NJ; j++)
#pragma unroll
          for (int r = 0; r < 4; r++)
#pragma unroll
            for (int e = 0; e < S::VL; e += 4) {
              floatx4* const d = (floatx4*)&s.o[c * S::OS + dh * S::DW + j * 16 * S::VL + S::VL * (4 * g + r) + e];
              floatx4 v = {o[j][e][r] * f, o[j][e + 1][r] * f, o[j][e + 2][r] * f, o[j][e + 3][r] * f};
              if (r4) v += *d;
              *d = v;
            }
      }
      __syncthreads();
    }
    for (int h = w; h < it.heads; h += 4)
      for (int d = lane; d < hd; d += 64) odd |= !finite(s.o[h * S::OS + d]);
    if (__syncthreads_or(odd))
      paged_walk<T, D>(a, it, lo + (int64_t)tile0 * S::TK, min(hi, lo + (int64_t)tile1 * S::TK), s);

    float* const y = a.y + (int64_t)it.row * row_out + (int64_t)it.head0 * a.hd;
    // with the sink: its weight beside the sum's, both against the larger maximum
    auto finish = [&](int h, float m2, float l2, float& f2) {
      f2 = 1.f;
      if (is_shared<A> && l2 == 0.f) {  // (no key has a weight: zeros, whatever the sink)
        f2 = 0.f;
        return;
      }
      if (a.sinks) {
        const float sk = a.sinks[it.head0 + h] * LOG2E;
        if (sk > m2) {
          f2 = exp2_fast(m2 - sk);
          l2 = l2 * f2 + 1.f;
        } else if (sk != -__builtin_inff()) {  // (switched off: no weight, where no key has one either)
          l2 += exp2_fast(sk - m2);
        }
      }
      f2 = l2 != 0.f ? f2 / l2 : 0.f;
    };
    if (tile0 == 0 && tile1 == n) {
      if constexpr (is_shared<A>) {
        for (int j = 4 * t; pre && j < it.heads * a.hd; j += 1024) {
          const int h = j / a.hd, d = j - h * a.hd;
          float v[4];
#pragma unroll
          for (int e = 0; e < 4; e++) v[e] = s.o[h * S::OS + d + e];
          with_prefix(it, h, d, s.m[h], s.l[h], v);
#pragma unroll
          for (int e = 0; e < 4; e++) y[j + e] = v[e];
        }
      }
      for (int h = w + (pre ? 16 : 0); h < it.heads; h += 4) {
        float f2;
        finish(h, s.m[h], s.l[h], f2);
        for (int d = lane; d < hd; d += 64) y[h * a.hd + d] = f2 == 0.f ? 0.f : s.o[h * S::OS + d] * f2;
      }
      __syncthreads();
    } else {
      const int ps = 16 * a.hd + 32;  // floats of a piece
      float* const pc = a.part + (int64_t)(2 * b + (tile0 ? 0 : 1)) * ps;
      for (int h = w; h < it.heads; h += 4)
        for (int d = lane; d < hd; d += 64) store_agent(pc + h * a.hd + d, s.o[h * S::OS + d]);
      if (t < 16) {
        store_agent(pc + 16 * a.hd + t, s.m[t]);
        store_agent(pc + 16 * a.hd + 16 + t, s.l[t]);
      }
      // the blocks of the item's first and last tile
      auto block_of = [&](uint32_t i) {
        uint32_t k = (uint32_t)((double)i * B / all);
        while (k > 0 && first(k) > i) k--;
        while (first(k + 1) <= i) k++;
        return k;
      };
      const uint32_t u0 = before + item * (n + OV) + OV, b0 = block_of(u0), np = block_of(u0 + n - 1) - b0 + 1;
      auto piece = [&](uint32_t i) { return a.part + (int64_t)(2 * (b0 + i) + (i == 0)) * ps; };
      // pieces i0, i0 + step, .. (cnt of them, at most 64) joined in that order: into
      // the output, or into the first of them
      auto join = [&](uint32_t i0, uint32_t step, uint32_t cnt, bool out) {
        // 4 values of 16 pieces a thread, the first on their way while the weights are formed
        const int total = it.heads * a.hd;
        uint64_t x[16][2];
        auto fetch = [&](int i, uint32_t j0) {
#pragma unroll
          for (uint32_t k = 0; k < 16; k++) {
            const double* const e = (const double*)(piece(i0 + step * min(j0 + k, cnt - 1)) + i);
            x[k][0] = __builtin_bit_cast(uint64_t, load_agent(e));
            x[k][1] = __builtin_bit_cast(uint64_t, load_agent(e + 1));
          }
        };
        if (4 * t < total) fetch(4 * t, 0);
        float* const wt = s.o;  // [64][16]: a piece's weight for each head, 0 past the last
        {
          const int h = t >> 4;
          float pm[4], pl[4], M2 = -__builtin_inff(), L = 0.f;
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const uint32_t j = (t & 15) + 16 * i;
            const float* const e = piece(i0 + step * min(j, cnt - 1)) + 16 * a.hd + h;
            pm[i] = j < cnt ? load_agent(e) : -__builtin_inff();
            pl[i] = j < cnt ? load_agent(e + 16) : 0.f;
            M2 = fmaxf(M2, pm[i]);
          }
          M2 = fmaxf(M2, xpart<1>(M2));
          M2 = fmaxf(M2, xpart<2>(M2));
          M2 = fmaxf(M2, xpart<4>(M2));
          M2 = fmaxf(M2, xpart<8>(M2));
          const float s2 = M2 == -__builtin_inff() ? 0.f : M2;
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const float f2 = exp2_fast(pm[i] - s2);
            L += f2 * pl[i];
            wt[((t & 15) + 16 * i) * 16 + h] = f2;
          }
          L = wave_sum(L, 16);
          __syncthreads();
          if ((t & 15) == 0) {
            s.m[h] = M2;
            s.l[h] = L;
            if (!out) {
              store_agent(piece(i0) + 16 * a.hd + h, M2);
              store_agent(piece(i0) + 16 * a.hd + 16 + h, L);
            }
          }
        }
        __syncthreads();
        for (int i = 4 * t; i < total; i += 1024) {
          const int h = i / a.hd;
          float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
          for (uint32_t j0 = 0; j0 < cnt; j0 += 16) {
            if (i != 4 * t || j0) fetch(i, j0);
#pragma unroll
            for (uint32_t k = 0; k < 16; k++) {
              const float f2 = wt[(j0 + k) * 16 + h];
#pragma unroll
              for (int e = 0; e < 4; e++) {
                const float p = bits_float((uint32_t)(x[k][e / 2] >> (32 * (e & 1))));
                v[e] = __builtin_fmaf(f2, f2 != 0.f ? p : 0.f, v[e]);  // (a part of no weight may hold an infinity)
              }
            }
          }
          if (out && pre) {
            with_prefix(it, h, i - h * a.hd, s.m[h], s.l[h], v);
#pragma unroll
            for (int e = 0; e < 4; e++) y[i + e] = v[e];
          } else if (out) {
            float f2;
            finish(h, s.m[h], s.l[h], f2);
#pragma unroll
            for (int e = 0; e < 4; e++) y[i + e] = f2 == 0.f ? 0.f : v[e] * f2;
          } else {
#pragma unroll
            for (int e = 0; e < 4; e++) store_agent(piece(i0) + i + e, v[e]);
          }
        }
      };
      // 16 pieces are joined by the last of their blocks, then those by the last of all
      const uint32_t mine = b - b0, i0 = mine & ~15u, cnt = min(16u, np - i0);
      int* const group = a.done + 32 * (b0 + i0) + (i0 == 0);
      if (last_block(group, (int)cnt)) {
        const uint32_t groups = (np + 15) / 16;
        join(i0, 1, cnt, groups == 1);
        if (t == 0) __hip_atomic_store(group, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (groups > 1 && last_block(a.done + 32 * b0 + 2, (int)groups)) {
          join(0, 16, groups, true);
          if (t == 0) __hip_atomic_store(a.done + 32 * b0 + 2, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
      }
      __syncthreads();
    }
    u += upto - at;
    if (u >= end) {
      if (OV && whole) break;
      return;
    }
    if (tile1 == n && item + 1 == per) {  // the next sequence with a key
      before = u;
      do n = tiles_of(++seq, lo, hi);
      while (n == 0);
    }
  }
  }
}

}  // namespace ihip
