// paged_shared.hip - attention of one new token of each sequence where groups of
// sequences share their first tokens: a launch over the prefixes, each read once for
// all of its group's queries, and one over the sequences' own tokens, which joins them.
// Built once for each type of pages (IHIP_SHARED_T: 0 single, 1 half, 2 bf16, 3 8-bit).
#include "paged_attention.h"

using namespace ihip;

// Columns (a member's query head each) of a block: 16 CT. As many as the loop over keys holds
// in the registers of two blocks a CU: heads of 128 two tiles (32 chats behind 4096 tokens 26
// us; four tiles and one block a CU 33, four and two blocks 53), of 64 four (128 sequences
// behind 30011 240 us; two and three blocks a CU 245, two and four 310), of 256 in 8-bit
// pages one (three prompts of 9001 68 us; two and one block 95 where one took 80). Others of
// 256 have two and one block (halves 97 us; one and two blocks 135 where two took 111). What
// lives from an item's start to its end does not fit beside that loop: the compiler spills up to 61
// registers (halves of 128 34, 8-bit heads of 256 26, and 67 of paged_own's; none of 512),
// which are stored and loaded once an item. Sizes between these have up to 11 loads a step.
template <int T, int D>
constexpr int shared_ct = PAGED_SHARED_TILES(D, T == 3);
template <int T, int D>
constexpr int shared_blocks = D <= 128 || (D == 256 && T == 3) ? 2 : 1;

template <int T, int D>
struct PrefixLds : AttnScales<T> {
  using S = AttnShape<T, D>;
  static constexpr int CT = shared_ct<T, D>;
  union {
    uintx4 q[CT][S::NP * S::DS * S::NF * 64];  // the query tiles as the matrix cores take them
    float o[CT][S::KG][16 * S::OS];            // behind the keys: a tile's sums, of the waves of each group of keys
  };
  float wm[4][CT * 16], wl[4][CT * 16];
  int odd;                 // whether sums are not all finite
  float m[CT * 16], l[CT * 16];  // the columns' maxima and sums
  uint32_t top[CT * 16];  // a column's largest magnitude, as bits
  int64_t at[CT * 16];  // a column's query and output, from q and y (rows of q_stride and heads * hd): row, -1 none
  int head[CT * 16];
  int keys[CT * 16];    // of a column: the prefix's tokens that its sequence has
  int64_t off[4][2][S::KS];
  floatx4 x[S::DS > 1 ? 2 : 1][S::DS > 1 ? 4 : 1][S::NT][64];
};

// a tile of 16 columns by the formula's own steps, where sums are not all finite
// (paged_walk's reasons)
template <int T, int D>
__device__ __forceinline__ void prefix_walk(const PagedSharedArgs& a, const int* table, int kv, int ct, int64_t j0,
                                            int64_t j1, PrefixLds<T, D>& s)
{
  using S = AttnShape<T, D>;
  constexpr int NV = D / 64;
  const int t = threadIdx.x, lane = t & 63, w = t >> 6;
  __shared__ float tmp[4 * D];
  for (int h = 0; h < 16; h++) {
    const int col = 16 * ct + h;
    if (s.at[col] < 0) continue;
    const float* const qp = a.q + s.at[col] * a.q_stride + (int64_t)s.head[col] * a.hd;
    float q[NV], acc[NV];
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const int d = lane + 64 * i;
      q[i] = d < a.hd ? qp[d] * a.scale : 0.f;
      acc[i] = 0.f;
    }
    float m = -__builtin_inff(), l = 0.f;
    const int64_t end = min(j1, (int64_t)s.keys[col]);
    for (int64_t j = j0 + w; j < end; j += 4) {
      const int page = table[(uint32_t)j / (uint32_t)a.page_size], in = (int)((uint32_t)j % (uint32_t)a.page_size);
      const int64_t at = paged_value(page, in, a.pages, a.page_stride, a.slot_stride);
      if (at < 0) continue;
      const int64_t row = (at + kv * a.head_stride) * S::ES;
      float x = 0.f, vscale = 1.f, kscale = 1.f;
      if constexpr (T == 3) {
        const int64_t sc = page * a.s_page + (int64_t)in * a.s_slot + kv * a.s_head;
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
      s.wm[w][col] = m;
      s.wl[w][col] = l;
    }
    __syncthreads();
    float M = -__builtin_inff(), L = 0.f, f[4];
    for (int i = 0; i < 4; i++) M = s.wm[i][col] > M || s.wm[i][col] != s.wm[i][col] ? s.wm[i][col] : M;
    for (int i = 0; i < 4; i++) {
      f[i] = s.wl[i][col] == 0.f ? 0.f : exp2_fast(s.wm[i][col] - M);
      L += f[i] * s.wl[i][col];
    }
    for (int d = t; d < a.hd; d += 256) {
      float v = 0.f;
      for (int i = 0; i < 4; i++)
        if (s.wl[i][col] != 0.f) v += f[i] * tmp[i * D + d];
      s.o[ct][0][h * S::OS + d] = v;
    }
    __syncthreads();
    // (as if one group of keys had them all)
    if (t < S::KG) {
      s.wm[t][col] = t == 0 ? M : -__builtin_inff();
      s.wl[t][col] = t == 0 ? L : 0.f;
    }
    __syncthreads();
  }
}

// The queries of a group's members for one KV head are the columns of one problem, which
// reads the prefix's keys and values once for 16 CT of them: scores K q^T and values V^T
// P as paged_attention's, a wave's keys and values in registers used for CT tiles of 16
// columns, the query tiles in LDS. All groups' tiles of keys are one row, shared out
// evenly over the grid. A block that has the whole of an item (KV head, columns) leaves
// it in y and sums; parts go to `pieces`, and the launch over the sequences' own tokens
// joins them. Bound by issue where a group is large (128 sequences behind 30011 tokens, 64
// heads of 64 over 8 in bf16 235 us: vector work 69%, matrix cores 40% of the SIMDs' time, of
// weights in three parts), by loads' latency where its columns are few (the sizes at
// shared_ct).
template <int T, int D, bool FULL>
__device__ __forceinline__ void paged_prefix_t(const PagedSharedArgs& a)
{
  using S = AttnShape<T, D>;
  constexpr int CT = shared_ct<T, D>, COLS = 16 * CT;
  __shared__ PrefixLds<T, D> s;
  const int t = threadIdx.x, lane = t & 63, c = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const uint32_t grid = gridDim.x;
  const int hd = FULL ? D : a.hd, row_out = a.heads * a.hd;

  // a group's items of a KV head and tiles of keys
  auto shape_of = [&](int grp, uint32_t& items, int64_t& common) {
    const int m0 = a.members[grp], m1 = a.members[grp + 1];
    common = paged_common(m0, m1, a.shared[grp], a.seqs, a.max_pages, a.page_size);
    items = common > 0 ? ((uint32_t)(m1 - m0) * a.group + COLS - 1) / COLS : 0;
    return (uint32_t)((common + S::TK - 1) / S::TK);
  };
  uint64_t total = 0;
  uint32_t n0 = 0, items0 = 0;  // of the first 64 groups, a lane each
  int64_t common0 = 0;
  for (int g0 = 0; g0 < a.groups; g0 += 64) {
    uint32_t items = 0, n = 0;
    int64_t common = 0;
    if (g0 + lane < a.groups) n = shape_of(g0 + lane, items, common);
    if (g0 == 0) n0 = n, items0 = items, common0 = common;
    total += wave_sum((uint64_t)n * items * (uint32_t)a.kvh, 64);
  }
  // (groups that overlap, which no caller has, may pass 32 bits)
  const uint32_t all = total < (1u << 31) ? __builtin_amdgcn_readfirstlane((uint32_t)total) : 0u;
  const uint32_t B = min(grid, all);
  // blocks that follow each other take the columns behind the same keys: onto one XCD (block
  // i runs on XCD i mod 8), whose L2 then has them (three prompts of 9001, 8-bit heads of 256:
  // 339 MiB fetched and 75 us, so 280 and 68)
  const uint32_t x = blockIdx.x, b = B == grid && grid % 8 == 0 ? x % 8 * (grid / 8) + x / 8 : x;
  if (b == 0 && t == 0) {
    a.plan[0] = (int)all;
    a.plan[1] = (int)B;
    a.plan[2] = CT;
  }
  if (b >= B && b) return;
  const PieceShare share(max(all, 1u), max(B, 1u));
  uint32_t u = B ? share.first(b) : UINT32_MAX;
  const uint32_t end = B ? share.first(b + 1) : 0u;
  // the group of tile u (and the plan, by the first block)
  int grp = -1;
  uint32_t before = 0, n = 0, items = 0;
  int64_t common = 0;
  uint32_t upto_all = 0;
  for (int g0 = 0; g0 < a.groups; g0 += 64) {
    if (g0 && g0 + lane < a.groups) n0 = shape_of(g0 + lane, items0, common0);
    else if (g0) n0 = items0 = 0;
    const uint32_t mine = n0 * items0 * a.kvh;
    uint32_t upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const uint32_t o = __shfl_up(upto, d, 64);
      if (lane >= d) upto += o;
    }
    if (b == 0 && w == 0 && g0 + lane < a.groups) {
      int* const e = a.plan + SHARED_PLAN + 3 * (g0 + lane);
      e[0] = (int)(upto_all + upto - mine);
      e[1] = (int)n0;
      e[2] = (int)items0;
    }
    const uint64_t there = __ballot(upto_all + upto > u);
    if (there && grp < 0) {
      const int f = __builtin_ctzll(there);
      grp = __builtin_amdgcn_readfirstlane(g0 + f);
      before = upto_all + __builtin_amdgcn_readlane(upto - mine, f);
      n = __builtin_amdgcn_readlane(n0, f);
      items = __builtin_amdgcn_readlane(items0, f);
      common = (int64_t)lane_value((uint64_t)common0, f);
      if (b) break;
    }
    upto_all += __builtin_amdgcn_readlane(upto, 63);
  }
  if (grp < 0) return;  // (no tile)

  for (;;) {
    const uint32_t item = (u - before) / n, tile0 = (u - before) - item * n;
    const uint32_t tile1 = min(n, tile0 + (end - u));
    const int kv = item / items, col0 = (int)(item - kv * items) * COLS;
    const int m0 = a.members[grp], cols = (a.members[grp + 1] - m0) * a.group;
    const char* const kb = a.kc + (int64_t)kv * a.head_stride * S::ES;
    const char* const vb = a.vc + (int64_t)kv * a.head_stride * S::ES;
    const float* sb = nullptr;
    float scale = 0.f;
    if constexpr (T == 3) sb = (lane < S::KS ? a.ks : a.vs) + (int64_t)kv * a.s_head;
    const int* const table = a.table + (int64_t)m0 * a.max_pages;
    const int kg = w / S::DS, dh = w % S::DS;
    const int64_t wlo = kg * S::KS;
    const int64_t jend = min(common, (int64_t)tile1 * S::TK);
    auto entry = [&](uint32_t tile) {
      const int64_t j = wlo + (int64_t)tile * S::TK + (lane & (S::KS - 1));
      return j < jend ? table[(uint32_t)j / (uint32_t)a.page_size] : -1;
    };
    auto locate = [&](uint32_t tile, int page) {
      const int64_t j = wlo + (int64_t)tile * S::TK + (lane & (S::KS - 1));
      const int in = (int)((uint32_t)j % (uint32_t)a.page_size);
      const int64_t at = paged_value(page, in, a.pages, a.page_stride, a.slot_stride);
      if (lane < S::KS) s.off[w][tile & 1][lane] = at < 0 ? 0 : at * S::ES;
      if constexpr (T == 3) scale = at < 0 ? 0.f : sb[page * a.s_page + (int64_t)in * a.s_slot];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      return (uint32_t)__ballot(at >= 0) & (uint32_t)((1ull << S::KS) - 1);
    };
    uint32_t tile = tile0;
    const int page0 = entry(tile);
    int page = entry(tile + 1);

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

    // the columns: a member's row, its head, the keys that it sees
    if (t < COLS) {
      const int col = col0 + t, seq = m0 + col / a.group;
      int64_t at = -1;
      int keys = 0;
      if (col < cols) {
        const int row = a.offsets ? paged_row(a.offsets[seq], a.offsets[seq + 1], a.rows) : paged_row(seq, seq + 1, a.rows);
        if (row >= 0 && a.lengths[seq] >= 0) {
          at = row;
          keys = (int)min((int64_t)a.lengths[seq], common);
        }
      }
      s.at[t] = at;
      s.head[t] = kv * a.group + col % a.group;
      s.keys[t] = keys;
      s.top[t] = 0;
    }
    lds_barrier();
    // the query tiles (stage_query's form), a thread's factors on their way at once
    constexpr int TILE = S::DS * S::NF * 64, R = CT * TILE / 256;
    float qv[R][S::FL];
#pragma unroll
    for (int r = 0; r < R; r++) {
      const int i = t + 256 * r, col = 16 * (i / TILE) + (i & 15), d0 = S::factor((i % TILE) >> 6, (i >> 4) & 3);
      const bool in = s.at[col] >= 0 && d0 < a.hd;
      const float* const q = a.q + (in ? s.at[col] * a.q_stride + (int64_t)s.head[col] * a.hd + d0 : 0);
#pragma unroll
      for (int e = 0; e < S::FL; e++) qv[r][e] = in ? q[e] : 0.f;
    }
    // (the first keys, on their way behind the queries)
    uint32_t steps = 0;
    if (S::DS > 1) {
      steps = tile1 - tile0;
    } else if (wlo + (int64_t)tile0 * S::TK < common) {
      const uint32_t mine = (uint32_t)((common - wlo + S::TK - 1) / S::TK);
      steps = min(tile1, mine) - tile0;
    }
    uint32_t there = locate(tile, page0);
    if (steps) load_keys(tile);
    if constexpr (T == 1 || T == 3) {
#pragma unroll
      for (int r = 0; r < R; r++) {
        const int i = t + 256 * r, col = 16 * (i / TILE) + (i & 15);
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < S::FL; e++) top = max(top, float_bits(fabsf(qv[r][e] * a.scale)));
        atomicMax(&s.top[col], top);
      }
      lds_barrier();
    }
    // the power of two that a column's queries are divided by: the largest below 2^14
    auto divisor = [&](int col) {
      const uint32_t top = s.top[col];
      const int e = top == 0 || top >= 0x7f800000u ? 14 : (int)(top >> 23) - 126;
      return ldexpf(1.f, max(e - 14, -120));
    };
#pragma unroll
    for (int r = 0; r < R; r++) {
      const int i = t + 256 * r, ct = i / TILE, j = i % TILE;
      float f = a.scale, v[S::FL];
      if constexpr (T == 1 || T == 3) f = 1.f / divisor(16 * ct + (i & 15));
#pragma unroll
      for (int e = 0; e < S::FL; e++) v[e] = T == 1 || T == 3 ? qv[r][e] * a.scale * f : qv[r][e] * f;
      if constexpr (T == 0) {
        s.q[ct][j] = uintx4{float_bits(v[0]), float_bits(v[1]), float_bits(v[2]), float_bits(v[3])};
      } else {
        uint32_t part[4][S::NP];
#pragma unroll
        for (int e = 0; e < 4; e++) split2<T>(v[2 * e], v[2 * e + 1], part[e]);
#pragma unroll
        for (int p = 0; p < S::NP; p++) s.q[ct][p * TILE + j] = uintx4{part[0][p], part[1][p], part[2][p], part[3][p]};
      }
    }
    lds_barrier();
    float sscale[CT];
    int keys[CT], least = INT32_MAX;  // of the lane's columns; the least of all
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
      sscale[ct] = T == 1 || T == 3 ? divisor(16 * ct + c) : 1.f;
      keys[ct] = s.keys[16 * ct + c];
      if (s.at[16 * ct + c] >= 0) least = min(least, keys[ct]);
    }
    least = -wave_max(-least);

    floatx4 o[CT][S::NJ][S::VL];
    float m[CT], l[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
      m[ct] = -__builtin_inff();
      l[ct] = 0.f;
#pragma unroll
      for (int i = 0; i < S::NJ; i++)
#pragma unroll
        for (int j = 0; j < S::VL; j++) o[ct][i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
    }
    float vtop = 0x1p-100f, vinv = 0x1p100f;
    for (uint32_t i = 0; i < steps; i++, tile++) {
      constexpr int NV = 4 * S::NT;
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
          for (int ct = 0; ct < CT; ct++)
#pragma unroll
            for (int j = 0; j < S::NJ; j++)
#pragma unroll
              for (int e = 0; e < S::VL; e++) o[ct][j][e] *= f;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int k = 0; k < S::NT; k++) {
          ksc[k] = *(const floatx4*)&s.sc[w][16 * k + 4 * g];
          vsc[k] = *(const floatx4*)&s.sc[w][32 + 16 * k + 4 * g] * (vinv * S::PS);
        }
      }
      // whether every column sees every key of the wave's step
      const bool plain = now == (uint32_t)((1ull << S::KS) - 1) && wlo + (int64_t)tile * S::TK + S::KS <= least;
      const int64_t key0 = wlo + (int64_t)tile * S::TK + 4 * g;
      there = locate(tile + 1, page);
      page = entry(tile + 2);
      floatx4 x[CT][S::NT];
#pragma unroll
      for (int ct = 0; ct < CT; ct++)
#pragma unroll
        for (int k = 0; k < S::NT; k++) x[ct][k] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < S::NF; j++) {
        uintx4 kf[S::NT];
#pragma unroll
        for (int k = 0; k < S::NT; k++) {
          if constexpr (T == 3) {
            const uintx2 lo = codes4(kr[k][j / 2][2 * (j & 1)] ^ 0x80808080u), hi = codes4(kr[k][j / 2][2 * (j & 1) + 1] ^ 0x80808080u);
            kf[k] = uintx4{lo[0], lo[1], hi[0], hi[1]};
          } else {
            kf[k] = kr[k][j];
          }
        }
#pragma unroll
        for (int ct = 0; ct < CT; ct++)
#pragma unroll
          for (int n2 = 0; n2 < S::NP; n2++) {
            const uintx4 q = s.q[ct][(n2 * S::DS * S::NF + dh * S::NF + j) * 64 + lane];
#pragma unroll
            for (int k = 0; k < S::NT; k++) {
              if constexpr (T == 0) {
#pragma unroll
                for (int e = 0; e < 4; e++)
                  x[ct][k] = __builtin_amdgcn_mfma_f32_16x16x4f32(bits_float(kf[k][e]), bits_float(q[e]), x[ct][k], 0, 0, 0);
              } else {
                x[ct][k] = mfma16<T>(kf[k], q, x[ct][k]);
              }
            }
          }
      }
      load_keys(tile + 1);
      products_done();
      if constexpr (S::DS > 1) {
        static_assert(S::DS == 1 || CT == 1, "one tile of columns where waves share a head");
#pragma unroll
        for (int k = 0; k < S::NT; k++) s.x[tile & 1][w][k][lane] = x[0][k];
        lds_barrier();
#pragma unroll
        for (int k = 0; k < S::NT; k++) x[0][k] += s.x[tile & 1][w ^ 1][k][lane];
      }
      // keys that are not there: values of zero (0 times NaN is NaN)
      if (T != 3 && now != (uint32_t)((1ull << S::KS) - 1)) {
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
          for (int j = 0; j < S::NJ; j++)
            if (!(now >> (16 * (k >> 2) + 4 * g + (k & 3)) & 1)) vr[k][j] = uintx4{0, 0, 0, 0};
      }
      // the values turned: 8 keys of a dimension side by side (once for all tiles of columns;
      // for one, where its products are, as they take as many registers as the values)
      auto turned = [&](int j, int e) {
        uintx4 v;
#pragma unroll
        for (int k = 0; k < 4; k++) {
          if constexpr (T == 3) {
            const uint32_t pair = __builtin_amdgcn_perm(vr[2 * k + 1][j][e / 4], vr[2 * k][j][e / 4],
                                                        e & 2 ? 0x07030602u : 0x05010400u) ^ 0x80808080u;
            v[k] = halves_of(__builtin_amdgcn_perm(0x64646464u, pair, e & 1 ? 0x04030402u : 0x04010400u));
          } else {
            v[k] = __builtin_amdgcn_perm(vr[2 * k + 1][j][e / 2], vr[2 * k][j][e / 2], e & 1 ? 0x07060302u : 0x05040100u);
          }
        }
        return v;
      };
      constexpr bool ONCE = T != 0 && CT > 1;
      uintx4 vt[ONCE ? S::NJ : 1][ONCE ? S::VL : 1];
      if constexpr (ONCE) {
#pragma unroll
        for (int j = 0; j < S::NJ; j++)
#pragma unroll
          for (int e = 0; e < S::VL; e++) vt[j][e] = turned(j, e);
      }
      // the scores' scale, what a column does not see, and whether a maximum rises
      float top[CT];
      bool rises = false;
#pragma unroll
      for (int ct = 0; ct < CT; ct++) {
        top[ct] = -__builtin_inff();
#pragma unroll
        for (int k = 0; k < NV; k++)
          x[ct][k >> 2][k & 3] *= T == 3 ? sscale[ct] * ksc[T == 3 ? k >> 2 : 0][k & 3] : sscale[ct];
      }
      if (!plain) {
#pragma unroll
        for (int ct = 0; ct < CT; ct++)
#pragma unroll
          for (int k = 0; k < NV; k++) {
            const bool in = (now >> (16 * (k >> 2) + 4 * g + (k & 3)) & 1) && key0 + 16 * (k >> 2) + (k & 3) < keys[ct];
            x[ct][k >> 2][k & 3] = in ? x[ct][k >> 2][k & 3] : -__builtin_inff();
          }
      }
#pragma unroll
      for (int ct = 0; ct < CT; ct++) {
#pragma unroll
        for (int k = 0; k < NV; k++) top[ct] = fmaxf(top[ct], x[ct][k >> 2][k & 3]);
        rises |= top[ct] > m[ct];
      }
      if (__any(rises)) {
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
          const float m2 = fmaxf(quad_max(top[ct]), m[ct]), f = m[ct] == -__builtin_inff() ? 0.f : exp2_fast(m[ct] - m2);
          m[ct] = m2;
          l[ct] *= f;
#pragma unroll
          for (int j = 0; j < S::NJ; j++)
#pragma unroll
            for (int e = 0; e < S::VL; e++) o[ct][j][e] *= f;
        }
      }
      // Weights and value products, without a branch: a tile's products run while the next
      // one's weights are formed.
#pragma unroll
      for (int ct = 0; ct < CT; ct++) {
        const float shift = m[ct] == -__builtin_inff() ? 0.f : m[ct];
        float p[NV];
#pragma unroll
        for (int k = 0; k < NV; k++) {
          p[k] = exp2_fast(x[ct][k >> 2][k & 3] - shift);
          l[ct] += p[k];
        }
        if constexpr (T == 0) {
#pragma unroll
          for (int k = 0; k < NV; k++)
#pragma unroll
            for (int j = 0; j < S::NJ; j++)
#pragma unroll
              for (int e = 0; e < 4; e++)
                o[ct][j][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(bits_float(vr[k][j][e]), p[k], o[ct][j][e], 0, 0, 0);
        } else {
          uint32_t part[4][S::NP];
#pragma unroll
          for (int k = 0; k < 4; k++) {
            if constexpr (T == 3)
              split2<T>(p[2 * k] * vsc[k >> 1][2 * k & 3], p[2 * k + 1] * vsc[k >> 1][(2 * k + 1) & 3], part[k]);
            else
              split2<T>(p[2 * k] * S::PS, p[2 * k + 1] * S::PS, part[k]);
          }
#pragma unroll
          for (int j = 0; j < S::NJ; j++)
#pragma unroll
            for (int e = 0; e < S::VL; e++) {
              uintx4 v;
              if constexpr (ONCE) v = vt[ONCE ? j : 0][ONCE ? e : 0];
              else v = turned(j, e);
#pragma unroll
              for (int n2 = 0; n2 < S::NP; n2++)
                o[ct][j][e] = mfma16<T>(v, uintx4{part[0][n2], part[1][n2], part[2][n2], part[3][n2]}, o[ct][j][e]);
            }
        }
      }
    }

    // the waves' sums meet: each group of keys' into LDS, where the query was, then added
    // up by all threads, 4 values of a column each time (loops that are not unrolled: the
    // code runs once a block, and fetching it is what it costs)
    products_done();
    const bool whole = tile0 == 0 && tile1 == n;
    float* const pc = a.pieces + (int64_t)(2 * b + (tile0 ? 0 : 1)) * COLS * (a.hd + 2);
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
      l[ct] = quad_sum(l[ct]);
      if (g == 0 && dh == 0) {
        s.wm[kg][16 * ct + c] = m[ct];
        s.wl[kg][16 * ct + c] = l[ct];
      }
    }
    lds_barrier();
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
      float M = s.wm[0][16 * ct + c];
#pragma unroll
      for (int i = 1; i < S::KG; i++) M = fmaxf(M, s.wm[i][16 * ct + c]);
      const float f = exp2_fast(m[ct] - (M == -__builtin_inff() ? 0.f : M)) * (1.f / S::PS) * (T == 3 ? vtop : 1.f);
#pragma unroll
      for (int j = 0; j < S::NJ; j++)
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
          for (int e = 0; e < S::VL; e += 4)
            *(floatx4*)&s.o[ct][kg][c * S::OS + dh * S::DW + j * 16 * S::VL + S::VL * (4 * g + r) + e] =
                floatx4{o[ct][j][e][r] * f, o[ct][j][e + 1][r] * f, o[ct][j][e + 2][r] * f, o[ct][j][e + 3][r] * f};
    }
    // (a tile's columns that are walked have theirs as one group of keys')
    auto sums = [&](int col) {
      float M2 = s.wm[0][col], L2 = 0.f;
#pragma unroll
      for (int i = 1; i < S::KG; i++) M2 = s.wm[i][col] > M2 || s.wm[i][col] != s.wm[i][col] ? s.wm[i][col] : M2;
      const float ms = M2 == -__builtin_inff() ? 0.f : M2;
#pragma unroll
      for (int i = 0; i < S::KG; i++) L2 += s.wl[i][col] == 0.f ? 0.f : s.wl[i][col] * exp2_fast(s.wm[i][col] - ms);
      s.m[col] = L2 == 0.f ? -__builtin_inff() : M2;
      s.l[col] = L2;
      return L2;
    };
    bool odd = false;
    if (t == 0) s.odd = 0;
    if (t < COLS) odd = s.at[t] >= 0 && !finite(sums(t));
    lds_barrier();
    auto value = [&](int ct, int i) {
      const float* const e = &s.o[ct][0][i / hd * S::OS + i % hd];
      floatx4 v = *(const floatx4*)e;
#pragma unroll
      for (int p = 1; p < S::KG; p++) v += *(const floatx4*)(e + p * 16 * S::OS);
      return v;
    };
#pragma unroll 1
    for (int i = 4 * t; i < CT * 16 * hd; i += 1024) {
      const floatx4 v = value(i / (16 * hd), i % (16 * hd));
      odd |= s.at[i / hd] >= 0 && !(finite(v[0]) && finite(v[1]) && finite(v[2]) && finite(v[3]));
    }
    // (again by the formula's steps, where sums are not all finite)
    if (__any(odd) && lane == 0) s.odd = 1;
    lds_barrier();
    const bool walked = s.odd != 0;
    if (walked) {
      for (int ct = 0; ct < CT; ct++) {
        prefix_walk<T, D>(a, table, kv, ct, (int64_t)tile0 * S::TK, jend, s);
        if (t < 16) sums(16 * ct + t);
      }
      __syncthreads();
    }
    // the columns' results: to y and sums, or to the pieces
    if (t < COLS && s.at[t] >= 0) {
      if (whole) {
        // (the maximum and the sum apart: one logarithm loses half a step of a large maximum)
        float* const e = a.sums + 2 * ((int64_t)(m0 + (col0 + t) / a.group) * a.heads + s.head[t]);
        e[0] = s.m[t];
        e[1] = s.l[t];
      } else {
        pc[COLS * a.hd + t] = s.m[t];
        pc[COLS * a.hd + COLS + t] = s.l[t];
      }
    }
#pragma unroll 1
    for (int i = 4 * t; i < CT * 16 * hd; i += 1024) {
      const int col = i / hd, d = i - col * hd, ct = col >> 4;
      if (s.at[col] < 0) continue;
      const floatx4 v = walked ? *(const floatx4*)&s.o[ct][0][(col & 15) * S::OS + d] : value(ct, i % (16 * hd));
      if (whole) {
        float* const y = a.y + s.at[col] * row_out + (int64_t)s.head[col] * a.hd + d;
#pragma unroll
        for (int e = 0; e < 4; e++) y[e] = v[e];
      } else {
        *(floatx4*)(pc + col * a.hd + d) = v;
      }
    }
    lds_barrier();
    u += tile1 - tile0;
    if (u >= end) return;
    if (tile1 == n && item + 1 == items * a.kvh) {  // the next group with a prefix
      before = u;
      do {
        if (++grp >= a.groups) return;
        n = shape_of(grp, items, common);
      } while (n == 0);
    }
  }
}

#define PAGED_SHARED2(NAME, T, D, SUFFIX, FULL)                                                                   \
  extern "C" __global__ __launch_bounds__(256, (shared_blocks<T, D>)) void paged_prefix_##NAME##_##D##SUFFIX(PagedSharedArgs a)          \
  {                                                                                                               \
    paged_prefix_t<T, D, FULL>(a);                                                                                \
  }                                                                                                               \
  extern "C" __global__ __launch_bounds__(256, (shared_blocks<T, D>)) void paged_own_##NAME##_##D##SUFFIX(PagedSharedArgs a)             \
  {                                                                                                               \
    paged_attention_t<T, D, FULL>(a);                                                                             \
  }
#define PAGED_SHARED1(NAME, T)                  \
  PAGED_SHARED2(NAME, T, 64, , true)            \
  PAGED_SHARED2(NAME, T, 64, _part, false)      \
  PAGED_SHARED2(NAME, T, 128, , true)           \
  PAGED_SHARED2(NAME, T, 128, _part, false)     \
  PAGED_SHARED2(NAME, T, 256, , true)           \
  PAGED_SHARED2(NAME, T, 256, _part, false)     \
  PAGED_SHARED2(NAME, T, 512, , true)           \
  PAGED_SHARED2(NAME, T, 512, _part, false)
#if IHIP_SHARED_T == 0
PAGED_SHARED1(f32, 0)
#elif IHIP_SHARED_T == 1
PAGED_SHARED1(f16, 1)
#elif IHIP_SHARED_T == 2
PAGED_SHARED1(bf16, 2)
#else
PAGED_SHARED1(q8, 3)
#endif
