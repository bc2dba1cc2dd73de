// logprobs.hip - log probabilities of given tokens, entropies and the top
// alternatives of rows of logits, each logit read once.
#include "common.h"

using namespace ihip;

struct LogprobArgs {
  const float* x;
  int64_t stride;
  const int* ids;
  float *logprobs, *entropy;
  int* top_ids;
  float* top_logprobs;
  double* part;  // [rows][parts][3 + k]: a part's maximum, sums and alternatives
  int* done;     // [rows] counters, 8 ints apart, zero between launches
  int32_t rows, vocab, k, parts;
};

typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));
typedef float floatx4u __attribute__((ext_vector_type(4), aligned(4)));

// a logit's place in the order of the alternatives: larger values first (both
// zeros the same), NaN (0) behind -infinity; and back
__device__ __forceinline__ uint32_t order_of(float v)
{
  if (v != v) return 0u;
  const uint32_t b = float_bits(v + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float order_value(uint32_t o)
{
  if (o == 0u) return __builtin_nanf("");
  return bits_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

__device__ __forceinline__ uint64_t lane_value(uint64_t v, int lane)
{
  return (uint64_t)__builtin_amdgcn_readlane((uint32_t)(v >> 32), lane) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((uint32_t)v, lane);
}

// The alternatives of a wave: lane i holds the i-th best so far as (order, ~id), 0
// where there is none yet, so that a larger number is a better alternative; a
// tile's candidates meet in LDS first. The code is kept small: a block of one row
// runs it once, from a cold instruction cache (sorting networks written out took
// 18 us for one row of 151936 logits and one alternative where these loops take 12).
struct TopList {
  uint64_t v;
  uint64_t* buf;   // [64 + 256]
  uint64_t* list;  // [64]
  int n;           // waiting in buf (the same in every lane)

  // between a lane's LDS write and another's read: no instruction, but no
  // reordering or forwarding past it
  __device__ __forceinline__ void lanes_meet()
  {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
  // the lanes' numbers c where `in` (b: those lanes)
  __device__ __forceinline__ void add(uint64_t b, bool in, uint64_t c)
  {
    if (in) buf[n + __builtin_amdgcn_mbcnt_hi((uint32_t)(b >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)b, 0u))] = c;
    n += __popcll(b);
  }
  // the waiting ones into the list, 64 at a time: few one by one, more by counting
  // for each, and for each of the list, how many are better
  __device__ __forceinline__ void flush(int k)
  {
    const int lane = threadIdx.x & 63;
    lanes_meet();
#pragma unroll 1
    for (int i = 0; i < n; i += 64) {
      const int m = min(n - i, 64);
      uint64_t c = lane < m ? buf[i + lane] : 0;
      uint64_t b = __ballot(c > lane_value(v, k - 1));
      if (__popcll(b) > 12) {
        int cr = 0, vr = lane;
        list[lane] = v;
        lanes_meet();
#pragma unroll 4
        for (int j = 0; j < m; j++) {
          const uint64_t x = buf[i + j];
          cr += x > c;
          vr += x > v;
        }
        if (lane_value(v, 0))
#pragma unroll 4
          for (int j = 0; j < k; j++) cr += list[j] > c;
        lanes_meet();
        list[lane] = 0;
        lanes_meet();
        if (v && vr < k) list[vr] = v;
        if (c && cr < k) list[cr] = c;
        lanes_meet();
        v = list[lane];
        continue;
      }
      while (b) {
        const int l = __builtin_ctzll(b);
        const uint64_t best = lane_value(c, l);
        // descending: the first `at` stay, the others move by a lane (DPP over the wave)
        const int at = __popcll(__ballot(v > best));
        const uint32_t lo = __builtin_amdgcn_update_dpp(0u, (uint32_t)v, 0x138, 0xF, 0xF, false);
        const uint32_t hi = __builtin_amdgcn_update_dpp(0u, (uint32_t)(v >> 32), 0x138, 0xF, 0xF, false);
        if (lane == at) v = best;
        else if (lane > at) v = (uint64_t)hi << 32 | lo;
        if (lane == l) c = 0;
        b = __ballot(c > lane_value(v, k - 1));
      }
    }
    lanes_meet();
    n = 0;
  }
};

constexpr uint32_t ORDER_LEAST = 0x007fffffu;  // of -infinity

// a bound that k lanes reach: the largest number of 20 high bits that k lanes'
// values are no smaller than (a 2^-11 below the k-th largest at most)
__device__ __forceinline__ uint32_t kth_of_lanes(uint32_t v, int k)
{
  uint32_t t = 0;
#pragma unroll 1
  for (uint32_t bit = 0x80000000u; bit >= 0x1000u; bit >>= 1)
    if (__popcll(__ballot(v >= (t | bit))) >= k) t |= bit;
  return t ? max(t, ORDER_LEAST) : 0;
}

constexpr float LOWEST = -3.40282347e38f;
constexpr float LOG2E = 1.44269504088896340736f;

// a thread's sums (m their maximum): sum of e^(x - m) and of (x - m) e^(x - m)
struct Sums {
  float m;
  double s, w;
  __device__ __forceinline__ void rescale(float m2)
  {
    if (m2 == m) return;
    // the factor in single: its error is that of the sums so far alone, U (2 + |d|) of
    // what e^d leaves of them (a double exponential was a fifth of a short part's
    // instructions)
    const double d = (double)m - (double)m2;
    const double f = (double)__builtin_amdgcn_exp2f((m - m2) * LOG2E);
    w = f * (w + (s > 0 ? d * s : 0.0));
    s = f * s;
    m = m2;
  }
  // o's sums against the same maximum or a smaller one
  __device__ __forceinline__ void add(Sums o)
  {
    o.rescale(m);
    s += o.s;
    w += o.w;
  }
};

constexpr int TILE = 1024;  // a wave's logits of one step, 16 a lane

// A block takes a row, or one of `parts` of a row where the rows do not fill the
// chip; its waves take tiles of 1024 logits in turn, so that a wave sees ids in
// ascending order. One pass: a lane adds 16 logits in single against the wave's
// running maximum (their sums go on in double) and compares their maximum with
// the k-th best so far; few tiles after the first have a better one. The first
// tiles' bound is what each wave has a share of k of among its lanes' maxima, found by
// bits with ballots. HBM bound with many rows (1024 rows of 151936 logits 110 us, 5.7 TB/s,
// with one alternative 113, with 20 126); the alternatives' instructions with some
// tens of rows (61 of 201088 15 us without, 27 with 5); round trips and cold code with
// one (6.5 us without, 15 with 20, of which the parts' meeting takes 8).
extern "C" __global__ __launch_bounds__(256) void logprobs(LogprobArgs a)
{
  __shared__ Sums sums_s[4];
  __shared__ alignas(16) uint32_t share_s[4], kth_s[4];  // bounds: of a share of k, of k
  __shared__ uint64_t list_s[4][64], buf_s[4][64 + 256];
  const int r = blockIdx.y, part = blockIdx.x, t = threadIdx.x, lane = t & 63;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const float* const x = a.x + (int64_t)r * a.stride;
  // the part: whole tiles but for the row's last
  const int tiles = (a.vocab + TILE - 1) / TILE;
  const int t0 = (int)((int64_t)part * tiles / a.parts), t1 = (int)((int64_t)(part + 1) * tiles / a.parts);

  IHIP_STAMP_SCOPE;
  IHIP_STAMP(0);
  Sums sum = {LOWEST, 0.0, 0.0};
  TopList top = {0, buf_s[w], list_s[w], 0};
  floatx4u v[4], nv[4];
  auto load = [&](int tile, floatx4u* d) {
    const int base = tile * TILE + 4 * lane;
    if ((tile + 1) * TILE <= a.vocab) {
#pragma unroll
      for (int j = 0; j < 4; j++) d[j] = *(const floatx4u*)(x + base + 256 * j);
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int i = base + 256 * j + e;
          d[j][e] = i < a.vocab ? x[i] : -__builtin_inff();
        }
    }
  };
  if (t0 + w < t1) load(t0 + w, nv);
  // a first bound of the block: each of its waves has a share of k as large, among
  // the lanes' maxima of its first tile
  const int active = min(4, t1 - t0), share = (a.k + active - 1) / active;
  if (a.k) {
    float m = nv[0][0];
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
      for (int e = 0; e < 4; e++) m = fmaxf(m, nv[j][e]);
    uint32_t q = 0;
    if (w < active && (t0 + w + 1) * TILE <= a.vocab) q = kth_of_lanes(order_of(m), share);
    if (lane == 0) {
      share_s[w] = w < active ? q : 0xffffffffu;
      kth_s[w] = 0;
    }
    __syncthreads();
  }
  IHIP_STAMP(1);
  for (int tile = t0 + w; tile < t1; tile += 4) {
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = nv[j];
    if (tile + 4 < t1) load(tile + 4, nv);
    float m = v[0][0];
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
      for (int e = 0; e < 4; e++) m = fmaxf(m, v[j][e]);
    // one maximum for the wave's lanes: it grows in few tiles
    if (__any(m > sum.m)) sum.rescale(fmaxf(sum.m, wave_max(m)));
    float s[4], wsum[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      s[j] = wsum[j] = 0.f;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float d = v[j][e] - sum.m;
        const float p = __builtin_amdgcn_exp2f(d * LOG2E);
        s[j] += p;
        wsum[j] = __builtin_fmaf(fmaxf(d, LOWEST), p, wsum[j]);  // (-infinity times 0)
      }
    }
    sum.s += (double)((s[0] + s[1]) + (s[2] + s[3]));
    sum.w += (double)((wsum[0] + wsum[1]) + (wsum[2] + wsum[3]));
    if (a.k) {
      const bool start = tile == t0 + w;
      uint32_t least;
      const uintx4 q = *(const volatile uintx4*)share_s, f = *(const volatile uintx4*)kth_s;
      least = min(min(q[0], q[1]), min(q[2], q[3]));
      if (start) {
        // equal ones only until there are k; a wave that knows no bound takes its own
        if (!least && (tile + 1) * TILE <= a.vocab) least = kth_of_lanes(order_of(m), a.k);
      } else {
        // larger than the wave's own k-th, as ids ascend; no smaller than another
        // wave's, or than what each wave has its share of (what the waves last wrote: an
        // older bound holds too)
        least = max(max(least, max(max(f[0], f[1]), max(f[2], f[3]))), (uint32_t)(lane_value(top.v, a.k - 1) >> 32) + 1);
      }
      float bound = order_value(max(least, ORDER_LEAST));  // (NaN above infinity)
      if (start || __any(m >= bound)) {
        const int base = tile * TILE + 4 * lane;
        const uint32_t first = least;
        int equal = 0;
#pragma unroll 1
        for (int j = 0; j < 4; j++) {
#pragma unroll
          for (int e = 0; e < 4; e++) {
            if (__ballot(v[0][e] >= bound || least == 0)) {
              const int i = base + 256 * j + e;
              const uint32_t o = order_of(v[0][e]);
              const bool in = o >= least && i < a.vocab;
              if (start) equal += __popcll(__ballot(in && o == first));
              top.add(__ballot(in), in, (uint64_t)o << 32 | (uint32_t)~i);
            }
          }
          if (start && equal >= a.k) {
            least = first + 1;
            bound = order_value(max(least, ORDER_LEAST));
          }
          if (top.n > 64 || j == 3) top.flush(a.k);
          v[0] = v[1];
          v[1] = v[2];
          v[2] = v[3];
        }
        if (lane == 0) {
          share_s[w] = max(q[w], (uint32_t)(lane_value(top.v, share - 1) >> 32));
          kth_s[w] = (uint32_t)(lane_value(top.v, a.k - 1) >> 32);
        }
      }
    }
  }

  // the lanes' sums and the waves' meet, then, of a row in parts, the parts' in its
  // last block
  IHIP_STAMP(2);
  Sums z = sum;
#pragma unroll 1
  for (int parts = a.parts;; parts = 1) {
    z.s = wave_sum(z.s, 64);
    z.w = wave_sum(z.w, 64);
    if (lane == 0) sums_s[w] = z;
    list_s[w][lane] = top.v;
    __syncthreads();
    z = sums_s[lane & 3];
    // (a wave without a tile: no sums, the lowest maximum)
    z.rescale(fmaxf(fmaxf(sums_s[0].m, sums_s[1].m), fmaxf(sums_s[2].m, sums_s[3].m)));
    z.s = wave_sum(z.s, 4);
    z.w = wave_sum(z.w, 4);
    if (a.k) {
      // an alternative's place among all: behind its own list's, and the others' better ones
      // (the lists descend, so a number's place in one is a search)
      const uint64_t mine = top.v;
      int n[3] = {0, 0, 0};
#pragma unroll 1
      for (int step = 32; step; step >>= 1)
#pragma unroll
        for (int i = 0; i < 3; i++)
          if (list_s[(w + i + 1) & 3][n[i] + step - 1] > mine) n[i] += step;
      int rank = lane;
#pragma unroll
      for (int i = 0; i < 3; i++) rank += n[i] + (n[i] == 63 && list_s[(w + i + 1) & 3][63] > mine);
      buf_s[0][t < a.k ? t : 64] = 0;
      __syncthreads();
      if (lane < a.k && mine && rank < a.k) buf_s[0][rank] = mine;
      __syncthreads();
      top.v = lane < a.k ? buf_s[0][lane] : 0;
    }
    IHIP_STAMP(3);
    if (parts == 1) break;
    double* const p = a.part + ((int64_t)r * a.parts + part) * (3 + a.k);
    if (t < a.k) store_agent(p + 3 + t, __builtin_bit_cast(double, top.v));
    if (t == 0) {
      store_agent(p, (double)z.m);
      store_agent(p + 1, z.s);
      store_agent(p + 2, z.w);
    }
    if (!last_block(a.done + 8 * r, a.parts)) return;
    if (t == 0) __hip_atomic_store(a.done + 8 * r, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    IHIP_STAMP(4);
    const double* const q = a.part + (int64_t)r * a.parts * (3 + a.k);
    z = {LOWEST, 0.0, 0.0};
    top.v = 0;
    uint64_t c[4];  // the wave's first alternatives, on their way meanwhile
    const int all = a.parts * a.k;
    auto alternative = [&](int i0) {
      const int i = min(i0 + lane, all - 1), of = i / a.k;
      return __builtin_bit_cast(uint64_t, load_agent(q + (int64_t)of * (3 + a.k) + 3 + i - of * a.k));
    };
    if (a.k)
#pragma unroll
      for (int j = 0; j < 4; j++) c[j] = alternative(64 * w + 256 * j);
    for (int i0 = 64 * w; i0 < a.parts; i0 += 256) {
      const double* const e = q + (int64_t)min(i0 + lane, a.parts - 1) * (3 + a.k);
      const bool in = i0 + lane < a.parts;
      const float em = (float)load_agent(e);
      const double es = load_agent(e + 1), ew = load_agent(e + 2);
      z.rescale(fmaxf(z.m, wave_max(em)));
      z.add({em, in ? es : 0.0, in ? ew : 0.0});
    }
    if (a.k) {
      // a bound that k of them reach: some lanes' parts have their j-th that good
      const int lanes = min(a.parts, 64), j = (a.k + lanes - 1) / lanes;
      uint32_t best = 0;
      for (int i = lane; i < a.parts; i += 64)
        best = max(best, (uint32_t)(__builtin_bit_cast(uint64_t, load_agent(q + (int64_t)i * (3 + a.k) + 2 + j)) >> 32));
      const uint64_t bound = (uint64_t)kth_of_lanes(best, (a.k + j - 1) / j) << 32;
#pragma unroll 1
      for (int i0 = 64 * w; i0 < all; i0 += 256) {
        const bool in = i0 + lane < all && c[0] >= bound && c[0];
        top.add(__ballot(in), in, c[0]);
        if (top.n > 64) top.flush(a.k);
        c[0] = c[1];
        c[1] = c[2];
        c[2] = c[3];
        if (i0 + 1024 < all) c[3] = alternative(i0 + 1024);
      }
      top.flush(a.k);
    }
    IHIP_STAMP(5);
  }

  // s is NaN where a logit is NaN or +infinity, 0 where all are -infinity
  const bool none = z.s == 0.0;
  const double ls = log(z.s), m = z.m;
  auto lp = [&](float l) { return none ? -__builtin_inff() : (float)((double)l - m - ls); };
  if (t == 0) {
    if (a.logprobs) {
      const int id = a.ids[r];
      a.logprobs[r] = id >= 0 && id < a.vocab ? lp(x[id]) : __builtin_nanf("");
    }
    if (a.entropy) a.entropy[r] = none ? 0.f : (float)(ls - z.w / z.s);
  }
  if (t < a.k) {
    const uint64_t c = top.v;
    a.top_ids[(int64_t)r * a.k + t] = c ? (int)~(uint32_t)c : -1;
    a.top_logprobs[(int64_t)r * a.k + t] = c ? lp(order_value((uint32_t)(c >> 32))) : -__builtin_inff();
  }
  IHIP_STAMP(6);
}
