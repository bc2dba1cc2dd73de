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

// the alternatives of a wave: lane i holds the i-th best so far as (order, ~id),
// 0 where there is none yet, so that a larger number is a better alternative
struct TopList {
  uint64_t v;
  __device__ __forceinline__ void insert(uint64_t c)  // c the same in every lane
  {
    const int at = __popcll(__ballot(v > c));  // descending: the first `at` stay
    // the lane before: DPP shifts over the whole wave
    const uint32_t lo = __builtin_amdgcn_update_dpp(0u, (uint32_t)v, 0x138, 0xF, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0u, (uint32_t)(v >> 32), 0x138, 0xF, 0xF, false);
    const int lane = threadIdx.x & 63;
    if (lane == at) v = c;
    else if (lane > at) v = (uint64_t)hi << 32 | lo;
  }
  // every lane's c (0: none) that is better than the list's k-th
  __device__ __forceinline__ void insert_lanes(uint64_t c, int k)
  {
    for (;;) {
      const uint64_t b = __ballot(c > lane_value(v, k - 1));
      if (!b) return;
      const int l = __builtin_ctzll(b);
      insert(lane_value(c, l));
      if ((int)(threadIdx.x & 63) == l) c = 0;
    }
  }
};

// the k-th largest of the lanes' values, at least: the largest t with k lanes >= t
__device__ __forceinline__ uint32_t kth_of_lanes(uint32_t v, int k)
{
  uint32_t t = 0;
#pragma unroll 1
  for (uint32_t bit = 0x80000000u; bit; bit >>= 1)
    if (__popcll(__ballot(v >= (t | bit))) >= k) t |= bit;
  return t;
}

// a thread's sums: sum of e^(x - m) and of (x - m) e^(x - m)
struct Sums {
  float m;
  double s, w;
  __device__ __forceinline__ void rescale(float m2)
  {
    if (m2 == m) return;
    const double d = (double)m - (double)m2, f = exp(d);
    w = f * (w + (s > 0 ? d * s : 0.0));
    s = f * s;
    m = m2;
  }
  __device__ __forceinline__ void add(Sums o)
  {
    const float m2 = fmaxf(m, o.m);
    rescale(m2);
    o.rescale(m2);
    s += o.s;
    w += o.w;
  }
};

constexpr float LOWEST = -3.40282347e38f;
constexpr float LOG2E = 1.44269504088896340736f;
constexpr int TILE = 1024;  // a wave's logits of one step, 16 a lane

// A block takes a row, or one of `parts` of a row where the rows do not fill the
// chip; its waves take tiles of 1024 logits in turn, so that a wave sees ids in
// ascending order. One pass: a lane adds 16 logits in single against its own
// running maximum (their sums go on in double) and compares their maximum with
// the wave's k-th best so far; few tiles after the first have a better one, and
// those are inserted one by one into a list held across the lanes. The first
// tile's bound is the k-th largest of the lanes' maxima, found by bits with
// ballots. HBM bound: 4 bytes a logit.
extern "C" __global__ __launch_bounds__(256) void logprobs(LogprobArgs a)
{
  __shared__ Sums sums_s[4];
  __shared__ uint64_t list_s[4][64];
  const int r = blockIdx.y, part = blockIdx.x, t = threadIdx.x, lane = t & 63;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const float* const x = a.x + (int64_t)r * a.stride;
  // the part: whole tiles but for the row's last
  const int tiles = (a.vocab + TILE - 1) / TILE;
  const int t0 = (int)((int64_t)part * tiles / a.parts), t1 = (int)((int64_t)(part + 1) * tiles / a.parts);

  Sums sum = {LOWEST, 0.0, 0.0};
  TopList top = {0};
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
  for (int tile = t0 + w; tile < t1; tile += 4) {
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = nv[j];
    if (tile + 4 < t1) load(tile + 4, nv);
    float m = v[0][0];
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
      for (int e = 0; e < 4; e++) m = fmaxf(m, v[j][e]);
    if (m > sum.m) sum.rescale(m);
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
      const uint64_t kth = lane_value(top.v, a.k - 1);
      const int base = tile * TILE + 4 * lane;
      uint32_t least = (uint32_t)(kth >> 32) + 1;  // ids ascend: only what is larger
      bool look = true;
      if (kth >> 32) look = __any(m > order_value((uint32_t)(kth >> 32)));
      else least = (tile + 1) * TILE <= a.vocab ? kth_of_lanes(order_of(m), a.k) : 0;
      if (look) {
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const int i = base + 256 * j + e;
            const uint32_t o = order_of(v[j][e]);
            const bool in = o >= least && i < a.vocab;
            if (__any(in)) top.insert_lanes(in ? (uint64_t)o << 32 | (uint32_t)~i : 0, a.k);
          }
      }
    }
  }

  // the lanes' sums, then the waves'; the waves' lists
  auto lanes_meet = [&](Sums z) {
    const float m = wave_max(z.m);
    z.rescale(m);
    z.s = wave_sum(z.s, 64);
    z.w = wave_sum(z.w, 64);
    return z;
  };
  auto block_meets = [&](Sums z) {  // sums of the waves (in every lane), lists of the waves
    if (lane == 0) sums_s[w] = z;
    list_s[w][lane] = top.v;
    __syncthreads();
    z = sums_s[0];
    for (int i = 1; i < 4; i++) z.add(sums_s[i]);
    // an alternative's place among all: those before it in its own list, and the
    // better ones of the others'
    const uint64_t mine = top.v;
    int rank = lane;
    for (int i = 0; i < 4; i++) {
      if (i == w) continue;
      int n = 0;
#pragma unroll
      for (int step = 32; step; step >>= 1)
        if (list_s[i][n + step - 1] > mine) n += step;
      n += n == 63 && list_s[i][63] > mine;
      rank += n;
    }
    __syncthreads();
    if (t < 64) list_s[0][t] = 0;
    __syncthreads();
    if (mine && rank < a.k) list_s[0][rank] = mine;
    __syncthreads();
    return z;
  };
  Sums z = block_meets(lanes_meet(sum));

  if (a.parts > 1) {
    double* const p = a.part + ((int64_t)r * a.parts + part) * (3 + a.k);
    if (t < a.k) store_agent(p + 3 + t, __builtin_bit_cast(double, list_s[0][t]));
    if (t == 0) {
      store_agent(p, (double)z.m);
      store_agent(p + 1, z.s);
      store_agent(p + 2, z.w);
    }
    if (!last_block(a.done + 8 * r, a.parts)) return;
    const double* const q = a.part + (int64_t)r * a.parts * (3 + a.k);
    z = {LOWEST, 0.0, 0.0};
    top.v = 0;
    uint64_t bound = 0;  // the best of the parts' k-th: no worse one is among the k
    for (int i = lane; i < a.parts; i += 64) {
      const double* const e = q + (int64_t)i * (3 + a.k);
      if (w == 0) z.add({(float)load_agent(e), load_agent(e + 1), load_agent(e + 2)});
      if (a.k) {
        const uint64_t b = __builtin_bit_cast(uint64_t, load_agent(e + 2 + a.k));
        bound = b > bound ? b : bound;
      }
    }
    if (a.k) {
      bound = wave_max(bound);
      const int all = a.parts * a.k;
      for (int i0 = 64 * w; i0 < all; i0 += 256) {
        const int i = i0 + lane;
        uint64_t c = 0;
        if (i < all) c = __builtin_bit_cast(uint64_t, load_agent(q + (int64_t)(i / a.k) * (3 + a.k) + 3 + i % a.k));
        top.insert_lanes(c >= bound ? c : 0, a.k);
      }
    }
    __syncthreads();
    z = block_meets(lanes_meet(z));
    if (t == 0) __hip_atomic_store(a.done + 8 * r, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
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
    const uint64_t c = list_s[0][t];
    a.top_ids[(int64_t)r * a.k + t] = c ? (int)~(uint32_t)c : -1;
    a.top_logprobs[(int64_t)r * a.k + t] = c ? lp(order_value((uint32_t)(c >> 32))) : -__builtin_inff();
  }
}
