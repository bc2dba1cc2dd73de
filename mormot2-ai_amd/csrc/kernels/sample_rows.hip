// sample_rows.hip - a draw for each row of logits (TInferSampler.Next's filters and
// order, src/infer/mormot.ai.infer.sampler.pas:269-435), with settings and a random
// number of its own for every row.
#include "common.h"
#include "../sample_rows.h"

using namespace ihip;

typedef unsigned long long u64;

struct SampleSettings {  // ihip_sampling
  double temperature;
  int32_t top_k, reserved;
  double top_p, min_p;
  int64_t seed;
};

struct SampleRowsArgs {
  const float* x;
  int64_t stride;
  const SampleSettings* settings;
  const double* uniform;
  int* ids;
  float* probs;
  // of each row's parts: the largest logit and its first id, the sum of the weights 2^((x -
  // that) c), and their sums by octave; of each chunk of 256 the largest logit
  float* best;
  int* best_id;
  double* sum;
  uint32_t* octaves;
  float* chunk;
  struct SampleRow* row;       // what the parts come to
  int* heavy;                  // how many rows have bins, zero between launches, and which
  u64* bins;                   // [SAMPLE_HEAVY][SAMPLE_BINS]
  int* found;                  // [SAMPLE_HEAVY][1 + SAMPLE_CAP]: how many tokens, and which, of the bins that matter
  int32_t rows, vocab, parts, chunks;
  int32_t wide;   // rows aligned to 16 bytes
  int32_t per;    // tokens of a part
};

// a row behind its parts
enum { ROW_DONE, ROW_FEW, ROW_MANY, ROW_BINS };
struct SampleRow {
  double all;     // the sum of its weights (where the filters need it)
  float m, least; // its largest logit, and the least that the filters may keep
  int32_t state;  // answered; its candidates are sorted; are too many; and are in bins
  int32_t slot;   // of `bins`
};

constexpr int OCT = 32;          // octaves below a part's largest weight that are told apart
constexpr int OCT_ONE = 16;      // bits below the point of a weight over its octave
constexpr int CHUNK = 256;       // tokens of a chunk
constexpr int GROUP = 512;       // tokens of a part's sums that a row without filters leaves (where others have octaves)
constexpr int PT = 512;        // threads
constexpr int WAVES = PT / 64;
constexpr int CAP = SAMPLE_CAP;  // candidates that are sorted at once
constexpr int BINS = SAMPLE_BINS;  // of more of them
constexpr int MLP = 8;         // chunks of a wave on their way at once
constexpr double LOG2E_D = 1.4426950408889634074;

enum { ROW_BAD, ROW_GREEDY, ROW_FREE, ROW_FILTERED };

__device__ __forceinline__ bool finite_d(double v) { return fabs(v) < __builtin_inf(); }
__device__ __forceinline__ bool finite_f(float f) { return (float_bits(f) & 0x7f800000u) != 0x7f800000u; }

// what a row's settings ask for (TInferSampler.Create's checks; a temperature too close to
// 0 to divide by is greedy)
__device__ __forceinline__ int row_kind(const SampleSettings& s)
{
  if (!finite_d(s.temperature) || !finite_d(s.top_p) || !finite_d(s.min_p) || s.top_k < 0 || s.top_p <= 0 ||
      s.top_p > 1 || s.min_p < 0 || s.min_p >= 1)
    return ROW_BAD;
  if (s.temperature < 1e-30) return ROW_GREEDY;
  return s.top_k > 0 || s.top_p < 1 || s.min_p > 0 ? ROW_FILTERED : ROW_FREE;
}

// 2^(j / 32) into LDS
__device__ __forceinline__ void weight_roots(double* root)
{
  if (threadIdx.x < 32) root[threadIdx.x] = exp2(threadIdx.x / 32.0);
}

// 2^(s / 32) for s between -32000 and 0: s to its nearest whole number (by the rounding of
// a sum with 1.5 2^52, whose low word then is that number), 2 to the rest by 6 terms of its
// series (the first left out is below 3e-15), the power of two added to the exponent
__device__ __forceinline__ double weight32(double s, const double* root)
{
  constexpr double MAGIC = 6755399441055744.0, L = 0.69314718055994530942 / 32;
  const double z = s + MAGIC, f = s - (z - MAGIC);
  double p = L * L * L * L * L / 120;
  p = __builtin_fma(p, f, L * L * L * L / 24);
  p = __builtin_fma(p, f, L * L * L / 6);
  p = __builtin_fma(p, f, L * L / 2);
  p = __builtin_fma(p, f, L);
  p = __builtin_fma(p, f, 1.0);
  const int j = (int)(uint32_t)__builtin_bit_cast(uint64_t, z);
  const uint64_t r = __builtin_bit_cast(uint64_t, root[j & 31]);
  const uint32_t hi = (uint32_t)(r >> 32) + ((uint32_t)(j >> 5) << 20);
  return p * __builtin_bit_cast(double, (uint64_t)hi << 32 | (uint32_t)r);
}
constexpr double LEAST32 = -32000;  // 2^-1000: no weight beside any other

// the logit as an order-preserving key (-0 as +0)
__device__ __forceinline__ uint32_t row_key(float f)
{
  const uint32_t b = float_bits(f);
  int k = (int)(b ^ ((b >> 31) * 0x7fffffffu));
  if (k == -1) k = 0;
  return (uint32_t)k ^ 0x80000000u;
}
__device__ __forceinline__ float key_logit(uint32_t k)
{
  const uint32_t b = k ^ 0x80000000u;
  return bits_float(b ^ (((int32_t)b >> 31) & 0x7fffffffu));
}

__device__ __forceinline__ u64 lane_of(u64 v, int lane)
{
  return (u64)__builtin_amdgcn_readlane((uint32_t)(v >> 32), lane) << 32 | (uint32_t)__builtin_amdgcn_readlane((uint32_t)v, lane);
}

// v's sum over the lanes up to this one, in registers (v is 0 or positive, so that adding
// 0 changes nothing)
template <int CTRL, int ROWS, typename T>
__device__ __forceinline__ T scan_step(T v)
{
  const u64 b = __builtin_bit_cast(u64, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0u, (uint32_t)b, CTRL, ROWS, 0xF, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0u, (uint32_t)(b >> 32), CTRL, ROWS, 0xF, false);
  return v + __builtin_bit_cast(T, (u64)hi << 32 | lo);
}
template <typename T>
__device__ __forceinline__ T wave_scan(T v)
{
  static_assert(sizeof(T) == 8, "doubles and 64-bit words");
  v = scan_step<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8
  v = scan_step<0x112, 0xF>(v);
  v = scan_step<0x114, 0xF>(v);
  v = scan_step<0x118, 0xF>(v);
  v = scan_step<0x142, 0xA>(v);  // rows 0 and 2 into 1 and 3
  return scan_step<0x143, 0xC>(v);  // rows 0 and 1 into 2 and 3
}

__device__ __forceinline__ int wave_scan32(int v)
{
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
  return v + __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
}

// v's sum over the NT threads before this one, and over all of them
template <int NT, typename T>
__device__ __forceinline__ T scan_threads(T v, T* sh, T& all)
{
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  T s = v;
  if constexpr (sizeof(T) == 8) {
    s = wave_scan(v);
  } else {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const T o = __shfl_up(s, d, 64);
      if (lane >= d) s = s + o;
    }
  }
  __syncthreads();
  if (lane == 63) sh[w] = s;
  __syncthreads();
  T before = T(0);
  all = T(0);
  for (int i = 0; i < NT / 64; i++) {
    if (i < w) before = before + sh[i];
    all = all + sh[i];
  }
  return before + (s - v);
}

// bins of the logits between `least` and m, the largest first: differences, products and
// truncation keep the order
struct LogitBins {
  float m, least, steps;
  __device__ __forceinline__ LogitBins(float m, float least)
      : m(m), least(least), steps((float)((BINS - 1) / ((double)m - (double)least)))
  {
  }
  __device__ __forceinline__ int of(float l) const { return min((int)((m - l) * steps), BINS - 1); }
};

// a weight as a whole number: the sum with 2^52 rounds it, in its low bits
__device__ __forceinline__ u64 whole_weight(double wt, double one)
{
  return __builtin_bit_cast(u64, __builtin_fma(wt, one, 0x1p52)) - __builtin_bit_cast(u64, 0x1p52);
}

// what a part's octaves hold: nothing, whole tokens, or sums of weights
enum { OCT_NONE, OCT_COUNTS, OCT_SUMS };
__device__ __forceinline__ int octave_kind(const SampleSettings& s)
{
  return s.top_k > 0 ? OCT_COUNTS : s.top_p < 1 ? OCT_SUMS : OCT_NONE;
}

// ------------------------------------------------------------- sample_rows_part
// A part of a row: its tokens in registers, read once; the largest logits of chunks, the
// part's largest, then, for rows that need it, the sum of the weights in double, and how
// many tokens, or which sums, lie in each octave below the largest (in whole numbers, a
// lane's own places in LDS, so that no order changes them). A row with top-k needs
// counts alone, which singles tell well enough (sample_rows_finish leaves room for them); a
// greedy one neither. Bound by vector arithmetic (500 rows of 151936, three of eight with sums,
// three with counts: 67 us, 4.5 TB/s, the SIMDs busy throughout), then by HBM.
template <int IT>
__device__ __forceinline__ void sample_part_t(const SampleRowsArgs& a)
{
  __shared__ double root[32], part[4];
  __shared__ float top[4];
  __shared__ int first[4];
  __shared__ uint32_t oct[(OCT + 1) * 64];  // (the last: of the others, which no one looks at)
  const int t = threadIdx.x, lane = t & 63, w = t >> 6;
  const int row = blockIdx.y, p = blockIdx.x;
  const float* const x = a.x + (int64_t)row * a.stride;
  const int i0 = p * a.per;
  float v[IT][4];
#pragma unroll
  for (int i = 0; i < IT; i++) {
    const int at = i0 + i * 1024 + 4 * t;
    if (a.wide && at + 4 <= a.vocab) {
      const float4 l = *(const float4*)(x + at);
      v[i][0] = l.x; v[i][1] = l.y; v[i][2] = l.z; v[i][3] = l.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) v[i][e] = at + e < a.vocab ? x[at + e] : bits_float(0x7fc00000u);
    }
  }
  const SampleSettings set = a.settings[row];
  const int kind = row_kind(set);
  if (kind == ROW_BAD) return;
  const bool filtered = kind == ROW_FILTERED;
  const int deep = filtered ? octave_kind(set) : OCT_NONE;
  const bool sums = kind == ROW_FREE || deep == OCT_SUMS;
  if (sums) weight_roots(root);
  if (deep)
    for (int i = t; i < OCT * 64; i += 256) oct[i] = 0;
  float m = -__builtin_inff();
#pragma unroll
  for (int i = 0; i < IT; i++) {
    const float c = fmaxf(fmaxf(v[i][0], v[i][1]), fmaxf(v[i][2], v[i][3]));
    m = fmaxf(m, c);
    if (filtered) {
      const float cm = wave_max(fmaxf(c, -__builtin_inff()));
      const int chunk = (i0 + i * 1024) / CHUNK + w;
      if (lane == 0 && chunk < a.chunks) a.chunk[(int64_t)row * a.chunks + chunk] = cm;
    }
  }
  const float own = m;
  m = wave_max(m);
  if (lane == 0) top[w] = m;
  __syncthreads();
  m = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
  int id = INT32_MAX;
  if (own == m) {
#pragma unroll
    for (int i = IT - 1; i >= 0; i--)
#pragma unroll
      for (int e = 3; e >= 0; e--)
        if (v[i][e] == m) id = i0 + i * 1024 + 4 * t + e;
  }
  id = -wave_max(-id);
  double s = 0;
  if (sums && finite_f(m)) {
    const double c = LOG2E_D / set.temperature * 32, md = m;
    auto add = [&](bool octaves) {
#pragma unroll
      for (int i = 0; i < IT; i++) {
        double four = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          // (NaN and -infinity among the least: a weight of 2^-1000 changes no sum)
          const double wt = weight32(fmax(((double)v[i][e] - md) * c, LEAST32), root);
          four = four + wt;
          if (octaves) {
            const uint32_t hi = (uint32_t)(__builtin_bit_cast(uint64_t, wt) >> 32);
            const uint32_t o = min(1023u - (hi >> 20), (uint32_t)OCT);  // 2^-o <= weight < 2^(1 - o)
            atomicAdd(&oct[o * 64 + lane], ((hi >> 4) & 0xffffu) | 0x10000u);
          }
        }
        if (!octaves) {
          four = wave_sum(four, 64);
          if (lane == 0) ((double*)oct)[i * 4 + w] = four;
        }
        s = s + four;
      }
    };
    if (deep) add(true);
    else add(false);
    if (!deep) s = lane == 0 ? s : 0;  // (the wave's already)
    s = wave_sum(s, 64);
  } else if (deep && finite_f(m)) {
    const float c = (float)(LOG2E_D / set.temperature);
#pragma unroll
    for (int i = 0; i < IT; i++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float o = fminf(ceilf((m - v[i][e]) * c), (float)OCT);  // weight >= 2^-o, up to the rounding (NaN: OCT)
        atomicAdd(&oct[(int)o * 64 + lane], 1u);
      }
  }
  if (lane == 0) {
    part[w] = s;
    first[w] = id;
  }
  __syncthreads();
  const int64_t to = (int64_t)row * a.parts + p;
  if (t == 0) {
    a.best[to] = m;
    a.best_id[to] = min(min(first[0], first[1]), min(first[2], first[3]));
    a.sum[to] = (part[0] + part[1]) + (part[2] + part[3]);
  }
  if (kind == ROW_FREE && finite_f(m) && t < IT * 2) ((double*)a.octaves)[to * (OCT / 2) + t] = ((double*)oct)[2 * t] + ((double*)oct)[2 * t + 1];
  if (deep) {
    uint32_t n = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) n += oct[(t >> 3) * 64 + (t & 7) * 8 + j];
    n = wave_sum(n, 8);
    if ((t & 7) == 0) a.octaves[to * OCT + (t >> 3)] = n;
  }
}

extern "C" __global__ __launch_bounds__(256) void sample_rows_part_2048(SampleRowsArgs a) { sample_part_t<2>(a); }
extern "C" __global__ __launch_bounds__(256) void sample_rows_part_4096(SampleRowsArgs a) { sample_part_t<4>(a); }
extern "C" __global__ __launch_bounds__(256, 5) void sample_rows_part_8192(SampleRowsArgs a) { sample_part_t<8>(a); }

// ------------------------------------------------------------- sample_rows_finish
// A block a row, behind its parts (a launch of its own: as the work of a row's last block
// it held the other blocks' places while their results went to memory, 500 rows 107 us
// for 65 and 9). Greedy rows take the best of them; rows without
// filters find the part in which the draw falls and look through that one again; of the
// others come the sum of the weights and the logit above which the tokens surely hold
// what the filters keep (by the parts' octaves, or min-p's share), and, where those are
// too many to be sorted, a place for their bins.
extern "C" __global__ __launch_bounds__(256) void sample_rows_finish(SampleRowsArgs a)
{
  constexpr int NT = 256;
  __shared__ double root[32];
  __shared__ u64 octave[64];
  __shared__ uint32_t tokens[64];
  __shared__ double sums[NT / 64], base;
  __shared__ float topf[NT / 64];
  __shared__ int topi[NT / 64], found, seen, slot;
  const int t = threadIdx.x, lane = t & 63, w = t >> 6;
  const int row = blockIdx.x;
  const int64_t p0 = (int64_t)row * a.parts;
  const SampleSettings set = a.settings[row];
  const int kind = row_kind(set), deep = kind == ROW_FILTERED ? octave_kind(set) : OCT_NONE;
  const float* const x = a.x + (int64_t)row * a.stride;
  auto answer = [&](int id, double prob) {
    a.ids[row] = id;
    if (a.probs) a.probs[row] = (float)prob;
    a.row[row].state = ROW_DONE;
  };
  // (the first octaves of a thread on their way while the best is found)
  constexpr int AHEAD = 4;
  uint32_t on[AHEAD];
  float om[AHEAD];
  const int octs = a.parts * OCT;
#pragma unroll
  for (int i = 0; i < AHEAD; i++) {
    const int at = min(t + i * NT, octs - 1);
    on[i] = deep ? a.octaves[p0 * OCT + at] : 0u;
    om[i] = deep ? a.best[p0 + at / OCT] : 0.f;
  }
  if (kind == ROW_BAD) {
    if (t == 0) answer(-1, 0.0);
    return;
  }
  weight_roots(root);
  float m = -__builtin_inff();
  int id = INT32_MAX;
  for (int p = t; p < a.parts; p += NT) {
    const float pm = a.best[p0 + p];
    const int pi = a.best_id[p0 + p];
    if (pm > m || (pm == m && pi < id)) {
      m = pm;
      id = pi;
    }
  }
  if (t < 64) {
    octave[t] = 0;
    tokens[t] = 0;
  }
  {
    const float wm = wave_max(m);
    const int wi = -wave_max(m == wm ? -id : -INT32_MAX);
    if (lane == 0) {
      topf[w] = wm;
      topi[w] = wi;
    }
    __syncthreads();
    m = topf[0];
    for (int i = 1; i < NT / 64; i++) m = fmaxf(m, topf[i]);
    id = INT32_MAX;
    for (int i = 0; i < NT / 64; i++)
      if (topf[i] == m) id = min(id, topi[i]);
  }
  const int best = id == INT32_MAX ? 0 : id;  // (a row of NaN: 0)
  if (kind == ROW_GREEDY || !finite_f(m)) {
    if (t == 0) answer(best, 1.0);
    return;
  }
  const double c = LOG2E_D / set.temperature, c32 = c * 32, md = m;
  auto weight_of = [&](float l) {  // 0 for -infinity and NaN
    const double y = ((double)l - md) * c32;
    return y >= LEAST32 ? weight32(y, root) : 0.0;
  };

  // the sum of all weights, and that of the parts before this thread's
  const int pq = (a.parts + NT - 1) / NT;
  double before = 0, all = 0;
  auto part_sum = [&](int p) {
    const float pm = a.best[p0 + p];
    return finite_f(pm) ? a.sum[p0 + p] * weight_of(pm) : 0.0;
  };
  if (kind == ROW_FREE || deep == OCT_SUMS) {
    double mine = 0;
    for (int p = t * pq; p < min((t + 1) * pq, a.parts); p++) mine = mine + part_sum(p);
    before = scan_threads<NT>(mine, sums, all);
  }
  if (kind == ROW_FREE) {
    const double target = a.uniform[row] * all;
    // the first part whose sums pass the target; none (rounding, or a number of 1): the best
    if (t == 0) found = INT32_MAX;
    __syncthreads();
    for (int p = t * pq; p < min((t + 1) * pq, a.parts); p++) {
      const double add = part_sum(p);
      if (add > 0 && target < before + add) {
        atomicMin(&found, p);
        break;
      }
      before = before + add;
    }
    __syncthreads();
    const int part = found;
    if (part == INT32_MAX) {
      if (t == 0) answer(best, 1.0 / all);
      return;
    }
    if (part / pq == t) base = before;
    __syncthreads();
    // The group of its tokens, by a wave's lanes, then the group's tokens, two a thread. (Tokens
    // without a weight are in its group's sum, as 2^-1000 of the part's best each: a group
    // that turns out to have no other is passed over, and the next one whose sums pass the
    // target is taken, or, where none does, for roundings, the last one before.)
    const float pm = a.best[p0 + part];
    double mine = 0, upto = 0;
    uint64_t ahead = 0, behind = 0;
    if (w == 0) {
      const double* const g = (const double*)(a.octaves + (p0 + part) * OCT);
      mine = lane < a.per / GROUP ? g[lane] * weight_of(pm) : 0.0;
      upto = base + wave_scan(mine);
      ahead = __ballot(mine > 0 && target < upto);
      behind = __ballot(mine > 0) & ~ahead;
    }
    for (;;) {
      if (w == 0) {
        const int at = ahead ? __builtin_ctzll(ahead) : behind ? 63 - __builtin_clzll(behind) : -1;
        if (lane == max(at, 0)) {
          sums[0] = upto - mine;
          slot = at;
          found = INT32_MAX;
          seen = -1;
        }
        if (ahead) ahead &= ahead - 1;
        else if (behind) behind &= ~(1ull << at);
      }
      __syncthreads();
      const int group = slot;
      if (group < 0) {  // (not reached: the part's best has a weight)
        if (t == 0) answer(best, 1.0 / all);
        return;
      }
      const int i0 = part * a.per + group * GROUP + 2 * t;
      const double start = sums[0];
      double wt[2], group_all;
#pragma unroll
      for (int e = 0; e < 2; e++) wt[e] = i0 + e < a.vocab ? weight_of(x[i0 + e]) : 0.0;
      double run = start + scan_threads<NT>(wt[0] + wt[1], sums, group_all);
      int first = INT32_MAX, last = -1;
#pragma unroll
      for (int e = 0; e < 2; e++) {
        run = run + wt[e];
        if (wt[e] > 0) last = i0 + e;  // (the last one, where roundings leave none)
        if (wt[e] > 0 && target < run) first = min(first, i0 + e);
      }
      last = wave_max(last);
      first = -wave_max(-first);
      if (lane == 0) {
        atomicMax(&seen, last);
        atomicMin(&found, first);
      }
      __syncthreads();
      if (group_all > 0) {
        if (t == 0) {
          const int i = found != INT32_MAX ? found : seen;
          answer(i, weight_of(x[i]) / all);
        }
        return;
      }
      __syncthreads();
    }
  }

  // the octave below the best weight that surely holds k tokens, or top_p of the sum
  const bool by_p = set.top_p < 1, by_k = set.top_k > 0;
  double lo = -__builtin_inf();
  int state = ROW_FEW;
  if (deep) {
    auto enter = [&](int i, uint32_t n, float pm) {
      const int o = i % OCT;
      if (n == 0 || !finite_f(pm)) return;
      const double below = (md - (double)pm) * c;  // of the part's best
      const double k = ceil(below) + o;            // every weight of these is 2^-k at least
      if (k < 64) {
        atomicAdd(&tokens[(int)k], deep == OCT_COUNTS ? n : n >> 8);
        if (deep == OCT_SUMS) atomicAdd(&octave[(int)k], (u64)(ldexp(n * weight_of(pm), 40 - OCT_ONE - o)));
      }
    };
#pragma unroll
    for (int i = 0; i < AHEAD; i++)
      if (t + i * NT < octs) enter(t + i * NT, on[i], om[i]);
#pragma unroll 1
    for (int i = t + AHEAD * NT; i < octs; i += AHEAD * NT) {
#pragma unroll
      for (int j = 0; j < AHEAD; j++) {
        const int at = min(i + j * NT, octs - 1);
        on[j] = a.octaves[p0 * OCT + at];
        om[j] = a.best[p0 + at / OCT];
      }
#pragma unroll
      for (int j = 0; j < AHEAD; j++)
        if (i + j * NT < octs) enter(i + j * NT, on[j], om[j]);
    }
    __syncthreads();
    if (w == 0) {
      u64 mass = octave[lane];
      uint32_t n = tokens[lane];  // (of sums: 2^(OCT_ONE - 8) a token, for its place in the octave up to twice that)
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const u64 o = __shfl_up(mass, d, 64);
        const uint32_t on2 = __shfl_up(n, d, 64);
        if (lane >= d) mass += o, n += on2;
      }
      const bool enough = deep == OCT_COUNTS ? n >= (uint32_t)set.top_k : (double)mass * 0x1p-40 >= set.top_p * all * (1 + 1e-9);
      const uint64_t there = __ballot(enough);
      const int k = there ? __builtin_ctzll(there) : -1;
      if (lane == 0) found = k;
      if (lane == max(k, 0)) seen = !there || (deep == OCT_COUNTS ? n : n >> (OCT_ONE - 8)) > (uint32_t)CAP;
    }
    __syncthreads();
    // (counts are by singles: room for 2^-20 of their distance and of an octave)
    if (found >= 0) lo = md - (found + (deep == OCT_COUNTS ? (found + 1) * 0x1p-20 : 0.0)) / c;
    if (seen) state = ROW_MANY;
  }
  const double floor = set.min_p;
  if (floor > 0 && !(by_k && by_p)) {
    lo = fmax(lo, md + log2(floor) / c);
    state = ROW_FEW;  // (not known)
  }
  lo = lo - 1e-9 * (fabs(lo) + fabs(md));
  float least = (float)lo;
  if ((double)least > lo) least = key_logit(row_key(least) - 1);
  if (!(least > -3.4028235e38f)) least = -3.4028235e38f;  // (infinities and NaN are no candidates)
  // (Rows with top-k have no bins by the grid. Where their octaves do not hold k tokens - large k,
  // or a low temperature, at which few tokens lie within 2^-32 of their part's best - one
  // block walks the row several times: 16 rows of 151936 at temperature 0.1 with top-k 40
  // 765 us, 21 at 0.8.)
  if (state == ROW_MANY && !by_k) {
    if (t == 0) {
      slot = atomicAdd(a.heavy, 1);
      if (slot < SAMPLE_HEAVY) a.heavy[1 + slot] = row;
    }
    __syncthreads();
    if (slot < SAMPLE_HEAVY) {
      state = ROW_BINS;
      for (int i = t; i < BINS; i += NT) a.bins[(int64_t)slot * BINS + i] = 0;
      if (t == 0) a.found[(int64_t)slot * (1 + CAP)] = 0;
    }
  }
  if (t == 0) {
    SampleRow r;
    r.all = all;
    r.m = m;
    r.least = least;
    r.state = state;
    r.slot = state == ROW_BINS ? slot : -1;
    a.row[row] = r;
  }
}

// ------------------------------------------------------------- sample_rows_bins
// The tasks (a row with bins, a part of it) of this block, in order: each(slot, row, part)
template <typename F>
__device__ __forceinline__ void heavy_tasks(const SampleRowsArgs& a, F&& each)
{
  const int64_t all = (int64_t)min(a.heavy[0], SAMPLE_HEAVY) * a.parts;
  const int64_t i0 = all * blockIdx.x / gridDim.x, i1 = all * (blockIdx.x + 1) / gridDim.x;
  for (int64_t i = i0; i < i1; i++) {
    const int slot = (int)(i / a.parts), row = a.heavy[1 + slot];
    // (what an earlier call, whose launches failed, has left is nobody's)
    if (row >= 0 && row < a.rows && a.row[row].slot == slot) each(slot, row, (int)(i - (int64_t)slot * a.parts));
  }
}

// 4 of each 1024 of a part's tokens a thread: each(logits, id of the first)
template <typename F>
__device__ __forceinline__ void part_tokens(const SampleRowsArgs& a, int row, int part, F&& each)
{
  const float* const x = a.x + (int64_t)row * a.stride;
  for (int i0 = part * a.per; i0 < min((part + 1) * a.per, a.vocab); i0 += 1024) {
    const int at = i0 + 4 * threadIdx.x;
    float v[4];
    if (a.wide && at + 4 <= a.vocab) {
      const float4 l = *(const float4*)(x + at);
      v[0] = l.x; v[1] = l.y; v[2] = l.z; v[3] = l.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) v[e] = at + e < a.vocab ? x[at + e] : -__builtin_inff();
    }
    each(v, at);
  }
}

// The bins of the rows with too many candidates for one block: parts of them shared out
// over the grid, in LDS and then added up (whole numbers: in any order). On one block a
// row's 150000 weights in double take 60 us.
extern "C" __global__ __launch_bounds__(256) void sample_rows_bins(SampleRowsArgs a)
{
  __shared__ double root[32];
  __shared__ u64 mass[BINS];
  const int t = threadIdx.x;
  if (a.heavy[0] == 0) return;
  weight_roots(root);
  const double one = ldexp(1.0, sample_weight_bits(a.vocab));
  for (int i = t; i < BINS; i += 256) mass[i] = 0;
  __syncthreads();
  int cur = -1;
  auto flush = [&]() {
    __syncthreads();
    for (int i = t; i < BINS; i += 256) {
      if (mass[i]) atomicAdd(a.bins + (int64_t)cur * BINS + i, mass[i]);
      mass[i] = 0;
    }
    __syncthreads();
  };
  heavy_tasks(a, [&](int slot, int row, int part) {
    if (cur >= 0 && cur != slot) flush();
    cur = slot;
    const SampleRow r = a.row[row];
    const double c32 = LOG2E_D / a.settings[row].temperature * 32, md = r.m;
    const LogitBins bins(r.m, r.least);
    part_tokens(a, row, part, [&](const float (&v)[4], int) {
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (v[e] >= r.least) {
          const double wt = weight32(fmax(((double)v[e] - md) * c32, LEAST32), root);
          atomicAdd(&mass[bins.of(v[e])], whole_weight(wt, one));
        }
    });
  });
  if (cur >= 0) flush();
}

// The first bin whose weights, those of the larger bins with them, come to `upto` (or pass
// it), at most `last`; mass_to(i): those before bin i. -1: none. NT threads.
template <int NT, bool PASS, typename F>
__device__ __forceinline__ int first_bin(int* found, int last, double upto, F&& mass_to)
{
  __syncthreads();
  if (threadIdx.x == 0) *found = INT32_MAX;
  __syncthreads();
  for (int i = threadIdx.x; i <= last; i += NT)
    if (PASS ? mass_to(i + 1) > upto : mass_to(i + 1) >= upto) {
      atomicMin(found, i);
      break;
    }
  __syncthreads();
  const int b = *found;
  return b == INT32_MAX ? -1 : b;
}

// the bin in which top-p's share ends, and the one in which the draw then falls, as nearly
// as is known before that one's tokens are (-1: the same, or none)
template <int NT, typename F>
__device__ __forceinline__ int border_bins(int* found, double upto, double u, F&& mass_to, int& ahead)
{
  ahead = -1;
  const int b = first_bin<NT, false>(found, BINS - 1, upto, mass_to);
  if (b > 0) ahead = first_bin<NT, true>(found, b, u * upto, mass_to);
  if (ahead == b) ahead = -1;
  return b;
}

// ------------------------------------------------------------- sample_rows_find
// The tokens of the two bins that matter of each row with bins, by the grid's blocks (on one
// block 30 us a row); each forms the bins' running sums for itself.
extern "C" __global__ __launch_bounds__(256) void sample_rows_find(SampleRowsArgs a)
{
  constexpr int NT = 256, Q = BINS / NT;
  __shared__ u64 mass[BINS], scan[NT / 64];
  __shared__ int found;
  const int t = threadIdx.x;
  if (a.heavy[0] == 0) return;
  int cur = -1, b = -1, ahead = -1;
  const int bits = sample_weight_bits(a.vocab);
  heavy_tasks(a, [&](int slot, int row, int part) {
    const SampleRow r = a.row[row];
    if (cur != slot) {
      u64 m[Q], sum = 0, all;
#pragma unroll
      for (int i = 0; i < Q; i++) sum += m[i] = a.bins[(int64_t)slot * BINS + Q * t + i];
      u64 to = scan_threads<NT>(sum, scan, all);
#pragma unroll
      for (int i = 0; i < Q; i++) {
        mass[Q * t + i] = to;
        to += m[i];
      }
      b = border_bins<NT>(&found, a.settings[row].top_p * r.all, a.uniform[row],
                          [&](int i) { return ldexp((double)(i >= BINS ? all : mass[i]), -bits); }, ahead);
      cur = slot;
    }
    if (b < 0) return;  // (the threads alike)
    const LogitBins bins(r.m, r.least);
    int* const list = a.found + (int64_t)slot * (1 + CAP);
    part_tokens(a, row, part, [&](const float (&v)[4], int at) {
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int i = bins.of(v[e]);
        if (v[e] >= r.least && (i == b || i == ahead)) {
          const int to = atomicAdd(list, 1);
          if (to < CAP) list[1 + to] = at + e;
        }
      }
    });
  });
}

// ------------------------------------------------------------- sample_rows_pick
struct PickLds {
  double root[32], wave[WAVES], total;
  u64 scan[WAVES];
  int topi[WAVES], chunk[WAVES][MLP];
  int n, at, found, ties;
  uint32_t key;            // a search's result: the key,
  u64 above;               // the weights of larger keys
  u64 cand[CAP];           // key << 32 | ~id
  uint32_t ids[CAP];
  u64 mass[BINS];          // weights of a bin, then those of the bins before it
  uint32_t count[BINS];    // tokens likewise
};

// A sorted list of E values a thread of T (a wave's, or the block's), the largest first:
// value e of thread t is number e T + t. Steps of the bitonic network within a wave are
// register moves, those between waves go through LDS, those between a thread's values
// are its own.
template <int T, int E>
struct SortedList {
  static_assert(T == 64 || T == PT, "a wave or the block");
  u64 v[E];
  double wt[E], before[E];  // weights, and their sums before each
  double all;
  int n, t;

  __device__ __forceinline__ int at(int e) const { return e * T + t; }

  template <int K>
  __device__ __forceinline__ void step(int k)
  {
#pragma unroll
    for (int e = 0; e < E; e++) {
      const u64 o = xswap<K>(v[e]);
      const bool most = ((at(e) & K) == 0) == ((at(e) & k) == 0);
      v[e] = (o > v[e]) == most ? o : v[e];
    }
  }

  // the values at c, zeros behind them
  __device__ __forceinline__ void sort(u64* c, int count)
  {
    n = count;
    t = T == 64 ? threadIdx.x & 63 : threadIdx.x;
    int size = 64;
    while (size < n) size *= 2;
#pragma unroll
    for (int e = 0; e < E; e++) v[e] = at(e) < n ? c[at(e)] : 0;
    for (int k = 2; k <= size; k *= 2) {
      int j = k / 2;
#pragma unroll
      for (int d = E / 2; d > 0; d /= 2)
        if (j == d * T) {
#pragma unroll
          for (int e = 0; e < E; e++)
            if ((e & d) == 0) {
              const u64 a = v[e], b = v[e + d];
              const bool most = (at(e) & k) == 0;
              v[e] = (a > b) == most ? a : b;
              v[e + d] = (a > b) == most ? b : a;
            }
          j /= 2;
        }
      if constexpr (T > 64)
        for (; j >= 64; j /= 2) {
          __syncthreads();
#pragma unroll
          for (int e = 0; e < E; e++)
            if (e * T < size) c[at(e)] = v[e];
          __syncthreads();
#pragma unroll
          for (int e = 0; e < E; e++)
            if (e * T < size) {
              const u64 o = c[at(e) ^ j];
              const bool most = ((at(e) & j) == 0) == ((at(e) & k) == 0);
              v[e] = (o > v[e]) == most ? o : v[e];
            }
        }
      if (j >= 32) step<32>(k);
      if (j >= 16) step<16>(k);
      if (j >= 8) step<8>(k);
      if (j >= 4) step<4>(k);
      if (j >= 2) step<2>(k);
      step<1>(k);
    }
    if constexpr (T > 64) {  // (the drawn one is read there)
      __syncthreads();
#pragma unroll
      for (int e = 0; e < E; e++)
        if (e * T < size) c[at(e)] = v[e];
      __syncthreads();
    }
  }

  template <typename F>
  __device__ __forceinline__ void weigh(double* sh, F&& weight_of)
  {
    double sum = 0;
#pragma unroll
    for (int e = 0; e < E; e++) {
      wt[e] = before[e] = 0;
      if (e > 0 && e * T >= n) continue;  // (the threads' alike)
      wt[e] = at(e) < n ? weight_of(key_logit((uint32_t)(v[e] >> 32))) : 0.0;
      const double run = wave_scan(wt[e]);
      double part = 0, whole = __builtin_bit_cast(double, lane_of(__builtin_bit_cast(u64, run), 63));
      if constexpr (T > 64) {
        __syncthreads();
        if ((t & 63) == 63) sh[t >> 6] = run;
        __syncthreads();
        whole = 0;
        for (int i = 0; i < T / 64; i++) {
          if (i < t >> 6) part = part + sh[i];
          whole = whole + sh[i];
        }
      }
      before[e] = sum + part + (run - wt[e]);
      sum = sum + whole;
    }
    all = sum;
  }

  // how many say yes: yes(number, e)
  template <typename F>
  __device__ __forceinline__ int count(int* sh, F&& yes) const
  {
    int c = 0;
#pragma unroll
    for (int e = 0; e < E; e++)
      if (e == 0 || e * T < n) c += __popcll(__ballot(at(e) < n && yes(at(e), e)));
    if constexpr (T > 64) {
      __syncthreads();
      if ((t & 63) == 0) sh[t >> 6] = c;
      __syncthreads();
      c = 0;
      for (int i = 0; i < T / 64; i++) c += sh[i];
    }
    return c;
  }

  // f(e) of number i
  template <typename V, typename F>
  __device__ __forceinline__ V of(int i, V* sh, F&& f) const
  {
    V got = V(0);
    if constexpr (T == 64) {
#pragma unroll
      for (int e = 0; e < E; e++)
        if (i / T == e) got = __shfl(f(e), i & 63, 64);
    } else {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < E; e++)
        if (at(e) == i) *sh = f(e);
      __syncthreads();
      got = *sh;
    }
    return got;
  }
  // the weights of the first `count`
  __device__ __forceinline__ double sum_of(int count, double* sh) const
  {
    return count >= n ? all : of<double>(count, sh, [&](int e) { return before[e]; });
  }
};

// the bins' weights and tokens into those before each bin (with `above` and `count` before
// the first)
__device__ __forceinline__ void scan_bins(PickLds& s, u64 above, uint32_t count, u64& mass_all, uint32_t& count_all)
{
  constexpr int Q = BINS / PT;
  const int t = threadIdx.x;
  u64 m[Q], mass = 0;
  uint32_t n[Q], tokens = 0;
#pragma unroll
  for (int i = 0; i < Q; i++) {
    m[i] = s.mass[Q * t + i];
    n[i] = s.count[Q * t + i];
    mass += m[i];
    tokens += n[i];
  }
  u64 mb = above + scan_threads<PT>(mass, s.scan, mass_all);
  uint32_t nb = count + scan_threads<PT>(tokens, (uint32_t*)s.topi, count_all);
#pragma unroll
  for (int i = 0; i < Q; i++) {
    s.mass[Q * t + i] = mb;
    s.count[Q * t + i] = nb;
    mb += m[i];
    nb += n[i];
  }
  mass_all += above;
  count_all += count;
  __syncthreads();
}

// One block a filtered row. The candidates are gathered from the chunks that reach
// `least`, sorted, and cut in TInferSampler's order by sums in double. Of more of them
// than CAP the bins' weights (whole numbers, so that their order changes nothing) say in
// which bin each border and the draw lie: that bin's tokens are gathered and sorted in
// turn. Logits so much alike that a bin passes CAP are searched by their keys.
template <bool WIDE>
__device__ __forceinline__ void sample_pick_t(const SampleRowsArgs& a)
{
  __shared__ PickLds s;
  IHIP_STAMP_SCOPE;
  IHIP_STAMP(0);
  const int t = threadIdx.x, lane = t & 63, w = t >> 6;
  const int row = blockIdx.x;
  const float* const cmax = a.chunk + (int64_t)row * a.chunks;
  const SampleRow head = a.row[row];
  const SampleSettings set = a.settings[row];
  const double u = a.uniform[row];
  if (row == 0 && t == 0) a.heavy[0] = 0;  // (of the next launch)
  if (head.state == ROW_DONE) return;
  // chunk i of a wave's 64 of a turn of PT: WAVES apart, so that the waves share them alike
  const int mine0 = lane * WAVES + w;
  const float cm0 = mine0 < a.chunks ? cmax[mine0] : -__builtin_inff();  // (of the first turn)
  auto answer = [&](int id, double prob) {
    a.ids[row] = id;
    if (a.probs) a.probs[row] = (float)prob;
  };
  const float* const x = a.x + (int64_t)row * a.stride;
  weight_roots(s.root);
  if (t == 0) s.n = 0;
  __syncthreads();
  IHIP_STAMP(1);
  const float m = head.m, least = head.least;
  const double all = head.all, md = m, c = LOG2E_D / set.temperature, c32 = c * 32;
  auto weight_of = [&](float l) {
    const double y = ((double)l - md) * c32;
    return y >= LEAST32 ? weight32(y, s.root) : 0.0;
  };
  const bool by_p = set.top_p < 1, by_k = set.top_k > 0;
  const double floor = set.min_p;
  bool many = head.state != ROW_FEW;
  // The tokens of the chunks that reach `least`: each(four logits of the lane, the first
  // one's id), MLP chunks of a wave on their way at once. (The code is short, as it comes
  // from a cold cache: chunks move up through the registers instead of being unrolled.)
  auto tokens = [&](auto&& each) {
    for (int c0 = 0; c0 < a.chunks; c0 += PT) {
      const float cm = c0 == 0 ? cm0 : c0 + mine0 < a.chunks ? cmax[c0 + mine0] : -__builtin_inff();
      uint64_t there = __ballot(cm >= least);
      const uint64_t last = __ballot(c0 + mine0 == a.chunks - 1);
      if ((a.vocab & (CHUNK - 1)) && there & last) {  // the row's end, part of a chunk
        there &= ~last;
        const int i0 = (a.chunks - 1) * CHUNK + 4 * lane;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = i0 + e < a.vocab ? x[i0 + e] : -__builtin_inff();
        each(v, i0);
      }
      while (there) {
        float v[MLP][4];
        const int got = min(__popcll(there), MLP);
        uint64_t rest = there;
#pragma unroll
        for (int k = 0; k < MLP; k++) {
          const float* const p = x + (c0 + w + WAVES * __builtin_ctzll(rest)) * CHUNK + 4 * lane;
          if (rest & (rest - 1)) rest &= rest - 1;  // (the last one again)
          if constexpr (WIDE) {
            const float4 l = *(const float4*)p;
            v[k][0] = l.x; v[k][1] = l.y; v[k][2] = l.z; v[k][3] = l.w;
          } else {
#pragma unroll
            for (int e = 0; e < 4; e++) v[k][e] = p[e];
          }
        }
#pragma unroll 1
        for (int k = 0; k < got; k++) {
          each(v[0], (c0 + w + WAVES * __builtin_ctzll(there)) * CHUNK + 4 * lane);
          there &= there - 1;
#pragma unroll
          for (int i = 0; i + 1 < MLP; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) v[i][e] = v[i + 1][e];
        }
      }
    }
  };
  auto read_list = [&]() {
    for (int i = t; i < min(s.n, CAP); i += PT) {
      const uint32_t id = s.ids[i];
      s.cand[i] = (u64)row_key(x[id]) << 32 | (uint32_t)~id;
    }
    __syncthreads();
  };
  // The tokens that say yes into the list, as far as they find place; s.n counts them. A
  // round's chunks are looked at together, a bit a value, as most have few such tokens,
  // while the next round's are on their way; the ids go into the list, whose logits are
  // read again at the end.
  auto gather = [&](auto&& yes) {
    for (int c0 = 0; c0 < a.chunks; c0 += PT) {
      const float cm = c0 == 0 ? cm0 : c0 + mine0 < a.chunks ? cmax[c0 + mine0] : -__builtin_inff();
      uint64_t there = __ballot(cm >= least);
      const bool end = a.vocab & (CHUNK - 1);
      float v[MLP][4];
      int mine, got;  // the round's chunks, in lane k too, and how many
      auto load = [&](float (&v)[MLP][4]) {
        got = 0;
#pragma unroll
        for (int k = 0; k < MLP; k++) {
          const int chunk = c0 + w + WAVES * (there ? __builtin_ctzll(there) : 0);
          got += there != 0;
          there &= there - 1;
          if (lane == k) mine = chunk;
          const float* const p = x + chunk * CHUNK + 4 * lane;
          if (end && chunk == a.chunks - 1) {  // the row's end, part of a chunk
#pragma unroll
            for (int e = 0; e < 4; e++) v[k][e] = chunk * CHUNK + 4 * lane + e < a.vocab ? p[e] : -__builtin_inff();
          } else if constexpr (WIDE) {
            const float4 l = *(const float4*)p;
            v[k][0] = l.x; v[k][1] = l.y; v[k][2] = l.z; v[k][3] = l.w;
          } else {
#pragma unroll
            for (int e = 0; e < 4; e++) v[k][e] = p[e];
          }
        }
      };
      if (there) load(v);
      else continue;
      for (;;) {
        const int now = got, chunks = mine;
        float next[MLP][4];
        const bool more = there != 0;
        if (more) load(next);
        uint32_t in = 0;
#pragma unroll
        for (int k = 0; k < MLP; k++)
#pragma unroll
          for (int e = 0; e < 4; e++)
            in |= (uint32_t)((v[k][e] >= least) & yes(v[k][e])) << (4 * k + e);  // (no branches)
        if (now < MLP) in &= (1u << 4 * now) - 1;
        const int n = __popc(in), upto = wave_scan32(n), round = __builtin_amdgcn_readlane(upto, 63);
        if (round) {
          int to = 0;
          if (lane == 0) to = atomicAdd(&s.n, round);
          to = __builtin_amdgcn_readfirstlane(to) + upto - n;
          if (lane < MLP) s.chunk[w][lane] = chunks;
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          __builtin_amdgcn_wave_barrier();
          for (; in; in &= in - 1, to++) {
            const int bit = __builtin_ctz(in);
            if (to < CAP) s.ids[to] = s.chunk[w][bit >> 2] * CHUNK + 4 * lane + (bit & 3);
          }
        }
        if (!more) break;
#pragma unroll
        for (int k = 0; k < MLP; k++)
#pragma unroll
          for (int e = 0; e < 4; e++) v[k][e] = next[k][e];
      }
    }
    __syncthreads();
    read_list();
  };
  int n = 0;
  if (!many) {
    gather([](float) { return true; });
    n = s.n;
    many = n > CAP;
  }

  IHIP_STAMP(3);
  const int bits = sample_weight_bits(a.vocab);
  const double one = ldexp(1.0, bits);
  auto whole = [&](float l) { return whole_weight(weight_of(l), one); };
  const LogitBins bins(m, least);
  u64 mass_all = 0;
  uint32_t count_all = 0;
  if (many) {
    for (int i = t; i < BINS; i += PT) {
      s.mass[i] = head.state == ROW_BINS ? a.bins[(int64_t)head.slot * BINS + i] : 0;
      s.count[i] = 0;
    }
    __syncthreads();
    if (head.state != ROW_BINS)
      tokens([&](const float (&v)[4], int) {
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (v[e] >= least) {
            const int b = bins.of(v[e]);
            atomicAdd(&s.mass[b], whole(v[e]));
            if (by_k) atomicAdd(&s.count[b], 1u);
          }
      });
    __syncthreads();
    scan_bins(s, 0, 0, mass_all, count_all);
  }
  IHIP_STAMP(4);
  // tokens and weights before a bin, and those with it
  auto tokens_to = [&](int b) { return b >= BINS ? count_all : s.count[b]; };
  auto mass_to = [&](int b) { return ldexp((double)(b >= BINS ? mass_all : s.mass[b]), -bits); };
  // Few: one list, and its borders one after another
  auto few = [&](auto& list) {
    list.sort(s.cand, n);
    list.weigh(s.wave, weight_of);
    IHIP_STAMP(5);
    int keep = n;
    double total = list.all;
    if (by_k && n > set.top_k) {
      const uint32_t kth = list.template of<uint32_t>(set.top_k - 1, &s.key, [&](int e) { return (uint32_t)(list.v[e] >> 32); });
      keep = list.count(s.topi, [&](int, int e) { return (uint32_t)(list.v[e] >> 32) >= kth; });
      total = list.sum_of(keep, &s.total);
    }
    if (by_p) {
      const double upto = set.top_p * (by_k ? total : all);
      keep = list.count(s.topi, [&](int i, int e) { return i < keep && (i == 0 || list.before[e] < upto); });
    }
    if (floor > 0) keep = list.count(s.topi, [&](int i, int e) { return i < keep && (i == 0 || list.wt[e] >= floor); });
    if (by_p || floor > 0) total = list.sum_of(keep, &s.total);
    const double target = u * total;
    // (sums do not fall: those before the drawn one are the others that pass)
    int i = list.count(s.topi, [&](int i, int e) { return i < keep && !(target < list.before[e] + list.wt[e]); });
    if (i >= keep) i = 0;  // none: the best
    IHIP_STAMP(7);
    const u64 got = list.template of<u64>(i, &s.above, [&](int e) { return list.v[e]; });
    if (t == 0) answer((int)~(uint32_t)got, weight_of(key_logit((uint32_t)(got >> 32))) / total);
  };
  if (!many) {
    if (n <= 64) {
      if (w > 0) return;
      SortedList<64, 1> list;
      few(list);
    } else if (n <= 128) {
      if (w > 0) return;
      SortedList<64, 2> list;
      few(list);
    } else {
      SortedList<PT, CAP / PT> list;
      few(list);
    }
    return;
  }

  // The borders of the filters and the draw, each in one bin: the tokens kept are those of
  // the bins before `last` and `kept` of its own. The list holds the tokens of one bin, or,
  // as the draw's bin is nearly known when the border's is gathered, those of two: the
  // first `split` of them are of bin `ahead`, the others of bin `cur`.
  int cur = -1, ahead = -1, split = 0, last = BINS - 1, kept = INT32_MAX;
  double mass = all, total = mass_to(BINS);
  bool alike = false;
  SortedList<PT, CAP / PT> list;
#pragma unroll 1
  for (int phase = 0; phase < 4; phase++) {
    int b = 0, next = -1;
    double upto = 0;
    if (phase == 0) {  // top-k: the bin of the kth token
      if (!by_k) continue;
      b = first_bin<PT, false>(&s.found, last, (double)set.top_k, [&](int i) { return (double)tokens_to(i); });
      mass = total;
      if (b < 0) continue;  // (it keeps all)
    } else if (phase == 1) {  // top-p: the bin in which the sum passes its share
      if (!by_p) continue;
      upto = set.top_p * mass;
      b = border_bins<PT>(&s.found, upto, u, mass_to, next);
      if (b < 0 || b > last) continue;
    } else if (phase == 2) {  // min-p: the bin of the smallest weight
      if (!(floor > 0)) continue;
      b = bins.of((float)fmax(md + log2(floor) / c, (double)least));
      if (b > last) continue;
    } else {
      upto = u * total;
      b = first_bin<PT, true>(&s.found, last, upto, mass_to);
      if (b < 0) b = last;
    }
    if (b != cur && b != ahead) {
      cur = b;
      ahead = next;
      if (phase == 1 && head.state == ROW_BINS) {  // (sample_rows_find has them)
        const int* const got = a.found + (int64_t)head.slot * (1 + CAP);
        if (t == 0) s.n = got[0];
        for (int i = t; i < CAP; i += PT) s.ids[i] = (uint32_t)min(max(got[1 + i], 0), a.vocab - 1);
        __syncthreads();
        read_list();
      } else {
        if (t == 0) s.n = 0;
        __syncthreads();
        gather([&](float l) {
          const int i = bins.of(l);
          return (i == b) | (i == ahead);
        });
      }
      if (s.n > CAP) {
        alike = true;
        break;
      }
      list.sort(s.cand, s.n);
      list.weigh(s.wave, weight_of);
      split = ahead < 0 ? 0 : list.count(s.topi, [&](int, int e) { return bins.of(key_logit((uint32_t)(list.v[e] >> 32))) < b; });
      IHIP_STAMP(5);
    }
    // the bin's part of the list
    const int i0 = b == cur ? split : 0, i1 = b == cur ? list.n : split;
    const double base = mass_to(b) - list.sum_of(i0, &s.total);
    const int lim = b == last && kept < i1 - i0 ? i0 + kept : i1;
    if (phase == 3) {
      IHIP_STAMP(6);
      int i = i0 + list.count(s.topi, [&](int i, int e) { return i >= i0 && i < lim && !(upto < base + list.before[e] + list.wt[e]); });
      // (none: the best; a rounding between bins: the last)
      if (i >= lim) i = b == 0 ? i0 : max(lim - 1, i0);
      IHIP_STAMP(7);
      if (t == 0) {
        const u64 got = s.cand[i];
        answer((int)~(uint32_t)got, weight_of(key_logit((uint32_t)(got >> 32))) / total);
      }
      return;
    }
    const uint32_t kth = phase == 0 ? (uint32_t)(s.cand[min(set.top_k - (int)tokens_to(b), list.n) - 1] >> 32) : 0u;
    kept = list.count(s.topi, [&](int i, int e) {
      const bool in = phase == 0 ? (uint32_t)(list.v[e] >> 32) >= kth : phase == 1 ? base + list.before[e] < upto : list.wt[e] >= floor;
      return i >= i0 && i < lim && (in || (i == i0 && b == 0));
    });
    last = b;
    total = base + list.sum_of(i0 + kept, &s.total);
    if (phase == 0) mass = total;
  }
  if (!alike) return;  // (not reached)

  // Logits so much alike that they cannot be sorted: the key at which the running count or
  // weight, the largest key first, of the candidates from `from` on (and of a weight of
  // `floor` at least) passes `want`, or the smallest of them, by rounds of 2048 bins
  const uint32_t key_best = row_key(m);
  uint32_t from = row_key(least), end = 0;
  u64 kept_mass = 0;
  mass = all;
#pragma unroll 1
  for (int phase = 0; phase < 3; phase++) {
    if (phase == 0 && !by_k) continue;
    u64 want = phase == 0 ? (u64)set.top_k : ~0ull;
    const double upto = ldexp(set.top_p * mass, bits);
    if (phase == 1 && by_p) want = (u64)ceil(fmin(upto, 0x1p62));
    const u64 target = phase == 2 ? min((u64)fmin(fmax(u * (double)kept_mass, 0.0), 0x1p62), kept_mass - 1) : 0;
    if (phase == 2) {
      want = target + 1;
      from = end;
    }
    uint32_t klo = from, khi = key_best;
    u64 above = 0;
    uint32_t count = 0;
    for (;;) {
      int shift = 0;
      while (((khi - klo) >> shift) >= (uint32_t)BINS) shift++;
      __syncthreads();
      for (int i = t; i < BINS; i += PT) {
        s.mass[i] = 0;
        s.count[i] = 0;
      }
      __syncthreads();
      tokens([&](const float (&v)[4], int) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const uint32_t k = row_key(v[e]);
          if (!(v[e] >= least) || k < klo || k > khi) continue;
          if (phase > 0 && floor > 0 && k != key_best && !(weight_of(v[e]) >= floor)) continue;
          const uint32_t b = (khi - k) >> shift;
          atomicAdd(&s.mass[b], whole(v[e]));
          atomicAdd(&s.count[b], 1u);
        }
      });
      __syncthreads();
      if (t == 0) {
        s.found = INT32_MAX;
        s.at = 0;
      }
      scan_bins(s, above, count, mass_all, count_all);
      // the first bin that passes, else the last one that holds any
      for (int i = t; i < BINS; i += PT) {
        const uint32_t upto_n = tokens_to(i + 1);
        const u64 upto_m = i + 1 < BINS ? s.mass[i + 1] : mass_all;
        if (upto_n == s.count[i]) continue;
        if (phase == 0 ? upto_n >= want : upto_m >= want) atomicMin(&s.found, i);
        atomicMax(&s.at, i);
      }
      __syncthreads();
      const int b = s.found != INT32_MAX ? s.found : s.at;
      if (t == 0) {
        s.above = s.mass[b];
        s.n = (int)s.count[b];
        s.ties = (int)(tokens_to(b + 1) - s.count[b]);
      }
      __syncthreads();
      above = s.above;
      count = (uint32_t)s.n;
      const uint32_t top = khi - ((uint32_t)b << shift);
      if (shift == 0) {
        khi = top;
        break;
      }
      const uint32_t width = (1u << shift) - 1;
      klo = top - klo > width ? top - width : klo;
      khi = top;
    }
    // `khi` and its ties
    const u64 tie = max(whole(key_logit(khi)), (u64)1), ties = (u64)max(s.ties, 1);
    if (phase == 0) {
      from = khi;
      mass = ldexp((double)(above + tie * ties), -bits);
    } else if (phase == 1) {
      u64 r = ties;
      if (by_p) {
        const double need = upto - (double)above;
        r = need > 0 ? (u64)fmin(ceil(need / (double)tie), (double)ties) : 1;
        r = max(r, (u64)1);
      }
      end = khi;
      kept_mass = above + r * tie;
    } else {
      const int nth = (int)min((target - min(above, target)) / tie, ties - 1);
      __syncthreads();
      // the nth token of that key by id: a run of tokens a thread
      const int each = (a.vocab + PT - 1) / PT;
      int found = 0, tot;
      const int i1 = min((t + 1) * each, a.vocab);
      for (int i = t * each; i < i1; i++) found += finite_f(x[i]) && row_key(x[i]) == khi;
      int at = scan_threads<PT>(found, s.topi, tot);
      if (at <= nth && nth < at + found)
        for (int i = t * each; i < i1; i++)
          if (finite_f(x[i]) && row_key(x[i]) == khi && at++ == nth) {
            answer(i, weight_of(x[i]) / ldexp((double)kept_mass, -bits));
            break;
          }
    }
    __syncthreads();
  }
}

extern "C" __global__ __launch_bounds__(PT, 4) void sample_rows_pick(SampleRowsArgs a) { sample_pick_t<false>(a); }
extern "C" __global__ __launch_bounds__(PT, 4) void sample_rows_pick_wide(SampleRowsArgs a) { sample_pick_t<true>(a); }
