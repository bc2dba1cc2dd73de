// sample_rows.hip - a draw for each row of logits (TInferSampler.Next's filters and
// order, src/infer/mormot.ai.infer.sampler.pas:269-435), with settings and a random
// number of its own for every row.
#include "common.h"
#include "../sample_rows.h"

using namespace ihip;

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
  int32_t rows, vocab, parts, chunks;
  int32_t wide;   // rows aligned to 16 bytes
  int32_t per;    // tokens of a part
};

constexpr int OCT = 32;          // octaves below a part's largest weight that are told apart
constexpr int OCT_ONE = 17;      // a weight of 1 in its octave's sum, as a power of two
constexpr int CHUNK = 256;       // tokens of a chunk
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

// 2^y for y <= 0: y as a multiple of 1 / 16 and the rest, whose powers sum to 4e-16 of the
// result in 7 terms; 0 below 2^-1100
__device__ __forceinline__ double weight(double y, const double* root)
{
  const double s = fmax(y, -1100.0) * 16.0, n = rint(s), f = (s - n) * (0.69314718055994530942 / 16);
  double p = 1.0 / 720;
  p = __builtin_fma(p, f, 1.0 / 120);
  p = __builtin_fma(p, f, 1.0 / 24);
  p = __builtin_fma(p, f, 1.0 / 6);
  p = __builtin_fma(p, f, 0.5);
  p = __builtin_fma(p, f, 1.0);
  p = __builtin_fma(p, f, 1.0);
  const int j = (int)n;
  return ldexp(root[j & 15] * p, j >> 4);
}

// 2^(j / 16) into LDS
__device__ __forceinline__ void weight_roots(double* root)
{
  if (threadIdx.x < 16) root[threadIdx.x] = exp2(threadIdx.x / 16.0);
}

// ------------------------------------------------------------- sample_rows_part
// A part of a row: its tokens in registers, read once; the largest logits of chunks, the
// part's largest, then the weights' sum in double and, where a filter asks how deep it has
// to look, their sums by octave (in whole numbers, a lane's own places in LDS, so that no
// order changes them).
template <int IT>
__device__ __forceinline__ void sample_part_t(const SampleRowsArgs& a)
{
  __shared__ double root[16], part[4];
  __shared__ float top[4];
  __shared__ int first[4];
  __shared__ uint32_t oct[OCT * 64];
  const int t = threadIdx.x, lane = t & 63, w = t >> 6;
  const int row = blockIdx.y, p = blockIdx.x;
  const SampleSettings set = a.settings[row];
  const int kind = row_kind(set);
  if (kind == ROW_BAD) return;
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
  const bool filtered = kind == ROW_FILTERED, deep = filtered && (set.top_k > 0 || set.top_p < 1);
  if (kind != ROW_GREEDY) {
    weight_roots(root);
    if (deep)
      for (int i = t; i < OCT * 64; i += 256) oct[i] = 0;
  }
  float m = -__builtin_inff();
#pragma unroll
  for (int i = 0; i < IT; i++) {
    const float c = fmaxf(fmaxf(v[i][0], v[i][1]), fmaxf(v[i][2], v[i][3]));
    if (filtered) {
      const float cm = wave_max(c == c ? c : -__builtin_inff());
      const int chunk = (i0 + i * 1024) / CHUNK + w;
      if (lane == 0 && chunk < a.chunks) a.chunk[(int64_t)row * a.chunks + chunk] = cm;
    }
    m = fmaxf(m, c);
  }
  m = wave_max(m);
  if (lane == 0) top[w] = m;
  __syncthreads();
  m = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
  int id = INT32_MAX;
#pragma unroll
  for (int i = IT - 1; i >= 0; i--)
#pragma unroll
    for (int e = 3; e >= 0; e--)
      if (v[i][e] == m) id = i0 + i * 1024 + 4 * t + e;
  id = -wave_max(-id);
  double s = 0;
  if (kind != ROW_GREEDY && finite_f(m)) {
    const double c = LOG2E_D / set.temperature, md = m;
#pragma unroll
    for (int i = 0; i < IT; i++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const double y = v[i][e] == v[i][e] ? ((double)v[i][e] - md) * c : -__builtin_inf();
        const double wt = weight(y, root);
        s = s + wt;
        if (deep) {
          const double up = ceil(y);  // 2^(up - 1) < weight <= 2^up
          if (up > -(double)OCT) atomicAdd(&oct[-(int)up * 64 + lane], (uint32_t)ldexp(wt, OCT_ONE - (int)up));
        }
      }
    s = wave_sum(s, 64);
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
  if (deep) {
    uint32_t n = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) n += oct[(t >> 3) * 64 + (t & 7) * 8 + j];
    n = wave_sum(n, 8);
    if ((t & 7) == 0) a.octaves[to * OCT + (t >> 3)] = n;
  }
}

extern "C" __global__ __launch_bounds__(256) void sample_rows_part_2048(SampleRowsArgs a) { sample_part_t<2>(a); }
extern "C" __global__ __launch_bounds__(256) void sample_rows_part_8192(SampleRowsArgs a) { sample_part_t<8>(a); }

// ------------------------------------------------------------- sample_rows_pick
constexpr int PT = 1024;       // threads
constexpr int CAP = 4096;      // candidates that are sorted
constexpr int BINS = 2048;     // of a search over more of them

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

struct PickLds {
  double root[16], wave[PT / 64], total;
  float topf[PT / 64];
  int topi[PT / 64];
  unsigned long long omass[64], ocount[64];
  int n, octave, found;
  uint32_t key;            // a search's result: the key,
  unsigned long long above, count;  // the weights and tokens of larger keys
  union {
    uint64_t cand[CAP];    // key << 32 | ~id
    struct {
      unsigned long long mass[BINS];
      uint32_t count[BINS];
    } bin;
    int ties[PT];
  };
};

// v's sum over the threads before this one, and over all of them
template <typename T>
__device__ __forceinline__ T scan_threads(T v, T* sh, T& all)
{
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  T s = v;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const T o = __shfl_up(s, d, 64);
    if (lane >= d) s = s + o;
  }
  __syncthreads();
  if (lane == 63) sh[w] = s;
  __syncthreads();
  T before = T(0);
  all = T(0);
  for (int i = 0; i < PT / 64; i++) {
    if (i < w) before = before + sh[i];
    all = all + sh[i];
  }
  return before + (s - v);
}

// One block a row, behind its parts' results. Greedy rows take the best of them; rows
// without filters find the part in which the draw falls and look through that one again.
// With filters the candidates are the tokens above a logit that surely holds what the
// filters keep (by the parts' octaves, or min-p's share), gathered from the chunks that
// reach it, sorted, and cut in TInferSampler's order by sums in double. More of them than
// CAP are not sorted: kept and drawn tokens are found by searches over their keys, in
// sums of whole numbers.
extern "C" __global__ __launch_bounds__(PT) void sample_rows_pick(SampleRowsArgs a)
{
  __shared__ PickLds s;
  const int t = threadIdx.x, lane = t & 63, w = t >> 6;
  const int row = blockIdx.x;
  const SampleSettings set = a.settings[row];
  const int kind = row_kind(set);
  auto answer = [&](int id, double prob) {
    a.ids[row] = id;
    if (a.probs) a.probs[row] = (float)prob;
  };
  if (kind == ROW_BAD) {
    if (t == 0) answer(-1, 0.0);
    return;
  }
  const float* const x = a.x + (int64_t)row * a.stride;
  const int64_t p0 = (int64_t)row * a.parts;
  weight_roots(s.root);
  // the best of the parts
  float m = -__builtin_inff();
  int id = INT32_MAX;
  for (int p = t; p < a.parts; p += PT) {
    const float pm = a.best[p0 + p];
    const int pi = a.best_id[p0 + p];
    if (pm > m || (pm == m && pi < id)) {
      m = pm;
      id = pi;
    }
  }
  {
    const float wm = wave_max(m);
    const int wi = -wave_max(m == wm ? -id : -INT32_MAX);
    if (lane == 0) {
      s.topf[w] = wm;
      s.topi[w] = wi;
    }
    __syncthreads();
    m = s.topf[0];
    for (int i = 1; i < PT / 64; i++) m = fmaxf(m, s.topf[i]);
    id = INT32_MAX;
    for (int i = 0; i < PT / 64; i++)
      if (s.topf[i] == m) id = min(id, s.topi[i]);
  }
  const int best = id == INT32_MAX ? 0 : id;  // (a row of NaN: 0)
  if (kind == ROW_GREEDY || !finite_f(m)) {
    if (t == 0) answer(best, 1.0);
    return;
  }
  const double c = LOG2E_D / set.temperature, md = m, u = a.uniform[row];
  auto weight_of = [&](float l) { return l == l ? weight(((double)l - md) * c, s.root) : 0.0; };

  // the sum of all weights, and where this thread's parts begin
  const int pq = (a.parts + PT - 1) / PT;
  double mine = 0, all;
  for (int p = t * pq; p < min((t + 1) * pq, a.parts); p++) {
    const float pm = a.best[p0 + p];
    if (finite_f(pm)) mine = mine + a.sum[p0 + p] * weight(((double)pm - md) * c, s.root);
  }
  double before = scan_threads(mine, s.wave, all);
  if (kind == ROW_FREE) {
    const double target = u * all;
    // the first part whose sums pass the target; none (rounding, or u of 1): the best token
    if (t == 0) s.found = INT32_MAX;
    __syncthreads();
    for (int p = t * pq; p < min((t + 1) * pq, a.parts); p++) {
      const float pm = a.best[p0 + p];
      const double add = finite_f(pm) ? a.sum[p0 + p] * weight(((double)pm - md) * c, s.root) : 0.0;
      if (add > 0 && target < before + add) {
        atomicMin(&s.found, p);
        break;
      }
      before = before + add;
    }
    __syncthreads();
    const int part = s.found;
    if (part == INT32_MAX) {
      if (t == 0) answer(best, 1.0 / all);
      return;
    }
    if (part / pq == t) s.total = before;
    __syncthreads();
    const double base = s.total;
    // its tokens in order, `each` a thread
    const int each = a.per / PT;
    double sum = 0;
    for (int e = 0; e < each; e++) {
      const int i = part * a.per + t * each + e;
      if (i < a.vocab) sum = sum + weight_of(x[i]);
    }
    double part_all;
    double run = base + scan_threads(sum, s.wave, part_all);
    if (t == 0) s.found = INT32_MAX, s.n = -1;
    __syncthreads();
    for (int e = 0; e < each; e++) {
      const int i = part * a.per + t * each + e;
      const double wt = i < a.vocab ? weight_of(x[i]) : 0.0;
      if (wt > 0) {
        atomicMax(&s.n, i);  // (the last one, where roundings leave none)
        run = run + wt;
        if (target < run) {
          atomicMin(&s.found, i);
          break;
        }
      }
    }
    __syncthreads();
    if (t == 0) {
      const int i = s.found != INT32_MAX ? s.found : s.n >= 0 ? s.n : best;
      answer(i, weight_of(x[i]) / all);
    }
    return;
  }

  // the octave below the best weight that surely holds k tokens and top_p of the sum
  const bool by_p = set.top_p < 1, by_k = set.top_k > 0;
  const bool sure_p = by_p && !by_k;  // (behind top-k the mass is that of what it keeps)
  double lo = -__builtin_inf();
  if (by_k || by_p) {
    if (t < 64) s.omass[t] = s.ocount[t] = 0;
    __syncthreads();
    for (int i = t; i < a.parts * OCT; i += PT) {
      const int p = i / OCT, b = i - p * OCT;
      const uint32_t n = a.octaves[(p0 + p) * OCT + b];
      const float pm = a.best[p0 + p];
      if (n == 0 || !finite_f(pm)) continue;
      const double below = (md - (double)pm) * c;  // of the part's best
      const double k = ceil(below) + b;            // every weight of these is above 2^-(k + 1)
      if (k < 63) {
        atomicAdd(&s.omass[(int)k + 1], (unsigned long long)(n * weight(-below - b, s.root) * 0x1p23));
        atomicAdd(&s.ocount[(int)k + 1], (unsigned long long)n);
      }
    }
    __syncthreads();
    if (w == 0) {
      unsigned long long mass = s.omass[lane], count = s.ocount[lane];
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const unsigned long long om = __shfl_up(mass, d, 64), oc = __shfl_up(count, d, 64);
        if (lane >= d) mass += om, count += oc;
      }
      const bool enough = (!by_k || (count >> OCT_ONE) >= (unsigned long long)set.top_k) &&
                          (!sure_p || (double)mass * 0x1p-40 >= set.top_p * all * (1 + 1e-9));
      const uint64_t there = __ballot(enough);
      if (lane == 0) s.octave = there ? __builtin_ctzll(there) : -1;
    }
    __syncthreads();
    if (s.octave >= 0) lo = md - s.octave / c;
  }
  if (set.min_p > 0 && !(by_k && by_p)) lo = fmax(lo, md + log2(set.min_p) / c);
  lo = lo - 1e-9 * (fabs(lo) + fabs(md));
  float least = (float)lo;
  if ((double)least > lo) least = key_logit(row_key(least) - 1);
  if (!(least > -3.4028235e38f)) least = -3.4028235e38f;  // (infinities and NaN are no candidates)

  // every token of the row from `least` on: each(logit, id), lanes over a chunk's tokens
  auto tokens = [&](auto&& each) {
    for (int c0 = w * 64; c0 < a.chunks; c0 += PT) {
      const float cm = c0 + lane < a.chunks ? a.chunk[(int64_t)row * a.chunks + c0 + lane] : -__builtin_inff();
      for (uint64_t there = __ballot(cm >= least); there; there &= there - 1) {
        const int i0 = (c0 + __builtin_ctzll(there)) * CHUNK + 4 * lane;
        float v[4];
        if (a.wide && i0 + 4 <= a.vocab) {
          const float4 l = *(const float4*)(x + i0);
          v[0] = l.x; v[1] = l.y; v[2] = l.z; v[3] = l.w;
        } else {
#pragma unroll
          for (int e = 0; e < 4; e++) v[e] = i0 + e < a.vocab ? x[i0 + e] : -__builtin_inff();
        }
        each(v, i0);
      }
    }
  };
  if (t == 0) s.n = 0;
  __syncthreads();
  tokens([&](const float (&v)[4], int i0) {
    uint64_t in[4];
    int n = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      in[e] = __ballot(v[e] >= least && finite_f(v[e]));
      n += __popcll(in[e]);
    }
    int at = 0;
    if (lane == 0 && n) at = atomicAdd(&s.n, n);
    at = __builtin_amdgcn_readfirstlane(at);
    const uint64_t below = (1ull << lane) - 1;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int to = at + __popcll(in[e] & below);
      if ((in[e] >> lane & 1) && to < CAP) s.cand[to] = (uint64_t)row_key(v[e]) << 32 | (uint32_t)~(i0 + e);
      at += __popcll(in[e]);
    }
  });
  __syncthreads();
  const int n = s.n;
  if (n <= CAP) {
    // sorted: the largest key first, the lowest id on a tie
    int size = 64;
    while (size < n) size *= 2;
    for (int i = n + t; i < size; i += PT) s.cand[i] = 0;
    __syncthreads();
    for (int k = 2; k <= size; k *= 2)
      for (int j = k / 2; j > 0; j /= 2) {
        for (int i = t; i < size / 2; i += PT) {
          const int l = 2 * i - (i & (j - 1)), r = l + j;
          const uint64_t x0 = s.cand[l], x1 = s.cand[r];
          if ((x0 < x1) == ((l & k) == 0)) {
            s.cand[l] = x1;
            s.cand[r] = x0;
          }
        }
        __syncthreads();
      }
    // 4 a thread, in order, and their running sums
    constexpr int E = CAP / PT;
    uint32_t key[E];
    double wt[E], sum = 0, cand_all;
#pragma unroll
    for (int e = 0; e < E; e++) {
      const int i = t * E + e;
      key[e] = i < n ? (uint32_t)(s.cand[i] >> 32) : 0u;
      wt[e] = i < n ? weight_of(key_logit(key[e])) : 0.0;
      sum = sum + wt[e];
    }
    double run = scan_threads(sum, s.wave, cand_all);
    int keep = n;
    if (by_k && n > set.top_k) {
      const uint32_t kth = (uint32_t)(s.cand[set.top_k - 1] >> 32);
      int c2 = 0;
#pragma unroll
      for (int e = 0; e < E; e++) c2 += t * E + e < n && key[e] >= kth;
      int tot;
      __syncthreads();
      (void)scan_threads(c2, s.topi, tot);
      keep = tot;
    }
    // the sum of the first `count` of them
    auto sum_of = [&](int count) {
      double r = run, got = 0;
#pragma unroll
      for (int e = 0; e < E; e++) {
        r = r + wt[e];
        if (t * E + e == count - 1) got = r;
      }
      __syncthreads();
      if (count > 0 && (count - 1) / E == t) s.total = got;
      __syncthreads();
      return s.total;
    };
    if (by_p) {
      const double mass = by_k ? sum_of(keep) : all, upto = set.top_p * mass;
      double r = run;
      int c2 = 0;
#pragma unroll
      for (int e = 0; e < E; e++) {
        c2 += t * E + e < keep && (t * E + e == 0 || r < upto);
        r = r + wt[e];
      }
      int tot;
      __syncthreads();
      (void)scan_threads(c2, s.topi, tot);
      keep = tot;
    }
    if (set.min_p > 0) {
      int c2 = 0;
#pragma unroll
      for (int e = 0; e < E; e++) c2 += t * E + e < keep && (t * E + e == 0 || wt[e] >= set.min_p);
      int tot;
      __syncthreads();
      (void)scan_threads(c2, s.topi, tot);
      keep = tot;
    }
    const double total = sum_of(keep), target = u * total;
    if (t == 0) s.found = INT32_MAX;
    __syncthreads();
    double r = run;
    int first = INT32_MAX;
#pragma unroll
    for (int e = 0; e < E; e++) {
      r = r + wt[e];
      if (t * E + e < keep && target < r) first = min(first, t * E + e);
    }
    if (first != INT32_MAX) atomicMin(&s.found, first);
    __syncthreads();
    if (t == 0) {
      const uint64_t got = s.cand[s.found == INT32_MAX ? 0 : s.found];  // (none: the best)
      answer((int)~(uint32_t)got, weight_of(key_logit((uint32_t)(got >> 32))) / total);
    }
    return;
  }

  // Many candidates: weights as whole numbers, so that sums do not depend on their order
  const int bits = sample_weight_bits(a.vocab);
  const uint32_t key_best = row_key(m);
  auto whole = [&](float l) { return (unsigned long long)(ldexp(weight_of(l), bits)); };
  // The key at which the running count or weight, the largest key first, of the candidates
  // between `from` and the best with a weight of `floor` at least passes `want` (or the
  // smallest of them), by rounds of 2048 bins; s.key, s.above, s.count
  auto search = [&](bool counts, unsigned long long want, uint32_t from, double floor) {
    uint32_t klo = from, khi = key_best;
    unsigned long long above = 0, count = 0;
    for (;;) {
      int shift = 0;
      while (((khi - klo) >> shift) >= (uint32_t)BINS) shift++;
      __syncthreads();
      for (int i = t; i < BINS; i += PT) {
        s.bin.mass[i] = 0;
        s.bin.count[i] = 0;
      }
      __syncthreads();
      tokens([&](const float (&v)[4], int) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
          if (!(v[e] >= least) || !finite_f(v[e])) continue;
          const uint32_t key = row_key(v[e]);
          if (key < klo || key > khi) continue;
          if (floor > 0 && key != key_best && !(weight_of(v[e]) >= floor)) continue;
          const uint32_t b = (khi - key) >> shift;
          atomicAdd(&s.bin.mass[b], whole(v[e]));
          atomicAdd(&s.bin.count[b], 1u);
        }
      });
      __syncthreads();
      // two bins a thread, the largest keys first
      const unsigned long long m0 = s.bin.mass[2 * t], m1 = s.bin.mass[2 * t + 1];
      const unsigned long long n0 = s.bin.count[2 * t], n1 = s.bin.count[2 * t + 1];
      unsigned long long mall, nall;
      unsigned long long* const sh = (unsigned long long*)s.wave;
      const unsigned long long mb = above + scan_threads(m0 + m1, sh, mall);
      const unsigned long long nb = count + scan_threads(n0 + n1, sh, nall);
      if (t == 0) s.found = INT32_MAX;
      __syncthreads();
      // the first bin that passes, else the last one that holds any
      const bool h0 = n0 && (counts ? nb + n0 >= want : mb + m0 >= want), h1 = n1 && (counts ? nb + n0 + n1 >= want : mb + m0 + m1 >= want);
      if (h0 || h1) atomicMin(&s.found, 2 * t + (h0 ? 0 : 1));
      __syncthreads();
      int b = s.found;
      __syncthreads();
      if (b == INT32_MAX) {
        if (t == 0) s.found = -1;
        __syncthreads();
        if (n0 || n1) atomicMax(&s.found, 2 * t + (n1 ? 1 : 0));
        __syncthreads();
        b = s.found;
        __syncthreads();
      }
      if (b < 0) b = 0;  // (none at all: the best's own bin)
      if (b / 2 == t) {
        s.above = mb + (b & 1 ? m0 : 0);
        s.count = nb + (b & 1 ? n0 : 0);
      }
      __syncthreads();
      above = s.above;
      count = s.count;
      const uint32_t top = khi - ((uint32_t)b << shift);
      if (shift == 0) {
        if (t == 0) {
          s.key = top;
          s.octave = (int)s.bin.count[b];  // its ties
        }
        __syncthreads();
        return;
      }
      const uint32_t width = (1u << shift) - 1;
      klo = top - klo > width ? top - width : klo;
      khi = top;
    }
  };
  uint32_t from = row_key(least);
  const double floor = set.min_p;
  // (a sum of the whole weights stands for `all` in double: below 2^63)
  double mass = all;
  if (by_k) {
    search(true, (unsigned long long)set.top_k, from, 0.0);
    from = s.key;
    if (by_p) {
      const unsigned long long tie = whole(key_logit(s.key));
      mass = ldexp((double)(s.above + tie * (unsigned long long)s.octave), -bits);
    }
  }
  // what is kept: the keys above `end`, and `ties` of it
  uint32_t end = 0;
  unsigned long long kept = 0;  // their weights
  if (by_p) {
    const double upto = ldexp(set.top_p * mass, bits);
    search(false, (unsigned long long)ceil(fmin(upto, 0x1p62)), from, floor);
    end = s.key;
    const unsigned long long tie = max(whole(key_logit(end)), 1ull);
    const double need = upto - (double)s.above;
    unsigned long long r = need > 0 ? (unsigned long long)ceil(need / (double)tie) : 1ull;
    r = min(max(r, 1ull), (unsigned long long)max(s.octave, 1));
    kept = s.above + r * tie;
  } else {
    search(false, ~0ull, from, floor);  // all of them
    end = s.key;
    kept = s.above + max(whole(key_logit(end)), 1ull) * (unsigned long long)max(s.octave, 1);
  }
  __syncthreads();
  // the draw: the key whose weights pass the target, and which of its ties
  const unsigned long long target = (unsigned long long)fmin(fmax(u * (double)kept, 0.0), 0x1p62);
  search(false, min(target, kept - 1) + 1, end, floor);
  const uint32_t drawn = s.key;
  const unsigned long long tie = max(whole(key_logit(drawn)), 1ull);
  const unsigned long long rest = min(target, kept - 1) - min(s.above, min(target, kept - 1));
  const int nth = (int)min(rest / tie, (unsigned long long)max(s.octave, 1) - 1);
  __syncthreads();
  // the nth token of that key by id: a run of tokens a thread
  const int each = (a.vocab + PT - 1) / PT;
  int found = 0, tot;
  const int i1 = min((t + 1) * each, a.vocab);
  for (int i = t * each; i < i1; i++) found += finite_f(x[i]) && row_key(x[i]) == drawn;
  int at = scan_threads(found, s.topi, tot);
  if (at <= nth && nth < at + found)
    for (int i = t * each; i < i1; i++)
      if (finite_f(x[i]) && row_key(x[i]) == drawn && at++ == nth) {
        answer(i, weight_of(x[i]) / ldexp((double)kept, -bits));
        break;
      }
}
