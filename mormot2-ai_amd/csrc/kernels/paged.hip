// paged.hip - several sequences decoded together over one paged cache: the
// plan of a step, q/k/v of the new rows into the pages, attention over them.
#include "common.h"
#include "../paged.h"

using namespace ihip;

// ------------------------------------------------------------- paged_slots
struct SlotArgs {
  const int *past, *count;
  int *table, *ring;
  const int64_t* ends;
  int64_t* ends_out;
  int *offsets, *lengths, *positions, *slots, *failed;
  int* plan;  // [5][seqs], then 3: the plan between the two launches
  int32_t seqs, max_pages, page_size, pages, rows;
  int32_t here;  // 1: the rows in this launch too
};

constexpr int SLOT_THREADS = 1024, SLOT_PER = 4;  // sequences: 4 a thread
static_assert(SLOT_THREADS * SLOT_PER == 4096, "IHIP_PAGED_SEQS");

// the sums of v over the threads before this one; total: over all of them
__device__ __forceinline__ int64_t scan_block(int64_t v, int64_t& total)
{
  __shared__ int64_t part[SLOT_THREADS / 64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int64_t s = v;
  for (int d = 1; d < 64; d *= 2) {
    const int64_t o = __shfl_up(s, d, 64);
    if (lane >= d) s += o;
  }
  __syncthreads();
  if (lane == 63) part[w] = s;
  __syncthreads();
  int64_t before = 0;
  total = 0;
  for (int i = 0; i < SLOT_THREADS / 64; i++) {
    if (i < w) before += part[i];
    total += part[i];
  }
  return before + s - v;
}

// the plan of the sequences, in LDS: row[s] the first row, move[s] the first
// of the page moves (pages taken, or put back), rank[s] the first page's place
// among the taken (or, of an ended sequence, among the put back), past[s], and
// state[s]: 0 nothing moves and no row has a slot, 1 live, 2 ended
struct SlotPlan {
  int *row, *move, *rank, *past, *state;
  int rows, moves, first, last;  // all rows, all moves, ends[0] and ends[1] modulo pages
};

__device__ __forceinline__ SlotPlan slot_plan(int* p, int n)
{
  return {p, p + n, p + 2 * n, p + 3 * n, p + 4 * n, 0, 0, 0, 0};
}

// the last s of the n with first[s] <= i (first ascending, first[0] <= i)
__device__ __forceinline__ int slot_find(const int* first, int n, int i)
{
  int lo = 0, hi = n;  // first[lo] <= i < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= i) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ int ring_at(uint32_t base, uint32_t i, uint32_t pages)
{
  const uint32_t at = base + i;  // both below 2^31
  return (int)(at >= pages ? at % pages : at);
}

// rows and page moves i0, i0 + step, ... of the plan
__device__ __forceinline__ void slot_rows(const SlotArgs& a, const SlotPlan& p, int i0, int step)
{
  const uint32_t ps = a.page_size;
  for (int64_t i = i0; i < p.moves; i += step) {
    const int s = slot_find(p.move, a.seqs, (int)i), j = (int)i - p.move[s];
    int* const t = a.table + (int64_t)s * a.max_pages;
    const uint32_t at = (uint32_t)p.rank[s] + (uint32_t)j;
    if (p.state[s] == 2) a.ring[ring_at(p.last, at, a.pages)] = t[j];
    else t[((uint32_t)p.past[s] + ps - 1) / ps + j] = a.ring[ring_at(p.first, at, a.pages)];
  }
  for (int64_t i = i0; i < a.rows; i += step) {
    int pos = -1, slot = -1;
    if (i < p.rows) {
      const int s = slot_find(p.row, a.seqs, (int)i);
      // (a sequence beyond every table has no slot; its positions end at the largest)
      const uint32_t at = (uint32_t)p.past[s] + (uint32_t)((int)i - p.row[s]);
      pos = at <= INT32_MAX ? (int)at : INT32_MAX;
      if (p.state[s] == 1) {
        // a page the sequence had, or one it takes in this step: from the ring, as
        // another thread writes the table's entry
        const int have = (int)(((uint32_t)p.past[s] + ps - 1) / ps), j = (int)((uint32_t)pos / ps);
        const int page = j < have ? a.table[(int64_t)s * a.max_pages + j]
                                  : a.ring[ring_at(p.first, p.rank[s] + j - have, a.pages)];
        if (page >= 0 && page < a.pages) slot = page * (int)ps + (int)((uint32_t)pos % ps);
      }
    }
    a.positions[i] = pos;
    a.slots[i] = slot;
  }
}

// one block: two scans over the sequences (rows and pages put back; then the
// pages taken, which depend on the rows that fit), the plan in LDS. Everything
// that a caller may pass as input and output is read before the barrier behind
// which it is written. Latency bound.
extern "C" __global__ __launch_bounds__(SLOT_THREADS) void paged_slots(SlotArgs a)
{
  extern __shared__ int slot_lds[];
  SlotPlan p = slot_plan(slot_lds, a.seqs);
  const int t = threadIdx.x, ps = a.page_size;
  const int64_t width = a.max_pages, cap = width * ps;
  const int64_t first = a.ends[0], last = a.ends[1];
  int64_t free_pages = first >= 0 && last > first ? last - first : 0;
  if (free_pages > a.pages) free_pages = a.pages;
  p.first = first >= 0 ? (int)(first % a.pages) : 0;
  p.last = last >= 0 ? (int)(last % a.pages) : 0;

  int past[SLOT_PER], live[SLOT_PER];
  int64_t fresh[SLOT_PER], have[SLOT_PER], rows = 0, back = 0;
#pragma unroll
  for (int i = 0; i < SLOT_PER; i++) {
    const int s = t * SLOT_PER + i;
    past[i] = s < a.seqs ? a.past[s] : -1;
    const int n = s < a.seqs && a.count ? a.count[s] : 1;
    live[i] = past[i] < 0 ? 0 : n < 0 ? 2 : 1;
    fresh[i] = live[i] == 1 ? n : 0;
    have[i] = live[i] ? ((int64_t)past[i] + ps - 1) / ps : 0;
    if (live[i] == 2) {  // no more than the table holds
      if (have[i] > width) have[i] = width;
      back += have[i];
    }
    rows += fresh[i];
  }
  int64_t all_rows, all_back, all_want, want = 0;
  int64_t row = scan_block(rows, all_rows), put = scan_block(back, all_back);
  int64_t need[SLOT_PER];
  {
    int64_t r = row;
#pragma unroll
    for (int i = 0; i < SLOT_PER; i++) {
      r += fresh[i];
      need[i] = 0;
      if (live[i] == 1) {
        const int64_t upto = past[i] + fresh[i];
        if (upto > cap || r > a.rows) live[i] = 3;  // has no place
        else need[i] = (upto + ps - 1) / ps - have[i];
      }
      want += need[i];
    }
  }
  int64_t take = scan_block(want, all_want);
  int64_t moved = 0, taken = 0, lost = 0;
  back = 0;
#pragma unroll
  for (int i = 0; i < SLOT_PER; i++) {
    const int s = t * SLOT_PER + i;
    const int64_t at = take, put_at = put;
    take += need[i];
    if (live[i] == 2) {
      // the ring holds the pool's pages once: what would pass that is no page in use
      put += have[i];
      if (put > a.pages - free_pages) have[i] = 0;
      back += have[i];
    }
    if (need[i] && take > free_pages) {
      live[i] = 3;
      need[i] = 0;
    }
    taken += need[i];
    lost += live[i] == 3;
    moved += live[i] == 2 ? have[i] : need[i];
    if (s < a.seqs) {
      p.rank[s] = (int)(live[i] == 2 ? (put_at < a.pages ? put_at : 0) : at < a.pages ? at : 0);
      p.past[s] = past[i];
      p.state[s] = live[i] == 1 ? 1 : live[i] == 2 ? 2 : 0;
      p.row[s] = (int)(row < INT32_MAX ? row : INT32_MAX);
    }
    row += fresh[i];
  }
  int64_t all_moved, all_taken, all_lost;
  int64_t move = scan_block(moved, all_moved);
  scan_block(back, all_back);
  scan_block(taken, all_taken);
  scan_block(lost, all_lost);
#pragma unroll
  for (int i = 0; i < SLOT_PER; i++) {
    const int s = t * SLOT_PER + i;
    if (s < a.seqs) p.move[s] = (int)move;
    move += live[i] == 2 ? have[i] : need[i];
  }
  p.rows = (int)(all_rows < INT32_MAX ? all_rows : INT32_MAX);
  p.moves = (int)all_moved;
  __syncthreads();  // the inputs are read, the plan is in LDS
#pragma unroll
  for (int i = 0; i < SLOT_PER; i++) {
    const int s = t * SLOT_PER + i;
    if (s >= a.seqs) break;
    a.offsets[s] = p.row[s];
    a.lengths[s] = live[i] == 1 ? (int)(past[i] + fresh[i]) : live[i] == 3 ? past[i] : -1;
  }
  if (t == 0) {
    a.offsets[a.seqs] = p.rows;
    a.ends_out[0] = first + all_taken;
    a.ends_out[1] = last + all_back;
    if (a.failed) a.failed[0] = (int)all_lost;
  }
  if (a.here) {
    slot_rows(a, p, t, SLOT_THREADS);
    return;
  }
  for (int i = t; i < 5 * a.seqs; i += SLOT_THREADS) a.plan[i] = slot_lds[i];
  if (t == 0) {
    int* const e = a.plan + 5 * a.seqs;
    e[0] = p.rows;
    e[1] = p.moves;
    e[2] = p.first;
    e[3] = p.last;
  }
}

// the rows of a step with prompts, by as many blocks as they fill: the plan
// from paged_slots' launch
extern "C" __global__ __launch_bounds__(256) void paged_slots_rows(SlotArgs a)
{
  extern __shared__ int slot_lds[];
  for (int i = threadIdx.x; i < 5 * a.seqs; i += 256) slot_lds[i] = a.plan[i];
  SlotPlan p = slot_plan(slot_lds, a.seqs);
  const int* const e = a.plan + 5 * a.seqs;
  p.rows = e[0];
  p.moves = e[1];
  p.first = e[2];
  p.last = e[3];
  __syncthreads();
  slot_rows(a, p, blockIdx.x * 256 + threadIdx.x, gridDim.x * 256);
}

// ------------------------------------------------------------ paged_qkrope
struct PagedRopeArgs {
  const float *q, *k, *v;
  float* q_out;
  const float *qn, *kn, *freq;
  const int *positions, *slots;
  char *kc, *vc;
  int64_t q_stride, k_stride, v_stride, out_stride;
  int64_t pages, page_stride, slot_stride, head_stride;
  double eps, scale;
  int32_t rows, heads, kvh, hd, page_size;
  int32_t half;         // rotating pairs
  int32_t interleaved;  // pairs (2 i, 2 i + 1), else (i, i + half)
  int32_t wide;         // 16-byte loads and stores
  int32_t seg;          // lanes of a head (a power of two, 8 values each)
  int32_t parts;        // blocks of a row
};

// cosine and sine of an angle of up to 2^31 radians, in double: the angle less
// its nearest multiple of pi / 2 (the product exact in the fused steps, pi / 2 in
// two parts), then their Taylor series on [-pi / 4, pi / 4], whose first left-out
// terms are below 1e-13 and 1e-14
__device__ __forceinline__ void turn(double angle, double& c, double& s)
{
  const double n = rint(angle * 0.63661977236758134308);
  double r = __builtin_fma(-n, 1.57079632679489655800, angle);
  r = __builtin_fma(-n, 6.12323399573676603587e-17, r);
  const double z = r * r;
  double p = 1.0 / 6227020800.0;
  p = __builtin_fma(p, z, -1.0 / 39916800.0);
  p = __builtin_fma(p, z, 1.0 / 362880.0);
  p = __builtin_fma(p, z, -1.0 / 5040.0);
  p = __builtin_fma(p, z, 1.0 / 120.0);
  p = __builtin_fma(p, z, -1.0 / 6.0);
  const double sn = __builtin_fma(p * z, r, r);
  double g = -1.0 / 87178291200.0;
  g = __builtin_fma(g, z, 1.0 / 479001600.0);
  g = __builtin_fma(g, z, -1.0 / 3628800.0);
  g = __builtin_fma(g, z, 1.0 / 40320.0);
  g = __builtin_fma(g, z, -1.0 / 720.0);
  g = __builtin_fma(g, z, 1.0 / 24.0);
  g = __builtin_fma(g, z, -0.5);
  const double cn = __builtin_fma(g, z, 1.0);
  const int m = (int)((int64_t)n & 3);
  const double cc = m & 1 ? sn : cn, ss = m & 1 ? cn : sn;
  c = m == 1 || m == 2 ? -cc : cc;
  s = m & 2 ? -ss : ss;
}

__device__ __forceinline__ uint16_t float_to_bf16(float f)
{
  const uint32_t b = float_bits(f);
  if ((b & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((b >> 16) | 0x40u);  // NaN stays one
  return (uint16_t)((b + 0x7fffu + ((b >> 16) & 1u)) >> 16);
}

// N (2 or 4) consecutive values of a cache row; T: 0 float, 1 half, 2 bf16
template <int T>
__device__ __forceinline__ void store4(char* p, const float (&v)[4])
{
  if constexpr (T == 0) {
    *(float4*)p = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; i++) h[i] = T == 1 ? float_to_half(v[i]) : float_to_bf16(v[i]);
    *(uint2*)p = make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
  }
}
template <int T>
__device__ __forceinline__ void store1(char* p, float v)
{
  if constexpr (T == 0) *(float*)p = v;
  else *(uint16_t*)p = T == 1 ? float_to_half(v) : float_to_bf16(v);
}

// A block forms the row's cosines and sines once, in LDS, then walks the row's
// heads (q, k, then v), 8 values (4 pairs) a lane, a head in `seg` lanes, so that
// the norm is a sum over aligned lanes. Sums, angles and the rotation are in
// double (full rate on this chip) and rounded once to single, then to the
// cache's type. Bound by HBM: 4 bytes in and 4 (q) or the cache's (k, v) out.
template <int T>
__device__ __forceinline__ void paged_qkrope_t(const PagedRopeArgs& a)
{
  constexpr int ES = T == 0 ? 4 : 2;
  __shared__ double2 cs[256];
  const int row = blockIdx.x, t = threadIdx.x;
  const int pos = a.positions[row];
  if (pos < 0) return;  // (the block's threads alike)
  const int64_t base = paged_slot_value(a.slots[row], a.page_size, a.pages, a.page_stride, a.slot_stride);
  if (t < a.half) {
    double c, s;
    turn((double)a.freq[t] * (double)pos, c, s);
    cs[t] = make_double2(c * a.scale, s * a.scale);
  }
  __syncthreads();
  const int seg = a.seg, all = (a.heads + 2 * a.kvh) * seg, hd = a.hd;
  for (int i = blockIdx.y * 256 + t; i < all; i += a.parts * 256) {
    const int h = i / seg, u = i & (seg - 1);  // the head, the lane's unit of 8 values
    const int kind = h < a.heads ? 0 : h < a.heads + a.kvh ? 1 : 2;
    const int hh = kind == 0 ? h : kind == 1 ? h - a.heads : h - a.heads - a.kvh;
    const float* in = (kind == 0 ? a.q + row * a.q_stride : kind == 1 ? a.k + row * a.k_stride
                                                                    : a.v + row * a.v_stride) + hh * hd;
    const float* w = kind == 0 ? a.qn : kind == 1 ? a.kn : nullptr;
    const bool on = u * 8 < hd;
    // where the unit's 4 pairs are: split over the halves, or consecutive
    const int half = kind == 2 ? 0 : a.half;
    const bool split = !a.interleaved && 4 * u < half;
    float x[8], wv[8];
    auto at = [&](int j, int e) {  // value e of pair j of the unit
      const int p = 4 * u + j;
      return split && p < half ? p + e * half : 2 * p + e;
    };
    if (on) {
      if (a.wide) {
        const int i0 = split ? 4 * u : 8 * u, i1 = split ? half + 4 * u : 8 * u + 4;
        const float4 v0 = *(const float4*)(in + i0), v1 = *(const float4*)(in + i1);
        const float l[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
        float g[8] = {1, 1, 1, 1, 1, 1, 1, 1};
        if (w) {
          const float4 w0 = *(const float4*)(w + i0), w1 = *(const float4*)(w + i1);
          g[0] = w0.x; g[1] = w0.y; g[2] = w0.z; g[3] = w0.w;
          g[4] = w1.x; g[5] = w1.y; g[6] = w1.z; g[7] = w1.w;
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
          x[2 * j] = split ? l[j] : l[2 * j];
          x[2 * j + 1] = split ? l[4 + j] : l[2 * j + 1];
          wv[2 * j] = split ? g[j] : g[2 * j];
          wv[2 * j + 1] = split ? g[4 + j] : g[2 * j + 1];
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; j++) {
          x[j] = in[at(j / 2, j & 1)];
          wv[j] = w ? w[at(j / 2, j & 1)] : 1.f;
        }
      }
    }
    double inv = 1.0;
    if (w) {
      double s = 0;
#pragma unroll
      for (int j = 0; j < 8; j++)
        if (on) s = __builtin_fma((double)x[j], (double)x[j], s);
      inv = 1.0 / sqrt(wave_sum(s, seg) / (double)hd + a.eps);
    }
    if (!on) continue;
    float o[8];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const double x0 = (double)x[2 * j] * inv * (double)wv[2 * j];
      const double x1 = (double)x[2 * j + 1] * inv * (double)wv[2 * j + 1];
      const bool rot = 4 * u + j < half;
      const double2 e = rot ? cs[4 * u + j] : make_double2(1.0, 0.0);
      o[2 * j] = rot ? (float)(x0 * e.x - x1 * e.y) : (float)x0;
      o[2 * j + 1] = rot ? (float)(x1 * e.x + x0 * e.y) : (float)x1;
    }
    if (kind == 0) {
      float* out = a.q_out + row * a.out_stride + hh * hd;
      if (a.wide) {
        const int i0 = split ? 4 * u : 8 * u, i1 = split ? half + 4 * u : 8 * u + 4;
        *(float4*)(out + i0) = split ? make_float4(o[0], o[2], o[4], o[6]) : make_float4(o[0], o[1], o[2], o[3]);
        *(float4*)(out + i1) = split ? make_float4(o[1], o[3], o[5], o[7]) : make_float4(o[4], o[5], o[6], o[7]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; j++) out[at(j / 2, j & 1)] = o[j];
      }
    } else if (base >= 0) {
      char* out = (kind == 1 ? a.kc : a.vc) + (base + hh * a.head_stride) * ES;
      if (a.wide) {
        const int i0 = split ? 4 * u : 8 * u, i1 = split ? half + 4 * u : 8 * u + 4;
        const float v0[4] = {o[0], split ? o[2] : o[1], split ? o[4] : o[2], split ? o[6] : o[3]};
        const float v1[4] = {split ? o[1] : o[4], split ? o[3] : o[5], split ? o[5] : o[6], o[7]};
        store4<T>(out + i0 * ES, v0);
        store4<T>(out + i1 * ES, v1);
      } else {
#pragma unroll
        for (int j = 0; j < 8; j++) store1<T>(out + at(j / 2, j & 1) * ES, o[j]);
      }
    }
  }
}

extern "C" __global__ __launch_bounds__(256) void paged_qkrope_f32(PagedRopeArgs a) { paged_qkrope_t<0>(a); }
extern "C" __global__ __launch_bounds__(256) void paged_qkrope_f16(PagedRopeArgs a) { paged_qkrope_t<1>(a); }
extern "C" __global__ __launch_bounds__(256) void paged_qkrope_bf16(PagedRopeArgs a) { paged_qkrope_t<2>(a); }

// --------------------------------------------------------- paged_attention
struct PagedAttnArgs {
  const float* q;
  const char *kc, *vc;
  const int *table, *lengths;
  float* y;
  const float* sinks;
  int64_t q_stride, pages, page_stride, slot_stride, head_stride, window;
  float scale;
  int32_t seqs, heads, kvh, hd, page_size, max_pages;
};

template <int T>
__device__ __forceinline__ float load1(const char* p)
{
  if constexpr (T == 0) return *(const float*)p;
  else if constexpr (T == 1) return half_to_float(*(const uint16_t*)p);
  else return bits_float((uint32_t)*(const uint16_t*)p << 16);
}

// one block per (head, sequence): wave w takes keys w, w + 4, ..., its lanes the
// dimensions, with a running maximum, sum and values; the waves meet at the end
template <int T>
__device__ __forceinline__ void paged_attention_t(const PagedAttnArgs& a)
{
  constexpr int ES = T == 0 ? 4 : 2, NV = 8;
  __shared__ float acc_s[4][512];
  __shared__ float ml[4][2];
  const int h = blockIdx.x, s = blockIdx.y, t = threadIdx.x, lane = t & 63, w = t >> 6;
  const int len = a.lengths[s], hd = a.hd;
  if (len < 0) return;
  int64_t lo, hi;
  paged_range(len, a.window, a.max_pages, a.page_size, &lo, &hi);
  const int64_t hoff = (int64_t)(h / (a.heads / a.kvh)) * a.head_stride;
  float q[NV], acc[NV];
#pragma unroll
  for (int i = 0; i < NV; i++) {
    const int d = lane + 64 * i;
    q[i] = d < hd ? a.q[s * a.q_stride + (int64_t)h * hd + d] : 0.f;
    acc[i] = 0.f;
  }
  float m = -__builtin_inff(), l = 0.f;
  for (int64_t j = lo + w; j < hi; j += 4) {
    const uint32_t pg = (uint32_t)j / (uint32_t)a.page_size;
    const int64_t at = paged_value(a.table[(int64_t)s * a.max_pages + pg], (int)((uint32_t)j % (uint32_t)a.page_size),
                                   a.pages, a.page_stride, a.slot_stride);
    if (at < 0) continue;
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < NV; i++)
      if (lane + 64 * i < hd) x = __builtin_fmaf(q[i], load1<T>(a.kc + (at + hoff + lane + 64 * i) * ES), x);
    x = wave_sum(x, 64) * a.scale;
    const float m2 = x > m || x != x ? x : m;
    const float f = m == -__builtin_inff() ? 0.f : expf(m - m2), p = x == -__builtin_inff() ? 0.f : expf(x - m2);
    l = l * f + p;
    m = m2;
#pragma unroll
    for (int i = 0; i < NV; i++)
      if (lane + 64 * i < hd) acc[i] = __builtin_fmaf(p, load1<T>(a.vc + (at + hoff + lane + 64 * i) * ES), acc[i] * f);
  }
#pragma unroll
  for (int i = 0; i < NV; i++) acc_s[w][lane + 64 * i] = acc[i];
  if (lane == 0) {
    ml[w][0] = m;
    ml[w][1] = l;
  }
  __syncthreads();
  float M = a.sinks ? a.sinks[h] : -__builtin_inff();
  for (int i = 0; i < 4; i++) M = ml[i][0] > M || ml[i][0] != ml[i][0] ? ml[i][0] : M;
  float den = a.sinks && lo < hi ? expf(a.sinks[h] - M) : 0.f, f[4];
  for (int i = 0; i < 4; i++) {
    f[i] = ml[i][1] == 0.f ? 0.f : expf(ml[i][0] - M);
    den += f[i] * ml[i][1];
  }
  for (int d = t; d < hd; d += 256) {
    float v = 0;
    for (int i = 0; i < 4; i++)
      if (ml[i][1] != 0.f) v += f[i] * acc_s[i][d];
    a.y[((int64_t)s * a.heads + h) * hd + d] = den != 0.f ? v / den : 0.f;
  }
}

extern "C" __global__ __launch_bounds__(256) void paged_attention_f32(PagedAttnArgs a) { paged_attention_t<0>(a); }
extern "C" __global__ __launch_bounds__(256) void paged_attention_f16(PagedAttnArgs a) { paged_attention_t<1>(a); }
extern "C" __global__ __launch_bounds__(256) void paged_attention_bf16(PagedAttnArgs a) { paged_attention_t<2>(a); }
