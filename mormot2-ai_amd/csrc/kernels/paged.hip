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
  int* plan;  // [5][seqs], then SlotPlan's numbers: the plan between the two launches
  int* meet;  // a counter of its blocks and a flag, zero between launches
  int32_t seqs, max_pages, page_size, pages, rows;
  int32_t here;  // 1: the rows in this launch too
};

constexpr int SLOT_THREADS = 1024;  // and up to 4 sequences a thread: IHIP_PAGED_SEQS

// one step of a scan over the wave: v and what lane - CTRL's shift holds (0 beyond
// the row of 16; broadcasts of a row's last lane: to the rows of `rows`)
template <int CTRL, int ROWS>
__device__ __forceinline__ int64_t scan_step(int64_t v)
{
  const uint32_t lo = __builtin_amdgcn_update_dpp(0u, (uint32_t)v, CTRL, ROWS, 0xF, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0u, (uint32_t)((uint64_t)v >> 32), CTRL, ROWS, 0xF, false);
  return v + (int64_t)((uint64_t)hi << 32 | lo);
}

// N values: each one's sum over the threads before this one, and over all of them
template <int N>
__device__ __forceinline__ void scan_block(const int64_t (&v)[N], int64_t (&before)[N], int64_t (&all)[N])
{
  __shared__ int64_t part[SLOT_THREADS / 64][4];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, waves = blockDim.x >> 6;
  int64_t s[N];
#pragma unroll
  for (int i = 0; i < N; i++) {
    s[i] = scan_step<0x111, 0xF>(v[i]);     // row_shr 1, 2, 4, 8
    s[i] = scan_step<0x112, 0xF>(s[i]);
    s[i] = scan_step<0x114, 0xF>(s[i]);
    s[i] = scan_step<0x118, 0xF>(s[i]);
    s[i] = scan_step<0x142, 0xA>(s[i]);     // rows 0 and 2 into 1 and 3
    s[i] = scan_step<0x143, 0xC>(s[i]);     // rows 0 and 1 into 2 and 3
    before[i] = s[i] - v[i];
    all[i] = 0;
  }
  __syncthreads();
  if (lane == 63)
#pragma unroll
    for (int i = 0; i < N; i++) part[w][i] = s[i];
  __syncthreads();
#pragma unroll 1
  for (int k = 0; k < waves; k++)
#pragma unroll
    for (int i = 0; i < N; i++) {
      if (k < w) before[i] += part[k][i];
      all[i] += part[k][i];
    }
}

// the plan of the sequences, in LDS: row[s] the first row, move[s] the first
// of the page moves (pages taken, or put back), rank[s] the first page's place
// among the taken (or, of an ended sequence, among the put back), past[s], and
// state[s]: 0 nothing moves and no row has a slot, 1 live, 2 ended
struct SlotPlan {
  int *row, *move, *rank, *past, *state;
  int rows, moves, first, last;  // all rows, all moves, ends[0] and ends[1] modulo pages
  int back, room;  // entries put back, pages that the ring has place for
  int closed;      // 1: sequences end, 2: and not all of their tables' entries find a place
};

__device__ __forceinline__ SlotPlan slot_plan(int* p, int n)
{
  return {p, p + n, p + 2 * n, p + 3 * n, p + 4 * n, 0, 0, 0, 0, 0, 0, 0};
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

__device__ __forceinline__ bool page_there(const SlotArgs& a, int page) { return page >= 0 && page < a.pages; }

// (through to memory: another block may write the entry again, put_back)
__device__ __forceinline__ void ring_store(const SlotArgs& a, const SlotPlan& p, uint32_t at, int page)
{
  __hip_atomic_store(a.ring + ring_at(p.last, at, a.pages), page, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// page moves i0, i0 + step, ... of the plan; whether an entry put back is no page of the
// pool
__device__ __forceinline__ bool slot_moves(const SlotArgs& a, const SlotPlan& p, int i0, int step)
{
  const uint32_t ps = a.page_size;
  bool hole = false;
  for (int64_t i = i0; i < p.moves; i += step) {
    const int s = slot_find(p.move, a.seqs, (int)i), j = (int)i - p.move[s];
    int* const t = a.table + (int64_t)s * a.max_pages;
    const uint32_t at = (uint32_t)p.rank[s] + (uint32_t)j;
    if (p.state[s] == 2) {
      const int page = t[j];
      hole |= !page_there(a, page);
      ring_store(a, p, at, page);
    } else {
      t[((uint32_t)p.past[s] + ps - 1) / ps + j] = a.ring[ring_at(p.first, at, a.pages)];
    }
  }
  return hole;
}

// rows i0, i0 + step, ... of the plan
__device__ __forceinline__ void slot_rows(const SlotArgs& a, const SlotPlan& p, int i0, int step)
{
  const uint32_t ps = a.page_size;
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
        if (page_there(a, page)) slot = page * (int)ps + (int)((uint32_t)pos % ps);
      }
    }
    a.positions[i] = pos;
    a.slots[i] = slot;
  }
}

// The ended sequences' pages into the ring once more, by one block, where a table has
// entries that are no page of the pool (holes, which are no free pages) or where with
// them the entries passed the ring's place: those that are pages alone, in order. Rare,
// so that the others' way has no look at the tables before the plan is made (with it
// 500 sequences 28 us for 15).
__device__ __forceinline__ void put_back(const SlotArgs& a, const SlotPlan& p)
{
  const int t = threadIdx.x, lane = t & 63, waves = blockDim.x >> 6, per = (a.seqs + blockDim.x - 1) / blockDim.x;
  auto entries = [&](int s, auto&& each) {
    const int n = p.state[s] == 2 ? (int)min(((uint32_t)p.past[s] + a.page_size - 1) / (uint32_t)a.page_size, (uint32_t)a.max_pages) : 0;
    int kept = 0;
#pragma unroll 1
    for (int j = lane; j - lane < n; j += 64) {
      const int page = j < n ? a.table[(int64_t)s * a.max_pages + j] : -1;
      const uint64_t there = __ballot(page_there(a, page));
      if (page_there(a, page))
        each(kept + __builtin_amdgcn_mbcnt_hi((uint32_t)(there >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)there, 0u)), page);
      kept += __popcll(there);
    }
    return kept;
  };
  for (int s = t >> 6; s < a.seqs; s += waves) {
    const int kept = entries(s, [](int, int) {});
    if (lane == 0) p.rank[s] = kept;
  }
  __syncthreads();
  int64_t mine = 0, before[1], all[1];
  for (int s = t * per; s < min((t + 1) * per, a.seqs); s++) mine += p.rank[s];
  scan_block<1>({mine}, before, all);
  int64_t put = before[0], back = 0;
  for (int s = t * per; s < min((t + 1) * per, a.seqs); s++) {
    const int n = p.rank[s];
    p.move[s] = put + n <= p.room ? (int)put : -1;
    if (put + n <= p.room) back += n;
    put += n;
  }
  scan_block<1>({back}, before, all);
  if (t == 0) a.ends_out[1] += all[0] - p.back;
  for (int s = t >> 6; s < a.seqs; s += waves) {
    const int at = p.move[s];
    if (at >= 0) entries(s, [&](int i, int page) { ring_store(a, p, at + i, page); });
  }
}

// One block: scans over the sequences (rows and pages put back; the pages taken,
// which depend on the rows that fit; the moves), the plan in LDS. Everything that a
// caller may pass as input and output is read before the barrier behind which it is
// written. Latency bound: the lengths, then a table entry or a free page, then the
// stores, then whether any page put back was none. 64 sequences' decode step 7.4 us; 500
// with 150000 rows 6.2 us and 9.4 for paged_slots_rows.
template <int SLOT_PER>
__device__ __forceinline__ void paged_slots_t(const SlotArgs& a)
{
  extern __shared__ int slot_lds[];
  SlotPlan p = slot_plan(slot_lds, a.seqs);
  const int t = threadIdx.x, ps = a.page_size;
  const int64_t cap = (int64_t)a.max_pages * ps;
  const int64_t first = a.ends[0], last = a.ends[1];
  int64_t free_pages = first >= 0 && last > first ? last - first : 0;
  if (free_pages > a.pages) free_pages = a.pages;
  // (a 64-bit remainder is a long way around, for a ring turned 2^32 times)
  auto turned = [&](int64_t v) { return v >> 32 ? (int)(v % a.pages) : (int)((uint32_t)v % (uint32_t)a.pages); };
  p.first = first >= 0 ? turned(first) : 0;
  p.last = last >= 0 ? turned(last) : 0;

  int past[SLOT_PER], live[SLOT_PER], fresh[SLOT_PER], have[SLOT_PER];
  int64_t rows = 0, back = 0;
#pragma unroll
  for (int i = 0; i < SLOT_PER; i++) {
    const int s = t * SLOT_PER + i;
    past[i] = s < a.seqs ? a.past[s] : -1;
    const int n = s < a.seqs && a.count ? a.count[s] : 1;
    live[i] = past[i] < 0 ? 0 : n < 0 ? 2 : 1;
    fresh[i] = live[i] == 1 ? n : 0;
    have[i] = live[i] ? (int)(((uint32_t)past[i] + ps - 1) / (uint32_t)ps) : 0;
    if (live[i] == 2) {  // no more than the table holds
      have[i] = min(have[i], a.max_pages);
      back += have[i];
    }
    rows += fresh[i];
  }
  int64_t first2[2], all2[2], first1[1], all1[1], first4[4], all4[4], want = 0;
  scan_block<2>({rows, back}, first2, all2);
  int64_t row = first2[0], put = first2[1];
  const int64_t all_rows = all2[0];
  int need[SLOT_PER];
  {
    int64_t r = row;
#pragma unroll
    for (int i = 0; i < SLOT_PER; i++) {
      r += fresh[i];
      need[i] = 0;
      if (live[i] == 1) {
        const int64_t upto = (int64_t)past[i] + fresh[i];
        if (upto > cap || r > a.rows) live[i] = 3;  // has no place
        else need[i] = (int)(((uint32_t)upto + ps - 1) / (uint32_t)ps) - have[i];
      }
      want += need[i];
    }
  }
  scan_block<1>({want}, first1, all1);
  int64_t take = first1[0];
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
  scan_block<4>({moved, back, taken, lost}, first4, all4);
  int64_t move = first4[0];
#pragma unroll
  for (int i = 0; i < SLOT_PER; i++) {
    const int s = t * SLOT_PER + i;
    if (s < a.seqs) p.move[s] = (int)move;
    move += live[i] == 2 ? have[i] : need[i];
  }
  p.rows = (int)(all_rows < INT32_MAX ? all_rows : INT32_MAX);
  p.moves = (int)all4[0];
  p.back = (int)all4[1];
  p.room = (int)(a.pages - free_pages);
  p.closed = all2[1] ? all2[1] > p.back ? 2 : 1 : 0;
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
    a.ends_out[0] = first + all4[2];
    a.ends_out[1] = last + all4[1];
    if (a.failed) a.failed[0] = (int)all4[3];
  }
  if (a.here) {
    // (the moves by other waves than the first rows')
    const bool hole = slot_moves(a, p, blockDim.x - 1 - t, blockDim.x);
    slot_rows(a, p, t, blockDim.x);
    if (p.closed && __syncthreads_or(hole || p.closed == 2)) put_back(a, p);
    return;
  }
  for (int i = t; i < 5 * a.seqs; i += blockDim.x) a.plan[i] = slot_lds[i];
  if (t == 0) {
    int* const e = a.plan + 5 * a.seqs;
    e[0] = p.rows;
    e[1] = p.moves;
    e[2] = p.first;
    e[3] = p.last;
    e[4] = p.back;
    e[5] = p.room;
    e[6] = p.closed;
  }
}

// one sequence a thread up to 256 (a decode step of 64 6.7 us, four a thread, whose
// code is longer and comes from a cold cache, 8.3; both without the look at what is put
// back, 0.6 more), else four (500 sequences 6.0 us, one a thread, whose scans have four
// times the waves, 6.5)
extern "C" __global__ __launch_bounds__(SLOT_THREADS) void paged_slots_1(SlotArgs a) { paged_slots_t<1>(a); }
extern "C" __global__ __launch_bounds__(SLOT_THREADS) void paged_slots_4(SlotArgs a) { paged_slots_t<4>(a); }

// the rows of a step with prompts, by as many blocks as they fill, and as many again for
// the page moves, which are through with their meeting before the rows are: the plan from
// paged_slots' launch
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
  p.back = e[4];
  p.room = e[5];
  p.closed = e[6];
  __syncthreads();
  const int half = gridDim.x / 2, b = blockIdx.x;
  if (b < half) {
    slot_rows(a, p, b * 256 + threadIdx.x, half * 256);
    return;
  }
  const bool hole = slot_moves(a, p, (b - half) * 256 + threadIdx.x, half * 256);
  if (!p.closed) return;
  // what the blocks found meets in the last of them
  if (__syncthreads_or(hole) && threadIdx.x == 0)
    __hip_atomic_store(a.meet + 1, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  if (!last_block(a.meet, half)) return;
  const int any = __hip_atomic_load(a.meet + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (threadIdx.x == 0) {
    __hip_atomic_store(a.meet, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(a.meet + 1, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  if (any || p.closed == 2) put_back(a, p);
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

// consecutive values of a cache row; T: 0 float, 1 half, 2 bf16
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
// cache's type (halves and bf16 so in two steps, a 2^-13 or 2^-16 of a step more
// than in one). Bound by HBM: 4 bytes in and 4 (q) or the cache's (k, v) out; 8000
// rows of 64 + 8 heads of 64 into a bf16 cache 59 us (5.2 TB/s, beside 4.7 of a large
// copy), 32 rows of 32 + 4 heads of 128 4.8 us (launch and two round trips).
template <int T>
__device__ __forceinline__ void paged_qkrope_t(const PagedRopeArgs& a)
{
  constexpr int ES = T == 0 ? 4 : 2;
  __shared__ double2 cs[256];
  const int row = blockIdx.x, t = threadIdx.x;
  const int pos = a.positions[row];
  if (pos < 0) return;  // (the block's threads alike)
  const int64_t base = paged_slot_value(a.slots[row], a.page_size, a.pages, a.page_stride, a.slot_stride);
  for (int i = t; i < a.half; i += blockDim.x) {
    double c, s;
    turn((double)a.freq[i] * (double)pos, c, s);
    cs[i] = make_double2(c * a.scale, s * a.scale);
  }
  __syncthreads();
  const int seg = a.seg, all = (a.heads + 2 * a.kvh) * seg, hd = a.hd;
  for (int i = blockIdx.y * blockDim.x + t; i < all; i += a.parts * blockDim.x) {
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

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));
typedef uint32_t uintx2 __attribute__((ext_vector_type(2)));

constexpr float LOG2E = 1.44269504088896340736f;
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ bool finite(float x) { return (float_bits(x) & 0x7f800000u) != 0x7f800000u; }

template <int T>
__device__ __forceinline__ float load1(const char* p)
{
  if constexpr (T == 0) return *(const float*)p;
  else if constexpr (T == 1) return half_to_float(*(const uint16_t*)p);
  else return bits_float((uint32_t)*(const uint16_t*)p << 16);
}

template <int T>
__device__ __forceinline__ floatx4 mfma16(uintx4 a, uintx4 b, floatx4 c)
{
  if constexpr (T == 1)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// two singles as NP parts of the cache's type that add up to them: halves (the
// first towards zero, the second to nearest: 22 bits, of values scaled into a
// half's normal range) or bf16 (towards zero: all 24 bits)
template <int T>
__device__ __forceinline__ void split2(float x, float y, uint32_t* part)
{
  if constexpr (T == 1) {
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

// what a block works on: a sequence, one of its KV heads, 16 of that one's query heads
struct AttnItem {
  int s, row, kv;   // sequence, its row of q and y, KV head
  int heads;        // query heads of the tile
  int head0;        // the first of them
};

template <int T, int D>
struct AttnShape {
  static constexpr int ES = T == 0 ? 4 : 2;            // bytes of a value
  static constexpr int KS = T == 0 ? 16 : 32;          // keys of a wave's step
  static constexpr int DS = D == 512 ? 2 : 1;          // waves that share a head's dimensions (registers)
  static constexpr int DW = D / DS;                    // dimensions of a wave
  static constexpr int KG = 4 / DS;                    // groups of keys: the others' waves
  static constexpr int TK = KG * KS;                   // keys of a block's tile
  static constexpr int NT = KS / 16;                   // score tiles of a step
  static constexpr int QL = 16 / ES;                   // values of a key load
  static constexpr int NQ = DW / (4 * QL);             // key loads of a lane and key
  static constexpr int NP = T == 0 ? 1 : T == 1 ? 2 : 3;  // parts of a single value
  static constexpr int VL = T != 0 && D > 64 ? 8 : 4;  // values of a value load
  static constexpr int NJ = DW / (16 * VL);            // value loads of a lane and key
  static constexpr int OS = D + 4;                     // a head's row in o_s
  // weights enter the product times this: into the halves' normal range. The two parts
  // hold 22 bits of those down to 2^-18 of the largest; smaller ones are off by 2^-40 of
  // the largest at most
  static constexpr float PS = T == 1 ? 32768.f : 1.f;
};

template <int T, int D>
struct AttnLds {
  using S = AttnShape<T, D>;
  uintx4 q[S::NP * S::DS * S::NQ * 64];  // the query tile as the matrix cores take it, by lane
  float o[16 * S::OS];           // a piece's values
  float m[16], l[16];            // its maxima and sums
  float wm[4][16], wl[4][16];    // the waves'
  float qs[16];                  // powers of two that the queries were divided by
  int64_t off[4][2][S::KS];      // byte offsets of the steps' keys
  floatx4 x[S::DS > 1 ? 2 : 1][S::DS > 1 ? 4 : 1][S::NT][64];  // the waves' shares of the scores
};

// The heads of a piece whose sums are not all finite, again by the formula's own
// steps in single: the matrix cores' parts turn an infinity into NaN (0 times it
// is added), and a key of score -infinity has weight 0. Waves take keys in turn,
// lanes dimensions. Slow, and only for such data.
template <int T, int D>
__device__ __forceinline__ void paged_walk(const PagedAttnArgs& a, const AttnItem& it, int64_t j0, int64_t j1,
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
      const int64_t at = paged_value(a.table[(int64_t)it.s * a.max_pages + pg], (int)((uint32_t)j % (uint32_t)a.page_size),
                                     a.pages, a.page_stride, a.slot_stride);
      if (at < 0) continue;
      const int64_t row = (at + it.kv * a.head_stride) * S::ES;
      float x = 0.f;
#pragma unroll
      for (int i = 0; i < NV; i++)
        if (lane + 64 * i < a.hd) x = __builtin_fmaf(q[i], load1<T>(a.kc + row + (lane + 64 * i) * S::ES), x);
      x = wave_sum(x, 64);
      if (x == -__builtin_inff()) continue;
      const float m2 = x > m || x != x ? x : m;
      const float f = m == -__builtin_inff() ? 0.f : exp2_fast(m - m2), p = exp2_fast(x - m2);
      l = l * f + p;
      m = m2;
#pragma unroll
      for (int i = 0; i < NV; i++)
        if (lane + 64 * i < a.hd)
          acc[i] = __builtin_fmaf(p, load1<T>(a.vc + row + (lane + 64 * i) * S::ES), acc[i] * f);
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
  for (int i = t; i < S::DS * S::NQ * 64; i += 256) {
    const int c = i & 15, d0 = (i >> 6) * 4 * S::QL + ((i >> 4) & 3) * S::QL;
    float v[S::QL];
    const bool in = c < it.heads && d0 < a.hd;
    float f = a.scale;
    if constexpr (T == 1) f = 1.f / s.qs[c];
#pragma unroll
    for (int j = 0; j < S::QL; j++) {
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
      for (int n = 0; n < S::NP; n++) s.q[n * S::DS * S::NQ * 64 + i] = uintx4{part[0][n], part[1][n], part[2][n], part[3][n]};
    }
  }
  __syncthreads();
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
template <int T, int D, bool FULL>
__device__ __forceinline__ void paged_attention_t(const PagedAttnArgs& a)
{
  using S = AttnShape<T, D>;
  __shared__ AttnLds<T, D> s;
  const int t = threadIdx.x, lane = t & 63, c = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const uint32_t grid = gridDim.x, b = blockIdx.x, per = a.kvh * a.tiles;
  const int hd = FULL ? D : a.hd, row_out = a.heads * a.hd;

  // a sequence's row, -1 where it has none in this step
  auto row_of = [&](int seq) {
    return a.offsets ? paged_row(a.offsets[seq], a.offsets[seq + 1], a.rows) : paged_row(seq, seq + 1, a.rows);
  };
  auto tiles_of = [&](int seq, int64_t& lo, int64_t& hi) {
    lo = hi = 0;
    if (row_of(seq) < 0) return 0u;
    paged_range(a.lengths[seq], a.window, a.max_pages, a.page_size, &lo, &hi);
    return (uint32_t)((hi - lo + S::TK - 1) / S::TK);
  };
  // all tiles (each wave for itself); rows without a key are zeros
  uint32_t all = 0, n0 = 0, live = 0;  // tiles, those of the lane's first sequence; sequences with any
  int64_t lo0 = 0, hi0 = 0;  // of the first 64 sequences, a lane each
  for (int s0 = 0; s0 < a.seqs; s0 += 64) {
    const int seq = s0 + lane;
    uint32_t n = 0;
    bool zero = false;
    if (seq < a.seqs) {
      int64_t lo, hi;
      n = tiles_of(seq, lo, hi);
      if (s0 == 0) n0 = n, lo0 = lo, hi0 = hi;
      zero = n == 0 && a.lengths[seq] >= 0 && row_of(seq) >= 0 && (uint32_t)seq % grid == b;
    }
    all += n * per;
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
  const uint32_t B = all >= 32 * grid && all / 24 >= live * per ? min(grid, (uint32_t)a.cus) : min(grid, all);
  if (b >= B) return;
  const uint32_t quot = all / B, rem = all % B;
  auto first = [&](uint32_t i) { return i * quot + i * rem / B; };
  uint32_t u = first(b);
  const uint32_t end = first(b + 1);
  // the sequence of tile u
  int seq = 0;
  uint32_t before = 0, n = 0;  // tiles before the sequence, tiles of a KV head's item
  int64_t lo = 0, hi = 0;
  for (int s0 = 0;; s0 += 64) {
    uint32_t m = s0 == 0 ? n0 : 0;
    if (s0 > 0 && s0 + lane < a.seqs) m = tiles_of(s0 + lane, lo0, hi0);
    const uint32_t items = m;
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

  for (;;) {
    const uint32_t item = (u - before) / n, tile0 = (u - before) - item * n;
    const uint32_t tile1 = min(n, tile0 + (end - u));
    AttnItem it;
    it.s = seq;
    it.row = row_of(seq);
    it.kv = item / a.tiles;
    const int tile16 = item - it.kv * a.tiles;
    it.heads = min(16, a.group - 16 * tile16);
    it.head0 = it.kv * a.group + 16 * tile16;
    const char* const kb = a.kc + (int64_t)it.kv * a.head_stride * S::ES;
    const char* const vb = a.vc + (int64_t)it.kv * a.head_stride * S::ES;
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
      // other lanes read it: no instruction, but no reordering or forwarding past here
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      return (uint32_t)__ballot(at >= 0) & (uint32_t)((1ull << S::KS) - 1);
    };
    uint32_t tile = tile0;
    const int page0 = entry(tile);
    int page = entry(tile + 1);
    stage_query<T, D>(a, it, s);
    const float sscale = T == 1 ? s.qs[c] : 1.f;

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
          if constexpr (S::VL * S::ES == 16) {
            vr[k][j] = *(const uintx4*)v;
          } else {
            const uintx2 h = *(const uintx2*)v;
            vr[k][j] = uintx4{h[0], h[1], 0, 0};
          }
        }
      }
      const uint32_t now = there;
      there = locate(tile + 1, page);
      page = entry(tile + 2);
      floatx4 x[S::NT];
#pragma unroll
      for (int k = 0; k < S::NT; k++) x[k] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < S::NQ; j++) {
#pragma unroll
        for (int n2 = 0; n2 < S::NP; n2++) {
          const uintx4 q = s.q[(n2 * S::DS * S::NQ + dh * S::NQ + j) * 64 + lane];
#pragma unroll
          for (int k = 0; k < S::NT; k++) {
            if constexpr (T == 0) {
#pragma unroll
              for (int e = 0; e < 4; e++)
                x[k] = __builtin_amdgcn_mfma_f32_16x16x4f32(bits_float(kr[k][j][e]), bits_float(q[e]), x[k], 0, 0, 0);
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
            x[k][r] = x[k][r] * sscale;
            top = fmaxf(top, x[k][r]);
          }
      } else {
#pragma unroll
        for (int k = 0; k < NV; k++) {
          const bool in = now >> (16 * (k >> 2) + 4 * g + (k & 3)) & 1;
          x[k >> 2][k & 3] = in ? x[k >> 2][k & 3] * sscale : -__builtin_inff();
          top = fmaxf(top, x[k >> 2][k & 3]);
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
        for (int k = 0; k < 4; k++) split2<T>(p[2 * k] * S::PS, p[2 * k + 1] * S::PS, part[k]);
#pragma unroll
        for (int j = 0; j < S::NJ; j++)
#pragma unroll
          for (int e = 0; e < S::VL; e++) {
            uintx4 v;
#pragma unroll
            for (int k = 0; k < 4; k++)
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
    const float f = exp2_fast(m - Ms) * (1.f / S::PS);
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
      for (int h = w; h < it.heads; h += 4) {
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
      const uint32_t u0 = before + item * n, b0 = block_of(u0), np = block_of(u0 + n - 1) - b0 + 1;
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
          if (out) {
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
    u += tile1 - tile0;
    if (u >= end) return;
    if (tile1 == n && item + 1 == per) {  // the next sequence with a key
      before = u;
      do n = tiles_of(++seq, lo, hi);
      while (n == 0);
    }
  }
}

// heads between two sizes: two blocks a CU up to 128. The others have no bound, which
// costs the join of few long sequences (24 us became 32). On their own those up to 128
// take 189 to 256 registers, two blocks a CU - but for halves of 128, whose 260 leave
// one: 64 ragged sequences up to 4000 keys, 16 heads over 8, 140 us where bf16 takes 115,
// 200 of them 350 and 310.
#define PAGED_ATTENTION(NAME, T, D)                                                                         \
  extern "C" __global__ __launch_bounds__(256) void paged_attention_##NAME##_##D(PagedAttnArgs a)           \
  {                                                                                                         \
    paged_attention_t<T, D, true>(a);                                                                       \
  }                                                                                                         \
  extern "C" __global__ __launch_bounds__(256, D == 128 ? 2 : 1) void                                       \
  paged_attention_##NAME##_##D##_part(PagedAttnArgs a)                                                      \
  {                                                                                                         \
    paged_attention_t<T, D, false>(a);                                                                      \
  }
PAGED_ATTENTION(f32, 0, 64)
PAGED_ATTENTION(f32, 0, 128)
PAGED_ATTENTION(f32, 0, 256)
PAGED_ATTENTION(f32, 0, 512)
PAGED_ATTENTION(f16, 1, 64)
PAGED_ATTENTION(f16, 1, 128)
PAGED_ATTENTION(f16, 1, 256)
PAGED_ATTENTION(f16, 1, 512)
PAGED_ATTENTION(bf16, 2, 64)
PAGED_ATTENTION(bf16, 2, 128)
PAGED_ATTENTION(bf16, 2, 256)
PAGED_ATTENTION(bf16, 2, 512)
