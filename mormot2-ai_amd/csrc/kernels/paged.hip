// paged.hip - several sequences decoded together over one paged cache: the
// plan of a step, q/k/v of the new rows into the pages, attention over them.
#include <type_traits>

#include "common.h"
#include "../paged.h"
#include "paged_attention.h"

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

// 8-bit pages: codes in kc and vc, single scales of a token's heads
struct PagedRope8Args : PagedRopeArgs {
  float *ks, *vs;
  int64_t s_page, s_slot, s_head;
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

// 8 values of a head in `seg` lanes as codes, and the scale by which they count: 1 / 127
// of the head's largest magnitude, in single. A code is the nearest whole number to its
// value over the scale, the even one between two (the division of doubles is exact to
// its last place, so that a tie is one). Codes pass 127 only where the scale is subnormal
// and was rounded down by more than one in 254: they are cut to it. A NaN or an infinity
// makes the scale NaN, and the head reads as NaN. 8001 rows of 64 + 2 x 8 heads of 64 take
// 69 us, 4.8 TB/s with the queries in single (63% of the SIMDs' time in vector work).
__device__ __forceinline__ uint2 codes8(const double (&x)[8], bool on, int seg, float& scale)
{
  double m = 0;
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const double v = on ? fabs(x[j]) : 0.0;
    m = v > m || v != v ? v : m;
  }
  auto top = [&](double o) { m = o > m || o != o ? o : m; };
  if (seg > 1) top(xpart<1>(m));
  if (seg > 2) top(xpart<2>(m));
  if (seg > 4) top(xpart<4>(m));
  if (seg > 8) top(xpart<8>(m));
  if (seg > 16) top(xpart<16>(m));
  if (seg > 32) top(xpart<32>(m));
  scale = (float)(m / 127.0);
  const bool bad = (float_bits(scale) & 0x7f800000u) == 0x7f800000u;
  if (bad) scale = bits_float(0x7fc00000u);
  uint32_t b[2] = {0, 0};
  if (!bad && scale != 0.f) {
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const double c = fmin(fmax(rint(x[j] / (double)scale), -127.0), 127.0);
      b[j / 4] |= ((uint32_t)(int)c & 255u) << (8 * (j & 3));
    }
  }
  return make_uint2(b[0], b[1]);
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
// than in one; 8-bit codes from the doubles, codes8, a head's values in order through
// LDS where its pairs lie in two halves). Bound by HBM: 4 bytes in and 4 (q) or the cache's (k, v) out; 8000
// rows of 64 + 8 heads of 64 into a bf16 cache 59 us (5.2 TB/s, beside 4.7 of a large
// copy), 32 rows of 32 + 4 heads of 128 4.8 us (launch and two round trips).
template <int T, typename A>
__device__ __forceinline__ void paged_qkrope_t(const A& a)
{
  constexpr int ES = T == 0 ? 4 : T == 3 ? 1 : 2;
  typedef typename std::conditional<T == 3, double, float>::type real;  // a turned value
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
    if (T != 3 && !on) continue;
    real o[8];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const double x0 = (double)x[2 * j] * inv * (double)wv[2 * j];
      const double x1 = (double)x[2 * j + 1] * inv * (double)wv[2 * j + 1];
      const bool rot = 4 * u + j < half;
      const double2 e = rot ? cs[4 * u + j] : make_double2(1.0, 0.0);
      o[2 * j] = rot ? (real)(x0 * e.x - x1 * e.y) : (real)x0;
      o[2 * j + 1] = rot ? (real)(x1 * e.x + x0 * e.y) : (real)x1;
    }
    if constexpr (T == 3) {
      if (kind != 0) {
        __shared__ double line[256 * 8];
        if (half && !a.interleaved) {
          // (a head's lanes are a wave's)
#pragma unroll
          for (int j = 0; j < 8; j++)
            if (on) line[(t - u) * 8 + at(j / 2, j & 1)] = o[j];
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          __builtin_amdgcn_wave_barrier();
#pragma unroll
          for (int j = 0; j < 8; j++)
            if (on) o[j] = line[t * 8 + j];
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          __builtin_amdgcn_wave_barrier();
        }
        float scale;
        const uint2 codes = codes8(o, on, seg, scale);
        if (on && base >= 0) {
          *(uint2*)((kind == 1 ? a.kc : a.vc) + base + hh * a.head_stride + 8 * u) = codes;
          if (u == 0)
            (kind == 1 ? a.ks : a.vs)[paged_slot_value(a.slots[row], a.page_size, a.pages, a.s_page, a.s_slot) + hh * a.s_head] = scale;
        }
        continue;
      }
      if (!on) continue;
    }
    if (kind == 0) {
      float* out = a.q_out + row * a.out_stride + hh * hd;
      if (a.wide) {
        const int i0 = split ? 4 * u : 8 * u, i1 = split ? half + 4 * u : 8 * u + 4;
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; j++) f[j] = (float)o[j];
        *(float4*)(out + i0) = split ? make_float4(f[0], f[2], f[4], f[6]) : make_float4(f[0], f[1], f[2], f[3]);
        *(float4*)(out + i1) = split ? make_float4(f[1], f[3], f[5], f[7]) : make_float4(f[4], f[5], f[6], f[7]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; j++) out[at(j / 2, j & 1)] = (float)o[j];
      }
    } else if constexpr (T != 3) {
      if (base < 0) continue;
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
extern "C" __global__ __launch_bounds__(256) void paged_qkrope_q8(PagedRope8Args a) { paged_qkrope_t<3>(a); }

// -------------------------------------------------------------- paged_read
struct PagedReadArgs {
  const char *kc, *vc;
  const float *ks, *vs;
  const int *table, *first, *offsets;
  char *k_out, *v_out;
  int64_t pages, page_stride, slot_stride, head_stride, s_page, s_slot, s_head;
  int32_t rows, seqs, max_pages, page_size, hd, units, chunk;  // units of 16 bytes of a row's output, rows of a wave's turn
};

// The cached tokens of sequences as rows of single or half values. A wave takes `chunk`
// rows a turn, one a lane, for the rows' places (the sequence by search, its table's
// entry), then walks the rows' units, 16 bytes of output a lane, so that stores are
// contiguous and loads too within a head. Bound by HBM, mostly by what it writes: 48
// histories of up to 8200, 8 KV heads of 128 from 8-bit pages to single, 2.0 GB in 445 us,
// 4.6 TB/s (a large copy's 4.8); one of 1151 tokens to half 4.8 us, a launch.
template <int T, int OUT>
__device__ __forceinline__ void paged_read_t(const PagedReadArgs& a)
{
  constexpr int ES = T == 0 ? 4 : T == 3 ? 1 : 2, N = OUT == 0 ? 4 : 8;
  const int lane = threadIdx.x & 63;
  const int waves = gridDim.x * 4, wave = blockIdx.x * 4 + (threadIdx.x >> 6);
  const uint32_t units = a.units;
  for (int64_t r0 = (int64_t)wave * a.chunk; r0 < a.rows; r0 += (int64_t)waves * a.chunk) {
    const int n = (int)min((int64_t)a.chunk, a.rows - r0);
    // the lane's row: its place in values and in scales, -1 nothing there, -2 no row of the call
    int64_t at = -2, sat = 0;
    if (lane < n) {
      const int row = (int)r0 + lane;
      if (row >= a.offsets[0] && row < a.offsets[a.seqs]) {
        const int s = slot_find(a.offsets, a.seqs, row);
        const int64_t pos = (int64_t)(a.first ? a.first[s] : 0) + ((int64_t)row - a.offsets[s]);
        at = -1;
        if (pos >= 0 && pos < (int64_t)a.max_pages * a.page_size) {
          const int page = a.table[(int64_t)s * a.max_pages + (uint32_t)pos / (uint32_t)a.page_size];
          const int in = (int)((uint32_t)pos % (uint32_t)a.page_size);
          at = paged_value(page, in, a.pages, a.page_stride, a.slot_stride);
          if (T == 3 && at >= 0) sat = page * a.s_page + (int64_t)in * a.s_slot;
        }
      }
    }
    const uint32_t all = n * units;
    // 4 units a lane on their way at once, of k and of v
    for (uint32_t i0 = 0; i0 < all; i0 += 256) {
      uint64_t raw[2][4][T == 3 ? 1 : N * ES / 8];
      float sc[2][4];
      int64_t to[4];
      bool there[4];
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const uint32_t i = min(i0 + 64 * e + lane, all - 1), r = i / units, u = i - r * units;
        const int64_t from = __shfl(at, r, 64), sfrom = T == 3 ? __shfl(sat, r, 64) : 0;
        const uint32_t v = u * N, h = v / (uint32_t)a.hd, d = v - h * a.hd;
        to[e] = i0 + 64 * e + lane < all && from != -2 ? (r0 + r) * (int64_t)units + u : -1;
        there[e] = from >= 0;
        const int64_t src = there[e] ? (from + h * a.head_stride + d) * ES : 0;
#pragma unroll
        for (int x = 0; x < 2; x++) {
          const char* const p = (x ? a.vc : a.kc) + src;
          if constexpr (T == 3) {
            if constexpr (N == 4) raw[x][e][0] = *(const uint32_t*)p;
            else raw[x][e][0] = *(const uint64_t*)p;
            sc[x][e] = there[e] ? (x ? a.vs : a.ks)[sfrom + h * a.s_head] : 0.f;
          } else {
#pragma unroll
            for (int j = 0; j < N * ES / 8; j++) raw[x][e][j] = ((const uint64_t*)p)[j];
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 4; e++) {
        if (to[e] < 0) continue;
#pragma unroll
        for (int x = 0; x < 2; x++) {
          float f[N];
#pragma unroll
          for (int j = 0; j < N; j++) {
            const uint32_t w = (uint32_t)(raw[x][e][j * ES / 8] >> (8 * (j * ES % 8)));
            if constexpr (T == 0) f[j] = bits_float(w);
            else if constexpr (T == 1) f[j] = half_to_float(w & 0xffffu);
            else if constexpr (T == 2) f[j] = bits_float(w << 16);
            else f[j] = (float)(int8_t)w * sc[x][e];
            if (!there[e]) f[j] = 0.f;
          }
          char* const o = (x ? a.v_out : a.k_out) + to[e] * 16;
          if constexpr (OUT == 0) {
            *(float4*)o = make_float4(f[0], f[1], f[2], f[3]);
          } else {
            uint32_t h[4];
#pragma unroll
            for (int j = 0; j < 4; j++) h[j] = float_to_half(f[2 * j]) | (uint32_t)float_to_half(f[2 * j + 1]) << 16;
            *(uint4*)o = make_uint4(h[0], h[1], h[2], h[3]);
          }
        }
      }
    }
  }
}

#define PAGED_READ(NAME, T)                                                                                          \
  extern "C" __global__ __launch_bounds__(256) void paged_read_##NAME##_f32(PagedReadArgs a) { paged_read_t<T, 0>(a); } \
  extern "C" __global__ __launch_bounds__(256) void paged_read_##NAME##_f16(PagedReadArgs a) { paged_read_t<T, 1>(a); }
PAGED_READ(f32, 0)
PAGED_READ(f16, 1)
PAGED_READ(bf16, 2)
PAGED_READ(q8, 3)

// --------------------------------------------------------- paged_attention
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
