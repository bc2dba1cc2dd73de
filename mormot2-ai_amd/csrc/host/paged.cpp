// paged.cpp - several sequences decoded together over one paged cache: the
// plan of a step, q/k/v into the pages, attention over them, and the log
// probabilities of a row of logits. Arguments are checked before the context,
// so that a host without a device can check a call.
#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdio>
#include <string>

#include "internal.h"
#include "../paged.h"
#include "../sample_rows.h"

using namespace ihip;

namespace {

// the context's device made the caller's for the launches of one call
struct OnDevice {
  int before = -1;
  explicit OnDevice(const ihip_ctx* c)
  {
    int now = 0;
    if (hipGetDevice(&now) != hipSuccess || now == c->device) return;
    if (hipSetDevice(c->device) == hipSuccess) before = now;
  }
  ~OnDevice()
  {
    if (before >= 0) (void)hipSetDevice(before);
  }
};

int no_context(const char* who) { return fail(IHIP_E_ARG, std::string(who) + ": no context"); }

int refuse(const char* who, const char* why, int code = IHIP_E_ARG)
{
  return fail(code, std::string(who) + ": " + why);
}

// floats from a row to the next: rows times it stay far from 64 bits
constexpr int64_t STRIDE_MOST = (int64_t)1 << 36;

// whether the bytes [a, a + n) meet any of the rows of `width` bytes at s, s + stride, ..
bool overlaps(uint64_t a, __int128 n, uint64_t s, __int128 stride, __int128 width, int64_t rows)
{
  // row r is met where s + r stride < a + n and s + r stride + width > a
  const __int128 d = (__int128)a - (__int128)s;
  if (d + n <= 0 || (rows - 1) * stride + width <= d) return false;
  const __int128 first = d < width ? 0 : (d - width) / stride + 1, last = (d + n - 1) / stride;
  return first <= last && first < rows;
}

// a pool with its strides filled in, in values and in scales (of 8-bit pages)
struct Pool {
  int64_t page_stride = 0, slot_stride = 0, head_stride = 0;
  int64_t s_page = 0, s_slot = 0, s_head = 0;
  int64_t es = 0;  // bytes of a value
  const char* type = "";
};

const char* type_name(int t)
{
  return t == IHIP_F32 ? "f32" : t == IHIP_F16 ? "f16" : t == IHIP_BF16 ? "bf16" : t == IHIP_Q8_HEAD ? "q8" : nullptr;
}

// the scales of a pool's keys or values (the fields of other pools are not looked at)
uint64_t q8_scales(const ihip_pages* p, int values)
{
  return p->dtype != IHIP_Q8_HEAD ? 0 : values ? p->v_scale : p->k_scale;
}

int check_pool(const char* who, const ihip_pages* p, Pool* out)
{
  if (!p || !p->k || !p->v) return refuse(who, "no cache");
  out->type = type_name(p->dtype);
  if (!out->type) return refuse(who, "a cache that is not F32, F16 or BF16, nor Q8_HEAD", IHIP_E_UNSUPPORTED);
  if (p->head_dim < 8 || p->head_dim > 512 || p->head_dim % 8)
    return refuse(who, "head_dim is a multiple of 8 up to 512", IHIP_E_UNSUPPORTED);
  const bool q8 = p->dtype == IHIP_Q8_HEAD;
  if (q8 && p->head_dim % 16) return refuse(who, "head_dim of 8-bit pages is a multiple of 16", IHIP_E_UNSUPPORTED);
  if (p->kv_heads < 1 || p->kv_heads > 65535 || p->page_size < 1 || p->pages < 1 ||
      p->pages > INT32_MAX / p->page_size)
    return refuse(who, "kv_heads, page_size or pages out of range");
  const int64_t row = (int64_t)p->kv_heads * p->head_dim, es = p->dtype == IHIP_F32 ? 4 : q8 ? 1 : 2;
  out->es = es;
  out->head_stride = p->head_stride ? p->head_stride : p->head_dim;
  out->slot_stride = p->slot_stride ? p->slot_stride : row;
  out->page_stride = p->page_stride ? p->page_stride : row * p->page_size;
  for (int64_t s : {out->head_stride, out->slot_stride, out->page_stride})
    if (s < p->head_dim || s > (int64_t)1 << 40 || s * es % 16)
      return refuse(who, "a stride below head_dim or not of 16 bytes");
  // within a page 32 bits hold every offset
  if (out->slot_stride * (p->page_size - 1) + out->head_stride * (p->kv_heads - 1) + p->head_dim > INT32_MAX)
    return refuse(who, "a page of more than 2^31 values");
  if (p->k % 16 || p->v % 16) return refuse(who, "a cache that is not aligned to 16 bytes");
  if (q8) {
    if (!p->k_scale || !p->v_scale || (p->k_scale | p->v_scale) % 4)
      return refuse(who, "8-bit pages without scales, or scales not aligned to 4 bytes");
    if (out->head_stride % p->head_dim || out->slot_stride % p->head_dim || out->page_stride % p->head_dim)
      return refuse(who, "a stride of 8-bit pages that is no multiple of head_dim");
    out->s_page = out->page_stride / p->head_dim;
    out->s_slot = out->slot_stride / p->head_dim;
    out->s_head = out->head_stride / p->head_dim;
  }
  return 0;
}

// the sequences that share their first tokens (null: none do)
struct Groups {
  uint64_t members, shared;
  int64_t groups;
};

int paged_attention(const char* who, ihip_ctx* c, uint64_t q, int64_t q_stride, const ihip_pages* cache,
                    uint64_t table, int64_t max_pages, uint64_t lengths, uint64_t offsets, int64_t rows,
                    const Groups* groups, uint64_t y, int64_t seqs, int64_t heads, int64_t window,
                    uint64_t sinks, double scale)
{
  Pool p;
  if (int rc = check_pool(who, cache, &p)) return rc;
  const int64_t hd = cache->head_dim, kvh = cache->kv_heads;
  if (!q || !table || !lengths || !y || (groups && (!groups->members || !groups->shared)))
    return refuse(who, "a missing array");
  if (seqs > IHIP_PAGED_SEQS) return refuse(who, "more sequences than IHIP_PAGED_SEQS", IHIP_E_NOMEM);
  if (seqs < 1 || heads < 1 || heads > 65535 || heads % kvh || window < 0 || max_pages < 1 ||
      max_pages > INT32_MAX / cache->page_size || rows < 1 || rows > INT32_MAX)
    return refuse(who, "seqs, heads, window, max_pages or rows out of range");
  if (groups && (groups->groups < 1 || groups->groups > seqs)) return refuse(who, "groups out of range");
  if (groups && seqs * heads > SHARED_HEADS) return refuse(who, "more than 2^20 heads of sequences", IHIP_E_NOMEM);
  q_stride = q_stride ? q_stride : heads * hd;
  if (q_stride < heads * hd) return refuse(who, "a stride below a row");
  if (q_stride > STRIDE_MOST) return refuse(who, "a stride beyond 2^36");
  if ((q | y | sinks | lengths | offsets | table | (groups ? groups->members | groups->shared : 0)) % 4) return refuse(who, "arrays aligned to 4 bytes");
  if (overlaps(y, (__int128)rows * heads * hd * 4, q, q_stride * 4, heads * hd * 4, rows) &&
      (groups || !(y == q && q_stride == heads * hd)))
    return refuse(who, groups ? "y overlaps q" : "y overlaps q, and is not q's contiguous rows");
  // (the kernel's scores are in base 2, in single)
  const float scale2 = (float)((scale != 0 ? scale : 1.0 / std::sqrt((double)hd)) * 1.4426950408889634);
  if (!(scale >= 0) || !std::isfinite(scale2)) return refuse(who, "scale is 0 or positive, times log2 e within single");
  // the kernels take tiles of 128 keys of 16-bit and 8-bit caches, 64 of single ones,
  // half as many of heads beyond 256
  const int64_t group = heads / kvh, tiles = (group + 15) / 16;
  const int64_t tk = (cache->dtype == IHIP_F32 ? 64 : 128) / (hd > 256 ? 2 : 1);
  const int64_t keys = window > 0 ? std::min(window, max_pages * cache->page_size) : max_pages * cache->page_size;
  // (8-bit pages' and the groups' kernels count three more an item)
  const int64_t units = ((keys + tk - 1) / tk + (cache->dtype == IHIP_Q8_HEAD || groups ? 3 : 0)) * kvh * tiles;
  if (units > INT32_MAX / seqs) return refuse(who, "more than 2^31 tiles of keys", IHIP_E_NOMEM);
  if (!c) return no_context(who);
  OnDevice on(c);
  struct {
    const float* q;
    const char *kc, *vc;
    const int *table, *lengths, *offsets;
    float* y;
    const float* sinks;
    float* part;
    int* done;
    int64_t q_stride, pages, page_stride, slot_stride, head_stride, window;
    float scale;
    int32_t seqs, heads, kvh, hd, page_size, max_pages, group, tiles, rows, cus;
    uint64_t ks, vs;  // (of 8-bit pages' and the groups' kernels alone, as what follows)
    int64_t s_page, s_slot, s_head;
    uint64_t members, shared, pieces, sums, plan;  // (of the groups' kernels alone)
    int32_t groups, pad;
  } a = {(const float*)q, (const char*)cache->k, (const char*)cache->v, (const int*)table,
         (const int*)lengths, (const int*)offsets, (float*)y, (const float*)sinks, (float*)c->paged_part,
         (int*)(c->paged_part + PAGED_PART_BYTES), q_stride, cache->pages, p.page_stride,
         p.slot_stride, p.head_stride, window,
         scale2, (int32_t)seqs,
         (int32_t)heads, (int32_t)kvh, (int32_t)hd, cache->page_size, (int32_t)max_pages, (int32_t)group,
         (int32_t)tiles, (int32_t)rows, c->cus, q8_scales(cache, 0), q8_scales(cache, 1), p.s_page, p.s_slot, p.s_head,
         groups ? groups->members : 0, groups ? groups->shared : 0, c->paged_shared, c->paged_shared + SHARED_PIECE_BYTES,
         c->paged_shared + SHARED_PIECE_BYTES + SHARED_HEADS * 8, groups ? (int32_t)groups->groups : 0, 0};
  const int d = hd <= 64 ? 64 : hd <= 128 ? 128 : hd <= 256 ? 256 : 512;
  char name[40];
  // (a window's keys are few: every sequence reads its own)
  const bool prefix = groups && window == 0;
  if (prefix) {
    const int64_t cols = 16 * PAGED_SHARED_TILES(d, cache->dtype == IHIP_Q8_HEAD);
    snprintf(name, sizeof name, "paged_prefix_%s_%d%s", p.type, d, hd == d ? "" : "_part");
    int64_t blocks = (int64_t)c->cus * resident_blocks(c, name, 256);
    blocks = std::min<int64_t>({blocks, PAGED_BLOCKS, (int64_t)(SHARED_PIECE_BYTES / (2 * cols * (hd + 2) * 4)), units * seqs});
    if (int rc = launch(c, name, dim3((unsigned)blocks), dim3(256), &a)) return rc;
  }
  snprintf(name, sizeof name, "paged_%s_%s_%d%s", prefix ? "own" : "attention", p.type, d, hd == d ? "" : "_part");
  // as many blocks as reside at once, and as there are tiles and pieces for them
  int64_t blocks = (int64_t)c->cus * resident_blocks(c, name, 256);
  blocks = std::min<int64_t>({blocks, PAGED_BLOCKS, (int64_t)(PAGED_PART_BYTES / (2 * (16 * hd + 32) * 4)), units * seqs});
  return launch(c, name, dim3((unsigned)blocks), dim3(256), &a);
}

}  // namespace

extern "C" {

int ihip_enqueue_paged_slots(ihip_ctx* c, uint64_t past, uint64_t count, int64_t seqs, uint64_t table,
                             int64_t max_pages, int64_t page_size, uint64_t ring, int64_t pages,
                             uint64_t ends, uint64_t ends_out, uint64_t offsets, uint64_t lengths,
                             uint64_t positions, uint64_t slots, int64_t rows, uint64_t failed)
{
  const char* who = "ihip_enqueue_paged_slots";
  if (!past || !table || !ring || !ends || !ends_out || !offsets || !lengths || !positions || !slots)
    return refuse(who, "a missing array");
  if (seqs > IHIP_PAGED_SEQS) return refuse(who, "more sequences than IHIP_PAGED_SEQS", IHIP_E_NOMEM);
  if (seqs < 1 || rows < 1 || rows > INT32_MAX || page_size < 1 || page_size > INT32_MAX || pages < 1 ||
      pages > INT32_MAX / page_size || max_pages < 1 || max_pages > INT32_MAX / page_size)
    return refuse(who, "seqs, rows, page_size, pages or max_pages out of range");
  if (ends % 8 || ends_out % 8) return refuse(who, "ends are int64, aligned to 8 bytes");
  if ((past | count | table | ring | offsets | lengths | positions | slots | failed) % 4)
    return refuse(who, "arrays aligned to 4 bytes");
  if (!c) return no_context(who);
  OnDevice on(c);
  struct {
    const int *past, *count;
    int *table, *ring;
    const int64_t* ends;
    int64_t* ends_out;
    int *offsets, *lengths, *positions, *slots, *failed;
    int *plan, *meet;
    int32_t seqs, max_pages, page_size, pages, rows, here;
  } a = {(const int*)past, (const int*)count, (int*)table, (int*)ring, (const int64_t*)ends,
         (int64_t*)ends_out, (int*)offsets, (int*)lengths, (int*)positions, (int*)slots, (int*)failed,
         (int*)c->paged_plan, (int*)(c->paged_plan + PAGED_PLAN_BYTES), (int32_t)seqs, (int32_t)max_pages, (int32_t)page_size, (int32_t)pages,
         (int32_t)rows, rows <= PAGED_ROWS_HERE};
  const size_t shmem = (size_t)seqs * 5 * 4;
  // a thread for the kernel's sequences, and where this block writes the rows one for
  // a row and a wave beside them for the pages that move
  const int per = seqs <= 256 ? 1 : 4;
  const int64_t threads = std::max<int64_t>((seqs + per - 1) / per, a.here ? std::min<int64_t>(rows + 64, 1024) : 256);
  int rc = launch(c, per == 1 ? "paged_slots_1" : "paged_slots_4", dim3(1), dim3((unsigned)((threads + 63) / 64 * 64)), &a, shmem);
  if (rc || a.here) return rc;
  return launch(c, "paged_slots_rows", dim3(2 * (unsigned)std::min<int64_t>(4 * c->cus, (rows + 1023) / 1024)),
                dim3(256), &a, shmem);
}

int ihip_enqueue_paged_qkrope(ihip_ctx* c, uint64_t q, int64_t q_stride, uint64_t k, int64_t k_stride,
                              uint64_t v, int64_t v_stride, int64_t rows, int64_t heads, uint64_t qn,
                              uint64_t kn, double eps, const ihip_rope* rope, uint64_t positions,
                              uint64_t slots, const ihip_pages* cache, uint64_t q_out)
{
  const char* who = "ihip_enqueue_paged_qkrope";
  Pool p;
  if (int rc = check_pool(who, cache, &p)) return rc;
  const int64_t hd = cache->head_dim, kvh = cache->kv_heads;
  if (!q || !k || !v || !positions || !slots) return refuse(who, "a missing array");
  // (a grid of 256 threads a row counts its threads in 32 bits)
  if (rows < 1 || rows > 1 << 23 || heads < 1 || heads > 65535 || heads % kvh)
    return refuse(who, "rows or heads out of range");
  const int64_t qw = heads * hd, kw = kvh * hd;
  q_stride = q_stride ? q_stride : qw;
  k_stride = k_stride ? k_stride : kw;
  v_stride = v_stride ? v_stride : kw;
  if (q_stride < qw || k_stride < kw || v_stride < kw) return refuse(who, "a stride below a row");
  if (std::max({q_stride, k_stride, v_stride}) > STRIDE_MOST) return refuse(who, "a stride beyond 2^36");
  const uint64_t aligned = q | k | v | q_out | qn | kn;
  if ((aligned | positions | slots) % 4) return refuse(who, "arrays aligned to 4 bytes");
  // (a row's values are read and written by several blocks and waves in any order)
  const __int128 out = (__int128)rows * qw * 4;
  if (q_out && ((overlaps(q_out, out, q, q_stride * 4, qw * 4, rows) && !(q_out == q && q_stride == qw)) ||
                overlaps(q_out, out, k, k_stride * 4, kw * 4, rows) || overlaps(q_out, out, v, v_stride * 4, kw * 4, rows)))
    return refuse(who, "q_out overlaps q, k or v, and is not q's contiguous rows");
  if (!(eps >= 0) || !std::isfinite(eps)) return refuse(who, "eps");
  int64_t dims = 0;
  if (rope) {
    dims = rope->dims ? rope->dims : hd;
    if (!rope->freq || rope->freq % 4 || dims < 2 || dims > hd || dims & 1)
      return refuse(who, "rope: freq, or dims odd or beyond head_dim");
    if (!std::isfinite(rope->scale)) return refuse(who, "rope: scale");
  }
  if (!c) return no_context(who);
  OnDevice on(c);
  struct {
    const float *q, *k, *v;
    float* q_out;
    const float *qn, *kn, *freq;
    const int *positions, *slots;
    char *kc, *vc;
    int64_t q_stride, k_stride, v_stride, out_stride;
    int64_t pages, page_stride, slot_stride, head_stride;
    double eps, scale;
    int32_t rows, heads, kvh, hd, page_size, half, interleaved, wide, seg, parts;
    uint64_t ks, vs;  // (of 8-bit pages' kernel alone, as what follows)
    int64_t s_page, s_slot, s_head;
  } a = {(const float*)q, (const float*)k, (const float*)v, (float*)(q_out ? q_out : q), (const float*)qn,
         (const float*)kn, (const float*)(rope ? rope->freq : 0), (const int*)positions, (const int*)slots,
         (char*)cache->k, (char*)cache->v, q_stride, k_stride, v_stride, q_out ? qw : q_stride,
         cache->pages, p.page_stride, p.slot_stride, p.head_stride, eps,
         rope && rope->scale != 0 ? rope->scale : 1.0, (int32_t)rows, (int32_t)heads, (int32_t)kvh,
         (int32_t)hd, cache->page_size, (int32_t)(dims / 2), rope ? rope->interleaved != 0 : 0,
         // 16-byte loads: rows aligned, and no unit of 4 pairs that only half turns
         aligned % 16 == 0 && (q_stride | k_stride | v_stride) % 4 == 0 &&
             (!rope || rope->interleaved || dims % 8 == 0),
         1, 1, q8_scales(cache, 0), q8_scales(cache, 1), p.s_page, p.s_slot, p.s_head};
  while (a.seg * 8 < hd) a.seg *= 2;  // lanes of a head: 8 values each
  const int64_t lanes = (heads + 2 * kvh) * a.seg;
  // a block of 256 lanes a row (512 lanes, which leave no remainder, take 66 us for
  // 8000 rows of 64 + 8 heads, 256 54); where the rows leave the chip empty, more
  // blocks share a row's heads
  a.parts = (int32_t)std::max<int64_t>(1, std::min<int64_t>((lanes + 255) / 256, 2 * c->cus / rows));
  char name[32];
  snprintf(name, sizeof name, "paged_qkrope_%s", p.type);
  return launch(c, name, dim3((unsigned)rows, (unsigned)a.parts), dim3(256), &a);
}

int ihip_enqueue_paged_attention(ihip_ctx* c, uint64_t q, int64_t q_stride, const ihip_pages* cache,
                                 uint64_t table, int64_t max_pages, uint64_t lengths, uint64_t y,
                                 int64_t seqs, int64_t heads, int64_t window, uint64_t sinks, double scale)
{
  return ihip_enqueue_paged_attention_at(c, q, q_stride, cache, table, max_pages, lengths, 0, seqs, y, seqs, heads,
                                         window, sinks, scale);
}

int ihip_enqueue_paged_attention_at(ihip_ctx* c, uint64_t q, int64_t q_stride, const ihip_pages* cache,
                                    uint64_t table, int64_t max_pages, uint64_t lengths, uint64_t offsets,
                                    int64_t rows, uint64_t y, int64_t seqs, int64_t heads, int64_t window,
                                    uint64_t sinks, double scale)
{
  return paged_attention("ihip_enqueue_paged_attention", c, q, q_stride, cache, table, max_pages, lengths, offsets, rows,
                         nullptr, y, seqs, heads, window, sinks, scale);
}

int ihip_enqueue_paged_attention_shared(ihip_ctx* c, uint64_t q, int64_t q_stride, const ihip_pages* cache,
                                        uint64_t table, int64_t max_pages, uint64_t lengths, uint64_t offsets,
                                        int64_t rows, uint64_t members, uint64_t shared, int64_t groups, uint64_t y,
                                        int64_t seqs, int64_t heads, int64_t window, uint64_t sinks, double scale)
{
  const Groups g = {members, shared, groups};
  return paged_attention("ihip_enqueue_paged_attention_shared", c, q, q_stride, cache, table, max_pages, lengths, offsets,
                         rows, &g, y, seqs, heads, window, sinks, scale);
}

int ihip_enqueue_paged_read(ihip_ctx* c, const ihip_pages* cache, uint64_t table, int64_t max_pages,
                            uint64_t first, uint64_t offsets, int64_t seqs, int64_t rows, int out_type,
                            uint64_t k_out, uint64_t v_out)
{
  const char* who = "ihip_enqueue_paged_read";
  Pool p;
  if (int rc = check_pool(who, cache, &p)) return rc;
  if (!table || !offsets || !k_out || !v_out) return refuse(who, "a missing array");
  if (out_type != IHIP_F32 && out_type != IHIP_F16) return refuse(who, "rows are F32 or F16", IHIP_E_UNSUPPORTED);
  if (seqs > IHIP_PAGED_SEQS) return refuse(who, "more sequences than IHIP_PAGED_SEQS", IHIP_E_NOMEM);
  if (seqs < 1 || rows < 1 || rows > INT32_MAX || max_pages < 1 || max_pages > INT32_MAX / cache->page_size)
    return refuse(who, "seqs, rows or max_pages out of range");
  if ((table | first | offsets) % 4) return refuse(who, "arrays aligned to 4 bytes");
  if ((k_out | v_out) % 16) return refuse(who, "rows aligned to 16 bytes");
  const int64_t hd = cache->head_dim, kvh = cache->kv_heads, width = kvh * hd, os = out_type == IHIP_F32 ? 4 : 2;
  const __int128 out = (__int128)rows * width * os;
  const __int128 held = ((__int128)(cache->pages - 1) * p.page_stride + p.slot_stride * (cache->page_size - 1) + p.head_stride * (kvh - 1) + hd) * p.es;
  const __int128 scales = held / (p.es * hd) * 4;
  auto meets = [](__int128 a, __int128 n, __int128 b, __int128 m) { return a < b + m && b < a + n; };
  bool over = meets(k_out, out, v_out, out);
  for (uint64_t o : {k_out, v_out})
    over |= meets(o, out, cache->k, held) || meets(o, out, cache->v, held) ||
            (cache->dtype == IHIP_Q8_HEAD && (meets(o, out, cache->k_scale, scales) || meets(o, out, cache->v_scale, scales)));
  if (over) return refuse(who, "rows that overlap each other or the cache");
  if (!c) return no_context(who);
  OnDevice on(c);
  struct {
    uint64_t kc, vc, ks, vs, table, first, offsets, k_out, v_out;
    int64_t pages, page_stride, slot_stride, head_stride, s_page, s_slot, s_head;
    int32_t rows, seqs, max_pages, page_size, hd, units, chunk;
  } a = {cache->k, cache->v, q8_scales(cache, 0), q8_scales(cache, 1), table, first, offsets, k_out, v_out,
         cache->pages, p.page_stride, p.slot_stride, p.head_stride, p.s_page, p.s_slot, p.s_head,
         (int32_t)rows, (int32_t)seqs, (int32_t)max_pages, cache->page_size, (int32_t)hd, (int32_t)(width * os / 16), 1};
  // a wave's rows: as many as leave 16 waves a CU, up to 16
  a.chunk = (int32_t)std::max<int64_t>(1, std::min<int64_t>(16, rows / (16 * c->cus)));
  const int64_t turns = (rows + a.chunk - 1) / a.chunk;
  char name[32];
  snprintf(name, sizeof name, "paged_read_%s_%s", p.type, out_type == IHIP_F32 ? "f32" : "f16");
  return launch(c, name, dim3((unsigned)std::min<int64_t>((turns + 3) / 4, 64 * c->cus)), dim3(256), &a);
}

int ihip_enqueue_sample_rows(ihip_ctx* c, uint64_t logits, int64_t rows, int64_t vocab, int64_t stride,
                             uint64_t settings, uint64_t uniform, uint64_t ids, uint64_t probs)
{
  const char* who = "ihip_enqueue_sample_rows";
  if (!logits || !settings || !uniform || !ids) return refuse(who, "a missing array");
  if (rows < 1 || rows > (int64_t)1 << 24 || vocab < 1 || vocab > 1 << 22)
    return refuse(who, "rows or vocab out of range");
  stride = stride ? stride : vocab;
  if (stride < vocab) return refuse(who, "a stride below a row");
  if (stride > STRIDE_MOST) return refuse(who, "a stride beyond 2^36");
  if ((logits | ids | probs) % 4) return refuse(who, "arrays aligned to 4 bytes");
  if ((settings | uniform) % 8) return refuse(who, "settings and random numbers are doubles, aligned to 8 bytes");
  // (a row's token is written while others are read)
  for (uint64_t o : {ids, probs})
    if (o && (overlaps(o, (__int128)rows * 4, logits, (__int128)stride * 4, (__int128)vocab * 4, rows) ||
              overlaps(o, (__int128)rows * 4, settings, sizeof(ihip_sampling), sizeof(ihip_sampling), rows) ||
              overlaps(o, (__int128)rows * 4, uniform, 8, 8, rows) || (o == probs && overlaps(probs, (__int128)rows * 4, ids, 4, 4, rows))))
      return refuse(who, "ids or probs overlap another array");
  if (!c) return no_context(who);
  OnDevice on(c);
  // parts of 8192 tokens, of 4096 or 2048 where they would leave the chip's CUs empty
  const int64_t most_parts = rows * ((vocab + 8191) / 8192);
  const int64_t per = most_parts < 2 * c->cus ? 2048 : most_parts < 8 * c->cus ? 4096 : 8192;
  const int64_t parts = (vocab + per - 1) / per, chunks = (vocab + 255) / 256;
  // a row's results: a double, two words and 32 octaves a part, a word a chunk, its sums
  const int64_t bytes = parts * (8 + 8 + 32 * 4) + chunks * 4 + 24;
  const int64_t most = std::min<int64_t>({rows, 65535, (int64_t)(SAMPLE_ROWS_BYTES / bytes)});
  struct {
    const float* x;
    int64_t stride;
    const ihip_sampling* settings;
    const double* uniform;
    int* ids;
    float* probs;
    float* best;
    int* best_id;
    double* sum;
    uint32_t* octaves;
    float* chunk;
    uint64_t row;
    int* heavy;
    uint64_t bins, found;
    int32_t rows, vocab, parts, chunks, wide, per;
  } a = {};
  a.stride = stride;
  a.bins = c->sample_rows;
  a.found = a.bins + SAMPLE_HEAVY * SAMPLE_BINS * 8;
  a.row = a.bins + SAMPLE_HEAVY_BYTES;
  a.sum = (double*)(a.row + 24 * most);
  a.heavy = (int*)(c->sample_rows + SAMPLE_HEAVY_BYTES + SAMPLE_ROWS_BYTES);
  a.best = (float*)(a.sum + most * parts);
  a.best_id = (int*)(a.best + most * parts);
  a.octaves = (uint32_t*)(a.best_id + most * parts);
  a.chunk = (float*)(a.octaves + most * parts * 32);
  a.vocab = (int32_t)vocab;
  a.parts = (int32_t)parts;
  a.chunks = (int32_t)chunks;
  a.wide = logits % 16 == 0 && stride % 4 == 0;
  a.per = (int32_t)per;
  for (int64_t r = 0; r < rows; r += most) {
    const int64_t n = std::min<int64_t>(rows - r, most);
    a.x = (const float*)logits + r * stride;
    a.settings = (const ihip_sampling*)settings + r;
    a.uniform = (const double*)uniform + r;
    a.ids = (int*)ids + r;
    a.probs = probs ? (float*)probs + r : nullptr;
    a.rows = (int32_t)n;
    int rc = launch(c, per == 2048 ? "sample_rows_part_2048" : per == 4096 ? "sample_rows_part_4096" : "sample_rows_part_8192", dim3((unsigned)parts, (unsigned)n),
                    dim3(256), &a);
    if (!rc) rc = launch(c, "sample_rows_finish", dim3((unsigned)n), dim3(256), &a);
    for (const char* heavy : {"sample_rows_bins", "sample_rows_find"})
      if (!rc) rc = launch(c, heavy, dim3((unsigned)c->cus), dim3(256), &a);
    if (!rc) rc = launch(c, a.wide ? "sample_rows_pick_wide" : "sample_rows_pick", dim3((unsigned)n), dim3(512), &a);
    if (rc) return rc;
  }
  return 0;
}

int ihip_enqueue_logprobs(ihip_ctx* c, uint64_t logits, int64_t rows, int64_t vocab, int64_t stride,
                          uint64_t ids, uint64_t logprobs, uint64_t entropy, int64_t k,
                          uint64_t top_ids, uint64_t top_logprobs)
{
  const char* who = "ihip_enqueue_logprobs";
  if (k < 0 || k > IHIP_LOGPROBS_TOP) return refuse(who, "more alternatives than IHIP_LOGPROBS_TOP", IHIP_E_NOMEM);
  if (!logits || (logprobs && !ids) || (k && (!top_ids || !top_logprobs)) || (!logprobs && !entropy && !k))
    return refuse(who, "a missing array");
  if (rows < 1 || rows > INT32_MAX || vocab < 1 || vocab > 1 << 22)
    return refuse(who, "rows or vocab out of range");
  stride = stride ? stride : vocab;
  if (stride < vocab) return refuse(who, "a stride below a row");
  if (stride > STRIDE_MOST || rows > (int64_t)1 << 24) return refuse(who, "rows beyond 2^24 or a stride beyond 2^36");
  if ((logits | ids | logprobs | entropy | top_ids | top_logprobs) % 4)
    return refuse(who, "arrays aligned to 4 bytes");
  if (!c) return no_context(who);
  OnDevice on(c);
  // The rows' parts: blocks for the whole chip (2048 instead of 1024: 61 rows of
  // 201088 35.9 us, 26.1), but no part so short that its first tile and its list cost
  // more than the blocks gain: 4096 logits for a few rows, 8192 from 16 rows (16 of
  // 151936 in 37 parts 16.9 us, in 18 16.5), 24576 from 256 (512 of 32000 in two parts
  // 29.5, in one 25.6; 300 of 151936 in one 57.3, in three 47.6)
  int64_t parts = 1;
  if (rows < LOGPROBS_BLOCKS) {
    const int64_t least = rows < 16 ? 4096 : rows < 256 ? 8192 : 24576;
    parts = std::max<int64_t>(1, std::min<int64_t>(vocab / least, LOGPROBS_BLOCKS / rows));
  }
  struct {
    const float* x;
    int64_t stride;
    const int* ids;
    float *logprobs, *entropy;
    int* top_ids;
    float* top_logprobs;
    double* part;
    int* done;
    int32_t rows, vocab, k, parts;
  } a = {(const float*)logits, stride, (const int*)ids, (float*)logprobs, (float*)entropy,
         (int*)top_ids, (float*)top_logprobs, (double*)c->logprobs_part,
         (int*)(c->logprobs_part + LOGPROBS_PART_BYTES), (int32_t)rows, (int32_t)vocab, (int32_t)k,
         (int32_t)parts};
  // rows in a grid's y, 65535 a launch
  for (int64_t r = 0; r < rows; r += 65535) {
    const int64_t n = std::min<int64_t>(rows - r, 65535);
    auto b = a;
    b.x += r * stride;
    if (ids) b.ids += r;
    if (logprobs) b.logprobs += r;
    if (entropy) b.entropy += r;
    if (k) {
      b.top_ids += r * k;
      b.top_logprobs += r * k;
    }
    if (int rc = launch(c, "logprobs", dim3((unsigned)parts, (unsigned)n), dim3(256), &b)) return rc;
  }
  return 0;
}

}  // extern "C"
