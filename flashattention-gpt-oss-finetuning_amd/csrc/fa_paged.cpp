// fa_paged.cpp - the C ABI of the paged key-value cache (include/fa_gfx950.h): host-side validation, workspace sizing and
// launch shapes.  Nothing is launched and no HIP call made before the arguments have been checked.
#include <algorithm>
#include <cmath>
#include <cstdint>

#include "../../include/fa_gfx950.h"
#include "fa_args.h"
#include "fa_paged.h"

namespace {

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
bool strides_ok(const int64_t* s, int n, int elem_bytes) {
  for (int i = 0; i < n; ++i)
    if (s[i] < 0 || (s[i] & (16 / elem_bytes - 1)) != 0) return false;
  return true;
}
int elem_bytes(int32_t dtype) { return dtype == FA_DTYPE_F32 ? 4 : dtype == FA_DTYPE_FP8_E4M3 ? 1 : 2; }
size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

int check_cache(const fa_paged_cache& c) {
  if (!c.k || !c.v || !c.table || !c.lens) return FA_ERR_NULL;
  if (c.batch < 1 || c.heads_kv < 1) return FA_ERR_SHAPE;
  if (c.pages < 1 || c.page_size < 1 || c.table_width < 1) return FA_ERR_PAGES;
  const int D = c.head_dim;
  if (D != 16 && D != 32 && D != 64 && D != 128) return FA_ERR_HEAD_DIM;
  if (c.dtype < FA_DTYPE_BF16 || c.dtype > FA_DTYPE_F32) return FA_ERR_DTYPE;
  const int eb = elem_bytes(c.dtype);
  if (eb == 1 && D < 64) return FA_ERR_HEAD_DIM;
  if (!aligned(c.k, 16) || !aligned(c.v, 16) || !aligned(c.table, 4) || !aligned(c.lens, 4) || c.table_stride < 0 ||
      !strides_ok(c.k_stride, 3, eb) || !strides_ok(c.v_stride, 3, eb))
    return FA_ERR_ALIGN;
  if (int64_t(c.table_width) * c.page_size >= fa::kPagedMaxTokens || c.heads_kv >= 1 << 24) return FA_ERR_OVERFLOW;
  return FA_OK;
}

// a call's element type against its cache's
bool types_ok(int32_t dtype, int32_t cache) {
  if (dtype != FA_DTYPE_BF16 && dtype != FA_DTYPE_F16 && dtype != FA_DTYPE_F32) return false;
  return cache == dtype || (cache == FA_DTYPE_FP8_E4M3 && dtype != FA_DTYPE_F32);
}

fa::PagedCache cache_args(const fa_paged_cache& c) {
  fa::PagedCache r{};
  const int eb = elem_bytes(c.dtype);
  r.k = static_cast<uint8_t*>(c.k);
  r.v = static_cast<uint8_t*>(c.v);
  for (int i = 0; i < 3; ++i) {
    r.sk[i] = c.k_stride[i] * eb;
    r.sv[i] = c.v_stride[i] * eb;
  }
  r.table = c.table;
  r.lens = c.lens;
  r.table_stride = c.table_stride;
  r.B = c.batch;
  r.pages = c.pages;
  r.page_size = c.page_size;
  r.table_width = c.table_width;
  r.Hkv = c.heads_kv;
  r.max_len = c.table_width * c.page_size;
  r.div = fa::page_div(uint32_t(c.page_size));
  return r;
}

int status(hipError_t e) { return e == hipSuccess ? FA_OK : FA_ERR_LAUNCH; }

// Which launch serves a call.  Sequences that see at most whole_keys() keys are taken whole, a workgroup each, in one launch; twice
// as many where there are kManyWgs (KV head, share of its heads, sequence) triples.  Ragged batches are no reason to split here: the
// bound is what the longest can be.  Times in us, whole / split, with 8 KV heads and D = 64 (4 and D = 128):
//   bf16: 1 sequence of 1001 tokens 9.1 / 9.8, of 1500 11.0 / 9.7, of 2048 12.9 / 9.8; 4 of 2048 14.2 / 12.4;
//     16 (128 workgroups) of 1500 13.3 / 19.2, of 2048 15.9 / 21.4; 64 (512 workgroups) of 2048 51.7 / 54.1, of 4096 98 / 96
//   bf16 D = 128: 1 of 600 10.1 / 9.9, of 1000 13.8 / 10.0; 16 (64 workgroups) of 700 12.6 / 18.8, of 1000 15.0 / 19.5
//   e4m3: 8 (64 workgroups) of 1500 10.2 / 11.4, of 2000 12.2 / 11.4; 16 of 2000 12.9 / 14.5
//   e4m3 D = 128: 1 of 600 8.0 / 9.2, of 1000 10.4 / 9.3; 16 (64 workgroups) of 1000 10.8 / 11.6, of 1500 14.1 / 13.2
//   float32: 1 of 600 12.6 / 10.0 (the lines cross at about 380); 8 (64 workgroups) of 500 11.2 / 10.7; 16 of 500 11.9 / 13.3
//   float32 D = 128: 1 of 600 21.6 / 12.4; 16 (64 workgroups) of 400 18.8 / 14.2
//   64 heads over one, bf16: 1 of 600 9.5 / 10.6, of 1000 11.9 / 10.4; 16 of 1000 12.5 / 12.6, of 1500 15.4 / 16.3
int whole_keys(int D, int cache_bytes) {
  return cache_bytes == 4 ? (D > 64 ? 128 : 256) : D * cache_bytes > 128 ? 512 : D > 64 ? 768 : 1024;
}
constexpr int kManyWgs = 64;
// Whole sequences are taken by 8 waves while there are at most as many workgroups as compute units (1 sequence of 1001
// tokens: 10.5 us with 4 waves, 9.1 with 8; but 64 of 256: 9.8 and 12.5), and by a wave each where there are kSingleWgs of at
// most kSingleUnits units (256 sliding-layer sequences 20.9 us with 4 waves, 15.6 with one; 1024 of them 83 and 62).
constexpr int kSingleWgs = 1024, kSingleUnits = 2;
// Split calls: workgroups for each compute unit.  With 1 / 2 / 3 of them 32 ragged sequences (261 MB) take 53 / 49 / 55 us, e4m3
// D = 128 (123 MB) 27 / 25 / 29, four of up to 128K tokens (876 MB) 158 / 149 / 150.  Rows of 32 bytes make a tile as much work for a
// quarter of the bytes: 137 us with 2, 113 with 3 (537 MB).  A unit more a workgroup costs a short call more than its piece
// does (1 sequence of 2048 tokens: 10.3 us with at least two units each, 9.8 with one).
constexpr int kPartsPerCu = 2, kPartsNarrow = 3, kLeastUnits = 1;
// Where a page has its slots before its heads, the workgroups of a part's KV heads read neighbouring pieces of the same rows, and
// twice as many and shorter runs keep them closer together, once the call is large.  With 2 / 4 a compute unit (bf16, 8 heads of
// D = 64): 261 MB 49 / 49 us, 342 MB 65.6 / 65.0, 420 MB 79.6 / 77.2, 502 MB 95 / 92, 876 MB 158 / 150; the second launch takes 0.3 more.
// So the second half of the parts is used above kManyBytes of K and V, and where a slot's row has kManyRow bytes at least, in
// entries of kManyEntry at most (about 700 MB): 16 heads of D = 64 281 / 236, of D = 32 180 / 163, 32 of D = 16 286 / 272; e4m3 16 heads of D = 64
// 181 / 163, 8 of D = 128 136 / 129; float32 8 heads of D = 32 141 / 130.  Shorter rows: 4 heads of D = 64 135 / 138, 8 of D = 32 173 / 190, 16 of
// D = 16 309 / 341, 2 of D = 32 229 / 261; e4m3 8 heads of D = 64 168 / 175.  Longer entries, of which a compute unit has fewer workgroups at a
// time: D = 128, 4 heads 92 / 99 (502 MB), 8 heads 244 / 247; float32 4 heads of D = 128 245 / 264, of D = 64 130 / 127.
constexpr int64_t kManyBytes = int64_t(384) << 20;
constexpr int kManyRow = 1024, kManyEntry = 128;
// Loads of a call that reads more than this are marked as read once, so that they do not run through the 256 MB last-level
// cache: 537 MB take 90 us so and 100 otherwise, 261 MB 49 and 54.  Below, the next step finds the keys there: three caches of 71 MB
// in turn take 18.1 us each, 19.8 with marked loads.
constexpr int64_t kKeepBytes = int64_t(96) << 20;

// K and V bytes of a unit of keys, all KV heads.
int64_t unit_bytes(const fa_paged_cache& c) {
  return int64_t(fa::kPagedUnit) * 2 * c.head_dim * elem_bytes(c.dtype) * c.heads_kv;
}

struct Plan {
  int max_units, row_tiles, rt, parts, few, many_units;
  size_t starts, part_o, part_ml, norm, logits;  // bytes
  size_t bytes() const { return std::max<size_t>(256, starts + part_o + part_ml + norm + logits); }
};

int plan(const fa_paged_attention_params* p, Plan* r) {
  if (!p) return FA_ERR_NULL;
  const fa_paged_cache& c = p->cache;
  const int rc = check_cache(c);
  if (rc != FA_OK) return rc;
  if (!p->q || !p->o) return FA_ERR_NULL;
  if (p->heads_q < 1 || p->heads_q % c.heads_kv != 0 || p->max_len < 1) return FA_ERR_SHAPE;
  if (!types_ok(p->dtype, c.dtype)) return FA_ERR_DTYPE;
  if (p->window < 1 && p->sink < 1) return FA_ERR_MASK;
  const bool q8 = c.dtype == FA_DTYPE_FP8_E4M3;
  if (!std::isfinite(p->softmax_scale) || (q8 && (!std::isfinite(float(p->softmax_scale * c.k_descale)) || !std::isfinite(float(c.v_descale)))))
    return FA_ERR_SCALE;
  const int eb = elem_bytes(p->dtype);
  if (!aligned(p->q, 16) || !aligned(p->o, 16) || !strides_ok(p->q_stride, 2, eb) || !strides_ok(p->o_stride, 2, eb) ||
      !aligned(p->sinks, 4) || !aligned(p->weight_sums, 4))
    return FA_ERR_ALIGN;
  const int max_len = int(std::min<int64_t>(int64_t(c.table_width) * c.page_size, p->max_len));
  if (p->weight_sums) {
    if (p->sums_stride[0] < 0 || p->sums_stride[1] < 0) return FA_ERR_ALIGN;
    if (p->sums_width < max_len) return FA_ERR_PAGES;
  }
  const int64_t most = std::min<int64_t>(max_len, int64_t(std::max(p->window, 0)) + std::max(p->sink, 0));
  const int G = p->heads_q / c.heads_kv;
  r->max_units = fa::paged_units(int(most));
  r->row_tiles = (G + 15) / 16;
  r->rt = r->row_tiles > 1 && fa::paged_pairs(c.head_dim, elem_bytes(c.dtype)) ? 2 : 1;
  const int64_t streams = int64_t(c.heads_kv) * ((r->row_tiles + r->rt - 1) / r->rt), units = int64_t(c.batch) * r->max_units;
  if (units >= (int64_t(1) << 30) || !fa::grid_fits(std::max(streams, int64_t(p->heads_q)) * c.batch)) return FA_ERR_OVERFLOW;
  r->parts = r->few = r->many_units = 0;
  if (most > whole_keys(c.head_dim, elem_bytes(c.dtype)) * (streams * c.batch >= kManyWgs ? 2 : 1)) {
    const int64_t want = std::max<int64_t>(1, int64_t(c.head_dim * elem_bytes(c.dtype) <= 32 ? kPartsNarrow : kPartsPerCu) * fa::device_cus() / streams);
    // (whole rounds of the 8 XCDs: the workgroups of a part, which read the same or neighbouring entries, then share an L2; pages
    // with the slots before the heads, 876 MB: 166 us with a KV head an XCD, 158 so)
    r->parts = int((std::min(want, (units + kLeastUnits - 1) / kLeastUnits) + 7) / 8 * 8);
    r->few = r->parts;
    r->many_units = int(std::min<int64_t>(kManyBytes / unit_bytes(c), INT32_MAX));
    const int64_t entry = int64_t(c.head_dim) * elem_bytes(c.dtype);
    if (c.k_stride[1] < c.k_stride[2] && entry <= kManyEntry && entry * c.heads_kv >= kManyRow && units > r->many_units) r->parts *= 2;
    if (!fa::grid_fits(streams * r->parts)) return FA_ERR_OVERFLOW;
  }
  const size_t slots = size_t(c.heads_kv) * r->row_tiles * r->parts * 2;
  r->starts = r->parts ? align256((size_t(c.batch) + 1) * sizeof(int32_t)) : 0;
  r->part_o = align256(slots * 16 * c.head_dim * sizeof(float));
  r->part_ml = align256(slots * 32 * sizeof(float));
  r->norm = r->logits = 0;
  if (p->weight_sums) {
    r->norm = align256(size_t(c.batch) * p->heads_q * 2 * sizeof(float));
    r->logits = align256(size_t(units) * p->heads_q * fa::kPagedUnit * sizeof(float));
    // (the second launch: a workgroup a query head, and one for each 1024 keys of a (sequence, KV head))
    if (!fa::grid_fits((p->heads_q + int64_t(r->max_units + 7) / 8 * c.heads_kv) * c.batch)) return FA_ERR_OVERFLOW;
  }
  return FA_OK;
}

// Weights that a thread of the selection holds.  Up to 16384 entries one workgroup takes a (sequence, KV head) in one launch.  More
// are cut into chunks: the smallest that leave a CU one workgroup, for each reads the counts of all chunks of its head.  With 4 / 8 /
// 16 (whole evictions): 8 heads of 32000 entries 29 / 34 / 40 us, 8 of 131071 42 / 42 / 48, 64 of 50000 116 / 82 / 65, 128 of 32000
// 104 / 80 / 66, 240 of 50000 372 / 276 / 241.
int select_each(int64_t heads, int64_t tokens) {
  if (tokens <= 16384) return tokens <= 4096 ? 4 : tokens <= 8192 ? 8 : 16;
  for (int each = 4; each < 16; each *= 2)
    if ((tokens + 1024 * each - 1) / (1024 * each) <= 256 / heads) return each;
  return 16;
}

// An eviction's launches and the bytes of its workspace.
struct EvictRoom {
  int each, chunks;
  size_t kept, state, counts;
};
EvictRoom evict_room(int64_t heads, int32_t keep, int64_t tokens) {
  EvictRoom r{};
  r.each = select_each(heads, tokens);
  r.chunks = int((tokens + 1024 * r.each - 1) / (1024 * r.each));
  r.kept = align256(size_t(heads) * keep * sizeof(int32_t));
  if (r.chunks > 1) {
    r.state = align256(size_t(heads) * r.chunks * fa::kSelectState * sizeof(int32_t));
    r.counts = align256(size_t(heads) * r.chunks * 3 * 2048 * sizeof(uint16_t));
  }
  return r;
}

// The tokens that a sequence can have in an eviction.
int64_t evict_tokens(const fa_paged_evict_params* p) {
  const int64_t table = int64_t(p->cache.table_width) * p->cache.page_size;
  return p->max_len > 0 ? std::min<int64_t>(table, p->max_len) : table;
}

// Everything of an eviction but its workspace.
int check_evict(const fa_paged_evict_params* p, EvictRoom* room) {
  if (!p) return FA_ERR_NULL;
  const fa_paged_cache& c = p->cache;
  const int rc = check_cache(c);
  if (rc != FA_OK) return rc;
  if (!p->sums || !p->new_sums || !p->new_table || !p->new_lens) return FA_ERR_NULL;
  if (p->max_len < 0) return FA_ERR_SHAPE;
  const int64_t tokens = evict_tokens(p);
  if (p->keep < 1 || p->sink < 0 || p->recent < 0 || int64_t(p->sink) + p->recent > p->keep || p->sums_width < tokens ||
      p->new_table_width < 1 || int64_t(p->new_table_width) * c.page_size < p->keep)
    return FA_ERR_PAGES;
  const int64_t heads = int64_t(c.batch) * c.heads_kv;
  if (p->keep >= fa::kPagedMaxTokens || !fa::grid_fits(heads)) return FA_ERR_OVERFLOW;
  if (!aligned(p->sums, 4) || !aligned(p->new_sums, 4) || !aligned(p->new_table, 4) || !aligned(p->new_lens, 4) ||
      p->new_table_stride < 0)
    return FA_ERR_ALIGN;
  for (int i = 0; i < 2; ++i)
    if (p->sums_stride[i] < 0 || p->new_sums_stride[i] < 0) return FA_ERR_ALIGN;
  // workgroups of the launches: 1024 threads a chunk, and one for each kGatherPieces of kept entries
  const int64_t chunk = fa::kGatherPieces / (c.head_dim * elem_bytes(c.dtype) / 16);
  *room = evict_room(heads, p->keep, tokens);
  if (!fa::grid_fits(heads * room->chunks, 1024) || !fa::grid_fits(heads * ((p->keep + chunk - 1) / chunk))) return FA_ERR_OVERFLOW;
  return FA_OK;
}

}  // namespace

extern "C" {

int fa_paged_append(const fa_paged_cache* c, const void* k, const void* v, const int64_t k_stride[2],
                    const int64_t v_stride[2], int32_t rows, int32_t dtype, const int32_t* cu_seqlens, void* stream) {
  if (!c || !k_stride || !v_stride) return FA_ERR_NULL;
  const int rc = check_cache(*c);
  if (rc != FA_OK) return rc;
  if (rows < 0 || (!cu_seqlens && rows != c->batch)) return FA_ERR_SHAPE;
  if (!types_ok(dtype, c->dtype)) return FA_ERR_DTYPE;
  const int eb = elem_bytes(dtype);
  if (!aligned(k, 16) || !aligned(v, 16) || !aligned(cu_seqlens, 4) || !strides_ok(k_stride, 2, eb) || !strides_ok(v_stride, 2, eb))
    return FA_ERR_ALIGN;
  fa::AppendArgs a{};
  if (c->dtype == FA_DTYPE_FP8_E4M3) {
    a.k_inv = float(1.0 / c->k_descale);
    a.v_inv = float(1.0 / c->v_descale);
    if (!std::isfinite(c->k_descale) || !std::isfinite(c->v_descale) || !std::isfinite(a.k_inv) || !std::isfinite(a.v_inv))
      return FA_ERR_SCALE;
  }
  if (rows == 0) return FA_OK;
  if (!k || !v) return FA_ERR_NULL;
  a.c = cache_args(*c);
  a.k = static_cast<const uint8_t*>(k);
  a.v = static_cast<const uint8_t*>(v);
  for (int i = 0; i < 2; ++i) {
    a.sk[i] = k_stride[i] * eb;
    a.sv[i] = v_stride[i] * eb;
  }
  a.cu = cu_seqlens;
  a.rows = rows;
  if (!fa::grid_fits((int64_t(rows) + 3) / 4)) return FA_ERR_OVERFLOW;
  return status(fa::launch_paged_append(a, dtype, c->dtype, c->head_dim, static_cast<hipStream_t>(stream)));
}

size_t fa_paged_workspace_bytes(const fa_paged_attention_params* p) {
  Plan r;
  return plan(p, &r) == FA_OK ? r.bytes() : 0;
}

int fa_paged_attention(const fa_paged_attention_params* p, void* workspace, size_t workspace_bytes, void* stream) {
  Plan r;
  const int rc = plan(p, &r);
  if (rc != FA_OK) return rc;
  if (!workspace || !aligned(workspace, 256) || workspace_bytes < r.bytes()) return FA_ERR_WORKSPACE;
  const fa_paged_cache& c = p->cache;
  const bool q8 = c.dtype == FA_DTYPE_FP8_E4M3;
  fa::PagedAttnArgs a{};
  a.c = cache_args(c);
  a.c.max_len = std::min(a.c.max_len, p->max_len);
  a.q = static_cast<const uint8_t*>(p->q);
  a.o = static_cast<uint8_t*>(p->o);
  const int eb = elem_bytes(p->dtype);
  for (int i = 0; i < 2; ++i) {
    a.sq[i] = p->q_stride[i] * eb;
    a.so[i] = p->o_stride[i] * eb;
    a.ssum[i] = p->sums_stride[i];
  }
  a.sinks = p->sinks;
  a.sums = p->weight_sums;
  a.Hq = p->heads_q;
  a.G = p->heads_q / c.heads_kv;
  a.row_tiles = r.row_tiles;
  a.rt = r.rt;
  a.W = std::min(std::max(p->window, 0), a.c.max_len);
  a.S = std::min(std::max(p->sink, 0), a.c.max_len);
  a.c2 = float(double(p->softmax_scale) * 1.4426950408889634 * (q8 ? c.k_descale : 1.0));
  a.oscale = q8 ? float(c.v_descale) : 1.f;
  a.max_units = r.max_units;
  a.parts = r.parts;
  a.few = r.few;
  a.many_units = r.many_units;
  a.least = kLeastUnits;
  const int64_t wgs = int64_t(c.heads_kv) * ((r.row_tiles + r.rt - 1) / r.rt) * c.batch;
  if (r.parts) a.waves = 4;
  else if (wgs <= fa::device_cus() && fa::paged_eight(c.head_dim, elem_bytes(c.dtype), r.rt)) a.waves = 8;
  else a.waves = r.rt == 1 && wgs >= kSingleWgs && r.max_units <= kSingleUnits ? 1 : 4;
  a.keep_units = int(std::min<int64_t>(kKeepBytes / unit_bytes(c), INT32_MAX));
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  a.starts = reinterpret_cast<int*>(ws);
  a.part_o = reinterpret_cast<float*>(ws += r.starts);
  a.part_ml = reinterpret_cast<float*>(ws += r.part_o);
  a.norm = reinterpret_cast<float*>(ws += r.part_ml);
  a.logits = reinterpret_cast<float*>(ws += r.norm);
  return status(fa::launch_paged_attention(a, p->dtype, c.dtype, c.head_dim, static_cast<hipStream_t>(stream)));
}

size_t fa_paged_evict_workspace_bytes(int32_t batch, int32_t heads_kv, int32_t keep, int32_t tokens) {
  if (batch < 1 || heads_kv < 1 || keep < 1 || tokens < 1) return 0;
  const EvictRoom r = evict_room(int64_t(batch) * heads_kv, keep, tokens);
  return r.kept + r.state + r.counts;
}

int fa_check_paged_evict(const fa_paged_evict_params* p) {
  EvictRoom room;
  return check_evict(p, &room);
}

int fa_paged_evict(const fa_paged_evict_params* p, void* workspace, size_t workspace_bytes, void* stream) {
  EvictRoom room;
  const int rc = check_evict(p, &room);
  if (rc != FA_OK) return rc;
  const fa_paged_cache& c = p->cache;
  if (!workspace || !aligned(workspace, 256) || workspace_bytes < room.kept + room.state + room.counts) return FA_ERR_WORKSPACE;
  fa::EvictArgs a{};
  a.c = cache_args(c);
  a.c.max_len = int(evict_tokens(p));
  a.sums = p->sums;
  a.new_sums = p->new_sums;
  for (int i = 0; i < 2; ++i) {
    a.ssum[i] = p->sums_stride[i];
    a.snew[i] = p->new_sums_stride[i];
  }
  a.sums_width = p->sums_width;
  a.new_table = p->new_table;
  a.new_table_stride = p->new_table_stride;
  a.new_lens = p->new_lens;
  a.keep = p->keep;
  a.S = p->sink;
  a.R = p->recent;
  a.each = room.each;
  a.chunks = room.chunks;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  a.kept = reinterpret_cast<int*>(ws);
  a.state = reinterpret_cast<int*>(ws + room.kept);
  a.counts = reinterpret_cast<uint16_t*>(ws + room.kept + room.state);
  return status(fa::launch_paged_evict(a, c.head_dim * elem_bytes(c.dtype), static_cast<hipStream_t>(stream)));
}

}  // extern "C"
