// fa_paged.h - kernel argument blocks of the paged key-value cache, shared by the C ABI (fa_paged.cpp) and the kernels.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fa_paged_plan.h"

namespace fa {

// The cache as the kernels read it.  Strides are in bytes; offsets are formed in 64 bits.
struct PagedCache {
  uint8_t* k;
  uint8_t* v;
  int64_t sk[3], sv[3];   // page, head, slot
  const int* table;       // [B][table_width], rows table_stride entries apart
  const int* lens;
  int64_t table_stride;
  int B, pages, page_size, table_width, Hkv;
  int max_len;            // lens are cut off here; at most table_width * page_size
  PageDiv div;
};

struct AppendArgs {
  PagedCache c;
  const uint8_t* k;
  const uint8_t* v;
  int64_t sk[2], sv[2];   // head, row
  const int* cu;          // NULL: row b belongs to sequence b
  int rows;
  float k_inv, v_inv;     // e4m3 pages: reciprocals of the descales
};

// Two tiles of heads and their sums fit a wave's registers: more than 16 heads a group then share what is read.
constexpr bool paged_pairs(int D, int cache_bytes) { return cache_bytes <= 2 && D * cache_bytes <= 128; }
// A wave of a workgroup of 8 has 256 registers: no room for two tiles of heads with D = 128, nor for 16-bit and
// float32 rows of that.
constexpr bool paged_eight(int D, int cache_bytes, int rt) {
  return cache_bytes == 4 ? D <= 64 : D * cache_bytes <= 128 && (D <= 64 || rt == 1);
}

struct PagedAttnArgs {
  PagedCache c;
  const uint8_t* q;
  uint8_t* o;
  int64_t sq[2], so[2];   // batch, head
  const float* sinks;     // NULL, or [Hq] learned logits
  float* sums;            // NULL, or accumulated weights [B][Hkv][max_len]
  int64_t ssum[2];
  int Hq, G, row_tiles;   // heads a group, tiles of 16 heads in it
  int W, S;
  float c2;               // softmax scale * log2(e) * K's descale: scores are exp2(c2 * q.k)
  float oscale;           // V's descale
  int max_units;          // units of a sequence of max_len tokens
  // split calls: the runs a (KV head, row tile) is cut into, 0 where every workgroup takes a whole sequence
  int parts, least;
  int few, many_units;    // calls of at most many_units units use the first `few` of the parts only
  int waves;              // of a workgroup: 1 (only with rt = 1), 4 or 8 (paged_eight)
  int rt;                 // tiles of heads that a workgroup takes: 1, or 2 (paged_pairs)
  int keep_units;         // calls that read more units a KV head than this mark their loads as read once
  // workspace
  int* starts;            // split calls: [B] the sequences' first units, and the units of a part
  float* part_o;          // [Hkv row_tiles][parts][2][16][D]
  float* part_ml;         // [Hkv row_tiles][parts][2][2][16]: what weights were taken against (log2 domain), their sum
  float* norm;            // with sums: [B][Hq] the same and 1 / sum, of the sequences that one workgroup took whole
  float* logits;          // with sums: [Hkv][B][max_units][G][kPagedUnit] (log2 domain)
};

constexpr int kGatherPieces = 512;  // 16-byte pieces of K, and of V, that a workgroup of the gather moves

constexpr int kSelectState = 8;     // numbers that a workgroup of the selection hands on to the next launch

struct EvictArgs {
  PagedCache c;
  const float* sums;
  float* new_sums;
  int64_t ssum[2], snew[2];
  int sums_width;
  const int* new_table;
  int64_t new_table_stride;
  int* new_lens;
  int keep, S, R;
  int each, chunks;       // chunks of 1024 each entries, a (sequence, KV head); each is 4, 8 or 16
  // workspace
  int* kept;              // [B][Hkv][keep] entries kept, in order
  int* state;             // with several chunks: [B][Hkv][chunks][kSelectState]
  uint16_t* counts;       // with several chunks: [B][Hkv][3 digits][chunks][2048]
};

// dtype and cache are fa_dtype values
hipError_t launch_paged_append(const AppendArgs& a, int dtype, int cache, int D, hipStream_t s);
hipError_t launch_paged_attention(const PagedAttnArgs& a, int dtype, int cache, int D, hipStream_t s);
// row_bytes: of a head's entry
hipError_t launch_paged_evict(const EvictArgs& a, int row_bytes, hipStream_t s);

}  // namespace fa
