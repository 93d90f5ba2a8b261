// fa_paged_cache.hip - what fills and thins out a paged key-value cache: new rows (fa_paged_append) and eviction by
// accumulated attention weight (fa_paged_evict).  Copies and a selection: memory bounds all of them.
//
// paged_append_kernel.  Row i of sequence b's n new rows goes to position lens[b] - n + i.  A wave takes a row: it finds the
// row's sequence by one ballot over cu_seqlens and the page once, then its lanes copy the 16-byte pieces of
// every head's K and V: a prompt of 16384 rows (67 MB moved) 13.0 us, 5.2 TB/s; into e4m3 pages, D = 128 (35 MB), 10.6; a
// decoding step of 64 rows 3.1, all latency.  Two rows a wave gained nothing (12.6, 11.2, 4.0, with 12.7, 10.5, 2.8 for one).  Rows of few
// pieces leave lanes idle: 16384 rows of one head, 8 MB with D = 64 and 4 with D = 32, take 7 us either way.  e4m3 pages get
// the codes of clamp(x * fl32(1 / descale), -448, 448), as quantize_fp8's.
//
// paged_select_kernel.  Of a (sequence, KV head)'s n entries the first S and the last R stay, and of the others the
// keep - S - R of the largest weight, the lower index first among equals (NaN counts as the largest).  Entries on no page are
// none of the sequence's: attention masks them, and a kept one would get a place that it cannot fill.  One look over the
// sequence's row of the table (1 us in the first launch) says whether there are any; only then are those on pages counted.  The weights are
// mapped to unsigned numbers of the same order; three digits of them, from the top, find the smallest one that stays and
// how many equal to it do; then the entries that stay are numbered in order.  8 sequences of up to 8192 tokens, 8 heads:
// 11.7 us, barriers and dependent steps on 64 of 256 compute units; one of 131071: four launches, 31.5 us in all.
// paged_gather_kernel.  Entry r of those kept goes to position r on the pages of the new table.  Those are other pages
// than the old ones, so no entry is read after it is overwritten and all are copied at once: 2048 entries of 8 sequences
// (66 MB moved) 13.5 us, 4.9 TB/s, a large copy's rate being 4.9.
#include <hip/hip_runtime.h>

#include "../../include/fa_gfx950.h"
#include "fa_common.h"
#include "fa_paged.h"

namespace fa {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ int seq_len(const PagedCache& c, int b) { return imin(imax(c.lens[b], 0), c.max_len); }

// ---- append ------------------------------------------------------------------------------------
constexpr float kE4m3Max = 448.f;

// Source elements of 16 bytes as float32.
struct SrcBF16 {
  static __device__ __forceinline__ float get(u32x4 v, int i) {
    const uint32_t w = v[i / 2];
    return BF16::to_f32(uint16_t(i % 2 ? w >> 16 : w));
  }
};
struct SrcF16 {
  static __device__ __forceinline__ float get(u32x4 v, int i) {
    const uint32_t w = v[i / 2];
    return F16::to_f32(uint16_t(i % 2 ? w >> 16 : w));
  }
};

// Eight codes.  The conversion gives every NaN the code 0xff; a NaN keeps its sign, as in quantize_fp8.
template <typename T>
__device__ __forceinline__ u32x2 encode8(u32x4 x, float inv) {
  float f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = T::get(x, i) * inv;
  auto clamp = [](float a) { return a < -kE4m3Max ? -kE4m3Max : a > kE4m3Max ? kE4m3Max : a; };
  u32x2 o;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(clamp(f[4 * w]), clamp(f[4 * w + 1]), 0, false);
    o[w] = uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(clamp(f[4 * w + 2]), clamp(f[4 * w + 3]), lo, true));
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (f[i] != f[i]) o[i / 4] ^= (~__builtin_bit_cast(uint32_t, f[i]) >> 31) << (8 * (i % 4) + 7);
  return o;
}

// The sequence of packed row `row` (cu: [B + 1] offsets) and how many of the sequence's rows lie behind it, or -1 where the
// row is no sequence's: the first b with cu[b + 1] > row, by ballots that narrow the range to a 64th.  Every lane of the
// wave calls.
__device__ __forceinline__ int row_seq(const int* cu, int B, int row, int& behind) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = B;  // it is among sequences [lo, lo + n)
  while (true) {
    const int step = (n + 63) / 64, at = imin(n, (lane + 1) * step);
    const int end = cu[lo + at];  // the end of the last sequence of the lane's share
    const unsigned long long m = __ballot(end > row);
    if (!m) return -1;
    const int l = __builtin_amdgcn_readfirstlane(__ffsll(m) - 1);
    lo += l * step;
    n = imin(step, n - l * step);
    if (n == 1) {
      behind = __builtin_amdgcn_readfirstlane(__shfl(end, l)) - row;
      return cu[lo] <= row ? lo : -1;
    }
  }
}

// PP: 16-byte pieces of a head's source row.  T: void for pages of the source's type, else the source's type for e4m3 pages.
template <int PP, typename T>
__global__ __launch_bounds__(kThreads) void paged_append_kernel(const AppendArgs a) {
  constexpr bool Q = !__is_same(T, void);
  const int lane = threadIdx.x & 63;
  const int row = __builtin_amdgcn_readfirstlane(int(blockIdx.x * (kThreads / 64) + threadIdx.x / 64));
  if (row >= a.rows) return;
  int b = row, behind = 1;
  if (a.cu) {
    b = row_seq(a.cu, a.c.B, row, behind);
    if (b < 0) return;
  }
  // (a row of a position before the sequence's first or past the table, or of an entry that is no page, is left out)
  const int64_t pos = int64_t(a.c.lens[b]) - behind;
  if (pos < 0 || pos >= a.c.max_len) return;
  const int pi = page_of(a.c.div, int(pos)), slot = int(pos) - pi * a.c.page_size;
  const int page = a.c.table[int64_t(b) * a.c.table_stride + pi];
  if (page < 0 || page >= a.c.pages) return;
  uint8_t* dk = a.c.k + int64_t(page) * a.c.sk[0] + int64_t(slot) * a.c.sk[2];
  uint8_t* dv = a.c.v + int64_t(page) * a.c.sv[0] + int64_t(slot) * a.c.sv[2];
  for (int i = lane; i < a.c.Hkv * PP; i += 64) {
    const int h = i / PP, piece = i % PP;
    const u32x4 k = ld16(a.k + int64_t(h) * a.sk[0] + int64_t(row) * a.sk[1] + 16 * piece);
    const u32x4 v = ld16(a.v + int64_t(h) * a.sv[0] + int64_t(row) * a.sv[1] + 16 * piece);
    if constexpr (Q) {
      *reinterpret_cast<u32x2*>(dk + int64_t(h) * a.c.sk[1] + 8 * piece) = encode8<T>(k, a.k_inv);
      *reinterpret_cast<u32x2*>(dv + int64_t(h) * a.c.sv[1] + 8 * piece) = encode8<T>(v, a.v_inv);
    } else {
      st16(dk + int64_t(h) * a.c.sk[1] + 16 * piece, k);
      st16(dv + int64_t(h) * a.c.sv[1] + 16 * piece, v);
    }
  }
}

template <int PP, typename T>
hipError_t append(const AppendArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((paged_append_kernel<PP, T>), dim3(unsigned((a.rows + 3) / 4)), dim3(kThreads), 0, s, a);
  return hipGetLastError();
}

// ---- evict -------------------------------------------------------------------------------------
constexpr int kSelectThreads = 1024;

// Unsigned numbers in the order of the weights: NaN above all, -0 as +0.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  if (x != x) return 0xffffffffu;
  if (x == 0.f) return 0x80000000u;
  return u >> 31 ? ~u : u | 0x80000000u;
}

// Digits of those numbers, from the top: 11, 11 and 10 bits.
constexpr int kDigits = 3, kBins = 2048;
__device__ __forceinline__ uint32_t digit_of(uint32_t u, int q) { return q == 0 ? u >> 21 : q == 1 ? u >> 10 & 2047 : u & 1023; }
__device__ __forceinline__ uint32_t digits_above(uint32_t u, int q) { return q == 0 ? 0u : q == 1 ? u >> 21 : u >> 10; }
__device__ __forceinline__ uint32_t with_digit(uint32_t prefix, uint32_t d, int q) { return prefix << (q == 2 ? 10 : 11) | d; }

constexpr int kSelectWaves = kSelectThreads / 64;

// A thread's entries of a chunk, in registers: entry first + EACH tid + e is x[e], u[e] its place in the order.
template <int EACH>
struct Entries {
  float x[EACH];
  uint32_t u[EACH];
  uint32_t live;  // bit e: it is an entry of the sequence, on a page
  uint32_t open;  // bit e: of these, it may be chosen; the others stay
};

struct SelectShared {
  uint32_t hist[kBins];
  int wave[2][kSelectWaves];
  int gaps[kSelectWaves], live[4][kSelectWaves];
  uint32_t digit;
  int need, prior, equal;
};

// The chunk's weights.  `width` of them are in memory, whatever n is, so these loads do not wait for lens.
template <int EACH>
__device__ __forceinline__ void read_entries(Entries<EACH>& t, const float* x, int first, int width) {
  typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));  // (rows start where the caller's strides put them)
  const int i0 = first + EACH * int(threadIdx.x);
  if (i0 + EACH <= width) {
#pragma unroll
    for (int e = 0; e < EACH; e += 4) {
      const f32x4 v = *reinterpret_cast<const f32x4_any*>(x + i0 + e);
#pragma unroll
      for (int c = 0; c < 4; ++c) t.x[e + c] = v[c];
    }
  } else {
#pragma unroll
    for (int e = 0; e < EACH; ++e) t.x[e] = i0 + e < width ? x[i0 + e] : 0.f;
  }
}

// How many of a sequence's positions before some are on a page.
struct Live {
  int gaps;                // is there a page of the sequence that the table does not name?
  int all, lo, hi, first;  // before its end n, before `lo`, `hi` and `first`, each of them at most n
};
// The same in every thread; a barrier is inside.  seen: table[tid], if the table is as wide.
__device__ __forceinline__ Live count_live(SelectShared& sh, const PagedCache& c, const int* table, int seen, int n, int lo, int hi, int first) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int pages = n > 0 ? page_of(c.div, n - 1) + 1 : 0;
  auto named = [&](int page) { return page >= 0 && page < c.pages; };
  bool gap = tid < pages && !named(seen);
  for (int p = tid + kSelectThreads; p < pages; p += kSelectThreads) gap |= !named(table[p]);
  if (const bool any = wave_any(gap); lane == 0) sh.gaps[wave] = any;
  __syncthreads();
  Live r{0, n, lo, hi, first};
#pragma unroll
  for (int w = 0; w < kSelectWaves; ++w) r.gaps |= sh.gaps[w];
  if (!r.gaps) return r;
  int x[4] = {0, 0, 0, 0};
  for (int p = tid; p < pages; p += kSelectThreads) {
    if (!named(table[p])) continue;
    const int at = p * c.page_size;
    auto of = [&](int end) { return imin(imax(end - at, 0), c.page_size); };
    x[0] += of(n);
    x[1] += of(lo);
    x[2] += of(hi);
    x[3] += of(first);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) x[i] += __shfl_xor(x[i], o);
    if (lane == 0) sh.live[i][wave] = x[i];
  }
  __syncthreads();
  r = Live{1, 0, 0, 0, 0};
  for (int w = 0; w < kSelectWaves; ++w) {
    r.all += sh.live[0][w];
    r.lo += sh.live[1][w];
    r.hi += sh.live[2][w];
    r.first += sh.live[3][w];
  }
  return r;
}

template <int EACH>
__device__ __forceinline__ void order_entries(Entries<EACH>& t, const PagedCache& c, const int* table, bool gaps, int first, int n, int lo, int hi) {
  const int i0 = first + EACH * int(threadIdx.x);
  t.live = t.open = 0;
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    t.u[e] = order_of(t.x[e]);
    t.live |= uint32_t(i0 + e < n) << e;
    t.open |= uint32_t(i0 + e >= lo && i0 + e < hi) << e;
  }
  if (gaps) {
    for (int e = 0; e < EACH && i0 + e < n; ++e) {
      const int page = table[page_of(c.div, i0 + e)];
      if (page < 0 || page >= c.pages) t.live &= ~(1u << e);
    }
    t.open &= t.live;
  }
}

// sh.hist, which is zero: how many open entries whose digits above digit q are `prefix` have each value of that digit.
__device__ __forceinline__ void clear_counts(SelectShared& sh) { sh.hist[threadIdx.x] = sh.hist[threadIdx.x + kSelectThreads] = 0; }
template <int EACH>
__device__ __forceinline__ void count_digits(SelectShared& sh, const Entries<EACH>& t, uint32_t prefix, int q) {
#pragma unroll
  for (int e = 0; e < EACH; ++e)
    if ((t.open >> e & 1) && digits_above(t.u[e], q) == prefix) atomicAdd(&sh.hist[digit_of(t.u[e], q)], 1u);
  __syncthreads();
}

// The sum over the workgroup's threads before this one, by one of two LDS rows.  A barrier is inside; the caller has one before the
// row is used again.
__device__ __forceinline__ int sum_before(SelectShared& sh, int row, int x) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int y = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int p = __shfl_up(y, o);
    if (lane >= o) y += p;
  }
  if (lane == 63) sh.wave[row][wave] = y;
  __syncthreads();
  int before = y - x;
#pragma unroll
  for (int w = 0; w < kSelectWaves; ++w) before += w < wave ? sh.wave[row][w] : 0;
  return before;
}

// cnt: entries in this thread's bins 2047 - 2 tid and 2046 - 2 tid; old: those of earlier chunks (MANY).  Finds the bin of
// the need-th entry from the largest: its digit; need becomes the number of its entries that stay; prior grows by the
// entries of earlier chunks in larger bins; equal: theirs in this bin.
template <bool MANY>
__device__ __forceinline__ uint32_t find_digit(SelectShared& sh, const int (&cnt)[2], const int (&old)[2], int& need, int& prior, int& equal) {
  const int tid = threadIdx.x;
  const int before = sum_before(sh, 0, cnt[0] + cnt[1]), before_old = MANY ? sum_before(sh, 1, old[0] + old[1]) : 0;
  if (before < need && before + cnt[0] + cnt[1] >= need) {  // (one thread: 1 <= need <= all entries)
    const int i = before + cnt[0] >= need ? 0 : 1;
    sh.digit = uint32_t(kBins - 1 - 2 * tid - i);
    sh.need = need - before - (i ? cnt[0] : 0);
    sh.prior = before_old + (i ? old[0] : 0);
    sh.equal = i ? old[1] : old[0];
  }
  __syncthreads();
  need = sh.need;
  if (MANY) {
    prior += sh.prior;
    equal = sh.equal;
  }
  return sh.digit;
}

// Numbers the chunk's entries that stay, in order, and writes them: those that are not open, the open ones above `least`, and
// of those equal to it the first `need` (equal of which are in earlier chunks).  rank: entries of earlier chunks that
// stay for another reason.
template <int EACH>
__device__ __forceinline__ void write_kept(SelectShared& sh, const Entries<EACH>& t, int first, int m, uint32_t least, int need, int rank, int equal,
                                           int* kept, float* y) {
  const int i0 = first + EACH * int(threadIdx.x);
  uint32_t stays = 0, equals = 0;
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const bool open = t.open >> e & 1;
    stays |= uint32_t((t.live >> e & 1) && (!open || t.u[e] > least)) << e;
    equals |= uint32_t(open && t.u[e] == least) << e;
  }
  // (both halves of the sums stay below 2^16: a chunk has at most 2^14 entries)
  const int before = sum_before(sh, 0, __popc(stays) | __popc(equals) << 16);
  rank += before & 0xffff;
  equal += before >> 16;
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const bool s = stays >> e & 1, q = equals >> e & 1;
    if (s || (q && equal < need)) {
      const int r = rank + imin(equal, need);
      if (unsigned(r) < unsigned(m)) {  // (always, unless the weights change under the running call)
        kept[r] = i0 + e;
        y[r] = t.x[e];
      }
    }
    rank += s;
    equal += q;
  }
}

// One chunk of 1024 EACH entries of a (sequence, KV head) a workgroup, in registers.  Where that is all of them (a.chunks = 1)
// one launch does everything.  Otherwise launch `stage` = 0, 1, 2 leaves the chunks' counts of digit `stage` in the
// workspace, from which every workgroup of the next launch finds the digit for itself, and launch 3 writes: no
// atomic in memory, nothing to clear, and nobody waits for another workgroup.
// The chunks of a head are as many workgroups apart as there are heads: with a multiple of 8 of them they run on one XCD and share the
// counts in its L2 (8 heads of 131071 entries 42.7 -> 41.3 us, of 32000 29.4 -> 26.8).
template <int EACH>
__global__ __launch_bounds__(kSelectThreads) void paged_select_kernel(const EvictArgs a, int stage) {
  constexpr int kChunk = EACH * kSelectThreads;
  __shared__ SelectShared sh;
  const int rows = a.c.B * a.c.Hkv, chunk = blockIdx.x / rows, row = blockIdx.x % rows, hkv = row % a.c.Hkv, b = row / a.c.Hkv;
  const int tid = threadIdx.x, first = chunk * kChunk;
  const bool last = a.chunks == 1 || stage == kDigits;
  const bool begin = a.chunks == 1 || stage == 0;
  const int* table = a.c.table + int64_t(b) * a.c.table_stride;
  // what this workgroup hands on to the next launch: its prefix, need and prior, and `live`
  int* state = a.state + (int64_t(row) * a.chunks + chunk) * kSelectState;
  // (loads return in order: what the first steps need is asked for before the weights)
  const int seen = begin && tid < a.c.table_width ? table[tid] : 0;
  Live live{};
  if (!begin) live = Live{state[3], state[4], state[5], state[6], state[7]};
  const int n = seq_len(a.c, b);
  Entries<EACH> t;
  read_entries(t, a.sums + int64_t(b) * a.ssum[0] + int64_t(hkv) * a.ssum[1], first, a.sums_width);
  clear_counts(sh);  // (a barrier, of count_live or of find_digit, is before their use)
  if (begin) live = count_live(sh, a.c, table, seen, n, imin(a.S, n), imax(n - a.R, 0), imin(first, n));
  if (!last && stage == 0 && tid == 0) {
    state[3] = live.gaps;
    state[4] = live.all;
    state[5] = live.lo;
    state[6] = live.hi;
    state[7] = live.first;
  }
  const bool evicts = live.all > a.keep;
  const int m = evicts ? a.keep : live.all;
  float* y = a.new_sums + int64_t(b) * a.snew[0] + int64_t(hkv) * a.snew[1];
  if (last) {
    if (hkv == 0 && chunk == 0 && tid == 0) a.new_lens[b] = m;
    const int end = chunk == a.chunks - 1 ? a.sums_width : imin(first + kChunk, a.sums_width);
    for (int i = imax(m, first) + tid; i < end; i += kSelectThreads) y[i] = 0.f;
  }
  // (entries to choose from: all but the first S and the last R, none where nothing is evicted or all stay by their place)
  const int choose = evicts ? a.keep - live.lo - (live.all - live.hi) : 0;
  if (first >= n || (choose == 0 && !last)) return;
  const int lo = evicts ? a.S : 0, hi = evicts ? n - a.R : 0;
  uint32_t prefix = choose > 0 ? 0u : 0xffffffffu;  // (nothing to choose: no number is above, and none equal is needed)
  int need = choose, prior = 0, equal = 0;
  if (choose > 0 && a.chunks > 1 && stage > 0) {
    const int chunks = (n + kChunk - 1) / kChunk;
    if (stage > 1) {
      prefix = uint32_t(state[0]);
      need = state[1];
      prior = state[2];
    }
    const uint32_t* of = reinterpret_cast<const uint32_t*>(a.counts + (int64_t(row) * kDigits + stage - 1) * a.chunks * kBins) + tid;
    int cnt[2] = {0, 0}, old[2] = {0, 0};
#pragma unroll 8
    for (int c = 0; c < chunks; ++c) {
      const uint32_t x = of[c * (kBins / 2)];
      if (c == chunk) {
        old[0] = cnt[0];
        old[1] = cnt[1];
      }
      cnt[0] += int(x & 0xffff);
      cnt[1] += int(x >> 16);
    }
    prefix = with_digit(prefix, find_digit<true>(sh, cnt, old, need, prior, equal), stage - 1);
    if (!last && tid == 0) {
      state[0] = int(prefix);
      state[1] = need;
      state[2] = prior;
    }
  }
  order_entries(t, a.c, table, live.gaps, first, n, lo, hi);
  if (!last) {  // counts: [digit][chunk][2047 - value]
    count_digits(sh, t, prefix, stage);
    reinterpret_cast<uint32_t*>(a.counts + ((int64_t(row) * kDigits + stage) * a.chunks + chunk) * kBins)[tid] =
        sh.hist[kBins - 1 - 2 * tid] | sh.hist[kBins - 2 - 2 * tid] << 16;
    return;
  }
  if (choose > 0 && a.chunks == 1) {
    for (int q = 0; q < kDigits; ++q) {
      if (q) {
        clear_counts(sh);
        __syncthreads();
      }
      count_digits(sh, t, prefix, q);
      const int cnt[2] = {int(sh.hist[kBins - 1 - 2 * tid]), int(sh.hist[kBins - 2 - 2 * tid])}, old[2] = {0, 0};
      prefix = with_digit(prefix, find_digit<false>(sh, cnt, old, need, prior, equal), q);
    }
  }
  // entries of earlier chunks that stay by their place
  const int fixed = evicts ? imin(live.first, live.lo) + imax(0, live.first - live.hi) : live.first;
  write_kept(sh, t, first, m, prefix, need, fixed + prior, equal, a.kept + int64_t(row) * a.keep, y);
}

// A workgroup has kThreads / pieces entries a round.  Rounds of 1 / 2 / 4 / 8: 15.7 / 13.6 / 15.6 / 18.4 us for 8 sequences, 17.2 / 16.6 /
// 17.9 / 21.0 for one of 16384 kept entries: the look-ups of some workgroups hide behind the copies of others.
constexpr int kGatherRounds = kGatherPieces / kThreads;

// The entries are taken in the order of the pages they go to: a head's one after the other, or (ACROSS, pages with their slots first)
// an entry of every head before the next ones, so that a workgroup writes whole rows.  By heads / ACROSS, slots first: 153 / 87 us
// for 15 sequences of 16 heads with D = 16 that keep 7642 entries, where an entry of one head is 32 bytes; 16.4 / 16.1 for one of
// 16384 with D = 64.
template <int PIECES, bool ACROSS>
__global__ __launch_bounds__(kThreads) void paged_gather_kernel(const EvictArgs a, int chunks) {
  constexpr int ROWS = kThreads / PIECES;
  const int chunk = blockIdx.x % chunks, s = blockIdx.x / chunks, b = ACROSS ? s : s / a.c.Hkv;
  const int n = seq_len(a.c, b), m = a.new_lens[b];
  const int* from = a.c.table + int64_t(b) * a.c.table_stride;
  const int* to = a.new_table + int64_t(b) * a.new_table_stride;
  const int piece = threadIdx.x % PIECES;
#pragma unroll
  for (int x = 0; x < kGatherRounds; ++x) {
    const int e = (chunk * kGatherRounds + x) * ROWS + int(threadIdx.x) / PIECES;
    const int r = ACROSS ? e / a.c.Hkv : e, hkv = ACROSS ? e % a.c.Hkv : s % a.c.Hkv;
    if (r >= m || r >= a.keep) continue;
    const int i = a.kept[(int64_t(b) * a.c.Hkv + hkv) * a.keep + r];
    if (i < 0 || i >= n) continue;  // (never, unless lens or weights change under the running call)
    const int pi = page_of(a.c.div, i), slot = i - pi * a.c.page_size, qi = page_of(a.c.div, r), new_slot = r - qi * a.c.page_size;
    const int page = from[pi], new_page = to[qi];
    if (page < 0 || page >= a.c.pages || new_page < 0 || new_page >= a.c.pages) continue;
    const u32x4 k = ld16(a.c.k + int64_t(page) * a.c.sk[0] + int64_t(hkv) * a.c.sk[1] + int64_t(slot) * a.c.sk[2] + 16 * piece);
    const u32x4 v = ld16(a.c.v + int64_t(page) * a.c.sv[0] + int64_t(hkv) * a.c.sv[1] + int64_t(slot) * a.c.sv[2] + 16 * piece);
    st16(a.c.k + int64_t(new_page) * a.c.sk[0] + int64_t(hkv) * a.c.sk[1] + int64_t(new_slot) * a.c.sk[2] + 16 * piece, k);
    st16(a.c.v + int64_t(new_page) * a.c.sv[0] + int64_t(hkv) * a.c.sv[1] + int64_t(new_slot) * a.c.sv[2] + 16 * piece, v);
  }
}

template <int PIECES>
hipError_t gather(const EvictArgs& a, hipStream_t s) {
  const int rows = kThreads / PIECES * kGatherRounds;
  const int64_t entries = int64_t(a.keep) * a.c.Hkv;
  if (a.c.sk[1] < a.c.sk[2] && entries < (int64_t(1) << 30)) {
    const int chunks = int((entries + rows - 1) / rows);
    hipLaunchKernelGGL((paged_gather_kernel<PIECES, true>), dim3(unsigned(chunks) * unsigned(a.c.B)), dim3(kThreads), 0, s, a, chunks);
  } else {
    const int chunks = (a.keep + rows - 1) / rows;
    hipLaunchKernelGGL((paged_gather_kernel<PIECES, false>), dim3(unsigned(chunks) * unsigned(a.c.B * a.c.Hkv)), dim3(kThreads), 0, s, a, chunks);
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_paged_append(const AppendArgs& a, int dtype, int cache, int D, hipStream_t s) {
  if (cache == FA_DTYPE_FP8_E4M3) {
    if (dtype == FA_DTYPE_BF16) return D == 64 ? append<8, SrcBF16>(a, s) : append<16, SrcBF16>(a, s);
    return D == 64 ? append<8, SrcF16>(a, s) : append<16, SrcF16>(a, s);
  }
  switch (D * (dtype == FA_DTYPE_F32 ? 4 : 2) / 16) {
    case 2: return append<2, void>(a, s);
    case 4: return append<4, void>(a, s);
    case 8: return append<8, void>(a, s);
    case 16: return append<16, void>(a, s);
    default: return append<32, void>(a, s);
  }
}

hipError_t launch_paged_evict(const EvictArgs& a, int row_bytes, hipStream_t s) {
  for (int stage = a.chunks == 1 ? kDigits : 0; stage <= kDigits; ++stage) {
    const dim3 grid(unsigned(a.chunks) * unsigned(a.c.B * a.c.Hkv)), block(kSelectThreads);
    if (a.each == 4) hipLaunchKernelGGL(paged_select_kernel<4>, grid, block, 0, s, a, stage);
    else if (a.each == 8) hipLaunchKernelGGL(paged_select_kernel<8>, grid, block, 0, s, a, stage);
    else hipLaunchKernelGGL(paged_select_kernel<16>, grid, block, 0, s, a, stage);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  switch (row_bytes / 16) {
    case 2: return gather<2>(a, s);
    case 4: return gather<4>(a, s);
    case 8: return gather<8>(a, s);
    case 16: return gather<16>(a, s);
    default: return gather<32>(a, s);
  }
}

}  // namespace fa
