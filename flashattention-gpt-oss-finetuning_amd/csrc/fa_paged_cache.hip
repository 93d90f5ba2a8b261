// fa_paged_cache.hip - what fills and thins out a paged key-value cache: new rows (fa_paged_append) and eviction by
// accumulated attention weight (fa_paged_evict).  Copies and a selection: memory bounds all of them.
//
// paged_append_kernel.  Row i of sequence b's n new rows goes to position lens[b] - n + i.  A wave takes a row: it finds the
// row's sequence by one ballot over cu_seqlens and the page once, then its lanes copy the 16-byte pieces of
// every head's K and V.  e4m3 pages get the codes of clamp(x * fl32(1 / descale), -448, 448), as quantize_fp8's.
//
// paged_select_kernel.  Of a (sequence, KV head)'s n entries the first S and the last R stay, and of the others the
// keep - S - R of the largest weight, the lower index first among equals (NaN counts as the largest).  The weights are
// mapped to unsigned numbers of the same order; four passes of 8 bits find the smallest one that stays, T, and how
// many equal to T do; a last pass in index order numbers the entries that stay.
// paged_gather_kernel.  Entry r of those kept goes to position r on the pages of the new table.  Those are other pages
// than the old ones, so no entry is read after it is overwritten and all are copied at once.
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
// row is no sequence's.  Every lane of the wave calls.
__device__ __forceinline__ int row_seq(const int* cu, int B, int row, int& behind) {
  const int lane = threadIdx.x & 63;
  for (int b0 = 0; b0 < B; b0 += 64) {
    const int end = b0 + lane < B ? cu[b0 + lane + 1] : -1;
    const unsigned long long m = __ballot(end > row);
    if (m) {
      const int l = __builtin_amdgcn_readfirstlane(__ffsll(m) - 1);
      behind = __builtin_amdgcn_readfirstlane(__shfl(end, l)) - row;
      return cu[b0 + l] <= row ? b0 + l : -1;
    }
  }
  return -1;
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
  const int n = a.c.Hkv * PP;
  for (int i = lane; i < 2 * n; i += 64) {
    const bool is_v = i >= n;
    const int p = is_v ? i - n : i, h = p / PP, piece = p % PP;
    const u32x4 x = is_v ? ld16(a.v + int64_t(h) * a.sv[0] + int64_t(row) * a.sv[1] + 16 * piece)
                         : ld16(a.k + int64_t(h) * a.sk[0] + int64_t(row) * a.sk[1] + 16 * piece);
    uint8_t* d = is_v ? a.c.v + int64_t(page) * a.c.sv[0] + int64_t(h) * a.c.sv[1] + int64_t(slot) * a.c.sv[2]
                      : a.c.k + int64_t(page) * a.c.sk[0] + int64_t(h) * a.c.sk[1] + int64_t(slot) * a.c.sk[2];
    if constexpr (Q) *reinterpret_cast<u32x2*>(d + 8 * piece) = encode8<T>(x, is_v ? a.v_inv : a.k_inv);
    else st16(d + 16 * piece, x);
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

__global__ __launch_bounds__(kSelectThreads) void paged_select_kernel(const EvictArgs a) {
  const int hkv = blockIdx.x % a.c.Hkv, b = blockIdx.x / a.c.Hkv;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n = seq_len(a.c, b), m = imin(n, a.keep);
  const float* x = a.sums + int64_t(b) * a.ssum[0] + int64_t(hkv) * a.ssum[1];
  float* y = a.new_sums + int64_t(b) * a.snew[0] + int64_t(hkv) * a.snew[1];
  int* kept = a.kept + (int64_t(b) * a.c.Hkv + hkv) * a.keep;
  if (hkv == 0 && tid == 0) a.new_lens[b] = m;
  for (int i = m + tid; i < a.sums_width; i += kSelectThreads) y[i] = 0.f;
  if (n <= a.keep) {
    for (int i = tid; i < n; i += kSelectThreads) {
      y[i] = x[i];
      kept[i] = i;
    }
    return;
  }
  __shared__ int hist[256];
  __shared__ uint32_t s_prefix;
  __shared__ int s_need;
  __shared__ uint32_t s_wave[kSelectThreads / 64];
  const int lo = a.S, hi = n - a.R;  // the entries to choose from; hi - lo > keep - S - R
  if (tid == 0) {
    s_prefix = 0;
    s_need = a.keep - a.S - a.R;
  }
  // the bits of the smallest number that stays, from the top; `need` counts those still to be found among
  // the numbers that share them
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    const uint32_t prefix = s_prefix;
    const int need = s_need;
    for (int i = lo + tid; i < hi; i += kSelectThreads) {
      const uint32_t u = order_of(x[i]);
      if (shift == 24 || u >> (shift + 8) == prefix) atomicAdd(&hist[u >> shift & 255], 1);
    }
    __syncthreads();
    if (wave == 0) {
      // digits from 255 down: lane l has digits 255 - 4l .. 252 - 4l
      int c[4], t = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) t += c[i] = hist[255 - 4 * lane - i];
      int before = t;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int z = __shfl_up(before, o);
        if (lane >= o) before += z;
      }
      before -= t;  // numbers of larger digits than this lane's
      // (need = 0: no number stays; T is then above all of them)
      if (need > 0 && before < need && before + t >= need) {
        int i = 0;
        while (before + c[i] < need) before += c[i++];
        s_prefix = prefix << 8 | uint32_t(255 - 4 * lane - i);
        s_need = need - before;
      }
    }
    __syncthreads();
  }
  const uint32_t T = s_prefix;
  const int need = s_need;
  const bool none = a.keep == a.S + a.R;
  int above = 0, equal = 0;  // entries before the tile that stay for good, and equal ones
  for (int i0 = 0; i0 < n; i0 += kSelectThreads) {
    const int i = i0 + tid;
    bool stays = false, eq = false;
    float w = 0.f;
    if (i < n) {
      w = x[i];
      const uint32_t u = order_of(w);
      stays = i < lo || i >= hi || (!none && u > T);
      eq = !stays && !none && u == T;
    }
    const unsigned long long ms = __ballot(stays), me = __ballot(eq);
    if (lane == 0) s_wave[wave] = uint32_t(__popcll(ms)) | uint32_t(__popcll(me)) << 16;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int v = 0; v < kSelectThreads / 64; ++v) {
      const uint32_t c = s_wave[v];
      before += v < wave ? c : 0u;
      all += c;
    }
    const unsigned long long below = (1ull << lane) - 1;
    const int sb = above + int(before & 0xffff) + __popcll(ms & below), eb = equal + int(before >> 16) + __popcll(me & below);
    if (stays || (eq && eb < need)) {
      const int r = sb + imin(eb, need);
      if (r < m) {  // (always, unless the weights change under the running call)
        kept[r] = i;
        y[r] = w;
      }
    }
    above += int(all & 0xffff);
    equal += int(all >> 16);
    __syncthreads();
  }
}

// Entries of a workgroup: kThreads / pieces a round.
constexpr int kGatherRounds = 4;

template <int PIECES>
__global__ __launch_bounds__(kThreads) void paged_gather_kernel(const EvictArgs a, int chunks) {
  constexpr int ROWS = kThreads / PIECES;
  const int chunk = blockIdx.x % chunks, s = blockIdx.x / chunks, hkv = s % a.c.Hkv, b = s / a.c.Hkv;
  const int n = seq_len(a.c, b), m = imin(n, a.keep);
  const int* kept = a.kept + int64_t(s) * a.keep;
  const int* from = a.c.table + int64_t(b) * a.c.table_stride;
  const int* to = a.new_table + int64_t(b) * a.new_table_stride;
  const int piece = threadIdx.x % PIECES;
#pragma unroll
  for (int x = 0; x < kGatherRounds; ++x) {
    const int r = (chunk * kGatherRounds + x) * ROWS + int(threadIdx.x) / PIECES;
    if (r >= m) continue;
    const int i = kept[r];
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
  const int rows = kThreads / PIECES * kGatherRounds, chunks = (a.keep + rows - 1) / rows;
  hipLaunchKernelGGL(paged_gather_kernel<PIECES>, dim3(unsigned(chunks) * unsigned(a.c.B * a.c.Hkv)), dim3(kThreads), 0, s, a, chunks);
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
  hipLaunchKernelGGL(paged_select_kernel, dim3(unsigned(a.c.B * a.c.Hkv)), dim3(kSelectThreads), 0, s, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  switch (row_bytes / 16) {
    case 2: return gather<2>(a, s);
    case 4: return gather<4>(a, s);
    case 8: return gather<8>(a, s);
    case 16: return gather<16>(a, s);
    default: return gather<32>(a, s);
  }
}

}  // namespace fa
