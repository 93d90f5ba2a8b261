// fa_paged_attn.hip - attention of one new token a sequence over a paged key-value cache (fa_paged_attention).
//
// For each (sequence, KV head) the G query heads of its group meet the n visible keys:
//     s[h, k] = scale q[h] . K[k],   lse[h] = log(sum_k exp s[h, k] + exp(sink[h])),   o[h] = sum_k exp(s[h, k] - lse[h]) V[k].
// 4 G operations a cache element, so the cache's bytes bound it: the kernel is built to keep them coming.
//
// paged_attn_kernel.  A workgroup of 4 or 8 waves takes a run of keys for 16 query heads (a group, padded); its waves
// take tiles of 32 keys in turn and meet only at the run's end.  In between no lane needs another's values:
//   * S^T = K Q^T as v_mfma_f32_16x16x32 with the keys as rows.  Lane l (r = l % 16, j = l / 16) supplies key rows r of two
//     16-key halves and gets, for head r, rows 4j..4j+3 of both.  Half T's row 4j + i is the tile's key 8j + 4T + i, so the
//     lane's eight scores are those of keys 8j..8j+7.
//   * O^T = V^T P^T with the head dim as rows: the lane's eight weights are the B operand as they lie, and the A
//     operand is eight V entries of keys 8j..8j+7, of which the lane loads D / 16 neighbouring dims each and pairs
//     two keys' halves (one v_perm per register).  Its C rows are the lane's own head again, so
//     maximum, sum and rescaling need no exchange.
// Weights are taken against a running reference, which is raised to the maximum only where a weight would exceed 2^8 (which 16
// bits and float32 hold as well as 1), after the first tiles hardly ever; only then do lanes exchange maxima.  float16
// has no numbers below 2^-24: there the reference lies 2^7 below the maximum, so that weights reach 2^15 and what a key
// can lose is 2^-32 of the largest weight of its wave's run, not 2^-25.
// K is loaded with neighbouring lanes on neighbouring 16-byte pieces and turned into fragments in the wave's own LDS: loaded
// as fragments (16 rows an instruction) 876 MB took 190 us, so 166, all else as it was.
// P goes into the 16-bit product as the sum of two 16-bit parts (P rounded, and what that left), so o carries its own
// rounding only; the second product costs matrix time that the loads leave idle.  It sees infinite values as the largest finite
// ones, for what the rounding left may be 0 or have the other sign: the first product decides (two operations a register of V:
// 32 ragged sequences 52.7 -> 53.4 us).  float32 uses v_mfma_f32_16x16x4.
//
// Keys are addressed through a wave's own LDS table of 64-bit offsets, 64 keys at a time: key -> page -> offset is worked
// out once a key, ahead of its use.  Keys on no page (an entry outside [0, pages)) and those past the end are marked in a
// mask; their scores become -inf and their V entries 0, whatever lies in memory (they are loaded from entry 0 of page 0).
//
// Runs.  With a workgroup a (KV head, sequence) long sequences would leave the chip idle, and with a fixed number of
// pieces a sequence ragged batches would.  Split calls deal out the units of all sequences evenly
// (fa_paged_plan.h): each workgroup finds its run by a prefix sum over lens, on the device, so the grid depends on
// sizes the host knows.  Pieces that are no whole sequence leave (maximum, sum, o) in the workspace, and
// paged_finish_kernel joins them.
//
// Measured (D = 64, bf16, 8 heads a group; rocprofv3): 32 ragged sequences, 261 MB of K and V, 49 to 51 us, 5.2 TB/s; four of up to 128K
// tokens, 876 MB, 138 us, 6.3 TB/s, with the heads before the slots in a page and 147 to 150, 5.9, with the slots first.  float32: 522 MB
// 93 us, 5.6 TB/s; with D = 128 119, 4.4.  The counters show 261 and 877 MB read: every entry once.  A plain kernel that only reads reaches 6.2 TB/s, 7.1 with loads marked as read
// once.  Without the products and the softmax (loads only) the kernel took the same time to 5%.
// What is left of a small call is latency: lens, table, K, four tiles, the waves' sums: one sliding-layer step 5.4 to 5.8 us.
#include <hip/hip_runtime.h>

#include "../../include/fa_gfx950.h"
#include "fa_common.h"
#include "fa_paged.h"

namespace fa {
namespace {

constexpr int kThreads = 256;
constexpr int kTile = 32;

__device__ __forceinline__ int seq_len(const PagedCache& c, int b) { return imin(imax(c.lens[b], 0), c.max_len); }

__device__ __forceinline__ int wave_prefix(int n, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(n, o);
    if (lane >= o) n += y;
  }
  return n;
}

__device__ __forceinline__ int units_of(const PagedAttnArgs& a, int b) {
  return b < a.c.B ? paged_units(visible(seq_len(a.c, b), a.W, a.S).count) : 0;
}

// The units of the sequences, 64 at a time over the lanes of a wave, all of which call.
struct Units {
  int n, upto;  // of this lane's sequence, and of the 64 up to it
  __device__ __forceinline__ int all() const { return __builtin_amdgcn_readfirstlane(__shfl(upto, 63)); }
};
__device__ __forceinline__ Units units_from(const PagedAttnArgs& a, int b0) {
  const int lane = threadIdx.x & 63, n = units_of(a, b0 + lane);
  return Units{n, wave_prefix(n, lane)};
}

// Units of all sequences; the first 64 sequences' are in `first`.
__device__ __forceinline__ int total_units(const PagedAttnArgs& a, const Units& first) {
  if (a.c.B <= 64) return first.all();
  int n = first.n;
#pragma unroll 4
  for (int b0 = 64; b0 < a.c.B; b0 += 64) n += units_of(a, b0 + (threadIdx.x & 63));
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) n += __shfl_xor(n, o);
  return __builtin_amdgcn_readfirstlane(n);
}

// The sequence that holds unit u < total, and its first unit.
__device__ __forceinline__ void find_unit(const PagedAttnArgs& a, Units x, int u, int& b, int& start) {
  int base = 0;
  for (int b0 = 0;;) {
    const unsigned long long m = __ballot(base + x.upto > u);
    if (m) {
      const int l = __builtin_amdgcn_readfirstlane(__ffsll(m) - 1);
      b = b0 + l;
      start = base + __builtin_amdgcn_readfirstlane(__shfl(x.upto - x.n, l));
      return;
    }
    base += x.all();
    b0 += 64;
    if (b0 >= a.c.B) break;
    x = units_from(a, b0);
  }
  b = 0;  // (not reached: u < total)
  start = 0;
}

// Element types.  EB, CB: bytes of a query and of a cache element.  kBelow: log2 of how far a new reference lies below the maximum.
struct PBF16 : BF16 {
  static constexpr int EB = 2, CB = 2;
  static constexpr float kBelow = 0.f;
  static constexpr uint16_t kLargest = 0x7f7f;
};
struct PF16 : F16 {
  static constexpr int EB = 2, CB = 2;
  static constexpr float kBelow = 7.f;
  static constexpr uint16_t kLargest = 0x7bff;
};
struct PBF16Q8 : BF16 {
  static constexpr int EB = 2, CB = 1;
  static constexpr float kBelow = 0.f;
  static __device__ __forceinline__ uint32_t widen(uint32_t x, bool hi) {
    return hi ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, true))
              : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, false));
  }
};
struct PF16Q8 : F16 {
  static constexpr int EB = 2, CB = 1;
  static constexpr float kBelow = 7.f;
  static __device__ __forceinline__ uint32_t widen(uint32_t x, bool hi) {
    return hi ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.0f, true))
              : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.0f, false));
  }
};
struct PF32 {
  static constexpr int EB = 4, CB = 4;
  static constexpr float kBelow = 0.f;
};

__device__ __forceinline__ float quarters_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float quarters_sum(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

template <bool ONCE, typename T>
__device__ __forceinline__ T fetch(const T* p) {
  if constexpr (ONCE) return __builtin_nontemporal_load(p);
  else return *p;
}

// Eight 16-bit numbers, the infinite ones (and NaN) as the largest finite ones of their sign: as integers, those of both signs are the
// ones above it, unsigned for the negative ones and signed for the others.
template <typename E>
__device__ __forceinline__ u32x4 finite8(u32x4 x) {
  typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
  typedef int16_t i16x8 __attribute__((ext_vector_type(8)));
  const u16x8 neg = __builtin_elementwise_min(__builtin_bit_cast(u16x8, x), u16x8(uint16_t(E::kLargest | 0x8000)));
  return __builtin_bit_cast(u32x4, __builtin_elementwise_min(__builtin_bit_cast(i16x8, neg), i16x8(int16_t(E::kLargest))));
}

// One wave's tile of 32 keys in registers.
template <typename E, int D>
struct Tile {
  static constexpr int ROW = D * E::CB;                      // bytes of an entry
  static constexpr int PR = ROW / 16;                        // 16-byte pieces of an entry
  static constexpr int NF = PR >= 4 ? PR / 4 : 1;            // of those that a lane supplies to the products
  static constexpr bool STAGED = E::CB < 4;                  // K goes through LDS
  static constexpr int NK = STAGED ? PR / 2 : 2 * NF;        // pieces of the tile that a lane loads
  static constexpr int VB = ROW / 16;                        // bytes of a V entry that a lane holds
  static constexpr int VD = VB >= 4 ? VB / 4 : 1;
  // tiles in flight (D = 32, 268 MB: 50.8 us with 2, 48.8 with 4; D = 64 in 16 bits no gain, D = 128 in 8 bits 24.6 and 31.4)
  static constexpr int AHEAD = ROW <= 64 ? 4 : 2;
  u32x4 k[NK];
  uint32_t v[8][VD];
  uint32_t live;  // bit i: key i of the tile is on a page (the same in every lane)
};

// A wave's state for RT tiles of 16 heads, which share the key tiles that it reads.
template <typename E, int D, int RT>
struct Wave {
  using T = Tile<E, D>;
  static constexpr int NC = D / 16;                          // dims a lane of the output holds of each 16 rows
  static constexpr bool F = E::EB == 4;
  static constexpr int NQ = F ? D / 16 : (D >= 32 ? D / 32 : 1);
  u32x4 q[RT][NQ];
  f32x4 acc[RT][NC];
  float m[RT], mref[RT], l[RT];  // running reference (log2 domain), the same with 0 for none, this lane's sum against it

  // Q as the B operand: head r of the tile, dims in the order in which the K pieces hold them.
  __device__ __forceinline__ void load_q(int x, const uint8_t* q_row, bool have) {
    const int j = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int f = 0; f < NQ; ++f) {
      // 16-byte piece 4f + j of the row; an e4m3 piece holds 16 dims, two pieces of q
      const int piece = E::CB == 1 ? 2 * (4 * (f / 2) + j) + f % 2 : 4 * f + j;
      q[x][f] = have && piece * 16 < D * E::EB ? ld16(q_row + 16 * piece) : zero16();
    }
  }
  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int x = 0; x < RT; ++x) {
#pragma unroll
      for (int c = 0; c < NC; ++c) acc[x][c] = f32x4{0.f, 0.f, 0.f, 0.f};
      m[x] = kNegInf;
      mref[x] = 0.f;
      l[x] = 0.f;
    }
  }

  // koff, voff: the tile's 32 offsets of K, and of V, in LDS.
  template <bool ONCE>
  static __device__ __forceinline__ void load(T& t, const uint8_t* k, const uint8_t* v, const int64_t* koff, const int64_t* voff,
                                              uint32_t live) {
    const int lane = threadIdx.x & 63, r = lane & 15, j = lane >> 4;
    t.live = live;
    if constexpr (T::STAGED) {  // neighbouring lanes take neighbouring pieces
#pragma unroll
      for (int n = 0; n < T::NK; ++n)
        t.k[n] = fetch<ONCE>(reinterpret_cast<const u32x4*>(k + koff[(64 * n + lane) / T::PR] + 16 * (lane % T::PR)));
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint8_t* p = k + koff[8 * (r >> 2) + 4 * h + (r & 3)];
#pragma unroll
        for (int n = 0; n < T::NF; ++n) t.k[h * T::NF + n] = fetch<ONCE>(reinterpret_cast<const u32x4*>(p + 64 * n + 16 * j));
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint8_t* p = v + voff[8 * j + e] + T::VB * r;
      if constexpr (T::VB == 2) {
        t.v[e][0] = fetch<ONCE>(reinterpret_cast<const uint16_t*>(p));
      } else if constexpr (T::VB == 4) {
        t.v[e][0] = fetch<ONCE>(reinterpret_cast<const uint32_t*>(p));
      } else if constexpr (T::VB == 8) {
        const u32x2 x = fetch<ONCE>(reinterpret_cast<const u32x2*>(p));
        t.v[e][0] = x[0];
        t.v[e][1] = x[1];
      } else {
#pragma unroll
        for (int w = 0; w < T::VB / 16; ++w) {
          const u32x4 x = fetch<ONCE>(reinterpret_cast<const u32x4*>(p + 16 * w));
#pragma unroll
          for (int i = 0; i < 4; ++i) t.v[e][4 * w + i] = x[i];
        }
      }
    }
  }

  // Eight keys' values of dim c of this lane as an A operand: v[e] holds D / 16 dims of key 8j + e.
  static __device__ __forceinline__ u32x4 v_frag(const uint32_t (&v)[8][NC >= 2 ? NC / 2 : 1], int c) {
    u32x4 f;
#pragma unroll
    for (int d = 0; d < 4; ++d)
      f[d] = __builtin_amdgcn_perm(v[2 * d + 1][c / 2], v[2 * d][c / 2], c % 2 ? 0x07060302u : 0x05040100u);
    return f;
  }

  // Place of piece p of the tile's key row in the staged tile: the rows 0..3 and 8..11 (and 4 or 16 more) that eight lanes
  // read at once, at the same piece, get different banks.
  static __device__ __forceinline__ int staged(int row, int p) {
    constexpr int PR = T::PR;
    const int s = PR >= 8 ? (row & 3) | (row >> 1 & 4) : PR == 4 ? (row >> 1 & 1) | (row >> 2 & 2) : row >> 3 & 1;
    return row * PR + (p ^ s);
  }

  // lds: the wave's room for a staged K tile; logits(x): where the lane's eight scores of head tile x go, or NULL
  template <typename L>
  __device__ __forceinline__ void step(T& t, float c2, u32x4* lds, L&& logits) {
    const int lane = threadIdx.x & 63, r = lane & 15, j = lane >> 4;
    u32x4 kf[2][T::NF];
    if constexpr (T::STAGED) {
#pragma unroll
      for (int n = 0; n < T::NK; ++n) lds[staged((64 * n + lane) / T::PR, lane % T::PR)] = t.k[n];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int n = 0; n < T::NF; ++n)
          kf[h][n] = 4 * n + j < T::PR ? lds[staged(8 * (r >> 2) + 4 * h + (r & 3), 4 * n + j)] : zero16();
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    } else {
#pragma unroll
      for (int n = 0; n < 2 * T::NF; ++n) kf[n / T::NF][n % T::NF] = t.k[n];
    }
    if (t.live != ~0u) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool ok = t.live >> (8 * j + e) & 1;
#pragma unroll
        for (int w = 0; w < T::VD; ++w) t.v[e][w] = ok ? t.v[e][w] : 0u;
      }
    }
    u32x4 hi[RT], lo[RT];  // the weights as B operands, in two 16-bit parts
    float p[RT][8];
#pragma unroll
    for (int x = 0; x < RT; ++x) {
      f32x4 s0 = {0.f, 0.f, 0.f, 0.f}, s1 = s0;
#pragma unroll
      for (int n = 0; n < T::NF; ++n) {
        if constexpr (F) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t k0 = kf[0][n][e], k1 = kf[1][n][e], qe = q[x][n][e];
            s0 = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, k0), __builtin_bit_cast(float, qe), s0, 0, 0, 0);
            s1 = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, k1), __builtin_bit_cast(float, qe), s1, 0, 0, 0);
          }
        } else if constexpr (E::CB == 1) {
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            u32x4 k0, k1;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              k0[2 * w] = E::widen(kf[0][n][2 * u + w], false);
              k0[2 * w + 1] = E::widen(kf[0][n][2 * u + w], true);
              k1[2 * w] = E::widen(kf[1][n][2 * u + w], false);
              k1[2 * w + 1] = E::widen(kf[1][n][2 * u + w], true);
            }
            s0 = E::mfma16(k0, q[x][2 * n + u], s0);
            s1 = E::mfma16(k1, q[x][2 * n + u], s1);
          }
        } else {
          s0 = E::mfma16(kf[0][n], q[x][n], s0);
          s1 = E::mfma16(kf[1][n], q[x][n], s1);
        }
      }
      float s[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[i] = s0[i] * c2;
        s[4 + i] = s1[i] * c2;
      }
      if (t.live != ~0u) {
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e] = t.live >> (8 * j + e) & 1 ? s[e] : kNegInf;
      }
      if (float* to = logits(x)) {
        *reinterpret_cast<f32x4*>(to) = f32x4{s[0], s[1], s[2], s[3]};
        *reinterpret_cast<f32x4*>(to + 4) = f32x4{s[4], s[5], s[6], s[7]};
      }
      float mx = s[0];
#pragma unroll
      for (int e = 1; e < 8; ++e) mx = fmaxf(mx, s[e]);
      if (wave_any(mx > m[x] + (8.f + E::kBelow))) {
        const float up = fmaxf(m[x], quarters_max(mx) - E::kBelow);
        const float scale = m[x] == kNegInf ? 0.f : fast_exp2(m[x] - up);
        l[x] *= scale;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[x][c][i] *= scale;
        m[x] = up;
        mref[x] = up == kNegInf ? 0.f : up;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[x][e] = fast_exp2(s[e] - mref[x]);
        l[x] += p[x][e];
      }
      if constexpr (!F) {
        hi[x] = pack8<E>(p[x]);
        float rest[8];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          rest[2 * w] = p[x][2 * w] - E::to_f32(uint16_t(hi[x][w]));
          rest[2 * w + 1] = p[x][2 * w + 1] - E::to_f32(uint16_t(hi[x][w] >> 16));
        }
        lo[x] = pack8<E>(rest);
      }
    }
    if constexpr (F) {
#pragma unroll
      for (int x = 0; x < RT; ++x)
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
          for (int c = 0; c < NC; ++c)
            acc[x][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, t.v[e][c]), p[x][e], acc[x][c], 0, 0, 0);
    } else {
      uint32_t w[8][NC >= 2 ? NC / 2 : 1];
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int d = 0; d < (NC >= 2 ? NC / 2 : 1); ++d) {
          if constexpr (E::CB == 1) w[e][d] = E::widen(t.v[e][d / 2], d % 2);
          else w[e][d] = t.v[e][d];
        }
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const u32x4 f = v_frag(w, c);
#pragma unroll
        for (int x = 0; x < RT; ++x) acc[x][c] = E::mfma16(f, hi[x], acc[x][c]);
        u32x4 g = f;
        if constexpr (E::CB == 2) g = finite8<E>(f);  // (e4m3 has no infinities)
#pragma unroll
        for (int x = 0; x < RT; ++x) acc[x][c] = E::mfma16(g, lo[x], acc[x][c]);
      }
    }
  }
};

// D / 16 output values of one head (float32) to o, in its type.
template <typename E, int N>
__device__ __forceinline__ void store_out(uint8_t* o, const float (&x)[N]) {
  if constexpr (E::EB == 4) {
    if constexpr (N == 1) *reinterpret_cast<float*>(o) = x[0];
    else if constexpr (N == 2) *reinterpret_cast<f32x2*>(o) = f32x2{x[0], x[1]};
    else {
#pragma unroll
      for (int i = 0; i < N; i += 4) *reinterpret_cast<f32x4*>(o + 4 * i) = f32x4{x[i], x[i + 1], x[i + 2], x[i + 3]};
    }
  } else if constexpr (N == 1) {
    *reinterpret_cast<uint16_t*>(o) = uint16_t(E::pack2(x[0], x[0]));
  } else {
    uint32_t w[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) w[i] = E::pack2(x[2 * i], x[2 * i + 1]);
    if constexpr (N == 2) *reinterpret_cast<uint32_t*>(o) = w[0];
    else if constexpr (N == 4) *reinterpret_cast<u32x2*>(o) = u32x2{w[0], w[1]};
    else st16(o, u32x4{w[0], w[1], w[2], w[3]});
  }
}

struct Yes {
  static constexpr bool value = true;
};
struct No {
  static constexpr bool value = false;
};

template <typename E, int D, int WAVES>
struct Shared {
  static constexpr int PAD = D + 4;  // float32 rows 4 banks apart
  union {
    struct {
      struct {
        int64_t k[64], v[64];
      } off[2];
      u32x4 k[Tile<E, D>::STAGED ? kTile * Tile<E, D>::PR : 1];
    } wave[WAVES];
    float o[WAVES][16][PAD];
  };
  float m[WAVES][16], l[WAVES][16];
};

template <typename E, int D, int WAVES, int RT>
__global__ __launch_bounds__(64 * WAVES) void paged_attn_kernel(const PagedAttnArgs a) {
  constexpr int NC = D / 16;
  __shared__ Shared<E, D, WAVES> sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, j = lane >> 4;
  const int parts = a.parts ? a.parts : a.c.B;
  const int stream = blockIdx.x / parts, part = blockIdx.x % parts;
  const int shares = (a.row_tiles + RT - 1) / RT;  // workgroups that a group's heads are shared out to
  const int hkv = stream / shares, h0 = stream % shares * (16 * RT);  // first head within the group
  const uint8_t* kb = a.c.k + int64_t(hkv) * a.c.sk[1];
  const uint8_t* vb = a.c.v + int64_t(hkv) * a.c.sv[1];

  int b, start, u, end;  // the run's sequence, its first unit, the run's units [u, end)
  int per = 0;
  bool once = false;
  if (a.parts == 0) {
    b = part;
    start = u = 0;
    end = 1;
  } else {
    const Units first = units_from(a, 0);
    const int total = total_units(a, first);
    per = units_per_part(total, total > a.many_units ? a.parts : a.few, a.least);
    once = total > a.keep_units;
    if (int64_t(part) * per >= total) return;
    u = part * per;
    end = imin(total, u + per);
    find_unit(a, first, u, b, start);
  }

  Wave<E, D, RT> w;
  // (b < B and v0 >= 0 hold by themselves, and so do the bounds in pieces_of, unless lens change under a running call: then the
  // results mean nothing, but no access leaves the tensors)
  while (u < end && b < a.c.B) {
    const Visible vis = visible(seq_len(a.c, b), a.W, a.S);
    const int units = paged_units(vis.count);
    if (a.parts == 0) end = units;
    const int stop = imin(end, start + units);
    const bool whole = u == start && stop == start + units;
    if (a.parts && stream == 0 && tid == 0) {  // for the second launch
      if (u == start) a.starts[b] = start;
      if (u == 0) a.starts[a.c.B] = per;
    }
    const int v0 = imax(0, (u - start) * kPagedUnit), v1 = imin(vis.count, (stop - start) * kPagedUnit);
#pragma unroll
    for (int x = 0; x < RT; ++x) {
      const int h = h0 + 16 * x + r;
      w.load_q(x, a.q + int64_t(b) * a.sq[0] + int64_t(hkv * a.G + (h < a.G ? h : 0)) * a.sq[1], h < a.G);
    }
    w.reset();
    const int* table = a.c.table + int64_t(b) * a.c.table_stride;
    // The wave's tiles are every 4th (8th) of the run.  A lane works out the place of one of the 64 keys of two of them (a
    // pair): its page is asked for one pair ahead of its offsets, which go to LDS just before the loads that use them.
    const int n = v1 - v0, tiles = (n + kTile - 1) / kTile, mine = (tiles - wave + WAVES - 1) / WAVES;
    auto ask = [&](int p, int& slot) {
      const int v = (wave + WAVES * (2 * p + (lane >> 5))) * kTile + (lane & 31);
      slot = 0;
      if (v >= n) return -1;
      const int key = visible_key(vis, v0 + v), pi = page_of(a.c.div, key);
      slot = key - pi * a.c.page_size;
      return table[pi];
    };
    // (bit l: the key of lane l is on a page)
    auto place = [&](int p, int page, int slot) -> unsigned long long {
      const bool ok = page >= 0 && page < a.c.pages;
      if (!ok) page = slot = 0;
      sh.wave[wave].off[p & 1].k[lane] = int64_t(page) * a.c.sk[0] + int64_t(slot) * a.c.sk[2];
      sh.wave[wave].off[p & 1].v[lane] = int64_t(page) * a.c.sv[0] + int64_t(slot) * a.c.sv[2];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (the wave's other lanes read them)
      return __ballot(ok);
    };
    auto logits = [&](int i) {  // of the wave's i-th tile
      const int at = v0 + (wave + WAVES * i) * kTile;
      return [=, &a](int x) -> float* {
        const int h = h0 + 16 * x + r;
        if (!a.sums || h >= a.G) return nullptr;
        return a.logits + (((int64_t(hkv) * a.c.B + b) * a.max_units + at / kPagedUnit) * a.G + h) * kPagedUnit + at % kPagedUnit + 8 * j;
      };
    };
    auto walk = [&](auto mode) {
      constexpr bool ONCE = decltype(mode)::value;
      constexpr int AHEAD = Tile<E, D>::AHEAD;
      Tile<E, D> t[AHEAD];
      unsigned long long live = 0;
      int slot, page = ask(0, slot);
      auto load = [&](Tile<E, D>& to, int i, bool first) {  // the wave's i-th tile; `first` of its pair
        if (i >= mine) return;
        const int p = i >> 1;
        if (first) {
          live = place(p, page, slot);
          page = ask(p + 1, slot);
        }
        const auto& off = sh.wave[wave].off[p & 1];
        w.template load<ONCE>(to, kb, vb, off.k + (first ? 0 : kTile), off.v + (first ? 0 : kTile), uint32_t(first ? live : live >> 32));
      };
#pragma unroll
      for (int d = 0; d < AHEAD; ++d) load(t[d], d, d % 2 == 0);
      for (int i = 0; i < mine; i += AHEAD) {
#pragma unroll
        for (int d = 0; d < AHEAD; ++d) {
          if (i + d < mine) w.step(t[d], a.c2, sh.wave[wave].k, logits(i + d));
          load(t[d], i + d + AHEAD, d % 2 == 0);
        }
      }
    };
    if (mine > 0) {
      if (once) walk(Yes{});
      else walk(No{});
    }

    // the waves' results, in wave order
#pragma unroll
    for (int x = 0; x < RT; ++x) {
      __syncthreads();
      const float l = quarters_sum(w.l[x]);
      if (j == 0) {
        sh.m[wave][r] = w.m[x];
        sh.l[wave][r] = l;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < NC; ++c) sh.o[wave][r][(4 * j + i) * NC + c] = w.acc[x][c][i];
      __syncthreads();
      for (int y = tid; y < 256; y += 64 * WAVES) {
        const int oh = y >> 4, od = (y & 15) * NC, h = h0 + 16 * x + oh;  // this thread's head and dims
        if (h >= a.G) continue;
        float m = kNegInf;
#pragma unroll
        for (int v = 0; v < WAVES; ++v) m = fmaxf(m, sh.m[v][oh]);
        const float ref = m == kNegInf ? 0.f : m;
        float sum = 0.f, o[NC] = {};
#pragma unroll
        for (int v = 0; v < WAVES; ++v) {
          const float f = fast_exp2(sh.m[v][oh] - ref);
          sum += f * sh.l[v][oh];
#pragma unroll
          for (int c = 0; c < NC; ++c) o[c] += f * sh.o[v][oh][od + c];
        }
        const int hq = hkv * a.G + h;
        if (whole) {
          float ls = sum, scale = 1.f;
          if (a.sinks) {
            const float sink = a.sinks[hq] * kLog2e, top = fmaxf(m, sink);
            if (top != kNegInf) {
              scale = fast_exp2(ref - top);
              ls = (m == kNegInf ? 0.f : sum * scale) + fast_exp2(sink - top);
              m = top;
            }
          }
          const float inv = ls == 0.f || sum == 0.f ? 0.f : scale * a.oscale / ls;
#pragma unroll
          for (int c = 0; c < NC; ++c) o[c] = sum == 0.f ? 0.f : o[c] * inv;
          store_out<E, NC>(a.o + int64_t(b) * a.so[0] + int64_t(hq) * a.so[1] + od * E::EB, o);
          if (a.sums && (y & 15) == 0)
            *reinterpret_cast<f32x2*>(a.norm + 2 * (int64_t(b) * a.Hq + hq)) = f32x2{m == kNegInf ? 0.f : m, ls == 0.f ? 0.f : 1.f / ls};
        } else {
          const int64_t slot = (int64_t(hkv) * a.row_tiles + h / 16) * a.parts * 2 + part_slot(part, per, start);
          float* po = a.part_o + (slot * 16 + oh) * D + od;
#pragma unroll
          for (int c = 0; c < NC; ++c) po[c] = o[c];
          if ((y & 15) == 0) {
            a.part_ml[slot * 32 + oh] = m;
            a.part_ml[slot * 32 + 16 + oh] = sum;
          }
        }
      }
    }
    __syncthreads();
    u = stop;
    start += units;
    ++b;
  }
}

// ---- the second launch ---------------------------------------------------------------------------
// Pieces of sequence b: those of the parts [first, last].
struct Pieces {
  int first, last, start, per;
};
__device__ __forceinline__ Pieces pieces_of(const PagedAttnArgs& a, int b) {
  Pieces p{0, 0, 0, 0};
  if (a.parts == 0) return p;
  p.start = a.starts[b];
  p.per = imax(1, a.starts[a.c.B]);
  p.first = imin(imax(p.start / p.per, 0), a.parts - 1);
  p.last = imin((p.start + units_of(a, b) - 1) / p.per, a.parts - 1);
  return p;
}

// Query head hq of sequence b, if it was cut: its pieces' results.  D / 4 threads take a piece; every thread adds its
// pieces in order, then the groups of threads are added in order.
template <typename E, int D, int THREADS>
__device__ __forceinline__ void join_head(const PagedAttnArgs& a, int b, int hq, float* smem) {
  constexpr int T = D / 4, GROUPS = THREADS / T;
  const Pieces ps = pieces_of(a, b);
  if (ps.first >= ps.last) return;
  const int hkv = hq / a.G, h = hq % a.G, oh = h % 16;
  const int64_t base = int64_t(hkv * a.row_tiles + h / 16) * a.parts * 2;
  const int tid = threadIdx.x, lane = tid & 63, group = tid / T, d = tid % T * 4;
  float m = kNegInf;
  for (int p = ps.first + lane; p <= ps.last; p += 64) m = fmaxf(m, a.part_ml[(base + part_slot(p, ps.per, ps.start)) * 32 + oh]);
#pragma unroll
  for (int x = 32; x >= 1; x >>= 1) m = fmaxf(m, __shfl_xor(m, x));
  const float sink = a.sinks ? a.sinks[hq] * kLog2e : kNegInf, top = fmaxf(m, sink), ref = top == kNegInf ? 0.f : top;
  float sum = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int p = ps.first + group; p <= ps.last; p += GROUPS) {
    const int64_t slot = base + part_slot(p, ps.per, ps.start);
    const float f = fast_exp2(a.part_ml[slot * 32 + oh] - ref);
    const f32x4 x = *reinterpret_cast<const f32x4*>(a.part_o + (slot * 16 + oh) * D + d);
    sum += f * a.part_ml[slot * 32 + 16 + oh];
    o += f * x;
  }
  // [group][D], [group] sums
#pragma unroll
  for (int i = 0; i < 4; ++i) smem[group * D + d + i] = o[i];
  if (d == 0) smem[GROUPS * D + group] = sum;
  __syncthreads();
  for (int i = tid; i < D; i += THREADS) {
    float x = 0.f, s = 0.f;
#pragma unroll 8
    for (int g = 0; g < GROUPS; ++g) {
      x += smem[g * D + i];
      s += smem[GROUPS * D + g];
    }
    const float ls = s + (sink == kNegInf ? 0.f : fast_exp2(sink - ref));
    const float out[1] = {s == 0.f ? 0.f : x * (a.oscale / ls)};
    store_out<E, 1>(a.o + int64_t(b) * a.so[0] + int64_t(hq) * a.so[1] + i * E::EB, out);
  }
}

// sums[b, hkv, key] += sum over the group's heads of 2^(logit - maximum) / sum: a thread takes keys, so there is no order to
// choose and no atomic.
constexpr int kSumKeys = 1024;
constexpr int kSumHeads = 16;  // heads at a time: 16 threads work out a head's maximum and the reciprocal of its sum
__device__ __forceinline__ void add_weights(const PagedAttnArgs& a, int b, int hkv, int chunk, float* smem) {
  const Visible vis = visible(seq_len(a.c, b), a.W, a.S);
  if (chunk * kSumKeys >= vis.count) return;
  // (a thread past the last key reads the last unit's room and writes nothing)
  const int v0 = chunk * kSumKeys + 4 * int(threadIdx.x), vr = imin(v0, (vis.count - 1) / 4 * 4);
  const float* x = a.logits + ((int64_t(hkv) * a.c.B + b) * a.max_units + vr / kPagedUnit) * a.G * kPagedUnit + vr % kPagedUnit;
  float* out = a.sums + int64_t(b) * a.ssum[0] + int64_t(hkv) * a.ssum[1];
  float w[4] = {0.f, 0.f, 0.f, 0.f}, old[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) old[c] = out[visible_key(vis, imin(v0 + c, vis.count - 1))];
  const Pieces ps = pieces_of(a, b);
  for (int g0 = 0; g0 < a.G; g0 += kSumHeads) {
    const int ng = imin(kSumHeads, a.G - g0);
    constexpr int HELD = 8;  // scores asked for before those are known
    f32x4 s[HELD];
#pragma unroll
    for (int i = 0; i < HELD; ++i) s[i] = *reinterpret_cast<const f32x4*>(x + (g0 + imin(i, ng - 1)) * kPagedUnit);
    if (g0) __syncthreads();
    const int g = g0 + int(threadIdx.x) / 16, sub = threadIdx.x & 15;
    if (g < a.G) {
      const int hq = hkv * a.G + g;
      float top, inv;
      if (ps.first >= ps.last) {
        const f32x2 v = *reinterpret_cast<const f32x2*>(a.norm + 2 * (int64_t(b) * a.Hq + hq));
        top = v[0];
        inv = v[1];
      } else {
        const float* ml = a.part_ml + int64_t(hkv * a.row_tiles + g / 16) * a.parts * 2 * 32 + g % 16;
        float m = a.sinks ? a.sinks[hq] * kLog2e : kNegInf;
        const float sink = m;
        for (int p = ps.first + sub; p <= ps.last; p += 16) m = fmaxf(m, ml[part_slot(p, ps.per, ps.start) * 32]);
#pragma unroll
        for (int y = 8; y >= 1; y >>= 1) m = fmaxf(m, __shfl_xor(m, y));
        const float ref = m == kNegInf ? 0.f : m;
        float l = sub == 0 && sink != kNegInf ? fast_exp2(sink - ref) : 0.f;
        for (int p = ps.first + sub; p <= ps.last; p += 16) {
          const int slot = part_slot(p, ps.per, ps.start) * 32;
          l += fast_exp2(ml[slot] - ref) * ml[slot + 16];
        }
#pragma unroll
        for (int y = 8; y >= 1; y >>= 1) l += __shfl_xor(l, y);
        top = ref;
        inv = l == 0.f ? 0.f : 1.f / l;
      }
      if (sub == 0) {
        smem[g - g0] = top;
        smem[kSumHeads + g - g0] = inv;
      }
    }
    __syncthreads();
    auto add = [&](f32x4 q, int i) {
      const float top = smem[i], inv = smem[kSumHeads + i];
#pragma unroll
      for (int c = 0; c < 4; ++c) w[c] += q[c] == kNegInf ? 0.f : fast_exp2(q[c] - top) * inv;
    };
#pragma unroll
    for (int i = 0; i < HELD; ++i)
      if (i < ng) add(s[i], i);
    for (int i = HELD; i < ng; ++i) add(*reinterpret_cast<const f32x4*>(x + (g0 + i) * kPagedUnit), i);
  }
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (v0 + c < vis.count) out[visible_key(vis, v0 + c)] = old[c] + w[c];
}

// Workgroups [0, joins) join heads, the ones behind them add weights.
template <typename E, int D, int THREADS>
__global__ __launch_bounds__(THREADS) void paged_finish_kernel(const PagedAttnArgs a, unsigned joins) {
  __shared__ float smem[THREADS * 4 + 64];
  if (blockIdx.x < joins) {
    join_head<E, D, THREADS>(a, blockIdx.x / a.Hq, blockIdx.x % a.Hq, smem);
    return;
  }
  if constexpr (THREADS == kThreads) {
    const unsigned i = blockIdx.x - joins, chunks = unsigned((a.max_units * kPagedUnit + kSumKeys - 1) / kSumKeys);
    add_weights(a, int(i / chunks / unsigned(a.c.Hkv)), int(i / chunks % unsigned(a.c.Hkv)), int(i % chunks), smem);
  }
}

template <typename E, int D>
hipError_t run(const PagedAttnArgs& a, hipStream_t s) {
  const unsigned B = unsigned(a.c.B), parts = a.parts ? unsigned(a.parts) : B;
  const unsigned streams = unsigned(a.c.Hkv) * unsigned((a.row_tiles + a.rt - 1) / a.rt);
  const auto launch = [&](auto kernel, int waves) { hipLaunchKernelGGL(kernel, dim3(streams * parts), dim3(64 * waves), 0, s, a); };
  if (a.rt == 2) {
    if constexpr (paged_pairs(D, E::CB)) {
      if constexpr (paged_eight(D, E::CB, 2)) {
        if (a.waves == 8) launch(paged_attn_kernel<E, D, 8, 2>, 8);
      }
      if (a.waves != 8) launch(paged_attn_kernel<E, D, 4, 2>, 4);
    }
  } else if (a.waves == 8) {
    if constexpr (paged_eight(D, E::CB, 1)) launch(paged_attn_kernel<E, D, 8, 1>, 8);
  } else if (a.waves == 1) {
    launch(paged_attn_kernel<E, D, 1, 1>, 1);
  } else {
    launch(paged_attn_kernel<E, D, 4, 1>, 4);
  }
  const hipError_t e = hipGetLastError();
  const unsigned joins = a.parts ? unsigned(a.Hq) * B : 0u;
  const unsigned adds = a.sums ? unsigned((a.max_units * kPagedUnit + kSumKeys - 1) / kSumKeys) * unsigned(a.c.Hkv) * B : 0u;
  if (e != hipSuccess || joins + adds == 0) return e;
  // a wave a head where the sequences have few pieces each
  if (adds == 0 && a.parts <= 4 * a.c.B) hipLaunchKernelGGL((paged_finish_kernel<E, D, 64>), dim3(joins), dim3(64), 0, s, a, joins);
  else hipLaunchKernelGGL((paged_finish_kernel<E, D, kThreads>), dim3(joins + adds), dim3(kThreads), 0, s, a, joins);
  return hipGetLastError();
}

template <typename E>
hipError_t run_d(const PagedAttnArgs& a, int D, hipStream_t s) {
  if constexpr (E::CB == 1) return D == 64 ? run<E, 64>(a, s) : run<E, 128>(a, s);
  else return D == 16 ? run<E, 16>(a, s) : D == 32 ? run<E, 32>(a, s) : D == 64 ? run<E, 64>(a, s) : run<E, 128>(a, s);
}

}  // namespace

hipError_t launch_paged_attention(const PagedAttnArgs& a, int dtype, int cache, int D, hipStream_t s) {
  if (dtype == FA_DTYPE_F32) return run_d<PF32>(a, D, s);
  if (dtype == FA_DTYPE_BF16) return cache == FA_DTYPE_FP8_E4M3 ? run_d<PBF16Q8>(a, D, s) : run_d<PBF16>(a, D, s);
  return cache == FA_DTYPE_FP8_E4M3 ? run_d<PF16Q8>(a, D, s) : run_d<PF16>(a, D, s);
}

}  // namespace fa
