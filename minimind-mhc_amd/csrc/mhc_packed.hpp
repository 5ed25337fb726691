// Packed sequences: what the attention kernels over them share.
#pragma once

#include "mhc_internal.hpp"

namespace mhc {

constexpr float kPackedLog2e = 1.44269504088896340736f;
// Below every score of finite inputs; finite, so that the difference of two maxima of rows
// that have seen no key yet is 0 and no NaN.
constexpr float kNoScore = -3e38f;

// The maximum a row's sums are taken under is raised only when a score exceeds it by more
// than 2^8 in the exponent: fp32 sums lose nothing by that, and most tiles rescale nothing.
constexpr float kPackedLazyMax = 8.f;
// fp16 probabilities are taken 2^6 times as large (the maximum is kept that much lower): at
// most 2^14 with the lazy maximum, and full precision down to 2^-20 of the largest.
template <bool F16>
constexpr float packed_head = F16 ? 6.f : 0.f;

typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_v __attribute__((ext_vector_type(2)));

__device__ __forceinline__ U32x4 ld16(const void* p) { return *static_cast<const U32x4*>(p); }
__device__ __forceinline__ float exp2_f(float x) { return __builtin_amdgcn_exp2f(x); }

// Row where sequence i of a packed tensor of T rows begins.  The bounds are device data
// that no host check has seen: clamped, they cannot lead out of the tensor.
__device__ __forceinline__ int seq_start(const int* cu, int i, int T) {
  return i == 0 ? 0 : min(max(cu[i], 0), T);
}

// log2 of a row's sum of exponentials, for the backward pass: infinite for a row without
// keys, whose probabilities then come out 0.
__device__ __forceinline__ float packed_lse(float m, float l) {
  return l == 0.f ? __builtin_inff() : m + __builtin_amdgcn_logf(l);
}
// Two outputs, rounded once, and (rest set, where a backward pass follows) what the rounding
// took from them: D = G . O is formed from both.  With the rounded output alone the error of
// D, the same for all keys of a row, was most of the error of dQ and dK (2.2e-3 of their
// size at short lengths, one rounding being 1.7e-3).
template <bool F16>
__device__ __forceinline__ uint32_t round2(float a, float b, uint32_t* rest) {
  const uint32_t w = pack2<F16>(a, b);
  if (rest) *rest = pack2<F16>(a - elem_lo<F16>(w), b - elem_hi<F16>(w));
  return w;
}
__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, dpp_f<kDppXor1>(v));
  v = fmaxf(v, dpp_f<kDppXor2>(v));
  v = fmaxf(v, dpp_f<kDppHalfMirror>(v));
  v = fmaxf(v, dpp_f<kDppRowMirror>(v));
  v = fmaxf(v, xor_lane16(v));
  return fmaxf(v, xor_lane32(v));
}

// A tile of M rows of one packed sequence.  Sequence i owns the tile numbers from
// start(i) / M + i on: enough for its rows wherever it starts, and found without a sum
// over the sequences before it.  The rows behind the last sequence are one more "sequence"
// (number B).  Every lane of the wave takes part: 64 bounds are looked at a step.
// packed_find also gives the sequence's rows in the other tensor (cu_o, To rows); used_t and
// used_o (or null) say how many of the rows are in use.
struct PackedTile {
  int seq, first, end;  // sequence, first row of the tile, end of the sequence's rows
  int start;            // first row of the sequence
  int used;             // its rows in use
};
// The other tensor's rows of a sequence: first row, how many (of them in use), none for the
// rows behind the last sequence.
struct PackedKeys {
  int start, len;
};
__device__ __forceinline__ void packed_find(const int* cu, int B, int T, int M, int tile, const int* cu_o, int To,
                                            const int* used_t, const int* used_o, PackedTile& t, PackedKeys& o) {
  const int lane = __lane_id();
  int lo = 0, hi = B + 1;
  while (hi - lo > 1) {
    const int step = (hi - lo - 1 + 63) / 64;
    const int64_t at = lo + (int64_t)(lane + 1) * step;
    const bool below = at < hi && seq_start(cu, (int)(at < hi ? at : lo), T) / M + at <= tile;
    const int n = __popcll(__ballot(below));
    lo += n * step;
    hi = min(hi, lo + step);
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  // all loads of the sequence's bounds before the first use of one
  const bool in = lo < B;
  const int next = in ? lo + 1 : lo, at = in ? lo : 0;
  const int s0 = cu[lo], s1 = cu[next], o0 = cu_o[lo], o1 = cu_o[next];
  const int ut = used_t && in ? used_t[at] : 0x7fffffff, uo = used_o && in ? used_o[at] : 0x7fffffff;
  t.seq = lo;
  t.start = lo == 0 ? 0 : min(max(s0, 0), T);
  t.end = max(in ? min(max(s1, 0), T) : T, t.start);
  t.first = t.start + (tile - (t.start / M + lo)) * M;
  o.start = lo == 0 ? 0 : min(max(o0, 0), To);
  o.len = in ? min(max(uo, 0), max(min(max(o1, 0), To) - o.start, 0)) : 0;
  t.used = in ? min(max(ut, 0), t.end - t.start) : 0;
}
// Tile numbers of T rows in B sequences.
inline int64_t packed_tiles(int64_t T, int64_t B, int M) { return T / M + B + 1; }

// An operand of ones: its product with the probabilities sums them on the matrix cores, over
// all lanes at once, and sums what the outputs are formed of, the rounded ones.
template <bool F16>
__device__ __forceinline__ U32x4 packed_ones() {
  const uint32_t w = F16 ? 0x3c003c00u : 0x3f803f80u;
  return U32x4{{w, w, w, w}};
}

// A tile of up to `rows` rows (stride `st` elements) from row r0 on, of a tensor's head whose
// first row is at p and which has n rows: 16 bytes at the byte offset `off` (of row and
// column) in it.  The descriptor's size cuts off the rows behind the last, which read as
// zeros: no comparison per lane, and no garbage beside probabilities of 0.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_rsrc(const uint16_t* p, int64_t st, int64_t r0, int n, int rows,
                                                            int hd) {
  const int left = (int)min((int64_t)rows, n - r0);
  return make_rsrc(p + r0 * st, left > 0 ? (uint32_t)(((left - 1) * st + hd) * 2) : 0u);
}

// The transposing LDS load: the 16 lanes of a group point at 4 rows x 16 columns, four
// columns a lane (lane r at row r / 4, column 4 (r % 4)), and lane r gets column r.
__device__ __forceinline__ u32x2_v lds_tr4(const uint16_t* p) {
  const s16x4_t w = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) s16x4_t*)const_cast<uint16_t*>(p));
  return __builtin_bit_cast(u32x2_v, w);
}

#define MHC_PACKED_HD(fn, a, s)                                          \
  switch (a.head_dim) {                                                  \
    case 64: return a.f16 ? fn<true, 64>(a, s) : fn<false, 64>(a, s);    \
    case 96: return a.f16 ? fn<true, 96>(a, s) : fn<false, 96>(a, s);    \
    case 128: return a.f16 ? fn<true, 128>(a, s) : fn<false, 128>(a, s); \
    default: return hipErrorInvalidValue;                                \
  }

}  // namespace mhc
