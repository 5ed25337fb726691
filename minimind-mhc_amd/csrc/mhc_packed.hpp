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
__device__ __forceinline__ void packed_bounds(const int* cu, int B, int T, int M, int seq, int tile, const int* cu_o,
                                              int To, const int* used_t, const int* used_o, PackedTile& t,
                                              PackedKeys& o) {
  // all loads of the sequence's bounds before the first use of one
  const bool in = seq < B;
  const int next = in ? seq + 1 : seq, at = in ? seq : 0;
  const int s0 = cu[seq], s1 = cu[next], o0 = cu_o[seq], o1 = cu_o[next];
  const int ut = used_t && in ? used_t[at] : 0x7fffffff, uo = used_o && in ? used_o[at] : 0x7fffffff;
  t.seq = seq;
  t.start = seq == 0 ? 0 : min(max(s0, 0), T);
  t.end = max(in ? min(max(s1, 0), T) : T, t.start);
  t.first = t.start + min(tile, (T - t.start) / M + 1) * M;
  o.start = seq == 0 ? 0 : min(max(o0, 0), To);
  o.len = in ? min(max(uo, 0), max(min(max(o1, 0), To) - o.start, 0)) : 0;
  t.used = in ? min(max(ut, 0), t.end - t.start) : 0;
}
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
  packed_bounds(cu, B, T, M, lo, tile - (seq_start(cu, lo, T) / M + lo), cu_o, To, used_t, used_o, t, o);
}

// The same by rank: the tiles of all sequences, those with the most work first (the last
// of a sequence's query tiles; backward: the first of its key tiles), so that the longest chains
// start at once and the short ones fill the ends.  A tile's level is its number in the
// sequence (`past`: and the tiles of keys before it); the rank's level is found by counting the
// tiles from each level up, four sequences a lane.  For up to 256 sequences; more of them
// even out by themselves.
constexpr int kRankSeqs = 256;
template <bool FIRST>
__device__ __forceinline__ void packed_rank(const int* cu, int B, int T, int M, int tiles, int rank, const int* cu_o,
                                            int To, const int* used_t, const int* used_o, PackedTile& t,
                                            PackedKeys& o) {
  if (B > kRankSeqs || T > 1 << 28) {
    packed_find(cu, B, T, M, FIRST ? rank : tiles - 1 - rank, cu_o, To, used_t, used_o, t, o);
    return;
  }
  constexpr int C = kRankSeqs / 64;
  const int lane = __lane_id();
  int start[C], len[C], other[C], olen[C], used[C];
  float n[C], past[C];  // small whole numbers, exact in fp32
  float most = 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int i = c * 64 + lane;
    start[c] = len[c] = other[c] = olen[c] = used[c] = 0;
    n[c] = past[c] = 0.f;
    if (c * 64 < B && i < B) {
      const int s0 = cu[i], s1 = cu[i + 1], o0 = cu_o[i], o1 = cu_o[i + 1];  // all before the first use
      const int ut = used_t ? used_t[i] : 0x7fffffff, uo = used_o ? used_o[i] : 0x7fffffff;
      start[c] = i == 0 ? 0 : min(max(s0, 0), T);
      len[c] = max(min(max(s1, 0), T) - start[c], 0);
      used[c] = min(max(ut, 0), len[c]);
      other[c] = i == 0 ? 0 : min(max(o0, 0), To);
      olen[c] = min(max(uo, 0), max(min(max(o1, 0), To) - other[c], 0));
      n[c] = (float)((len[c] + M - 1) / M);
      if (!FIRST) past[c] = (float)(max(olen[c] - len[c], 0) / M);
      most = fmaxf(most, n[c] + past[c]);
    }
  }
  auto count = [&](float level) {  // tiles of that level and above
    float x = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (c * 64 < B) x += fmaxf(n[c] + past[c] - fmaxf(level, past[c]), 0.f);
    return __builtin_amdgcn_readfirstlane((int)wave_sum(x));
  };
  const int total = count(0.f);
  if (rank >= total) {  // rows behind the last sequence
    packed_bounds(cu, B, T, M, B, rank - total, cu_o, To, used_t, used_o, t, o);
    return;
  }
  int lo = 0, hi = __builtin_amdgcn_readfirstlane((int)wave_max(most)), above = 0;  // count(lo) > rank >= count(hi)
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2, x = count((float)mid);
    if (x > rank) {
      lo = mid;
    } else {
      hi = mid;
      above = x;
    }
  }
  int k = rank - above;  // which of the level's tiles
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const bool has = past[c] <= (float)lo && (float)lo < past[c] + n[c];
    const uint64_t mask = __ballot(has);
    const int here = __popcll(mask);
    if (k >= 0 && k < here) {
      const uint64_t me = __ballot(has && __popcll(mask & ((1ull << lane) - 1)) == k);
      const int l = __ffsll((unsigned long long)me) - 1;
      const int level = lo - (int)__builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, past[c]), l));
      const int num = (int)__builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, n[c]), l));
      t.seq = c * 64 + l;
      t.start = __builtin_amdgcn_readlane(start[c], l);
      t.end = t.start + __builtin_amdgcn_readlane(len[c], l);
      t.used = __builtin_amdgcn_readlane(used[c], l);
      t.first = t.start + (FIRST ? num - 1 - level : level) * M;
      o.start = __builtin_amdgcn_readlane(other[c], l);
      o.len = __builtin_amdgcn_readlane(olen[c], l);
    }
    k -= here;
  }
}
// Whether a workgroup is two halves of four waves that share its tiles: where the launch has
// about one workgroup a CU, so the longest chain of tiles sets its time.  Forward: one sequence
// of 4096 tokens, 8 / 4 heads of 96 (264 workgroups), 71 us and 91 without; 12 sequences of 8192
// tokens together (564), 52 and 47.  dK and dV of those in one range (308): 102 and 139; of 3
// sequences of 16001 tokens, 8 heads of 64 (1032): 372 and 350.
inline bool packed_halves(unsigned workgroups) { return workgroups <= (unsigned)device_cus() * 5 / 4; }
// Tile numbers of T rows in B sequences.
__host__ __device__ inline int64_t packed_tiles(int64_t T, int64_t B, int M) { return T / M + B + 1; }

// An operand of ones: its product with the probabilities sums them on the matrix cores, over
// all lanes at once, and sums what the outputs are formed of, the rounded ones.
template <bool F16>
__device__ __forceinline__ U32x4 packed_ones() {
  const uint32_t w = F16 ? 0x3c003c00u : 0x3f803f80u;
  return U32x4{{w, w, w, w}};
}

// A tile of ROWS rows of one head in LDS, filled by direct-to-LDS loads: a wave's load
// writes 64 lanes x 16 bytes in a row, so rows lie without padding and their 16-byte slots are
// permuted instead (on the global side), so that 16 rows of one column spread over all 64 banks:
// an exclusive or with bits of the row where 8 or 16 slots make the row, a rotation by row / 4
// where 12 do.  The transposing reads (4 rows of 32 bytes a lane group) are not free of conflicts: two
// of a group's rows meet in the same 32 bytes modulo 256 at head_dim 64 and 128, two groups
// overlap by half at 96.  The counters show conflicts in 25 to 33% of the LDS's cycles there, and in 46 to 50%.
template <int HD>
__device__ __forceinline__ int tile_slot(int row, int slot) {
  if constexpr (HD == 64) return slot ^ ((row >> 1) & 7);
  else if constexpr (HD == 128) return slot ^ (row & 15);
  else return (slot + (row >> 2)) % 12;
}
template <int HD>
__device__ __forceinline__ int tile_column(int row, int place) {  // the slot that lies there
  if constexpr (HD == 96) return (place + 36 - (row >> 2)) % 12;  // 36: no negative remainder up to row 147
  else return tile_slot<HD>(row, place);
}
// `N` of the tile's 1 KiB units, from unit u0 on, by this wave.
template <int HD, int N>
struct TileLoader {
  uint32_t off[N];  // this lane's byte offset in the tile's rows
  __device__ __forceinline__ void init(int u0, int64_t st) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = (u0 + i) * 64 + __lane_id(), row = at / (HD / 8);
      off[i] = (uint32_t)(row * st + tile_column<HD>(row, at % (HD / 8)) * 8) * 2;
    }
  }
  // p: the tile's first row; left >= 1: rows that exist from there on (rows behind them
  // become copies of the last, uniform branch).
  __device__ __forceinline__ void issue(uint16_t* lds, const uint16_t* p, int u0, int64_t st, int rows, int left) const {
    const char* base = reinterpret_cast<const char*>(p);
    char* to = reinterpret_cast<char*>(lds) + u0 * 1024;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      uint32_t o = off[i];
      if (left < rows) {
        const int at = (u0 + i) * 64 + __lane_id(), row = at / (HD / 8);
        o = (uint32_t)(min(row, left - 1) * st + tile_column<HD>(row, at % (HD / 8)) * 8) * 2;
      }
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(base + o),
                                       (__attribute__((address_space(3))) void*)(to + i * 1024), 16, 0, 0);
    }
  }
};
// At most N direct-to-LDS loads of this wave in flight, and no LDS read; then every wave's.
template <int N>
__device__ __forceinline__ void tile_wait() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"i"(N) : "memory");
}
__device__ __forceinline__ void tile_barrier() {
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
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

// A lane's reads of a tile: 16 bytes of row 16 st + r at columns 32 c + 8 g (an operand
// whose rows are the tile's), and columns 16 d + r of the rows 32 h + 16 (j / 4) + 4 g + j % 4
// (an operand whose rows are the tile's columns; the rows are in the order in which a product
// leaves its results to a lane).
template <int HD>
struct TileReads {
  static constexpr int NK = HD == 96 ? 3 : HD / 32, NV = HD == 96 ? 6 : HD / 16;
  int k[NK], v[NV];  // elements
  __device__ __forceinline__ void init(int r, int g) {
    if constexpr (HD == 96) {  // rotated by row / 4: constants of the column and of the row add up modulo 12
#pragma unroll
      for (int i = 0; i < NK; ++i) k[i] = r * HD + (4 * i + g + (r >> 2)) % 12 * 8;
#pragma unroll
      for (int i = 0; i < NV; ++i) v[i] = (4 * g + (r >> 2)) * HD + (2 * i + ((r & 3) >> 1) + g) % 12 * 8 + 4 * (r & 1);
    } else {  // bits of the lane's part of the row only
#pragma unroll
      for (int i = 0; i < NK; ++i) k[i] = r * HD + tile_slot<HD>(r, 4 * i + g) * 8;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        v[i] = (4 * g + (r >> 2)) * HD + tile_slot<HD>(4 * g + (r >> 2), 2 * i + ((r & 3) >> 1)) * 8 + 4 * (r & 1);
    }
  }
  __device__ __forceinline__ U32x4 row16(const uint16_t* t, int st, int c) const {
    return *reinterpret_cast<const U32x4*>(t + k[HD == 96 ? (c + st) % 3 : c] + st * 16 * HD);
  }
  __device__ __forceinline__ U32x4 columns32(const uint16_t* t, int h, int d) const {
    U32x4 o;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const u32x2_v w = lds_tr4(t + v[HD == 96 ? (d + 2 * q + 4 * h) % 6 : d] + (h * 32 + q * 16) * HD);
      o.v[2 * q] = w.x;
      o.v[2 * q + 1] = w.y;
    }
    return o;
  }
};

}  // namespace mhc
