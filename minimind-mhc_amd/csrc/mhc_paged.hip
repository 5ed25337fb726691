// Attention of new tokens over a cache of pages: single tokens, drafted trees, chunks of prompts.
// Key x of a sequence lies in page table[x / page], row x % page; a page has 2^s >= 16 rows. The
// new rows' own keys are stored already, behind the `past` ones before them.
//   S_tj = scale q_t . k_j  for j < past, and for j - past a row of the same sequence that t sees
//   (causal: up to its own; a tree: its bits),  O_t = sum_j softmax(S_t)_j v_j
// 16-bit tensors, fp32 scores, sums and outputs.  The probabilities are a product's operand in two parts: rounded to
// 16 bits, and what the rounding took.  With the first part alone the outputs' error was 1.4 times that of their own
// rounding.  The second costs nothing up to 32 rows a sequence and kv head, where the keys' bytes bound the launch, and
// 1 to 24% above (8 trees of 30, heads of 128, 40.1 -> 40.4 us; chunks of 500, heads of 64, 45 -> 55; one tree of 64 over
// 65001 keys 58 -> 70).  Each product with the second part right behind that with the first: apart, two
// dozen registers more, and 3 to 5% slower at head_dim 128.  The outputs are rounded once.
#include "mhc_packed.hpp"

namespace mhc {
namespace {

constexpr int kPagedStages = 2;  // tiles of a ring: one in use, one in flight
// Up to so many sequences, workgroups are dealt out by the keys' lengths; of more, each block of rows is one
// workgroup over all of its keys.  Single tokens, 8 / 4 heads of 96, over 233 to 700 keys: 256 sequences 39.4 us, 257
// 36.9 (with 1 kv head, which leaves the chip half empty, 20.0 and 23.9).  A long one among short ones is
// what that costs: 65001 keys beside 100 each, 256 sequences 64 us, 257 1624.
constexpr int kPagedSeqs = 256;

// What a workgroup does: rows `first` and on (row = token * rep + head of the group) of a
// sequence, over part `split` of `splits` of the keys they see.
struct PagedUnit {
  int seq, start, n, past, len;
  int first, split, splits, blocks, base;
};
struct PagedSeq {
  int start, n, past, len;
};
__device__ __forceinline__ PagedSeq paged_seq(const PagedAttnArgs& a, int i, int s0, int s1, int past) {
  PagedSeq q;
  const int64_t cap = a.pages > 0 ? (int64_t)a.width << a.page_shift : 0;
  q.start = i == 0 ? 0 : min(max(s0, 0), a.Tq);
  q.n = max(min(max(s1, 0), a.Tq) - q.start, 0);
  q.past = (int)min((int64_t)max(past, 0), cap);
  q.len = (int)min((int64_t)q.past + q.n, cap);
  return q;
}
__device__ __forceinline__ int wave_scan(int v) {  // over the lanes up to this one
  const int lane = __lane_id();
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int o = __shfl_up(v, d);
    if (lane >= d) v += o;
  }
  return v;
}
// Unit number w of a kv head.  The keys of all sequences, times their blocks of rows, are cut
// into about a.slots ranges of the same length; a sequence shorter than one is one unit a block.
// The blocks of one range are neighbours.  Behind the sequences' units come those that clear the
// rows behind the last one (seq = B).  Workgroup `at` of XCD `xcd` takes the at-th of an eighth of
// the units: neighbours, which read the same keys, share its L2.
template <int KT>
__device__ __forceinline__ bool paged_find(const PagedAttnArgs& a, int xcd, int at_xcd, int& w, PagedUnit& u) {
  const int lane = __lane_id(), rep = a.heads / a.kv_heads, RB = a.block_rows;
  if (a.B > kPagedSeqs) {  // sequence i has the unit numbers from start(i) rep / RB + i on
    w = at_xcd * 8 + xcd;
    int lo = 0, hi = a.B + 1;
    while (hi - lo > 1) {
      const int step = (hi - lo - 1 + 63) / 64;
      const int64_t at = lo + (int64_t)(lane + 1) * step;
      const bool below = at < hi && (int64_t)seq_start(a.cu, (int)(at < hi ? at : lo), a.Tq) * rep / RB + at <= w;
      lo += __popcll(__ballot(below)) * step;
      hi = min(hi, lo + step);
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    const bool in = lo < a.B;
    const int first = seq_start(a.cu, lo, a.Tq);
    const PagedSeq q = paged_seq(a, lo, first, in ? a.cu[lo + 1] : a.Tq, in ? a.lengths[lo] : 0);
    u = PagedUnit{lo, q.start, q.n, q.past, q.len, 0, 0, 1, 1, 0};
    const int64_t at = (w - ((int64_t)first * rep / RB + lo)) * RB;
    if (at < 0 || at >= (int64_t)q.n * rep) return false;
    u.first = (int)at;
    return true;
  }
  constexpr int C = kPagedSeqs / 64;
  PagedSeq q[C];
  int blocks[C];
  float work = 0.f;  // of the lane's sequences, in tiles; past 2^24 rounded, the same in every workgroup
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int i = c * 64 + lane;
    q[c] = PagedSeq{0, 0, 0, 0};
    blocks[c] = 0;
    if (c * 64 < a.B && i < a.B) {
      const int s0 = a.cu[i], s1 = a.cu[i + 1], past = a.lengths[i];
      q[c] = paged_seq(a, i, s0, s1, past);
      blocks[c] = (int)(((int64_t)q[c].n * rep + RB - 1) / RB);
      work += (float)blocks[c] * (float)((q[c].len + KT - 1) / KT);
    }
  }
  int per = INT32_MAX;
  if (a.slots > 0) {  // a block's last range is half one on average
    float all = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) all += (float)blocks[c];
    const float want = fmaxf((float)a.slots - 0.5f * wave_sum(all), 0.5f * (float)a.slots);
    per = max((int)fminf(wave_sum(work) / want, 1e9f) + 1, a.least);
    per = __builtin_amdgcn_readfirstlane(per);
  }
  int splits[C], inc[C], all = 0;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    splits[c] = inc[c] = 0;
    if (c * 64 < a.B) {
      const int nt = (q[c].len + KT - 1) / KT;
      splits[c] = nt > per ? (nt + per - 1) / per : 1;
      inc[c] = all + wave_scan(blocks[c] * splits[c]);
      all = __builtin_amdgcn_readlane(inc[c], 63);
    }
  }
  const int end = seq_start(a.cu, a.B, a.Tq);
  // with the units of the rows behind the last sequence
  const int eighth = (all + (int)(((int64_t)(a.Tq - end) * rep + RB - 1) / RB) + 7) / 8;
  if (at_xcd >= eighth) return false;
  w = xcd * eighth + at_xcd;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    if (c * 64 >= a.B) break;
    const int first = inc[c] - blocks[c] * splits[c];
    const uint64_t who = __ballot(first <= w && w < inc[c]);
    if (who) {
      const int l = __ffsll((unsigned long long)who) - 1;
      u.seq = c * 64 + l;
      u.start = __builtin_amdgcn_readlane(q[c].start, l);
      u.n = __builtin_amdgcn_readlane(q[c].n, l);
      u.past = __builtin_amdgcn_readlane(q[c].past, l);
      u.len = __builtin_amdgcn_readlane(q[c].len, l);
      u.splits = __builtin_amdgcn_readlane(splits[c], l);
      u.blocks = __builtin_amdgcn_readlane(blocks[c], l);
      const int base = __builtin_amdgcn_readlane(first, l);
      u.base = base;
      u.split = min(max((w - base) / u.blocks, 0), u.splits - 1);  // the bounds of both: where cu decreases
      u.first = max((w - base) % u.blocks, 0) * RB;
      return true;
    }
  }
  // the rows behind the last sequence
  const int64_t at = (int64_t)(w - all) * RB;
  u = PagedUnit{a.B, end, a.Tq - end, 0, 0, 0, 0, 1, 1, 0};
  if (at < 0 || at >= (int64_t)u.n * rep) return false;
  u.first = (int)at;
  return true;
}

// The units of each sequence, [B]: its first row, its first unit, blocks of rows, ranges.
__device__ __forceinline__ int4* paged_units(const PagedAttnArgs& a) {
  return reinterpret_cast<int4*>(a.work + (int64_t)a.units * a.kv_heads * a.block_rows * (a.head_dim + 2));
}

// A wave's uniform read of the page table, by the scalar unit.
__device__ __forceinline__ int scalar_int(const int* p) {
  return *reinterpret_cast<const __attribute__((address_space(4))) int*>(reinterpret_cast<uintptr_t>(p));
}

// A workgroup takes 16 U RW rows (tokens times the query heads of one kv head) over a range of the
// keys.  RW waves share the tiles of KT keys, 16 U rows each; or (RW = 1) KW waves with the same rows
// take every KW-th tile, each with a ring of its own and no barrier, and join in LDS at the end.
// Tiles come by direct-to-LDS loads: a wave loads whole groups of 16 keys, which lie in one page, so
// a page number is one scalar read a group.  No wave leaves a step early: with a way out, for tiles
// that none of a wave's rows sees, the compiler spilled 56 registers at head_dim 128 (64 tokens over
// 65001 keys, 16 / 2 heads: 117 us instead of 51).
// Up to 32 rows the keys' bytes bound it: 64 single tokens over 725 to 2175 keys, 8 / 4 heads of 96, 146 MB, 33 us, 4.4 TB/s;
// trees of 16 there 37 us.  With more rows no unit is at its limit, products, softmax and LDS reads take turns: that tree of 64
// tokens 65 us, 530 TFLOP/s (of the busy CUs' cycles MFMA 43%, VALU 49%; CUs busy 80% of the launch); 6 chunks of 500
// over up to 4100 keys, heads of 64, 50 us, 380 TFLOP/s (38%, 59%; 70%).
template <int HD, int RW, int KW>
constexpr int paged_waves =  // of a SIMD, as the tiles' LDS lets in: two at most
    160 * 1024 / (KW * kPagedStages * 4 * (RW == 1 ? 32 : 64) * HD) * RW * KW >= 8 ? 2 : 1;
template <bool F16, int HD, int RW, int KW, int U>
__global__ __launch_bounds__(64 * RW * KW, (paged_waves<HD, RW, KW>)) void paged_kernel(PagedAttnArgs a) {
  constexpr int KT = RW == 1 ? 32 : 64;
  constexpr int NC = HD / 32, ND = HD / 16, NT = KT / 16, NH = KT / 32;
  constexpr int GW = NT / RW;               // groups of 16 keys that a wave loads of a tile
  constexpr int UG = HD / 32;               // 1 KiB units of a group
  constexpr int TILE = KT * HD;             // elements
  constexpr int WAVES = RW * KW, RB = 16 * U * RW;
  static_assert(RW == 1 || KW == 1, "waves that share a tile take the same steps");
  __shared__ __align__(16) uint16_t lds[KW][kPagedStages][2][TILE];
  static_assert(KW == 1 || sizeof(lds) >= WAVES * 16 * U * (HD + 2) * 4, "the waves' sums take the tiles' place");
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kw = wave / RW, rw = wave % RW;
  const int r = lane & 15, g = lane >> 4;
  const int rep = a.heads / a.kv_heads;
  // the heads of one unit go to one XCD, whose L2 then sees whole lines of a key's row:
  // workgroups are dealt to the 8 XCDs in turn
  const int in = blockIdx.x % (8 * a.kv_heads);
  const int kvh = in / 8;
  int w = 0;
  PagedUnit t;
  if (!paged_find<KT>(a, in % 8, blockIdx.x / (8 * a.kv_heads), w, t) || (unsigned)w >= (unsigned)a.units) return;
  for (int* x : {&t.seq, &t.start, &t.n, &t.past, &t.len, &t.first, &t.split, &t.splits, &w}) *x = __builtin_amdgcn_readfirstlane(*x);
  const int rows = t.n * rep;
  const int last_token = (min(t.first + RB, rows) - 1) / rep;
  const bool causal = a.tree == nullptr;
  const int seen = t.seq == a.B ? 0 : causal ? min(t.len, t.past + last_token + 1) : t.len;
  const int nt_all = (seen + KT - 1) / KT;
  const int per = (nt_all + t.splits - 1) / t.splits;
  const int t0 = min(t.split * per, nt_all), t1 = min(t0 + per, nt_all);
  const int steps = max((t1 - t0 - kw + KW - 1) / KW, 0);  // of this wave

  // ---- rows
  U32x4 qb[U][NC];
  int token[U];  // -1: no row
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int at = t.first + (rw * U + u) * 16 + r;
    const bool live = at < rows;
    token[u] = live ? at / rep : -1;
    const int h = kvh * rep + (live ? at % rep : 0);
    const uint16_t* q = static_cast<const uint16_t*>(a.q) + (int64_t)(t.start + max(token[u], 0)) * a.qs_t + h * a.qs_h + 8 * g;
#pragma unroll
    for (int c = 0; c < NC; ++c) qb[u][c] = ld16(q + 32 * c);
  }

  // ---- loading
  const int* table = a.page_table + (int64_t)min(t.seq, a.B - 1) * a.width;
  const int mask = (1 << a.page_shift) - 1;
  const char* kg = reinterpret_cast<const char*>(static_cast<const uint16_t*>(a.k) + kvh * a.s_h);
  const char* vg = reinterpret_cast<const char*>(static_cast<const uint16_t*>(a.v) + kvh * a.s_h);
  const int64_t page_b = 2 * a.s_p, row_b = 2 * a.s_t;  // of K and of V
  const int g0 = rw * GW;                                 // the wave's first group
  uint32_t off[GW * UG];
#pragma unroll
  for (int i = 0; i < GW * UG; ++i) {
    const int at = (g0 * UG + i) * 64 + lane, row = at / (HD / 8);
    off[i] = (uint32_t)((row & 15) * row_b + tile_column<HD>(row, at % (HD / 8)) * 16);
  }
  const int last_group = (max(seen, 1) - 1) & ~15;
  int page[GW];  // of the next tile to load
  auto look = [&](int i) {
    const int kt = min(t0 + i * KW + kw, t1 - 1);
#pragma unroll
    for (int y = 0; y < GW; ++y) page[y] = scalar_int(table + (min(kt * KT + 16 * (g0 + y), last_group) >> a.page_shift));
  };
  auto issue = [&](int i, uint16_t* __restrict__ kd, uint16_t* __restrict__ vd) {
    const int kt = min(t0 + i * KW + kw, t1 - 1);
    auto fetch = [&](const char* from, int y, uint16_t* to) {
#pragma unroll
      for (int z = 0; z < UG; ++z)
        __builtin_amdgcn_global_load_lds(
            (const __attribute__((address_space(1))) void*)(from + off[y * UG + z]),
            (__attribute__((address_space(3))) void*)(reinterpret_cast<char*>(to) + ((g0 + y) * UG + z) * 1024), 16, 0, 0);
    };
#pragma unroll
    for (int y = 0; y < GW; ++y) {
      const int p = (unsigned)page[y] < (unsigned)a.pages ? page[y] : 0;
      const int64_t from = p * page_b + (min(kt * KT + 16 * (g0 + y), last_group) & mask) * row_b;
      fetch(kg + from, y, kd);
      fetch(vg + from, y, vd);
    }
  };
  auto arrived = [&] {  // waits for the queries: in the loop that would be a wait for every tile in flight
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        u32x4_t w = __builtin_bit_cast(u32x4_t, qb[u][c]);
        asm volatile("" : "+v"(w));
        qb[u][c] = __builtin_bit_cast(U32x4, w);
      }
  };
  bool lost = false;  // whether a page of the range is none: then every tile looks which of its groups are
  if (steps > 0) {
    look(0);
    const int p0 = t0 * KT >> a.page_shift, p1 = min(t1 * KT - 1, last_group) >> a.page_shift;
    const int entry = table[min(p0 + lane, p1)];
    issue(0, lds[kw][0][0], lds[kw][0][1]);
    look(1);
    arrived();
    lost = __any((unsigned)entry >= (unsigned)a.pages);
    for (int p = p0 + 64; p <= p1; p += 64) lost |= __any((unsigned)table[min(p + lane, p1)] >= (unsigned)a.pages);
  } else {
    arrived();
  }
  const int wave_first = (t.first + rw * U * 16) / rep;  // token of the wave's first row
  const float scale = a.scale * kPackedLog2e;
  constexpr float kHead = packed_head<F16>;
  float m[U];
  f32x4_t l[U], o[U][ND];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    m[u] = kNoScore;
    l[u] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int d = 0; d < ND; ++d) o[u][d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  const U32x4 ones = packed_ones<F16>();
  TileReads<HD> at;
  at.init(r, g);

  const int plain = min(t.len, t.past + (causal ? wave_first + 1 : 0));  // keys that all of the wave's rows see
  // As restrict parameters the compiler sees that the stages differ; else it waits for every
  // load in flight before it reads one.
  auto step = [&](int i, const uint16_t* __restrict__ ks, const uint16_t* __restrict__ vs, uint16_t* __restrict__ kd,
                  uint16_t* __restrict__ vd) {
    const int kt = t0 + i * KW + kw, s0 = kt * KT;
    if (i + 1 < steps) issue(i + 1, kd, vd);
    look(i + 2);
    uint32_t none = 0;  // groups in no page
    if (lost) {
#pragma unroll
      for (int x = 0; x < NT; ++x)
        none |= (unsigned)scalar_int(table + (min(s0 + 16 * x, last_group) >> a.page_shift)) >= (unsigned)a.pages ? 1u << x : 0u;
    }
    // Bits of the lane's 4 NT keys, 16 st + 4 g + x at 4 st + x: those that are there, and those that
    // each row sees.  Formed here, before the products need the registers, and opaque: the compiler
    // would keep a scalar mask of every comparison.
    uint32_t there = ~0u, sees[U];
    const bool holes = s0 + KT > t.len || none;
    const bool edge = s0 + KT > plain || none;
    if (edge) {
      int g4 = 4 * g;  // opaque: what follows stays in this branch instead of in registers around the loop
      asm volatile("" : "+v"(g4));
#pragma unroll
      for (int st = 0; st < NT; ++st) {
        const int n = min(max(t.len - (s0 + 16 * st + g4), 0), 4);
        there &= ~((none >> st & 1 ? 15u : 15u & (15u << n)) << (4 * st));
      }
      asm volatile("" : "+v"(there));
#pragma unroll
      for (int u = 0; u < U; ++u) {
        uint32_t see = there;
        int tok = token[u];
        asm volatile("" : "+v"(tok));
        if (causal) {
#pragma unroll
          for (int st = 0; st < NT; ++st) {
            const int n = min(max(t.past + tok + 1 - (s0 + 16 * st + g4), 0), 4);
            see &= ~((15u & (15u << n)) << (4 * st));
          }
        } else {
          const uint64_t* row = a.tree + (int64_t)(t.start + max(tok, 0)) * a.words;
#pragma unroll
          for (int st = 0; st < NT; ++st) {
            const int j0 = s0 + 16 * st + g4 - t.past;  // of the sequence's rows
            const int w0 = j0 >> 6, w1 = (j0 + 3) >> 6;
            const uint64_t lo = w0 < 0 ? ~0ull : w0 < a.words ? row[w0] : 0, hi = w1 < 0 ? ~0ull : w1 < a.words ? row[w1] : 0;
            const int sh = j0 & 63;  // four bits of the two words from there on
            const uint32_t four = (uint32_t)(lo >> sh) | (w1 > w0 ? (uint32_t)(hi << (64 - sh)) : 0u);
            see &= ~((15u & ~four) << (4 * st));
          }
        }
        asm volatile("" : "+v"(see));
        sees[u] = see;
      }
    }
    f32x4_t s[U][NT];
#pragma unroll
    for (int st = 0; st < NT; ++st)
#pragma unroll
      for (int u = 0; u < U; ++u) s[u][st] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    // Operands are read from LDS before their products; the barriers keep the compiler from
    // sinking each read to its use, where every pair of products would wait.  At head_dim 128 half of
    // the tile at a time: all of it does not fit the registers beside the outputs.
    constexpr int KA = HD == 128 && NT > 2 ? 2 : NT;
#pragma unroll
    for (int s2 = 0; s2 < NT; s2 += KA) {
      U32x4 ka[KA][NC];
#pragma unroll
      for (int st = 0; st < KA; ++st)
#pragma unroll
        for (int c = 0; c < NC; ++c) ka[st][c] = at.row16(ks, s2 + st, c);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int sp = 0; sp < KA; sp += 2)
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int st = sp; st < sp + 2; ++st)
#pragma unroll
            for (int u = 0; u < U; ++u) s[u][s2 + st] = mfma16<F16>(ka[st][c], qb[u][c], s[u][s2 + st]);
    }
    U32x4 va[NH][ND];
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int d = 0; d < ND; ++d) va[0][d] = at.columns32(vs, 0, d);
    __builtin_amdgcn_sched_barrier(0);
    if (edge) {  // uniform
      asm volatile("");  // a branch: as selects they would be part of every step
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int st = 0; st < NT; ++st)
#pragma unroll
          for (int x = 0; x < 4; ++x)
            if (!(sees[u] >> (4 * st + x) & 1)) s[u][st][x] = -__builtin_inff();
    }
    // V rows that are no keys: probability 0 times what lies there could be NaN
    auto clear = [&](int hh) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const uint32_t four = there >> (4 * (2 * hh + q));
        const uint32_t k0 = (four & 1 ? 0xffffu : 0u) | (four & 2 ? 0xffff0000u : 0u);
        const uint32_t k1 = (four & 4 ? 0xffffu : 0u) | (four & 8 ? 0xffff0000u : 0u);
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          va[hh][d].v[2 * q] &= k0;
          va[hh][d].v[2 * q + 1] &= k1;
        }
      }
    };
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float mx = -__builtin_inff();
#pragma unroll
      for (int st = 0; st < NT; ++st)
#pragma unroll
        for (int j = 0; j < 4; ++j) mx = fmaxf(mx, s[u][st][j]);
      mx *= scale;
      if (__any(!(mx <= m[u] + kPackedLazyMax + kHead))) {
        mx = fmaxf(mx, xor_lane16(mx));
        mx = fmaxf(mx, xor_lane32(mx));
        mx = fmaxf(mx - kHead, m[u]);
        const float f = exp2_f(m[u] - mx);
        m[u] = mx;
#pragma unroll
        for (int j = 0; j < 4; ++j) l[u][j] *= f;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int j = 0; j < 4; ++j) o[u][d][j] *= f;
      }
    }
    U32x4 pf[U][NH], pr[U][NH];  // the probabilities rounded, and what the rounding took
    auto softmax = [&](int hh) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          float p[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) p[j] = exp2_f(fmaf(s[u][2 * hh + q][j], scale, -m[u]));
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const uint32_t w = pack2<F16>(p[2 * x], p[2 * x + 1]);
            pf[u][hh].v[2 * q + x] = w;
            pr[u][hh].v[2 * q + x] = pack2<F16>(p[2 * x] - elem_lo<F16>(w), p[2 * x + 1] - elem_hi<F16>(w));
          }
        }
    };
    auto outputs = [&](int hh) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        l[u] = mfma16<F16>(ones, pf[u][hh], l[u]);
        l[u] = mfma16<F16>(ones, pr[u][hh], l[u]);
      }
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          o[u][d] = mfma16<F16>(va[hh][d], pf[u][hh], o[u][d]);
          o[u][d] = mfma16<F16>(va[hh][d], pr[u][hh], o[u][d]);
        }
    };
    softmax(0);
    if (holes) clear(0);
    if constexpr (NH == 1) {
      outputs(0);
    } else {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int d = 0; d < ND; ++d) va[1][d] = at.columns32(vs, 1, d);
      __builtin_amdgcn_sched_barrier(0);
      // the first half's products with the second half's softmax between them
      outputs(0);
      softmax(1);
#pragma unroll
      for (int x = 0; x < U * ND + U; ++x) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x402, ND == 4 ? 4 : 3, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
      if (holes) clear(1);
      outputs(1);
    }
  };
  for (int i = 0; i < steps; ++i) {
    tile_wait<0>();
    if (RW > 1) tile_barrier();  // the tile has landed for every wave, and all are done with the one before
    const int stage = i & 1;
    step(i, lds[kw][stage][0], lds[kw][stage][1], lds[kw][1 - stage][0], lds[kw][1 - stage][1]);
  }

  // ---- results
  const bool whole = t.splits == 1;
  // for the join: where the sequence's units are
  if (a.slots > 0 && t.first == 0 && t.split == 0 && kvh == 0 && tid == 0 && t.seq < a.B)
    paged_units(a)[t.seq] = make_int4(t.start, t.base, t.blocks, t.splits);
  auto place = [&](int row) {  // of the output
    const int tok = row / rep;
    return ((int64_t)(t.start + tok) * a.heads + kvh * rep + row - tok * rep) * HD;
  };
  const int64_t part = ((int64_t)w * a.kv_heads + kvh) * RB;  // of the partial results' rows
  float* ml = a.work + (int64_t)a.units * a.kv_heads * RB * HD;
  if constexpr (KW == 1) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int in_block = (rw * U + u) * 16 + r, row = t.first + in_block;
      if (row >= rows) continue;
      if (!whole) {
        float* x = a.work + (part + in_block) * HD + 4 * g;
#pragma unroll
        for (int d = 0; d < ND; ++d) *reinterpret_cast<f32x4_t*>(x + 16 * d) = o[u][d];
        if (g == 0) *reinterpret_cast<float2*>(ml + 2 * (part + in_block)) = make_float2(m[u], l[u][0]);
        continue;
      }
      const float ls = l[u][0], inv = ls > 0.f || ls != ls ? 1.f / ls : 0.f;  // a row without keys: zeros
      uint16_t* out = static_cast<uint16_t*>(a.out) + place(row) + 4 * g;
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        uint2 x;
        x.x = pack2<F16>(o[u][d][0] * inv, o[u][d][1] * inv);
        x.y = pack2<F16>(o[u][d][2] * inv, o[u][d][3] * inv);
        *reinterpret_cast<uint2*>(out + 16 * d) = x;
      }
    }
  } else {
    // the waves' sums meet in LDS: [wave][rows][HD], then each row's maximum and sum
    __syncthreads();
    float* sums = reinterpret_cast<float*>(lds);
    float* marks = sums + WAVES * 16 * U * HD;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float* x = sums + ((wave * U + u) * 16 + r) * HD + 4 * g;
#pragma unroll
      for (int d = 0; d < ND; ++d) *reinterpret_cast<f32x4_t*>(x + 16 * d) = o[u][d];
      if (g == 0) *reinterpret_cast<float2*>(marks + 2 * ((wave * U + u) * 16 + r)) = make_float2(m[u], l[u][0]);
    }
    __syncthreads();
    for (int x = tid; x < RB * (HD / 4); x += 64 * WAVES) {
      const int in_block = x / (HD / 4), col = x % (HD / 4) * 4, row = t.first + in_block;
      if (row >= rows) break;
      float2 e[KW];
      float mx = kNoScore, ls = 0.f;
#pragma unroll
      for (int k = 0; k < KW; ++k) {
        e[k] = *reinterpret_cast<const float2*>(marks + 2 * (k * RB + in_block));
        mx = fmaxf(mx, e[k].x);
      }
      f32x4_t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < KW; ++k) {
        const float f = exp2_f(e[k].x - mx);
        const f32x4_t y = *reinterpret_cast<const f32x4_t*>(sums + (k * RB + in_block) * HD + col);
        ls += f * e[k].y;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] += f * y[j];
      }
      if (!whole) {
        *reinterpret_cast<f32x4_t*>(a.work + (part + in_block) * HD + col) = v;
        if (col == 0) *reinterpret_cast<float2*>(ml + 2 * (part + in_block)) = make_float2(mx, ls);
        continue;
      }
      const float inv = ls > 0.f || ls != ls ? 1.f / ls : 0.f;
      uint2 y;
      y.x = pack2<F16>(v[0] * inv, v[1] * inv);
      y.y = pack2<F16>(v[2] * inv, v[3] * inv);
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + place(row) + col) = y;
    }
  }
}

// Joins the ranges of a row: a lane takes four columns of one of its heads, a wave 64 such; with P > 1 the
// workgroup's P waves take every P-th range of the same 64, and the sums meet in LDS.  P follows the rows and the
// ranges that there can be.  Microseconds of a whole attention call with P = 1, 4, 16 (the rule's in brackets): one token
// over 65001 keys, 16 / 2 heads of 128, 35.0, 23.9, [22.9]; 8 rows over 65001, 8 / 4 heads of 96, 52.9, 31.5, [28.9]; 64 rows
// over 65001, 16 / 2 of 128, 75.4, [70.6], 78.0; 4 trees of 30 over 8001 26.0, [23.4], 25.8; 4 tokens over 8001 23.7,
// [18.6], 18.2; 16 over 4001 24.5, [23.6], 23.9; 100 rows over 4001 22.6, [20.5], 23.5; 64 trees of 16 over up to 2175 [36.5], 39.9, 64.0.
template <bool F16, int HD, int P>
__global__ __launch_bounds__(P == 16 ? 1024 : 256) void paged_join_kernel(PagedAttnArgs a) {
  __shared__ __align__(16) f32x4_t sums[P][64];
  __shared__ float2 marks[P][64];
  const int rep = a.heads / a.kv_heads, RB = a.block_rows;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned chunks = (a.heads * (HD / 4) + 63) / 64;  // Tq of them: under 2^31 with Tq * heads
  const unsigned at_wave = P == 1 ? blockIdx.x * 4 + wave : blockIdx.x;
  const int row = at_wave / chunks;
  if (row >= a.Tq) return;
  const float* ml = a.work + (int64_t)a.units * a.kv_heads * RB * HD;
  int lo = 0, hi = a.B + 1;  // the last sequence that begins at or before the row
  while (hi - lo > 1) {
    const int step = (hi - lo - 1 + 63) / 64;
    const int64_t at = lo + (int64_t)(lane + 1) * step;
    const bool below = at < hi && seq_start(a.cu, (int)(at < hi ? at : lo), a.Tq) <= row;
    lo += __popcll(__ballot(below)) * step;
    hi = min(hi, lo + step);
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  if (lo >= a.B) return;
  const int4 u = paged_units(a)[lo];
  // Where cu decreases, the row may be none of the sequence's, and a sequence without rows has no record: what
  // stands there is anything.  Within these bounds nothing below leaves the workspace.
  if (u.x < 0 || u.x > row || u.y < 0 || u.y >= a.units || u.z < 1 || u.z > a.units || u.w <= 1) return;
  const int blocks = u.z;
  const int x = (int)(at_wave % chunks) * 64 + lane;
  const bool live = x < a.heads * (HD / 4);
  const int head = live ? x / (HD / 4) : 0, col = live ? x % (HD / 4) * 4 : 0, kvh = head / rep;
  const int at = (row - u.x) * rep + head % rep, first = u.y + at / RB;
  const int splits = first < a.units ? min(u.w, (a.units - first + blocks - 1) / blocks) : 0;
  float mx = kNoScore, l = 0.f;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  auto add = [&](const float2& e, const f32x4_t& v) {
    const float mn = fmaxf(mx, e.x), f = exp2_f(mx - mn), k = exp2_f(e.x - mn);
    mx = mn;
    l = l * f + e.y * k;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = o[j] * f + v[j] * k;
  };
#pragma unroll 4
  for (int s = P == 1 ? 0 : wave; s < splits; s += P) {
    const int64_t part = ((int64_t)(first + s * blocks) * a.kv_heads + kvh) * RB + at % RB;
    add(*reinterpret_cast<const float2*>(ml + 2 * part), *reinterpret_cast<const f32x4_t*>(a.work + part * HD + col));
  }
  if constexpr (P > 1) {
    sums[wave][lane] = o;
    marks[wave][lane] = make_float2(mx, l);
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int s = 1; s < P; ++s) add(marks[s][lane], sums[s][lane]);
  }
  if (!live) return;
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  uint2 y;
  y.x = pack2<F16>(o[0] * inv, o[1] * inv);
  y.y = pack2<F16>(o[2] * inv, o[3] * inv);
  *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + ((int64_t)row * a.heads + head) * HD + col) = y;
}

// Blocks of rows, at most.
int64_t paged_row_blocks(const PagedAttnArgs& a) {
  return (int64_t)a.Tq * (a.heads / a.kv_heads) / a.block_rows + (a.B > 0 ? a.B : 1);
}
int64_t paged_blocks(const PagedAttnArgs& a) { return ((int64_t)a.units + 7) / 8 * 8 * a.kv_heads; }

template <bool F16, int HD, int RW, int KW, int U>
hipError_t run_paged(const PagedAttnArgs& a, hipStream_t s) {
  paged_kernel<F16, HD, RW, KW, U><<<dim3((unsigned)paged_blocks(a)), 64 * RW * KW, 0, s>>>(a);
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  if (a.slots > 0) {
    constexpr int KT = RW == 1 ? 32 : 64;
    const int64_t most = ((int64_t)a.width << a.page_shift) / (KT * a.least);  // ranges that the pages have room for
    if (most == 0) return hipGetLastError();
    const int64_t waves = (int64_t)a.Tq * ((a.heads * (HD / 4) + 63) / 64);
    if (waves > 8 * (int64_t)device_cus())
      paged_join_kernel<F16, HD, 1><<<dim3((unsigned)((waves + 3) / 4)), 256, 0, s>>>(a);
    else if (most < 64 || a.slots < 64 * paged_row_blocks(a))
      paged_join_kernel<F16, HD, 4><<<dim3((unsigned)waves), 256, 0, s>>>(a);
    else
      paged_join_kernel<F16, HD, 16><<<dim3((unsigned)waves), 1024, 0, s>>>(a);
  }
  return hipGetLastError();
}

template <bool F16, int HD>
hipError_t paged_hd(const PagedAttnArgs& a, hipStream_t s) {
  switch (a.block_rows) {
    case 16: return a.key_waves == 4 ? run_paged<F16, HD, 1, 4, 1>(a, s) : run_paged<F16, HD, 1, 1, 1>(a, s);
    case 32: return a.key_waves == 4 ? run_paged<F16, HD, 1, 4, 2>(a, s) : run_paged<F16, HD, 1, 1, 2>(a, s);
    case 64: return run_paged<F16, HD, 2, 1, 2>(a, s);
    default: return run_paged<F16, HD, 4, 1, 2>(a, s);
  }
}

}  // namespace

// How the work is cut; only totals are known here, the sequences' own lengths are read on the device.
// Rows of a workgroup follow from the mean rows a sequence, which suits sequences alike.  Others pay: 60 single tokens
// and 4 chunks of 500 in one call over 725 to 2175 keys, 8 / 4 heads of 96, with 16, 32, 64, 128 rows 95, 100, 89, [80] us,
// in calls of their own 29 and 38; 63 tokens and one chunk 54, [48], 58, 60, apart 30 and 26.
// Microseconds a call in a captured graph, join included, for 1, 2, 3, 4 workgroups a CU:
//   * Up to 32 rows a sequence and kv head, a wave each: 64 single tokens over 725 to 2175 keys, 8 / 4
//     heads of 96: -, 38.6, 37.6, 36.0 (5: 35.8, 6: 40); trees of 16 nodes there -, 45.8, 45.4, 43.9 (5: 45.2).
//     Where that would be more than 256 ranges of a sequence, four waves share one instead (one token
//     over 65001 keys, 16 / 2 heads of 128: 34.5 with 512 ranges, 24.7 with 128 of four waves).
//   * Up to 64 rows, two waves (from here on the same inputs on every call): 4 trees of 30 nodes over 2667 to 8001 keys
//     24.7, 22.3, 29.1, 29.3; one of 32 over 65001 keys 45.7, 32.3, 43.4, 43.8.
//   * More, four waves: 6 chunks of 500 over up to 4100 keys, heads of 64: 73, 55, 50, 56; of 96: 101, 71, 76, 76;
//     one tree of 64 nodes over 65001 keys, 16 / 2 heads of 128: 80, 67, 81, 81.
// Keys are not cut with four blocks of rows a place and more.  Cut and whole, sequences of a third to all of the longest's
// keys, 8 / 4 heads of 96: 96 chunks of 400 over 2000 keys (5.4 blocks a place) 389 and 367 us, 140 (7.9) 531 and 514.  Below
// four cutting costs about as much where lengths are that much alike (64 chunks, 3.6, 279 and 266; 128 trees of 30 over 700 keys, 1.9, 36.0
// and 32.3), but it is what keeps a long sequence among short ones from being one workgroup's.
// A range has 4 tiles at least, or 2 of the larger ones.  With 1, 2, 4, 8: a single token over 900 keys 9.9, 10.0, [11.4],
// 14.1 us; 8 trees of 5 12.5, 11.3, [12.0], 14.6; 32 tokens over 400 11.0, 11.0, [12.0], 13.9; two trees of 64 over 900 15.0, [16.7], 19.3,
// 25.6; a chunk of 300 22.3, [18.6], 18.7, 22.0.  (All the same inputs on every call.)
void paged_attn_plan(PagedAttnArgs& a) {
  const int rep = a.heads / a.kv_heads;
  const int64_t B = a.B > 0 ? a.B : 1, rows = (int64_t)a.Tq * rep, each = (rows + B - 1) / B;
  a.block_rows = each <= 16 ? 16 : each <= 32 ? 32 : each <= 64 ? 64 : 128;
  const int64_t blocks = paged_row_blocks(a);
  const int cu = a.block_rows <= 32 ? 4 : a.block_rows == 128 && a.head_dim == 64 ? 3 : 2;
  int64_t slots = ((int64_t)device_cus() * cu + a.kv_heads - 1) / a.kv_heads;
  a.key_waves = 1;
  if (a.block_rows <= 32 && slots > 256 * blocks) {
    a.key_waves = 4;
    slots /= 4;
  }
  a.slots = a.B > kPagedSeqs || blocks >= 4 * slots ? 0 : (int)slots;
  a.least = a.block_rows <= 32 ? 4 : 2;
  const int64_t units = a.slots + blocks + 2;
  a.units = units > INT32_MAX ? INT32_MAX : (int)units;
}
int64_t paged_attn_workspace(const PagedAttnArgs& a) {
  return a.slots > 0 ? (int64_t)a.units * a.kv_heads * a.block_rows * (a.head_dim + 2) * 4 + (int64_t)a.B * 16 : 0;
}
int64_t paged_attn_threads(const PagedAttnArgs& a) {
  const int64_t tiles = 256 * paged_blocks(a);
  const int64_t join = a.slots > 0 ? 256 * (int64_t)a.Tq * ((a.heads * (a.head_dim / 4) + 63) / 64) : 0;  // at most
  return tiles > join ? tiles : join;
}

hipError_t launch_paged_attn(PagedAttnArgs a, hipStream_t s) {
  // Few short sequences, as far as their pages have room: four waves share a range and nothing is joined
  // (one token, 8 / 4 heads of 96, over 300 keys: 11.8 us in ranges, 8.0 so; over 900: 12.3 and 12.7).
  if (a.block_rows <= 32 && (int64_t)a.width << a.page_shift <= 768 && paged_row_blocks(a) * a.kv_heads <= device_cus()) {
    a.slots = 0;
    a.key_waves = 4;
    a.units = (int)paged_row_blocks(a) + 2;
  }
  MHC_PACKED_HD(paged_hd, a, s)
}

}  // namespace mhc
