// Attention of new tokens over a cache of pages: single tokens, drafted trees, chunks of prompts.
// Key x of a sequence lies in page table[x / page], row x % page; a page has 2^s >= 16 rows. The
// new rows' own keys are stored already, behind the `past` ones before them.
//   S_tj = scale q_t . k_j  for j < past, and for j - past a row of the same sequence that t sees
//   (causal: up to its own; a tree: its bits),  O_t = sum_j softmax(S_t)_j v_j
// 16-bit tensors, fp32 scores, sums and outputs; the probabilities are rounded once as a product's
// operand, the outputs once.
#include "mhc_packed.hpp"

namespace mhc {
namespace {

constexpr int kPagedSeqs = 256;  // up to so many, workgroups are dealt out by the keys' lengths

// What a workgroup does: rows `first` and on (row = token * rep + head of the group) of a
// sequence, over part `split` of `splits` of the keys they see.
struct PagedUnit {
  int seq, start, n, past, len;
  int first, split, splits;
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
__device__ __forceinline__ double wave_total(double v) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
  return v;
}

// Unit number w of a kv head.  The keys of all sequences, times their blocks of rows, are cut
// into about a.slots ranges of the same length; a sequence shorter than one is one unit a block.
// Behind the sequences' units come those that clear the rows behind the last one (seq = B).
// `row` >= 0: instead the first unit of the block with that row (of Tq), w is set to it.
template <int KT>
__device__ __forceinline__ bool paged_find(const PagedAttnArgs& a, int& w, PagedUnit& u, int row) {
  const int lane = __lane_id(), rep = a.heads / a.kv_heads, RB = a.block_rows;
  if (a.B > kPagedSeqs) {  // sequence i has the unit numbers from start(i) rep / RB + i on
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
    u = PagedUnit{lo, q.start, q.n, q.past, q.len, 0, 0, 1};
    const int64_t at = (w - ((int64_t)first * rep / RB + lo)) * RB;
    if (at < 0 || at >= (int64_t)q.n * rep) return false;
    u.first = (int)at;
    return true;
  }
  constexpr int C = kPagedSeqs / 64;
  PagedSeq q[C];
  int blocks[C], units[C];
  double work = 0.0;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int i = c * 64 + lane;
    q[c] = PagedSeq{0, 0, 0, 0};
    blocks[c] = 0;
    if (c * 64 < a.B && i < a.B) {
      const int s0 = a.cu[i], s1 = a.cu[i + 1], past = a.lengths[i];
      q[c] = paged_seq(a, i, s0, s1, past);
      blocks[c] = (int)(((int64_t)q[c].n * rep + RB - 1) / RB);
      work += (double)blocks[c] * ((q[c].len + KT - 1) / KT);
    }
  }
  int per = INT32_MAX;
  if (a.slots > 0) per = max((int)fmin(wave_total(work) / a.slots, 1e9) + 1, a.least);
  int before = 0;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    if (c * 64 >= a.B) break;
    const int nt = (q[c].len + KT - 1) / KT;
    const int splits = nt > per ? (nt + per - 1) / per : 1;
    units[c] = blocks[c] * splits;
    const int inc = wave_scan(units[c]);
    bool mine;
    if (row >= 0) mine = q[c].n > 0 && row >= q[c].start && row < q[c].start + q[c].n;
    else mine = before + inc > w && before + inc - units[c] <= w;
    const uint64_t who = __ballot(mine);
    if (who) {
      const int l = __ffsll((unsigned long long)who) - 1;
      u.seq = c * 64 + l;
      u.start = __builtin_amdgcn_readlane(q[c].start, l);
      u.n = __builtin_amdgcn_readlane(q[c].n, l);
      u.past = __builtin_amdgcn_readlane(q[c].past, l);
      u.len = __builtin_amdgcn_readlane(q[c].len, l);
      u.splits = __builtin_amdgcn_readlane(splits, l);
      const int base = before + __builtin_amdgcn_readlane(inc - units[c], l);
      if (row >= 0) {
        u.split = 0;
        u.first = (row - u.start) * rep / RB * RB;
        w = base + u.first / RB * u.splits;
      } else {
        u.split = (w - base) % u.splits;
        u.first = (w - base) / u.splits * RB;
      }
      return true;
    }
    before += __builtin_amdgcn_readlane(inc, 63);
  }
  if (row >= 0) return false;
  // the rows behind the last sequence
  const int end = seq_start(a.cu, a.B, a.Tq);
  const int64_t at = (int64_t)(w - before) * RB;
  u = PagedUnit{a.B, end, a.Tq - end, 0, 0, 0, 0, 1};
  if (at >= (int64_t)u.n * rep) return false;
  u.first = (int)at;
  return true;
}

// A wave's uniform read of the page table, by the scalar unit.
__device__ __forceinline__ int scalar_int(const int* p) {
  return *reinterpret_cast<const __attribute__((address_space(4))) int*>(reinterpret_cast<uintptr_t>(p));
}

// A workgroup takes 16 U RW rows (tokens times the query heads of one kv head) over a range of the
// keys.  RW waves share the tiles of KT keys, 16 U rows each; KW such groups take every KW-th
// tile, and join in LDS at the end.  Tiles come by direct-to-LDS loads: a wave loads whole groups
// of 16 keys, which lie in one page, so a page number is one scalar read a group.
template <bool F16, int HD, int RW, int KW, int U, int S>
__global__ __launch_bounds__(64 * RW * KW, RW == 4 ? 2 : 1) void paged_kernel(PagedAttnArgs a) {
  constexpr int KT = RW == 1 ? 32 : 64;
  constexpr int NC = HD / 32, ND = HD / 16, NT = KT / 16, NH = KT / 32;
  constexpr int GW = NT / RW;               // groups of 16 keys that a wave loads of a tile
  constexpr int UG = HD / 32;               // 1 KiB units of a group
  constexpr int TILE = KT * HD;             // elements
  constexpr int WAVES = RW * KW, RB = 16 * U * RW;
  __shared__ __align__(16) uint16_t lds[KW][S][2][TILE];
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
  int w = blockIdx.x / (8 * a.kv_heads) * 8 + in % 8;
  PagedUnit t;
  if (w >= a.units || !paged_find<KT>(a, w, t, -1)) return;
  const int rows = t.n * rep;
  const int last_token = (min(t.first + RB, rows) - 1) / rep;
  const bool causal = a.tree == nullptr;
  const int seen = t.seq == a.B ? 0 : causal ? min(t.len, t.past + last_token + 1) : t.len;
  const int nt_all = (seen + KT - 1) / KT;
  const int per = (nt_all + t.splits - 1) / t.splits;
  const int t0 = min(t.split * per, nt_all), t1 = min(t0 + per, nt_all);
  const int steps = (t1 - t0 + KW - 1) / KW;

  // ---- loading
  const int* table = a.page_table + (int64_t)min(t.seq, a.B - 1) * a.width;
  const int mask = (1 << a.page_shift) - 1;
  const uint16_t* kg = static_cast<const uint16_t*>(a.k) + kvh * a.ks_h;
  const uint16_t* vg = static_cast<const uint16_t*>(a.v) + kvh * a.vs_h;
  uint32_t koff[GW * UG], voff[GW * UG];
#pragma unroll
  for (int i = 0; i < GW * UG; ++i) {
    const int at = ((rw * GW) * UG + i) * 64 + lane, row = at / (HD / 8), col = tile_column<HD>(row, at % (HD / 8)) * 8;
    koff[i] = (uint32_t)((row & 15) * a.ks_t + col) * 2;
    voff[i] = (uint32_t)((row & 15) * a.vs_t + col) * 2;
  }
  const int last_group = (max(seen, 1) - 1) & ~15;
  int page[NT];  // of the next tile to load
  auto look = [&](int i) {
    const int kt = min(t0 + i * KW + kw, t1 - 1);
#pragma unroll
    for (int x = 0; x < NT; ++x) page[x] = scalar_int(table + (min(kt * KT + 16 * x, last_group) >> a.page_shift));
  };
  uint64_t bad = 0;  // groups in no page, four bits a stage
  auto issue = [&](int i, int stage, uint16_t* __restrict__ kd, uint16_t* __restrict__ vd) {
    const int kt = min(t0 + i * KW + kw, t1 - 1);
    uint32_t none = 0;
#pragma unroll
    for (int x = 0; x < NT; ++x) none |= (unsigned)page[x] >= (unsigned)a.pages ? 1u << x : 0u;
    bad = (bad & ~(15ull << (4 * stage))) | ((uint64_t)none << (4 * stage));
#pragma unroll
    for (int y = 0; y < GW; ++y) {
      const int x = rw * GW + y;
      int p = page[0];
#pragma unroll
      for (int z = 1; z < NT; ++z)
        if (x == z) p = page[z];
      if ((unsigned)p >= (unsigned)a.pages) p = 0;
      const int row = min(kt * KT + 16 * x, last_group) & mask;
      const char* kp = reinterpret_cast<const char*>(kg + p * a.ks_p + row * a.ks_t);
      const char* vp = reinterpret_cast<const char*>(vg + p * a.vs_p + row * a.vs_t);
#pragma unroll
      for (int i2 = 0; i2 < UG; ++i2) {
        const int at = x * UG + i2;
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(kp + koff[y * UG + i2]),
                                         (__attribute__((address_space(3))) void*)(reinterpret_cast<char*>(kd) + at * 1024), 16, 0, 0);
      }
#pragma unroll
      for (int i2 = 0; i2 < UG; ++i2) {
        const int at = x * UG + i2;
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(vp + voff[y * UG + i2]),
                                         (__attribute__((address_space(3))) void*)(reinterpret_cast<char*>(vd) + at * 1024), 16, 0, 0);
      }
    }
    if (i + 1 < steps) look(i + 1);
  };
  if (steps > 0) {
    look(0);
#pragma unroll
    for (int i = 0; i < S - 1; ++i)
      if (i < steps) issue(i, i, lds[kw][i][0], lds[kw][i][1]);
  }

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
  const int wave_first = (t.first + rw * U * 16) / rep;  // tokens of the wave's rows
  const int wave_last = (min(t.first + (rw + 1) * U * 16, rows) - 1) / rep;
  const bool idle = t.first + rw * U * 16 >= rows;
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

  auto step = [&](int i, int stage, int next, const uint16_t* __restrict__ ks, const uint16_t* __restrict__ vs,
                  uint16_t* __restrict__ kd, uint16_t* __restrict__ vd) {
    const int kt = t0 + i * KW + kw, s0 = kt * KT;
    if (i + S - 1 < steps) issue(i + S - 1, next, kd, vd);
    if (kt >= t1 || idle || (causal && s0 > t.past + wave_last)) return;
    f32x4_t s[U][NT];
    U32x4 ka[NT][NC];
#pragma unroll
    for (int st = 0; st < NT; ++st)
#pragma unroll
      for (int c = 0; c < NC; ++c) ka[st][c] = at.row16(ks, st, c);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int st = 0; st < NT; ++st)
#pragma unroll
      for (int u = 0; u < U; ++u) s[u][st] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int sp = 0; sp < NT; sp += 2)
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int st = sp; st < sp + 2; ++st)
#pragma unroll
          for (int u = 0; u < U; ++u) s[u][st] = mfma16<F16>(ka[st][c], qb[u][c], s[u][st]);
    U32x4 va[NH][ND];
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int d = 0; d < ND; ++d) va[0][d] = at.columns32(vs, 0, d);
    __builtin_amdgcn_sched_barrier(0);
    const uint32_t none = (uint32_t)(bad >> (4 * stage)) & 15u;
    const bool edge = s0 + KT > t.past + (causal ? wave_first + 1 : 0) || none;  // uniform
    if (edge) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int st = 0; st < NT; ++st) {
          const int k0 = s0 + st * 16 + 4 * g, j0 = k0 - t.past;
          uint32_t bits = 15;  // of the lane's four keys
          if (causal) {
            const int more = token[u] - j0;  // keys k0 .. k0 + more
            bits = more >= 3 ? 15u : more < 0 ? 0u : (2u << more) - 1u;
          } else if (j0 > -4) {
            const uint64_t* row = a.tree + (int64_t)(t.start + max(token[u], 0)) * a.words;
            bits = 0;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int j = j0 + x;
              const bool own = j < 0 || (j < 64 * a.words && (row[min(max(j, 0) >> 6, a.words - 1)] >> (j & 63) & 1));
              bits |= own ? 1u << x : 0u;
            }
          }
          if (none >> st & 1) bits = 0;
          if (token[u] < 0) bits = 0;
#pragma unroll
          for (int x = 0; x < 4; ++x)
            if (!(bits >> x & 1) || k0 + x >= t.len) s[u][st][x] = -__builtin_inff();
        }
    }
    // V rows that are no keys: probability 0 times what lies there could be NaN
    const bool holes = s0 + KT > t.len || none;  // uniform
    auto clear = [&](int hh) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        uint32_t keep[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int k0 = s0 + 32 * hh + 16 * q + 4 * g + 2 * x;
          const bool no = none >> (2 * hh + q) & 1;
          keep[x] = (no || k0 >= t.len ? 0u : 0xffffu) | (no || k0 + 1 >= t.len ? 0u : 0xffff0000u);
        }
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          va[hh][d].v[2 * q] &= keep[0];
          va[hh][d].v[2 * q + 1] &= keep[1];
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
    U32x4 pf[U][NH];
#pragma unroll
    for (int hh = 0; hh < NH; ++hh) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          float p[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) p[j] = exp2_f(fmaf(s[u][2 * hh + q][j], scale, -m[u]));
          pf[u][hh].v[2 * q] = pack2<F16>(p[0], p[1]);
          pf[u][hh].v[2 * q + 1] = pack2<F16>(p[2], p[3]);
        }
      if (hh > 0) {
#pragma unroll
        for (int d = 0; d < ND; ++d) va[hh][d] = at.columns32(vs, hh, d);
      }
      if (holes) clear(hh);
#pragma unroll
      for (int u = 0; u < U; ++u) l[u] = mfma16<F16>(ones, pf[u][hh], l[u]);
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int u = 0; u < U; ++u) o[u][d] = mfma16<F16>(va[hh][d], pf[u][hh], o[u][d]);
    }
  };
  int stage = 0;
  for (int i = 0; i < steps; ++i) {
    constexpr int LOADS = 2 * GW * UG;
    if (S > 2 && i + S - 1 <= steps) tile_wait<(S - 2) * LOADS>();
    else tile_wait<0>();
    if (RW > 1) tile_barrier();  // the tile has landed for every wave, and all are done with the one before
    const int next = stage == 0 ? S - 1 : stage - 1;
    step(i, stage, next, lds[kw][stage][0], lds[kw][stage][1], lds[kw][next][0], lds[kw][next][1]);
    stage = stage == S - 1 ? 0 : stage + 1;
  }

  // ---- results
  const bool whole = t.splits == 1;
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

// Joins the ranges of one row and kv head: HD / 4 lanes take four columns each of a head.
template <bool F16, int HD, int KT>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttnArgs a) {
  const int rep = a.heads / a.kv_heads, RB = a.block_rows;
  const int row = blockIdx.x;
  const float* ml = a.work + (int64_t)a.units * a.kv_heads * RB * HD;
  PagedUnit u;
  int w = 0;
  if (!paged_find<KT>(a, w, u, row) || u.splits == 1) return;
  for (int x = threadIdx.x; x < a.heads * (HD / 4); x += 256) {
    const int head = x / (HD / 4), col = x % (HD / 4) * 4, kvh = head / rep;
    const int at = (row - u.start) * rep + head % rep;  // a head's row may begin the next block
    const int first = w + (at / RB - u.first / RB) * u.splits;
    if (first + u.splits > a.units) continue;  // bounds that decrease
    float mx = kNoScore, l = 0.f;
    f32x4_t o = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < u.splits; ++s) {
      const int64_t part = ((int64_t)(first + s) * a.kv_heads + kvh) * RB + at % RB;
      const float2 e = *reinterpret_cast<const float2*>(ml + 2 * part);
      const f32x4_t v = *reinterpret_cast<const f32x4_t*>(a.work + part * HD + col);
      const float mn = fmaxf(mx, e.x), f = exp2_f(mx - mn), k = exp2_f(e.x - mn);
      mx = mn;
      l = l * f + e.y * k;
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = o[j] * f + v[j] * k;
    }
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
    uint2 y;
    y.x = pack2<F16>(o[0] * inv, o[1] * inv);
    y.y = pack2<F16>(o[2] * inv, o[3] * inv);
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + ((int64_t)row * a.heads + head) * HD + col) = y;
  }
}

int64_t paged_blocks(const PagedAttnArgs& a) { return ((int64_t)a.units + 7) / 8 * 8 * a.kv_heads; }

template <bool F16, int HD, int RW, int KW, int U, int S>
hipError_t run_paged(const PagedAttnArgs& a, hipStream_t s) {
  paged_kernel<F16, HD, RW, KW, U, S><<<dim3((unsigned)paged_blocks(a)), 64 * RW * KW, 0, s>>>(a);
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  if (a.slots > 0) paged_join_kernel<F16, HD, RW == 1 ? 32 : 64><<<dim3((unsigned)a.Tq), 256, 0, s>>>(a);
  return hipGetLastError();
}

template <bool F16, int HD>
hipError_t paged_hd(const PagedAttnArgs& a, hipStream_t s) {
  constexpr int S1 = HD == 128 ? 2 : 3;
  switch (a.block_rows) {
    case 16: return run_paged<F16, HD, 1, 4, 1, S1>(a, s);
    case 32: return run_paged<F16, HD, 1, 4, 2, S1>(a, s);
    case 64: return run_paged<F16, HD, 2, 2, 2, 2>(a, s);
    default: return run_paged<F16, HD, 4, 1, 2, S1>(a, s);
  }
}

}  // namespace

void paged_attn_plan(PagedAttnArgs& a) {
  const int rep = a.heads / a.kv_heads;
  const int64_t B = a.B > 0 ? a.B : 1, rows = (int64_t)a.Tq * rep, each = (rows + B - 1) / B;
  a.block_rows = each <= 16 ? 16 : each <= 32 ? 32 : each <= 64 ? 64 : 128;
  const int64_t blocks = rows / a.block_rows + B;
  const int64_t want = ((int64_t)device_cus() + a.kv_heads - 1) / a.kv_heads;
  a.slots = a.B > kPagedSeqs || blocks >= 4 * want ? 0 : (int)want;
  a.least = a.block_rows <= 32 ? 4 : 2;
  const int64_t units = a.slots + blocks + 2;
  a.units = units > INT32_MAX ? INT32_MAX : (int)units;
}
int64_t paged_attn_workspace(const PagedAttnArgs& a) {
  return a.slots > 0 ? (int64_t)a.units * a.kv_heads * a.block_rows * (a.head_dim + 2) * 4 : 0;
}
int64_t paged_attn_threads(const PagedAttnArgs& a) {
  const int64_t tiles = 256 * paged_blocks(a), join = a.slots > 0 ? 256 * (int64_t)a.Tq : 0;
  return tiles > join ? tiles : join;
}

hipError_t launch_paged_attn(const PagedAttnArgs& a, hipStream_t s) { MHC_PACKED_HD(paged_hd, a, s) }

}  // namespace mhc
