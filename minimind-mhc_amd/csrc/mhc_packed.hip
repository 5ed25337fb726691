// Causal attention over packed sequences: forward.  q [Tq, heads, HD], k and v
// [Tk, kv_heads, HD] hold the sequences one after another (k and v perhaps in cache slots
// that are only partly used); the last query of a sequence sits at its last key.  16-bit
// tensors (bf16 or fp16), fp32 scores, sums and outputs, one rounding of the probabilities
// (they are a product's operand) and one of the output.
//   S_ij = scale q_i . k_j (j <= i + keys - queries),  O_i = sum_j softmax(S_i)_j v_j
#include "mhc_packed.hpp"

namespace mhc {
namespace {

// ------------------------------------------------------------- tiles of many queries
// A workgroup per (tile of 128 query rows of one kv head, range of the keys): HP query heads
// times 128 / HP positions, 32 rows a wave; with KS = 2 four more waves take every second key
// tile of the same rows and the halves join at the end.
//   * S^T = K Q^T and O^T = V^T P^T on v_mfma 16x16x32: a lane holds scores and outputs of
//     one query row, and S^T's registers, rounded, are P^T's operand as they stand.  V^T comes
//     from the row-major tile by the transposing LDS load.
//   * K and V tiles of 64 keys come through a ring of LDS stages by direct-to-LDS loads,
//     one tile (head_dim 128) or two ahead: through registers 0.5 us of a 1.7 us step was waiting.
//   * The second half's softmax stands between the first half's output products, so the
//     matrix cores and the VALU of a wave work side by side there.
// Two fp16 sequences of 11903 and 4480 tokens, 8 / 2 heads of 128: 336 to 395 us, 840 to 990 TFLOP/s
// (an 8192^3 product of the library 1268); matrix cores busy 49% of the time, the VALU 52%. Three
// of 16001 together, 8 heads of 64: 201 us, 650 TFLOP/s, 43% and 61%: the exponentials bound it. 16 prompts
// of 8192 together, 8 / 4 heads of 96: 37 us, of which the longest prompt's chain is 28.
template <bool F16, int HD, int HP, int KS>
__global__ __launch_bounds__(256 * KS, 2) void packed_fwd_kernel(PackedAttnArgs a) {
  constexpr int NC = HD / 32, ND = HD / 16, KT = 64;
  constexpr int PW = 128 / HP;
  constexpr int S = HD == 128 ? 2 : 3;     // stages
  constexpr int TILE = KT * HD;            // elements
  constexpr int UW = TILE * 2 / 1024 / 4;  // 1 KiB units of a tile a wave loads
  __shared__ __align__(16) uint16_t lds[KS][S][2][TILE];
  static_assert(KS == 1 || sizeof(lds) >= 4 * 64 * (2 * ND * 16 + 16), "the second half's sums take the tiles' place");
  const int tid = threadIdx.x & 255;
  const int half = KS == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int r = lane & 15, g = lane >> 4;
  const int groups = a.heads / HP;
  const int grp = blockIdx.x % groups;
  const int rest = blockIdx.x / groups;
  const int split = rest % a.splits;
  PackedTile t;
  PackedKeys kk;
  packed_rank<false>(a.cu_q, a.B, a.Tq, PW, a.qtiles, rest / a.splits, a.cu_k, a.Tk, nullptr, a.k_len, t, kk);
  if (t.first >= t.end) return;
  const int h = grp * HP + (HP == 2 ? wave >> 1 : 0);
  const int kvh = grp * HP / (a.heads / a.kv_heads);
  const int pb = t.first + (HP == 2 ? (wave & 1) * 32 : wave * 32);  // the wave's first row
  const int shift = kk.len - t.end;       // row x sees the keys up to x + shift
  const int last = min(t.first + PW, t.end) - 1 + shift;  // last key any row of the tile sees
  // this workgroup's range of the tile's keys, in whole key tiles
  const int nt_all = last < 0 ? 0 : last / KT + 1;
  const int per = (nt_all + a.splits - 1) / a.splits;
  const int t0 = split * per, t1 = min(t0 + per, nt_all);

  const int64_t ks_t = a.ks_t, vs_t = a.vs_t;
  const uint16_t* kg = static_cast<const uint16_t*>(a.k) + kk.start * ks_t + kvh * a.ks_h;
  const uint16_t* vg = static_cast<const uint16_t*>(a.v) + kk.start * vs_t + kvh * a.vs_h;
  TileLoader<HD, UW> kl, vl;
  kl.init(wave * UW, ks_t);
  vl.init(wave * UW, vs_t);
  // the i-th key tile of this half (a half without one loads the last again: the barriers and
  // waits are the same for all)
  auto issue = [&](int i, uint16_t* __restrict__ kd, uint16_t* __restrict__ vd) {
    const int kt = min(t0 + i * KS + half, t1 - 1);
    const int left = kk.len - kt * KT;
    kl.issue(kd, kg + (int64_t)kt * KT * ks_t, wave * UW, ks_t, KT, left);
    vl.issue(vd, vg + (int64_t)kt * KT * vs_t, wave * UW, vs_t, KT, left);
  };
  const int steps = t0 < t1 ? (t1 - t0 + KS - 1) / KS : 0;
  U32x4 qb[2][NC];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int64_t row = min(pb + u * 16 + r, t.end - 1);
    const uint16_t* q = static_cast<const uint16_t*>(a.q) + row * a.qs_t + h * a.qs_h + 8 * g;
#pragma unroll
    for (int c = 0; c < NC; ++c) qb[u][c] = ld16(q + 32 * c);
  }
#pragma unroll
  for (int i = 0; i < S - 1; ++i)
    if (i < steps) issue(i, lds[half][i][0], lds[half][i][1]);
  const float scale = a.scale * kPackedLog2e;
  constexpr float kHead = packed_head<F16>;
  float m[2] = {kNoScore, kNoScore};
  f32x4_t l[2] = {f32x4_t{0.f, 0.f, 0.f, 0.f}, f32x4_t{0.f, 0.f, 0.f, 0.f}};
  const U32x4 ones = packed_ones<F16>();
  f32x4_t o[2][ND];
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int d = 0; d < ND; ++d) o[u][d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  // this lane's places in a tile: K rows 16 st + r, columns 32 c + 8 g; V rows 4 g + r / 4 of
  // 16, columns 16 d + 4 (r % 4)
  TileReads<HD> at;
  at.init(r, g);

  // Step i: the tile in ks and vs, while one lands in kd and vd.  As restrict parameters the
  // compiler sees that they differ; else it waits for every load in flight at each step.
  auto step = [&](int i, const uint16_t* __restrict__ ks, uint16_t* __restrict__ vs, uint16_t* __restrict__ kd,
                  uint16_t* __restrict__ vd) {
    const int kt = t0 + i * KS + half, s0 = kt * KT;
    if (i + S - 1 < steps) issue(i + S - 1, kd, vd);
    // V rows that are not there: probability 0 times an infinite copy of the last would be
    // NaN.  Only a sequence's last tile has any (uniform over the workgroup's half; both
    // halves take part in the barrier).
    if (t0 * KT + (i + 1) * KS * KT > kk.len) {
      if (kt < t1) {
        for (int x = tid; x < KT * (HD / 8); x += 256)
          if (s0 + x / (HD / 8) >= kk.len) *reinterpret_cast<U32x4*>(&vs[x * 8]) = U32x4{};
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      tile_barrier();
    }
    if (kt >= t1 || pb >= t.end || s0 > pb + 31 + shift) return;  // no rows, or wholly above their diagonal
    // Operands are read from LDS a step ahead of their products; the barriers keep the
    // compiler from sinking each read to its use, where every pair of products would wait.
    f32x4_t s[2][4];
    U32x4 ka[4][NC];
#pragma unroll
    for (int st = 0; st < 4; ++st)
#pragma unroll
      for (int c = 0; c < NC; ++c) ka[st][c] = at.row16(ks, st, c);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int st = 0; st < 4; ++st) {
      s[0][st] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      s[1][st] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int sp = 0; sp < 4; sp += 2)
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int st = sp; st < sp + 2; ++st) {
          s[0][st] = mfma16<F16>(ka[st][c], qb[0][c], s[0][st]);
          s[1][st] = mfma16<F16>(ka[st][c], qb[1][c], s[1][st]);
        }
    U32x4 va[2][ND];
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int d = 0; d < ND; ++d) va[0][d] = at.columns32(vs, 0, d);
    __builtin_amdgcn_sched_barrier(0);
    if (s0 + KT - 1 > pb + shift) {  // uniform: only the tiles on the diagonal are compared
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int st = 0; st < 4; ++st)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (s0 + st * 16 + 4 * g + i > pb + u * 16 + r + shift) s[u][st][i] = -__builtin_inff();
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      float mx = -__builtin_inff();
#pragma unroll
      for (int st = 0; st < 4; ++st)
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
    U32x4 pf[2][2];
    auto softmax = [&](int hh) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          float p[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) p[j] = exp2_f(fmaf(s[u][2 * hh + q][j], scale, -m[u]));
          pf[u][hh].v[2 * q] = pack2<F16>(p[0], p[1]);
          pf[u][hh].v[2 * q + 1] = pack2<F16>(p[2], p[3]);
        }
    };
    auto outputs = [&](int hh) {
#pragma unroll
      for (int u = 0; u < 2; ++u) l[u] = mfma16<F16>(ones, pf[u][hh], l[u]);
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int u = 0; u < 2; ++u) o[u][d] = mfma16<F16>(va[hh][d], pf[u][hh], o[u][d]);
    };
    softmax(0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int d = 0; d < ND; ++d) va[1][d] = at.columns32(vs, 1, d);
    __builtin_amdgcn_sched_barrier(0);
    // the first half's products with the second half's softmax between them
    outputs(0);
    softmax(1);
#pragma unroll
    for (int x = 0; x < 2 * ND + 2; ++x) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x402, ND == 4 ? 4 : 3, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
    outputs(1);
  };
  int stage = 0;
  for (int i = 0; i < steps; ++i) {
    if (S > 2 && i + S - 1 <= steps) tile_wait<(S - 2) * 2 * UW>();
    else tile_wait<0>();
    tile_barrier();  // this step's tile has landed, and every wave is done with the one before
    const int next = stage == 0 ? S - 1 : stage - 1;
    step(i, lds[half][stage][0], lds[half][stage][1], lds[half][next][0], lds[half][next][1]);
    stage = stage == S - 1 ? 0 : stage + 1;
  }
  if constexpr (KS == 2) {  // the halves meet in LDS
    __syncthreads();
    float* x = reinterpret_cast<float*>(lds) + wave * 64 * (2 * ND * 4 + 4) + lane * 4;
    if (half == 1) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int d = 0; d < ND; ++d) *reinterpret_cast<f32x4_t*>(x + (u * ND + d) * 256) = o[u][d];
      *reinterpret_cast<f32x4_t*>(x + 2 * ND * 256) = f32x4_t{m[0], m[1], l[0][0], l[1][0]};
    }
    __syncthreads();
    if (half == 1) return;
    const f32x4_t ml = *reinterpret_cast<const f32x4_t*>(x + 2 * ND * 256);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const float mx = fmaxf(m[u], ml[u]);
      const float f = exp2_f(m[u] - mx), e = exp2_f(ml[u] - mx);
      m[u] = mx;
      l[u][0] = l[u][0] * f + ml[2 + u] * e;
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        const f32x4_t y = *reinterpret_cast<const f32x4_t*>(x + (u * ND + d) * 256);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[u][d][i] = o[u][d][i] * f + y[i] * e;
      }
    }
  }
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const float ls = l[u][0];
    const int row = pb + u * 16 + r;
    if (row >= t.end) continue;
    const int64_t at = (int64_t)row * a.heads + h;
    if (a.splits > 1) {
      const int64_t part = (int64_t)split * a.Tq * a.heads + at;
      float* w = a.work + part * HD + 4 * g;
#pragma unroll
      for (int d = 0; d < ND; ++d) *reinterpret_cast<f32x4_t*>(w + 16 * d) = o[u][d];
      if (g == 0) {
        float* ml = a.work + (int64_t)a.splits * a.Tq * a.heads * HD + 2 * part;
        ml[0] = m[u];
        ml[1] = ls;
      }
      continue;
    }
    const float inv = ls > 0.f || ls != ls ? 1.f / ls : 0.f;  // a row without keys: zeros
    uint16_t* out = static_cast<uint16_t*>(a.out) + at * HD + 4 * g;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      uint2 w, x;
      w.x = round2<F16>(o[u][d][0] * inv, o[u][d][1] * inv, a.rest ? &x.x : nullptr);
      w.y = round2<F16>(o[u][d][2] * inv, o[u][d][3] * inv, a.rest ? &x.y : nullptr);
      *reinterpret_cast<uint2*>(out + 16 * d) = w;
      if (a.rest) *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.rest) + at * HD + 4 * g + 16 * d) = x;
    }
    if (a.lse && g == 0) a.lse[(int64_t)h * a.Tq + row] = packed_lse(m[u], ls);
  }
}

// --------------------------------------------------------------- few queries, many keys
// A workgroup takes up to 16 rows (tokens times query heads of one kv head) and a range of
// the keys; its four waves take the range's 32-key tiles in turn, each with sums and LDS of
// its own (no barrier in the loop), and join at the end.  Bound by the cache's bytes, each
// read once: 64 single tokens over slots of 2176 rows, 4 kv heads of 96, 144 MB, 33 us, 4.4 TB/s
// (the first keys arrive some 5 us after the launch; 5.5 TB/s then).
template <bool F16, int HD>
__global__ __launch_bounds__(256) void packed_few_kernel(PackedAttnArgs a) {
  constexpr int NC = HD / 32, ND = HD / 16, KT = 32;
  constexpr int KST = HD + 8, VST = HD + 16;
  constexpr int PPT = KT * (HD / 8) / 64;
  constexpr int WAVE_LDS = KT * (KST + VST);  // elements
  static_assert(WAVE_LDS * 2 >= (16 * HD + 32) * 4, "the waves' sums take the tiles' place");
  __shared__ __align__(16) uint16_t lds[4][WAVE_LDS];
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int r = lane & 15, g = lane >> 4;
  const int rep = a.heads / a.kv_heads;
  const int HB = a.row_heads, nb = (rep + HB - 1) / HB;  // heads of a workgroup, workgroups of a kv head
  const int RT = 16 / HB;
  const int groups = a.kv_heads * nb;
  // the heads of one range go to one XCD, whose L2 then sees whole lines of a key's row:
  // workgroups are dealt to the 8 XCDs in turn
  const int block = blockIdx.x / (8 * groups), in = blockIdx.x % (8 * groups);
  const int grp = in / 8;
  const int rest = block * 8 + in % 8;
  const int split = rest % a.splits;
  const int tile = rest / a.splits;
  if (tile >= a.qtiles) return;
  PackedTile t;
  PackedKeys kk;
  packed_find(a.cu_q, a.B, a.Tq, RT, tile, a.cu_k, a.Tk, nullptr, a.k_len, t, kk);
  if (t.first >= t.end) return;
  const int kvh = grp / nb;
  const int hr = grp % nb * HB + r % HB;  // the lane's head in its group
  const int row = t.first + r / HB;
  const bool live = r < RT * HB && hr < rep && row < t.end;
  const int h = kvh * rep + (live ? hr : 0);
  const int shift = kk.len - t.end;
  const int last = min(t.first + RT, t.end) - 1 + shift;
  const int nt_all = last < 0 ? 0 : last / KT + 1;
  const int per = (nt_all + a.splits - 1) / a.splits;
  const int t0 = split * per, t1 = min(t0 + per, nt_all);

  const int64_t ks_t = a.ks_t, vs_t = a.vs_t;
  const uint16_t* kg = static_cast<const uint16_t*>(a.k) + kk.start * ks_t + kvh * a.ks_h;
  const uint16_t* vg = static_cast<const uint16_t*>(a.v) + kk.start * vs_t + kvh * a.vs_h;
  uint16_t* ks = lds[wave];
  uint16_t* vs = ks + KT * KST;
  U32x4 kr[PPT], vr[PPT];
  auto load = [&](int s0) {
#pragma unroll
    for (int p = 0; p < PPT; ++p) {
      const int piece = p * 64 + lane;
      const int at = min(s0 + piece / (HD / 8), kk.len - 1);
      const int col = (piece % (HD / 8)) * 8;
      kr[p] = ld16_nt(kg + at * ks_t + col);
      vr[p] = ld16_nt(vg + at * vs_t + col);
    }
  };
  if (t0 + wave < t1) load((t0 + wave) * KT);
  U32x4 qb[NC];
  {
    const uint16_t* q = static_cast<const uint16_t*>(a.q) + (int64_t)(live ? row : t.first) * a.qs_t + h * a.qs_h + 8 * g;
#pragma unroll
    for (int c = 0; c < NC; ++c) qb[c] = ld16(q + 32 * c);
  }
  const float scale = a.scale * kPackedLog2e;
  constexpr float kHead = packed_head<F16>;
  const int limit = live ? row + shift : -1;  // last key the lane's row sees
  float m = kNoScore;
  f32x4_t l = {0.f, 0.f, 0.f, 0.f};  // sums of the rounded probabilities, as in the tiles of many queries
  const U32x4 ones = packed_ones<F16>();
  f32x4_t o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) o[d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  for (int kt = t0 + wave; kt < t1; kt += 4) {
    const int s0 = kt * KT;
#pragma unroll
    for (int p = 0; p < PPT; ++p) {
      const int piece = p * 64 + lane;
      const int at = piece / (HD / 8);
      const int col = (piece % (HD / 8)) * 8;
      *reinterpret_cast<U32x4*>(&ks[at * KST + col]) = kr[p];
      *reinterpret_cast<U32x4*>(&vs[at * VST + col]) = vr[p];
    }
    if (s0 + KT > kk.len)  // rows that are not there: 0 x infinity would be NaN
#pragma unroll
      for (int p = 0; p < PPT; ++p) {
        const int piece = p * 64 + lane;
        const int at = piece / (HD / 8);
        if (s0 + at >= kk.len) *reinterpret_cast<U32x4*>(&vs[at * VST + (piece % (HD / 8)) * 8]) = U32x4{};
      }
    if (kt + 4 < t1) load(s0 + 4 * KT);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    f32x4_t s[2];
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      s[st] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < NC; ++c)
        s[st] = mfma16<F16>(*reinterpret_cast<const U32x4*>(&ks[(st * 16 + r) * KST + 32 * c + 8 * g]), qb[c], s[st]);
    }
#pragma unroll
    for (int st = 0; st < 2; ++st)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (s0 + st * 16 + 4 * g + i > limit) s[st][i] = -__builtin_inff();
    float mx = -__builtin_inff();
#pragma unroll
    for (int st = 0; st < 2; ++st)
#pragma unroll
      for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[st][i]);
    mx *= scale;
    if (__any(!(mx <= m + kPackedLazyMax + kHead))) {
      mx = fmaxf(mx, xor_lane16(mx));
      mx = fmaxf(mx, xor_lane32(mx));
      mx = fmaxf(mx - kHead, m);
      const float f = exp2_f(m - mx);
      m = mx;
#pragma unroll
      for (int i = 0; i < 4; ++i) l[i] *= f;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[d][i] *= f;
    }
    U32x4 pf;
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      float p[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) p[i] = exp2_f(fmaf(s[st][i], scale, -m));
      pf.v[2 * st] = pack2<F16>(p[0], p[1]);
      pf.v[2 * st + 1] = pack2<F16>(p[2], p[3]);
    }
    l = mfma16<F16>(ones, pf, l);
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      U32x4 va;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const u32x2_v w = lds_tr4(&vs[(q * 16 + 4 * g + (r >> 2)) * VST + 16 * d + 4 * (r & 3)]);
        va.v[2 * q] = w.x;
        va.v[2 * q + 1] = w.y;
      }
      o[d] = mfma16<F16>(va, pf, o[d]);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
  // the waves' sums meet in LDS: [16 rows][HD] and then each row's maximum and sum
  __syncthreads();
  float* mine = reinterpret_cast<float*>(lds[wave]);
#pragma unroll
  for (int d = 0; d < ND; ++d) *reinterpret_cast<f32x4_t*>(mine + r * HD + 16 * d + 4 * g) = o[d];
  if (g == 0) {
    mine[16 * HD + r] = m;
    mine[16 * HD + 16 + r] = l[0];
  }
  __syncthreads();
  // thread (row of 16, 1/16 of the columns)
  const int tr = tid >> 4, tc = tid & 15;
  const int ohr = grp % nb * HB + tr % HB, orow = t.first + tr / HB;
  if (tr >= RT * HB || ohr >= rep || orow >= t.end) return;
  float mx = kNoScore, ls = 0.f, f[4];
#pragma unroll
  for (int w = 0; w < 4; ++w) mx = fmaxf(mx, reinterpret_cast<const float*>(lds[w])[16 * HD + tr]);
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float* p = reinterpret_cast<const float*>(lds[w]);
    f[w] = exp2_f(p[16 * HD + tr] - mx);
    ls += f[w] * p[16 * HD + 16 + tr];
  }
  const int oh = kvh * rep + ohr;
  const int64_t at = (int64_t)orow * a.heads + oh;
  const int64_t part = (int64_t)split * a.Tq * a.heads + at;
  const float inv = a.splits > 1 ? 1.f : ls > 0.f || ls != ls ? 1.f / ls : 0.f;
#pragma unroll
  for (int c = 2 * tc; c < HD; c += 32) {
    float x = 0.f, y = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float* p = reinterpret_cast<const float*>(lds[w]) + tr * HD + c;
      x += f[w] * p[0];
      y += f[w] * p[1];
    }
    if (a.splits > 1) {
      *reinterpret_cast<float2*>(a.work + part * HD + c) = make_float2(x, y);
      continue;
    }
    uint32_t rest;
    *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + at * HD + c) =
        round2<F16>(x * inv, y * inv, a.rest ? &rest : nullptr);
    if (a.rest) *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.rest) + at * HD + c) = rest;
  }
  if (tc != 0) return;
  if (a.splits > 1) {
    float* ml = a.work + (int64_t)a.splits * a.Tq * a.heads * HD + 2 * part;
    ml[0] = mx;
    ml[1] = ls;
  } else if (a.lse) {
    a.lse[(int64_t)oh * a.Tq + orow] = packed_lse(mx, ls);
  }
}

// Joins the key ranges of one row and head: HD / 4 lanes take four columns each, the other
// lanes of the workgroup every 8th (16th) range, and the sums meet in LDS.
template <bool F16, int HD>
__global__ __launch_bounds__(256) void packed_merge_kernel(PackedAttnArgs a) {
  constexpr int LPR = HD <= 64 ? 16 : 32;
  constexpr int PAR = 256 / LPR;
  __shared__ __align__(16) float acc[PAR][HD + 4];
  const int64_t rows = (int64_t)a.Tq * a.heads;
  const int64_t at = blockIdx.x;
  const int col = threadIdx.x % LPR, sub = threadIdx.x / LPR;
  const bool live = col < HD / 4;
  const float* part = a.work + at * HD + (live ? 4 * col : 0);
  const float2* ml = reinterpret_cast<const float2*>(a.work + (int64_t)a.splits * rows * HD) + at;
  float mx = kNoScore, l = 0.f;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = sub; s < a.splits; s += PAR) {
    const float2 w = ml[s * rows];
    const f32x4_t v = *reinterpret_cast<const f32x4_t*>(part + s * rows * HD);
    const float mn = fmaxf(mx, w.x);
    const float f = exp2_f(mx - mn), e = exp2_f(w.x - mn);
    mx = mn;
    l = l * f + w.y * e;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = o[j] * f + v[j] * e;
  }
  if (live) *reinterpret_cast<f32x4_t*>(&acc[sub][4 * col]) = o;
  if (col == 0) {
    acc[sub][HD] = mx;
    acc[sub][HD + 1] = l;
  }
  __syncthreads();
  if (threadIdx.x >= HD / 2) return;
  float m = kNoScore, ls = 0.f, x = 0.f, y = 0.f;
  const int c = 2 * threadIdx.x;
#pragma unroll
  for (int s = 0; s < PAR; ++s) m = fmaxf(m, acc[s][HD]);
#pragma unroll
  for (int s = 0; s < PAR; ++s) {
    const float f = exp2_f(acc[s][HD] - m);
    ls += f * acc[s][HD + 1];
    x += f * acc[s][c];
    y += f * acc[s][c + 1];
  }
  const float inv = ls > 0.f || ls != ls ? 1.f / ls : 0.f;
  uint32_t rest;
  *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + at * HD + c) =
      round2<F16>(x * inv, y * inv, a.rest ? &rest : nullptr);
  if (a.rest) *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.rest) + at * HD + c) = rest;
  if (a.lse && c == 0) a.lse[at % a.heads * a.Tq + at / a.heads] = packed_lse(m, ls);
}

int64_t few_blocks(const PackedAttnArgs& a) {
  const int nb = (a.heads / a.kv_heads + a.row_heads - 1) / a.row_heads;
  return ((int64_t)a.qtiles * a.splits + 7) / 8 * 8 * a.kv_heads * nb;
}
int64_t tile_blocks(const PackedAttnArgs& a) { return (int64_t)a.qtiles * a.splits * (a.heads / a.row_heads); }

template <bool F16, int HD>
hipError_t packed_fwd_hd(const PackedAttnArgs& a, hipStream_t s) {
  if (a.few) {
    packed_few_kernel<F16, HD><<<dim3((unsigned)few_blocks(a)), 256, 0, s>>>(a);
  } else {
    const dim3 grid((unsigned)tile_blocks(a));
    const bool halves = packed_halves(grid.x);
    if (a.row_heads == 2) {
      if (halves) packed_fwd_kernel<F16, HD, 2, 2><<<grid, 512, 0, s>>>(a);
      else packed_fwd_kernel<F16, HD, 2, 1><<<grid, 256, 0, s>>>(a);
    } else {
      if (halves) packed_fwd_kernel<F16, HD, 1, 2><<<grid, 512, 0, s>>>(a);
      else packed_fwd_kernel<F16, HD, 1, 1><<<grid, 256, 0, s>>>(a);
    }
  }
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  if (a.splits > 1)
    packed_merge_kernel<F16, HD><<<dim3((unsigned)((int64_t)a.Tq * a.heads)), 256, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace

// Which kernel, how many heads a workgroup takes and into how many ranges the keys go. Only
// the totals are known here; the sequences' own lengths are read on the device.
// Times of the launches, join included:
//   * The kernel for few rows up to 8 rows (tokens times query heads of a kv head) a sequence on
//     average: 64 sequences over 2176-row slots, 8 / 4 heads of 96, 1 new token each 36.4 us (the other
//     kernel 39.4), 4 tokens 36.8 and 39.3, 8 tokens 54.3 and 39.4.
//   * Ranges: two workgroups a CU, none of under 128 (512) keys on average, 128 at most. Those 64 single
//     tokens in 1, 2, 4 and 8 ranges: 39.7, 36.7, 37.5, 42.1 us; 4 sequences of 4 tokens over 8000 keys each in 8, 16,
//     32 and 64: 23.6, 22.5, 18.0, 20.8; one token over 65001 keys, 16 / 2 heads of 128, in 64, 128, 256 and 512:
//     26.2, 20.8, 21.4, 29.4 (the join 3.9, 3.8, 5.2, 8.7 of them: hence the 128); one chunk of 512 tokens over
//     60000 keys, 16 / 2 heads of 128, in 2, 4, 8 and 16: 463, 262, 270, 277 (the products 960 TFLOP/s in 8); 8 of 128
//     over 4096 keys in 1, 4, 8 and 16: 64.3, 36.4, 35.9, 51.1.
void packed_attn_plan(PackedAttnArgs& a) {
  const int rep = a.heads / a.kv_heads;
  const int B = a.B > 0 ? a.B : 1;
  a.few = (int64_t)a.Tq * rep <= 8 * (int64_t)B;
  int groups, rows;
  if (a.few) {
    const int nb = (rep + 15) / 16;
    a.row_heads = (rep + nb - 1) / nb;
    groups = a.kv_heads * nb;
    rows = 16 / a.row_heads;
  } else {
    a.row_heads = rep % 2 == 0 ? 2 : 1;
    groups = a.heads / a.row_heads;
    rows = 128 / a.row_heads;
  }
  a.qtiles = (int)packed_tiles(a.Tq, a.B, rows);
  // workgroups with rows, about: at least one a sequence
  const int64_t full = ((int64_t)a.Tq + rows - 1) / rows, some = B < a.Tq ? B : a.Tq;
  const int64_t units = (full > some ? full : some) * groups;
  const int64_t keys = a.Tk / B;  // of a sequence, on average
  int64_t want = units > 0 ? (int64_t)device_cus() * 2 / units : 1;
  const int least = a.few ? 128 : 512;
  if (want > keys / least) want = keys / least;
  if (want > 128) want = 128;
  a.splits = want < 1 ? 1 : (int)want;
}
int64_t packed_attn_threads(const PackedAttnArgs& a) {
  const int64_t tiles = 256 * (a.few ? few_blocks(a) : tile_blocks(a));
  const int64_t merge = a.splits > 1 ? 256 * (int64_t)a.Tq * a.heads : 0;
  return tiles > merge ? tiles : merge;
}
int64_t packed_attn_workspace(const PackedAttnArgs& a) {
  return a.splits > 1 ? (int64_t)a.splits * a.Tq * a.heads * (a.head_dim + 2) * 4 : 0;
}

hipError_t launch_packed_attn(const PackedAttnArgs& a, hipStream_t s) { MHC_PACKED_HD(packed_fwd_hd, a, s) }

}  // namespace mhc
