// Causal attention over packed sequences: backward.  With P the probabilities (formed again
// from q, k and the forward's log sums) and G the output's gradient,
//   D_i = G_i . O_i,  dS_ij = P_ij (G_i . v_j - D_i),
//   dQ_i = scale sum_j dS_ij k_j,  dK_j = scale sum_i dS_ij q_i,  dV_j = sum_i P_ij G_i.
// One launch forms D and dQ by query tiles, a second dK and dV by key tiles, each summing
// its own rows' terms in registers (fp32): no atomics on sums, the same bits on every run.  P is
// formed twice for that: 7 products instead of 5.
//
// dS is an operand of products, so it is rounded to the tensors' type.  bf16 has fp32's range.
// An fp16 dS is multiplied by a power of two first, which the result is divided by: P of many
// keys times a gradient of 1e-3 lies below fp16's normal numbers (dQ over 8192 keys was off by 1e-2,
// for gradients of 1e-4 by 0.1).  No dS exceeds half the longest row of v times the length of its row of g
// (P_j sum_k P_k |dP_j - dP_k| <= P_j (1 - P_j) 2 |g| |v|), so the power that takes |g| |v| to 2^15 at most
// cannot overflow, and leaves 28 binary digits of normal numbers below.  dQ takes |g| of its own row, dK the
// longest row of g from the block of 1024 rows on where its keys are first seen.  This costs fp16 one
// launch (16001 rows, 8 heads of 64: 4.8 us of 749 a step).
#include "mhc_packed.hpp"

namespace mhc {
namespace {

// Rows of a block of g_top: few enough blocks that one load a lane reads those of a long sequence.
constexpr int kGradBlock = 1024;

// The exponent e with sqrt(w) 2^e in [2^14, 2^15), w = |g|^2 |v|^2; 0 where that is no positive number.
__device__ __forceinline__ int packed_exponent(float w) {
  return w > 0.f && w < __builtin_inff() ? 15 - ((__builtin_amdgcn_frexp_expf(w) + 1) >> 1) : 0;
}

// v_top: the longest of a tile's rows in use; 16 lanes a row (12 of them load at head_dim 96).  Also
// clears g_top, whose blocks the waves of the dQ kernel raise (a maximum: any order gives the same).
// 16001 rows, 8 heads of 64: 4.7 us.
template <int HD>
__global__ __launch_bounds__(256) void packed_v_top_kernel(PackedAttnArgs a) {
  __shared__ float top[4];
  const int kvh = blockIdx.x % a.kv_heads, tile = blockIdx.x / a.kv_heads;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.kv_heads * packed_tiles(a.Tq, a.B, kGradBlock);
       i += (int64_t)gridDim.x * 256)
    a.g_top[i] = 0.f;
  PackedTile t;
  PackedKeys o;
  packed_find(a.cu_k, a.B, a.Tk, 128, tile, a.cu_q, a.Tq, a.k_len, nullptr, t, o);
  if (t.first >= t.end) return;
  const int end = min(t.first + 128, t.start + t.used);
  const int sub = threadIdx.x & 15, row0 = t.first + (int)(threadIdx.x >> 4);
  U32x4 w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    w[i] = U32x4{};
    const int row = row0 + 16 * i;
    if (sub < HD / 8 && row < end)
      w[i] = ld16(static_cast<const uint16_t*>(a.v) + row * a.vs_t + kvh * a.vs_h + 8 * sub);
  }
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float x = elem_lo<true>(w[i].v[j]), y = elem_hi<true>(w[i].v[j]);
      s = fmaf(x, x, fmaf(y, y, s));
    }
    s += dpp_f<kDppXor1>(s);
    s += dpp_f<kDppXor2>(s);
    s += dpp_f<kDppHalfMirror>(s);
    s += dpp_f<kDppRowMirror>(s);
    most = fmaxf(most, s);
  }
  most = wave_max(most);
  if ((threadIdx.x & 63) == 0) top[threadIdx.x >> 6] = most;
  __syncthreads();
  if (threadIdx.x == 0)
    a.v_top[kvh * packed_tiles(a.Tk, a.B, 128) + tile] = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
}
// Of the first n keys of sequence seq, by one wave.
__device__ __forceinline__ float packed_v_top(const PackedAttnArgs& a, int kvh, int seq, int start, int n) {
  const float* p = a.v_top + kvh * packed_tiles(a.Tk, a.B, 128) + (start / 128 + seq);
  float most = 0.f;
  for (int i = __lane_id(); i < (n + 127) / 128; i += 64) most = fmaxf(most, p[i]);
  return wave_max(most);
}

// dQ: as the forward, one 4-wave workgroup per 128 query rows of one kv head, 32 rows a
// wave.  S^T = K Q^T and dP^T = V G^T put a lane's values all in one query row, and dS^T,
// rounded, is the operand of dQ^T = K^T dS^T as it stands.  Tiles, stages and halves as there.
// Three sequences of 16001 tokens together, 8 heads of 64: 229 us, 860 TFLOP/s of its three products
// (matrix cores busy 44%, VALU 59%); 12 of 8192, 8 / 4 heads of 96: 54 us.
template <bool F16, int HD, int HP, int KS>
__global__ __launch_bounds__(256 * KS, 2) void packed_dq_kernel(PackedAttnArgs a) {
  constexpr int NC = HD / 32, ND = HD / 16, KT = 64;
  constexpr int PW = 128 / HP;
  constexpr int S = HD == 128 ? 2 : 3;     // stages
  constexpr int TILE = KT * HD;            // elements
  constexpr int UW = TILE * 2 / 1024 / 4;  // 1 KiB units of a tile a wave loads
  __shared__ __align__(16) uint16_t lds_[KS][S][2][TILE];
  static_assert(KS == 1 || sizeof(lds_) >= 4 * 64 * 2 * ND * 16, "the second half's sums take the tiles' place");
  const int tid = threadIdx.x & 255;
  const int half = KS == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
  auto& lds = lds_[half];
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int r = lane & 15, g = lane >> 4;
  const int groups = a.heads / HP;
  const int grp = blockIdx.x % groups;
  PackedTile t;
  PackedKeys kk;
  packed_rank<false>(a.cu_q, a.B, a.Tq, PW, a.qtiles, blockIdx.x / groups, a.cu_k, a.Tk, nullptr, a.k_len, t, kk);
  if (t.first >= t.end) return;
  const int h = grp * HP + (HP == 2 ? wave >> 1 : 0);
  const int kvh = grp * HP / (a.heads / a.kv_heads);
  const int pb = t.first + (HP == 2 ? (wave & 1) * 32 : wave * 32);
  const int shift = kk.len - t.end;
  const int last = min(t.first + PW, t.end) - 1 + shift;
  const int nt_all = last < 0 ? 0 : last / KT + 1;
  const int nt = (nt_all - half + KS - 1) / KS, steps = (nt_all + KS - 1) / KS;  // this half's tiles

  const int64_t ks_t = a.ks_t, vs_t = a.vs_t;
  const uint16_t* kg = static_cast<const uint16_t*>(a.k) + kk.start * ks_t + kvh * a.ks_h;
  const uint16_t* vg = static_cast<const uint16_t*>(a.v) + kk.start * vs_t + kvh * a.vs_h;
  TileLoader<HD, UW> kl, vl;
  kl.init(wave * UW, ks_t);
  vl.init(wave * UW, vs_t);
  auto issue = [&](int i, uint16_t* __restrict__ kd, uint16_t* __restrict__ vd) {
    const int kt = i * KS + half, left = kk.len - kt * KT;
    kl.issue(kd, kg + (int64_t)kt * KT * ks_t, wave * UW, ks_t, KT, left);
    vl.issue(vd, vg + (int64_t)kt * KT * vs_t, wave * UW, vs_t, KT, left);
  };
  U32x4 qb[2][NC], gb[2][NC];
  float lse[2], delta[2], g2[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int row = pb + u * 16 + r;
    const int64_t at = min(row, t.end - 1);
    const uint16_t* q = static_cast<const uint16_t*>(a.q) + at * a.qs_t + h * a.qs_h + 8 * g;
    const int64_t off = (at * a.heads + h) * HD + 8 * g;
    const uint16_t* go = static_cast<const uint16_t*>(a.g_out) + off;
    const uint16_t* oo = static_cast<const uint16_t*>(a.out) + off;
    const uint16_t* ro = static_cast<const uint16_t*>(a.rest) + off;
    float d = 0.f, n = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      qb[u][c] = ld16(q + 32 * c);
      gb[u][c] = ld16(go + 32 * c);
      const U32x4 o = ld16(oo + 32 * c), rest = ld16(ro + 32 * c);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        d += elem_lo<F16>(gb[u][c].v[j]) * (elem_lo<F16>(o.v[j]) + elem_lo<F16>(rest.v[j]));
        d += elem_hi<F16>(gb[u][c].v[j]) * (elem_hi<F16>(o.v[j]) + elem_hi<F16>(rest.v[j]));
        if constexpr (F16) {
          const float x = elem_lo<F16>(gb[u][c].v[j]), y = elem_hi<F16>(gb[u][c].v[j]);
          n = fmaf(x, x, fmaf(y, y, n));
        }
      }
    }
    n += xor_lane16(n);
    g2[u] = n + xor_lane32(n);
    d += xor_lane16(d);
    d += xor_lane32(d);
    delta[u] = d;
    lse[u] = a.lse[(int64_t)h * a.Tq + at];
    if (half == 0 && g == 0 && row < t.end) a.delta[(int64_t)h * a.Tq + row] = d;
  }
#pragma unroll
  for (int i = 0; i < S - 1; ++i)
    if (i < nt) issue(i, lds[i][0], lds[i][1]);
  float out_scale[2] = {a.scale, a.scale};
  int g_most = 0;
  if constexpr (F16) {
    const float v2 = packed_v_top(a, kvh, t.seq, kk.start, max(last + 1, 0));
#pragma unroll
    for (int u = 0; u < 2; ++u) {  // P 2^e from here on
      const int e = packed_exponent(g2[u] * v2);
      lse[u] -= (float)e;
      out_scale[u] = __builtin_amdgcn_ldexpf(a.scale, -e);
    }
    // rows behind the last are copies of it; no negative floats: their bits are in their order
    g_most = __builtin_amdgcn_readfirstlane(__float_as_int(wave_max(fmaxf(g2[0], g2[1]))));
  }
  const float scale = a.scale * kPackedLog2e;
  f32x4_t dq[2][ND];
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int d = 0; d < ND; ++d) dq[u][d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  TileReads<HD> at;
  at.init(r, g);

  // step i: the tile in ks and vs, while one lands in kd and vd (which differ: restrict)
  auto step = [&](int i, const uint16_t* __restrict__ ks, const uint16_t* __restrict__ vs, uint16_t* __restrict__ kd,
                  uint16_t* __restrict__ vd) {
    const int s0 = (i * KS + half) * KT;
    if (i + S - 1 < nt) issue(i + S - 1, kd, vd);
    if (i >= nt || pb >= t.end || s0 > pb + 31 + shift) return;
    const bool diagonal = s0 + KT - 1 > pb + shift;
    f32x4_t s[2][2][2], dp[2][2][2];  // [half of the tile][16 query rows][16 keys]
    U32x4 kc[2][ND], pf[2][2];
    auto scores = [&](int hh) {
      constexpr int QS = HD == 128 ? 1 : 2;  // 16-key parts read ahead together (registers)
#pragma unroll
      for (int q0 = 0; q0 < 2; q0 += QS) {
        U32x4 ka[QS][NC], va[QS][NC];
#pragma unroll
        for (int q = 0; q < QS; ++q)
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            ka[q][c] = at.row16(ks, hh * 2 + q0 + q, c);
            va[q][c] = at.row16(vs, hh * 2 + q0 + q, c);
          }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int q = q0; q < q0 + QS; ++q)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            s[hh][u][q] = f32x4_t{0.f, 0.f, 0.f, 0.f};
            dp[hh][u][q] = f32x4_t{0.f, 0.f, 0.f, 0.f};
          }
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int q = 0; q < QS; ++q)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              s[hh][u][q0 + q] = mfma16<F16>(ka[q][c], qb[u][c], s[hh][u][q0 + q]);
              dp[hh][u][q0 + q] = mfma16<F16>(va[q][c], gb[u][c], dp[hh][u][q0 + q]);
            }
      }
    };
    auto mask = [&](int hh) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (s0 + hh * 32 + q * 16 + 4 * g + j > pb + u * 16 + r + shift) {
              s[hh][u][q][j] = -__builtin_inff();
              dp[hh][u][q][j] = 0.f;
            }
    };
    auto columns = [&](int hh) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int d = 0; d < ND; ++d) kc[hh][d] = at.columns32(ks, hh, d);
      __builtin_amdgcn_sched_barrier(0);
    };
    auto softmax = [&](int hh) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          float ds[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            ds[j] = exp2_f(fmaf(s[hh][u][q][j], scale, -lse[u])) * (dp[hh][u][q][j] - delta[u]);
          pf[hh][u].v[2 * q] = pack2<F16>(ds[0], ds[1]);
          pf[hh][u].v[2 * q + 1] = pack2<F16>(ds[2], ds[3]);
        }
    };
    auto outputs = [&](int hh) {
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int u = 0; u < 2; ++u) dq[u][d] = mfma16<F16>(kc[hh][d], pf[hh][u], dq[u][d]);
    };
    scores(0);
    if constexpr (HD == 128) {  // no registers for two halves side by side
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        if (hh) scores(1);
        columns(hh);
        if (diagonal) mask(hh);
        softmax(hh);
        outputs(hh);
      }
    } else {
      scores(1);
      columns(0);
      if (diagonal) {
        mask(0);
        mask(1);
      }
      softmax(0);
      columns(1);
      // the first half's products with the second half's probabilities between them
      outputs(0);
      softmax(1);
#pragma unroll
      for (int x = 0; x < 2 * ND; ++x) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x402, ND == 4 ? 8 : 6, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
      outputs(1);
    }
  };
  int stage = 0;
  for (int i = 0; i < steps; ++i) {
    if (S > 2 && i + S - 1 <= nt) tile_wait<(S - 2) * 2 * UW>();
    else tile_wait<0>();
    tile_barrier();
    const int next = stage == 0 ? S - 1 : stage - 1;
    step(i, lds[stage][0], lds[stage][1], lds[next][0], lds[next][1]);
    stage = stage == S - 1 ? 0 : stage + 1;
  }
  if constexpr (KS == 2) {
    __syncthreads();
    float* x = reinterpret_cast<float*>(lds_) + wave * 64 * (2 * ND * 4) + lane * 4;
    if (half == 1) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int d = 0; d < ND; ++d) *reinterpret_cast<f32x4_t*>(x + (u * ND + d) * 256) = dq[u][d];
    }
    __syncthreads();
    if (half == 1) return;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        const f32x4_t y = *reinterpret_cast<const f32x4_t*>(x + (u * ND + d) * 256);
#pragma unroll
        for (int j = 0; j < 4; ++j) dq[u][d][j] += y[j];
      }
  }
  if (F16 && pb < t.end && lane == 0)  // here: at the start the loop's first wait would be for it too
    atomicMax(reinterpret_cast<int*>(a.g_top) + kvh * packed_tiles(a.Tq, a.B, kGradBlock) +
                  (t.start / kGradBlock + t.seq + (pb - t.start) / kGradBlock),
              g_most);
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int row = pb + u * 16 + r;
    if (row >= t.end) continue;
    uint16_t* out = static_cast<uint16_t*>(a.g_q) + ((int64_t)row * a.heads + h) * HD + 4 * g;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      uint2 w;
      w.x = pack2<F16>(dq[u][d][0] * out_scale[u], dq[u][d][1] * out_scale[u]);
      w.y = pack2<F16>(dq[u][d][2] * out_scale[u], dq[u][d][3] * out_scale[u]);
      *reinterpret_cast<uint2*>(out + 16 * d) = w;
    }
  }
}

// dK and dV: one workgroup per 128 keys of one kv head, 32 keys a wave (head_dim 128: 16, or
// the sums would leave one wave a SIMD), whose rows of K and V stay in registers; the query rows that see them, of every head of the group,
// pass through LDS 32 at a time.  S = Q K^T and dP = G V^T put a lane's values all in one
// key, and P and dS, rounded, are the operands of dV^T = G^T P and dK^T = Q^T dS.
// An fp16 P is 2^14 times as large, which is taken out of dS as that gets its own power, and of
// dV at the end: a row of many keys has probabilities below fp16's smallest normal number.
// Three sequences of 16001 tokens together, 8 heads of 64: 346 us, 760 TFLOP/s of its four products
// (matrix cores busy 38%, VALU 50%); 12 of 8192, 8 / 4 heads of 96: 67 us and 14 for the join.
// KS = 2: four more waves take every second tile of rows, and the halves add up at the end.
// With a.ranges > 1 a workgroup takes one range of the rows' tiles and leaves its sums in fp32
// for packed_dkv_join_kernel.
template <int HD>
constexpr int packed_dkv_waves = HD == 128 ? 8 : 4;

template <bool F16, int HD, int KS>
__global__ __launch_bounds__(64 * packed_dkv_waves<HD> * KS, 2) void packed_dkv_kernel(PackedAttnArgs a) {
  constexpr int NC = HD / 32, ND = HD / 16, QT = 32, KW = 128;
  constexpr int S = 4;                     // stages
  constexpr int TILE = QT * HD;            // elements
  constexpr int NW = packed_dkv_waves<HD>, KU = KW / NW / 16;  // waves of a half, 16-key parts of a wave
  constexpr int UW = TILE * 2 / 1024 / (NW / 2);  // 1 KiB units a wave loads: half of the waves q, half g
  constexpr float kUp = F16 ? 14.f : 0.f, kDown = F16 ? 0x1p-14f : 1.f;
  __shared__ __align__(16) uint16_t lds_[KS][S][2 * TILE + 128];  // q, g, and the rows' 32 log sums and 32 D (fp32)
  static_assert(KS == 1 || sizeof(lds_) >= NW * 64 * 2 * KU * ND * 16, "the second half's sums take the tiles' place");
  const int tid = threadIdx.x & (64 * NW - 1);
  const int half = KS == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / (64 * NW));
  auto& lds = lds_[half];
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int r = lane & 15, g = lane >> 4;
  const int kvh = blockIdx.x % a.kv_heads;
  PackedTile t;
  PackedKeys qq;  // the sequence's query rows
  const int range = blockIdx.x / a.kv_heads % a.ranges;
  packed_rank<true>(a.cu_k, a.B, a.Tk, KW, 0, blockIdx.x / a.kv_heads / a.ranges, a.cu_q, a.Tq, a.k_len, nullptr, t, qq);
  if (t.first >= t.end) return;
  const PackedKeys kk{t.start, t.used};
  const int rep = a.heads / a.kv_heads;
  const int k0 = t.first - t.start;       // first key of the tile, in the sequence
  const int kb0 = k0 + wave * 16 * KU;    // of the wave
  const int shift = kk.len - qq.len;      // query x of the sequence sees the keys up to x + shift
  const int q_first = max(k0 - shift, 0);
  const int n_rows = t.seq < a.B && k0 < kk.len ? max(qq.len - q_first, 0) : 0;
  const int per_head = (n_rows + QT - 1) / QT;
  const int all = per_head * rep;         // tiles of rows, of all heads
  const int first = (int)((int64_t)all * range / a.ranges);
  const int nt = (int)((int64_t)all * (range + 1) / a.ranges) - first;  // of the range
  const int mine = (nt - half + KS - 1) / KS, steps = (nt + KS - 1) / KS;

  const bool loads_g = wave >= NW / 2;
  const int u0 = wave % (NW / 2) * UW;
  const int64_t row_st = loads_g ? (int64_t)a.heads * HD : a.qs_t, head_st = loads_g ? HD : a.qs_h;
  const uint16_t* src = static_cast<const uint16_t*>(loads_g ? a.g_out : a.q) + qq.start * row_st +
                        (int64_t)kvh * rep * head_st;
  TileLoader<HD, UW> tl;
  tl.init(u0, row_st);
  const int to = loads_g ? TILE : 0;
  int ih = 0, iq = 0;  // head and row tile of the next tile to load
  auto forth = [&](int n, int& hh, int& q) {  // n <= KS tiles on
    q += n;
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      const bool over = q >= per_head;
      q -= over ? per_head : 0;
      hh += over;
    }
  };
  if (nt > 0) {
    ih = first / per_head;
    iq = first % per_head;
    forth(half, ih, iq);
  }
  auto issue = [&](uint16_t* __restrict__ d) {
    const int q0 = q_first + iq * QT;
    const uint16_t* p0 = src + ih * head_st + q0 * row_st;
    tl.issue(d + to, p0, u0, row_st, QT, qq.len - q0);
    // every wave loads the rows' sums, so that each has as many loads in flight; the same
    // values to the same place
    const int row = min(q0 + (lane & 31), qq.len - 1);
    const float* p = (lane < 32 ? a.lse : a.delta) + (int64_t)(kvh * rep + ih) * a.Tq + qq.start + row;
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)p,
                                     (__attribute__((address_space(3))) void*)(d + 2 * TILE), 4, 0, 0);
    forth(KS, ih, iq);
  };
#pragma unroll
  for (int i = 0; i < S - 1; ++i)
    if (i < mine) issue(lds[i]);
  U32x4 kb[KU][NC], vb[KU][NC];
#pragma unroll
  for (int u = 0; u < KU; ++u) {
    const int64_t row = kk.start + max(min(kb0 + u * 16 + r, kk.len - 1), 0);
    const uint16_t* kp = static_cast<const uint16_t*>(a.k) + row * a.ks_t + kvh * a.ks_h + 8 * g;
    const uint16_t* vp = static_cast<const uint16_t*>(a.v) + row * a.vs_t + kvh * a.vs_h + 8 * g;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      kb[u][c] = ld16(kp + 32 * c);
      vb[u][c] = ld16(vp + 32 * c);
    }
  }
  float kd = 1.f, k_scale = a.scale;  // of dS, and of dK
  if constexpr (F16) {
    const float v2 = packed_v_top(a, kvh, t.seq, kk.start, kk.len);
    float most = 0.f;
    if (nt > 0) {
      const float* p = a.g_top + kvh * packed_tiles(a.Tq, a.B, kGradBlock) + (qq.start / kGradBlock + t.seq);
      for (int i = q_first / kGradBlock + lane; i <= (qq.len - 1) / kGradBlock; i += 64) most = fmaxf(most, p[i]);
    }
    most = wave_max(most);
    const int e = __builtin_amdgcn_readfirstlane(packed_exponent(most * v2));
    kd = __builtin_amdgcn_ldexpf(kDown, e);
    k_scale = __builtin_amdgcn_ldexpf(a.scale, -e);
  }
  const float scale = a.scale * kPackedLog2e;
  f32x4_t dk[KU][ND], dv[KU][ND];
#pragma unroll
  for (int u = 0; u < KU; ++u)
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      dk[u][d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      dv[u][d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
  TileReads<HD> at;
  at.init(r, g);
  auto step = [&](int q0, bool more, const uint16_t* __restrict__ qs, uint16_t* __restrict__ d) {
    if (more) issue(d);
    const uint16_t* gs = qs + TILE;
    if (kb0 >= kk.len || q0 + QT - 1 + shift < kb0) return;  // no keys, or none that these rows see
    // the diagonal, and the sequence's last rows, behind which lie copies of the last
    const bool edge = q0 + shift < kb0 + 16 * KU - 1 || q0 + QT > qq.len;
    f32x4_t s[2][KU], dp[2][KU];  // [16 query rows][16 keys]
    constexpr int QS = HD == 96 ? 1 : 2;  // 16-row parts read ahead together (registers)
#pragma unroll
    for (int q0_ = 0; q0_ < 2; q0_ += QS) {
      U32x4 qa[QS][NC], ga[QS][NC];
#pragma unroll
      for (int q = 0; q < QS; ++q)
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          qa[q][c] = at.row16(qs, q0_ + q, c);
          ga[q][c] = at.row16(gs, q0_ + q, c);
        }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int q = q0_; q < q0_ + QS; ++q)
#pragma unroll
        for (int u = 0; u < KU; ++u) {
          s[q][u] = f32x4_t{0.f, 0.f, 0.f, 0.f};
          dp[q][u] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int q = 0; q < QS; ++q)
#pragma unroll
          for (int u = 0; u < KU; ++u) {
            s[q0_ + q][u] = mfma16<F16>(qa[q][c], kb[u][c], s[q0_ + q][u]);
            dp[q0_ + q][u] = mfma16<F16>(ga[q][c], vb[u][c], dp[q0_ + q][u]);
          }
    }
    U32x4 gc[ND];
    f32x4_t l4[2], d4[2];
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      l4[q] = *reinterpret_cast<const f32x4_t*>(&gs[TILE + 2 * (q * 16 + 4 * g)]);
      d4[q] = *reinterpret_cast<const f32x4_t*>(&gs[TILE + 2 * (32 + q * 16 + 4 * g)]);
    }
#pragma unroll
    for (int d = 0; d < ND; ++d) gc[d] = at.columns32(gs, 0, d);
    __builtin_amdgcn_sched_barrier(0);
    if (edge) {
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int u = 0; u < KU; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int row = q0 + q * 16 + 4 * g + i;
            if (kb0 + u * 16 + r > row + shift || row >= qq.len) {
              s[q][u][i] = -__builtin_inff();
              dp[q][u][i] = 0.f;
            }
          }
    }
    U32x4 pf[KU], df[KU];
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int u = 0; u < KU; ++u) {
#pragma unroll
        for (int i = 0; i < 4; ++i) s[q][u][i] = exp2_f(fmaf(s[q][u][i], scale, kUp - l4[q][i]));
        pf[u].v[2 * q] = pack2<F16>(s[q][u][0], s[q][u][1]);
        pf[u].v[2 * q + 1] = pack2<F16>(s[q][u][2], s[q][u][3]);
      }
    auto terms = [&] {  // dS
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int u = 0; u < KU; ++u) {
          float ds[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            ds[i] = s[q][u][i] * (F16 ? fmaf(dp[q][u][i], kd, -d4[q][i] * kd) : dp[q][u][i] - d4[q][i]);
          df[u].v[2 * q] = pack2<F16>(ds[0], ds[1]);
          df[u].v[2 * q + 1] = pack2<F16>(ds[2], ds[3]);
        }
    };
    U32x4 qc[ND];
    auto columns = [&] {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int d = 0; d < ND; ++d) qc[d] = at.columns32(qs, 0, d);
      __builtin_amdgcn_sched_barrier(0);
    };
    auto values = [&] {
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int u = 0; u < KU; ++u) dv[u][d] = mfma16<F16>(gc[d], pf[u], dv[u][d]);
    };
    if constexpr (HD == 96) {  // with dV's products beside dS the registers spill
      terms();
      columns();
      values();
    } else {  // dV's products with dS between them
      columns();
      values();
      terms();
#pragma unroll
      for (int x = 0; x < KU * ND; ++x) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x402, ND == 4 ? 5 : 3, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int u = 0; u < KU; ++u) dk[u][d] = mfma16<F16>(qc[d], df[u], dk[u][d]);
  };
  int stage = 0, ch = 0, cq = nt > 0 ? first % per_head : 0;  // head and row tile of this step
  forth(half, ch, cq);
  for (int it = 0; it < steps; ++it) {
    if (it + S - 1 <= mine) tile_wait<(S - 2) * (UW + 1)>();
    else if (it + S - 2 <= mine) tile_wait<(S - 3) * (UW + 1)>();
    else tile_wait<0>();
    tile_barrier();
    const int next = stage == 0 ? S - 1 : stage - 1;
    if (it < mine) step(q_first + cq * QT, it + S - 1 < mine, lds[stage], lds[next]);
    stage = stage == S - 1 ? 0 : stage + 1;
    forth(KS, ch, cq);
  }
  if constexpr (KS == 2) {
    __syncthreads();
    float* x = reinterpret_cast<float*>(lds_) + wave * 64 * (2 * KU * ND * 4) + lane * 4;
    if (half == 1) {
#pragma unroll
      for (int u = 0; u < KU; ++u)
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          *reinterpret_cast<f32x4_t*>(x + (u * ND + d) * 256) = dk[u][d];
          *reinterpret_cast<f32x4_t*>(x + (KU * ND + u * ND + d) * 256) = dv[u][d];
        }
    }
    __syncthreads();
    if (half == 1) return;
#pragma unroll
    for (int u = 0; u < KU; ++u)
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        const f32x4_t y = *reinterpret_cast<const f32x4_t*>(x + (u * ND + d) * 256);
        const f32x4_t z = *reinterpret_cast<const f32x4_t*>(x + (KU * ND + u * ND + d) * 256);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          dk[u][d][i] += y[i];
          dv[u][d][i] += z[i];
        }
      }
  }
  // every row of the slot is written: those behind its length with zeros
#pragma unroll
  for (int u = 0; u < KU; ++u) {
    const int key = kb0 + u * 16 + r;
    const int row = t.start + key;
    if (row >= t.end) continue;
    const bool used = key < kk.len;
    const int64_t at = ((int64_t)row * a.kv_heads + kvh) * HD + 4 * g;
    const int64_t size = (int64_t)a.Tk * a.kv_heads * HD;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      f32x4_t x = {0.f, 0.f, 0.f, 0.f}, y = x;
      if (used) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[i] = dk[u][d][i] * k_scale;
          y[i] = dv[u][d][i] * kDown;
        }
      }
      if (a.ranges > 1) {
        float* part = a.work + 2 * range * size + at + 16 * d;
        *reinterpret_cast<f32x4_t*>(part) = x;
        *reinterpret_cast<f32x4_t*>(part + size) = y;
      } else {
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.g_k) + at + 16 * d) =
            make_uint2(pack2<F16>(x[0], x[1]), pack2<F16>(x[2], x[3]));
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.g_v) + at + 16 * d) =
            make_uint2(pack2<F16>(y[0], y[1]), pack2<F16>(y[2], y[3]));
      }
    }
  }
}

// The ranges' sums, in order, four elements of dK or dV a thread.
template <bool F16>
__global__ __launch_bounds__(256) void packed_dkv_join_kernel(PackedAttnArgs a) {
  const int64_t size = (int64_t)a.Tk * a.kv_heads * a.head_dim;
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;  // of dK, then of dV
  if (i >= 2 * size) return;
  f32x4_t x = *reinterpret_cast<const f32x4_t*>(a.work + i);
  for (int n = 1; n < a.ranges; ++n) {
    const f32x4_t y = *reinterpret_cast<const f32x4_t*>(a.work + 2 * n * size + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] += y[j];
  }
  uint16_t* out = i < size ? static_cast<uint16_t*>(a.g_k) + i : static_cast<uint16_t*>(a.g_v) + (i - size);
  *reinterpret_cast<uint2*>(out) = make_uint2(pack2<F16>(x[0], x[1]), pack2<F16>(x[2], x[3]));
}

template <bool F16, int HD>
hipError_t packed_bwd_hd(PackedAttnArgs a, hipStream_t s) {
  const int hp = (a.heads / a.kv_heads) % 2 == 0 ? 2 : 1;
  a.qtiles = (int)packed_tiles(a.Tq, a.B, 128 / hp);
  const dim3 grid((unsigned)((int64_t)a.qtiles * (a.heads / hp)));
  if (F16 && a.Tq > 0 && a.Tk > 0) {
    const dim3 tiles((unsigned)(packed_tiles(a.Tk, a.B, 128) * a.kv_heads));
    packed_v_top_kernel<HD><<<tiles, 256, 0, s>>>(a);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  if (a.Tq > 0) {
    const bool halves = packed_halves(grid.x);
    if (hp == 2) {
      if (halves) packed_dq_kernel<F16, HD, 2, 2><<<grid, 512, 0, s>>>(a);
      else packed_dq_kernel<F16, HD, 2, 1><<<grid, 256, 0, s>>>(a);
    } else {
      if (halves) packed_dq_kernel<F16, HD, 1, 2><<<grid, 512, 0, s>>>(a);
      else packed_dq_kernel<F16, HD, 1, 1><<<grid, 256, 0, s>>>(a);
    }
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  if (a.Tk == 0) return hipSuccess;
  const dim3 kgrid((unsigned)(packed_tiles(a.Tk, a.B, 128) * a.kv_heads * a.ranges));
  if (HD <= 96 && packed_halves(kgrid.x))  // at 128 a workgroup has eight waves as it is
    packed_dkv_kernel<F16, HD <= 96 ? HD : 64, 2><<<kgrid, 512, 0, s>>>(a);
  else
    packed_dkv_kernel<F16, HD, 1><<<kgrid, 64 * packed_dkv_waves<HD>, 0, s>>>(a);
  if (hipError_t e = hipGetLastError(); e != hipSuccess || a.ranges == 1) return e;
  const int64_t quads = (int64_t)a.Tk * a.kv_heads * HD / 2;
  packed_dkv_join_kernel<F16><<<dim3((unsigned)((quads + 255) / 256)), 256, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace

// Ranges that the query rows of a key tile are cut into: up to four workgroups a CU, none of
// under 8 tiles of rows (on average), beside whose products the ranges' sums (8 bytes an element
// each way) are small; 8 at most, which keeps the workspace to 64 bytes an element of k. (More would be
// faster where key tiles are few: dK, dV and their join of one sequence of 4096 tokens, 8 / 1 heads of 64, in 4, 8, 16
// and 31 ranges 154, 86, 72 and 70 us; of 2000 and 1000 tokens, 16 / 1 heads of 96, in 8 and 32 108 and 72; of one of
// 16000, 8 / 1 heads of 64, in 2, 4 and 8 1067, 849 and 611.)  A step of 12 sequences of 8192 tokens together, 8 / 4 heads of 96: 179 us with
// 3 ranges, 206 with one, 219 with 8; of 30 of 10000, 12 / 4 heads: 194, 231 and 254; of 2 sequences of 8000 tokens together, 8 / 2 heads of 128: 522 us
// with 4 ranges and 1120 with one; of 2 of 16000, 16 / 2 heads of 64: 1540 with 4, 2136 with 2, 2496
// with one; of 3 of 16001, 8 / 8 heads of 64 (four workgroups a CU as it is): 688 with 2, 664 with one.
void packed_bwd_plan(PackedAttnArgs& a) {
  const int64_t groups = (int64_t)a.Tk * a.kv_heads / 128 + 1;  // workgroups with work, about
  const int64_t chain = (int64_t)a.Tq / (a.B > 0 ? a.B : 1) * (a.heads / a.kv_heads) / 32;  // tiles of the longest, about
  int64_t want = 4 * (int64_t)device_cus() / groups;
  if (want > chain / 8) want = chain / 8;
  if (want > 8) want = 8;
  a.ranges = want < 1 ? 1 : (int)want;
}
int64_t packed_bwd_threads(const PackedAttnArgs& a) {
  const int hp = (a.heads / a.kv_heads) % 2 == 0 ? 2 : 1;
  const int64_t dq = 256 * packed_tiles(a.Tq, a.B, 128 / hp) * (a.heads / hp);
  const int64_t dkv = 512 * packed_tiles(a.Tk, a.B, 128) * a.kv_heads * a.ranges;
  return dq > dkv ? dq : dkv;  // the join has fewer: several ranges are for some 10^5 keys at most
}
// D, the longest rows of v and g by tiles, and the ranges' sums of dK and dV.
int64_t packed_bwd_workspace(PackedAttnArgs& a, float* workspace) {
  auto whole = [](int64_t n) { return (n + 3) / 4 * 4; };  // of 16 bytes
  const int64_t v_top = whole((int64_t)a.heads * a.Tq);
  const int64_t g_top = v_top + whole(packed_tiles(a.Tk, a.B, 128) * a.kv_heads);
  const int64_t sums = g_top + whole(packed_tiles(a.Tq, a.B, kGradBlock) * a.kv_heads);
  if (workspace) {
    a.delta = workspace;
    a.v_top = workspace + v_top;
    a.g_top = workspace + g_top;
    a.work = workspace + sums;
  }
  return (sums + (a.ranges > 1 ? 2 * a.ranges * (int64_t)a.Tk * a.kv_heads * a.head_dim : 0)) * 4;
}

hipError_t launch_packed_attn_bwd(const PackedAttnArgs& a, hipStream_t s) { MHC_PACKED_HD(packed_bwd_hd, a, s) }

}  // namespace mhc
