// Causal attention over packed sequences: backward.  With P the probabilities (formed again
// from q, k and the forward's log sums) and G the output's gradient,
//   D_i = G_i . O_i,  dS_ij = P_ij (G_i . v_j - D_i),
//   dQ_i = scale sum_j dS_ij k_j,  dK_j = scale sum_i dS_ij q_i,  dV_j = sum_i P_ij G_i.
// One launch forms D and dQ by query tiles, a second dK and dV by key tiles, each summing
// its own rows' terms in registers (fp32): no atomics, the same bits on every run.  P is
// formed twice for that: 7 products instead of 5.
#include "mhc_packed.hpp"

namespace mhc {
namespace {

// dQ: as the forward, one 4-wave workgroup per 128 query rows of one kv head, 32 rows a
// wave.  S^T = K Q^T and dP^T = V G^T put a lane's values all in one query row, and dS^T,
// rounded, is the operand of dQ^T = K^T dS^T as it stands.
template <bool F16, int HD, int HP>
__global__ __launch_bounds__(256, 2) void packed_dq_kernel(PackedAttnArgs a) {
  constexpr int NC = HD / 32, ND = HD / 16, KT = 64;
  constexpr int PW = 128 / HP;
  constexpr int KST = HD + 16, VST = HD + 8;
  constexpr int PPT = KT * (HD / 8) / 256;
  __shared__ __align__(16) uint16_t ks[2][KT * KST];
  __shared__ __align__(16) uint16_t vs[2][KT * VST];
  const int tid = threadIdx.x;
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
  const int nt = last < 0 ? 0 : last / KT + 1;

  const int64_t ks_t = a.ks_t, vs_t = a.vs_t;
  const uint16_t* kg = static_cast<const uint16_t*>(a.k) + kk.start * ks_t + kvh * a.ks_h;
  const uint16_t* vg = static_cast<const uint16_t*>(a.v) + kk.start * vs_t + kvh * a.vs_h;
  U32x4 kr[PPT], vr[PPT];
  auto load = [&](int s0) {
#pragma unroll
    for (int p = 0; p < PPT; ++p) {
      const int piece = p * 256 + tid;
      const int row = min(s0 + piece / (HD / 8), kk.len - 1);
      const int col = (piece % (HD / 8)) * 8;
      kr[p] = ld16(kg + row * ks_t + col);
      vr[p] = ld16(vg + row * vs_t + col);
    }
  };
  if (nt > 0) load(0);
  U32x4 qb[2][NC], gb[2][NC];
  float lse[2], delta[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int row = pb + u * 16 + r;
    const int64_t at = min(row, t.end - 1);
    const uint16_t* q = static_cast<const uint16_t*>(a.q) + at * a.qs_t + h * a.qs_h + 8 * g;
    const int64_t off = (at * a.heads + h) * HD + 8 * g;
    const uint16_t* go = static_cast<const uint16_t*>(a.g_out) + off;
    const uint16_t* oo = static_cast<const uint16_t*>(a.out) + off;
    const uint16_t* ro = static_cast<const uint16_t*>(a.rest) + off;
    float d = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      qb[u][c] = ld16(q + 32 * c);
      gb[u][c] = ld16(go + 32 * c);
      const U32x4 o = ld16(oo + 32 * c), rest = ld16(ro + 32 * c);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        d += elem_lo<F16>(gb[u][c].v[j]) * (elem_lo<F16>(o.v[j]) + elem_lo<F16>(rest.v[j]));
        d += elem_hi<F16>(gb[u][c].v[j]) * (elem_hi<F16>(o.v[j]) + elem_hi<F16>(rest.v[j]));
      }
    }
    d += xor_lane16(d);
    d += xor_lane32(d);
    delta[u] = d;
    lse[u] = a.lse[(int64_t)h * a.Tq + at];
    if (g == 0 && row < t.end) a.delta[(int64_t)h * a.Tq + row] = d;
  }
  const float scale = a.scale * kPackedLog2e;
  f32x4_t dq[2][ND];
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int d = 0; d < ND; ++d) dq[u][d] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  for (int kt = 0; kt < nt; ++kt) {
    const int buf = kt & 1;
    const int s0 = kt * KT;
#pragma unroll
    for (int p = 0; p < PPT; ++p) {
      const int piece = p * 256 + tid;
      const int row = piece / (HD / 8);
      const int col = (piece % (HD / 8)) * 8;
      *reinterpret_cast<U32x4*>(&ks[buf][row * KST + col]) = kr[p];
      *reinterpret_cast<U32x4*>(&vs[buf][row * VST + col]) = vr[p];
    }
    __syncthreads();
    if (kt + 1 < nt) load(s0 + KT);
    if (pb >= t.end || s0 > pb + 31 + shift) continue;
    const bool diagonal = s0 + KT - 1 > pb + shift;
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      f32x4_t s[2][2], dp[2][2];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          s[u][q] = f32x4_t{0.f, 0.f, 0.f, 0.f};
          dp[u][q] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const int row = hh * 32 + q * 16 + r;
          const U32x4 ka = *reinterpret_cast<const U32x4*>(&ks[buf][row * KST + 32 * c + 8 * g]);
          const U32x4 va = *reinterpret_cast<const U32x4*>(&vs[buf][row * VST + 32 * c + 8 * g]);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            s[u][q] = mfma16<F16>(ka, qb[u][c], s[u][q]);
            dp[u][q] = mfma16<F16>(va, gb[u][c], dp[u][q]);
          }
        }
      }
      if (diagonal) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (s0 + hh * 32 + q * 16 + 4 * g + i > pb + u * 16 + r + shift) {
                s[u][q][i] = -__builtin_inff();
                dp[u][q][i] = 0.f;
              }
      }
      U32x4 pf[2];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          float ds[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            ds[i] = exp2_f(fmaf(s[u][q][i], scale, -lse[u])) * (dp[u][q][i] - delta[u]);
          pf[u].v[2 * q] = pack2<F16>(ds[0], ds[1]);
          pf[u].v[2 * q + 1] = pack2<F16>(ds[2], ds[3]);
        }
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        U32x4 ka;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const u32x2_v w = lds_tr4(&ks[buf][(hh * 32 + q * 16 + 4 * g + (r >> 2)) * KST + 16 * d + 4 * (r & 3)]);
          ka.v[2 * q] = w.x;
          ka.v[2 * q + 1] = w.y;
        }
        dq[0][d] = mfma16<F16>(ka, pf[0], dq[0][d]);
        dq[1][d] = mfma16<F16>(ka, pf[1], dq[1][d]);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int row = pb + u * 16 + r;
    if (row >= t.end) continue;
    uint16_t* out = static_cast<uint16_t*>(a.g_q) + ((int64_t)row * a.heads + h) * HD + 4 * g;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      uint2 w;
      w.x = pack2<F16>(dq[u][d][0] * a.scale, dq[u][d][1] * a.scale);
      w.y = pack2<F16>(dq[u][d][2] * a.scale, dq[u][d][3] * a.scale);
      *reinterpret_cast<uint2*>(out + 16 * d) = w;
    }
  }
}

// dK and dV: one 4-wave workgroup per 128 keys of one kv head, 32 keys a wave, whose rows
// of K and V stay in registers; the query rows that see them, of every head of the group,
// pass through LDS 32 at a time.  S = Q K^T and dP = G V^T put a lane's values all in one
// key, and P and dS, rounded, are the operands of dV^T = G^T P and dK^T = Q^T dS.
// An fp16 P is 2^14 times as large, which is taken out of dS as it is formed and of dV at the
// end: a row of many keys has probabilities below fp16's smallest normal number.  dS has
// no bound and stays as it is: its terms under 2^-14 round at 2^-25, as any fp16 gradient does.
template <bool F16, int HD>
__global__ __launch_bounds__(256, HD <= 96 ? 2 : 1) void packed_dkv_kernel(PackedAttnArgs a) {
  constexpr int NC = HD / 32, ND = HD / 16, QT = 32, KW = 128;
  constexpr int ST = HD + 16;
  constexpr float kUp = F16 ? 14.f : 0.f, kDown = F16 ? 0x1p-14f : 1.f;
  constexpr int PPT = QT * (HD / 8) / 128;  // half the threads move q, half g
  __shared__ __align__(16) uint16_t qs[2][QT * ST];
  __shared__ __align__(16) uint16_t gs[2][QT * ST];
  __shared__ __align__(16) float ls[2][QT], ds_[2][QT];
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int r = lane & 15, g = lane >> 4;
  const int kvh = blockIdx.x % a.kv_heads;
  PackedTile t;
  PackedKeys qq;  // the sequence's query rows
  packed_rank<true>(a.cu_k, a.B, a.Tk, KW, 0, blockIdx.x / a.kv_heads, a.cu_q, a.Tq, a.k_len, nullptr, t, qq);
  if (t.first >= t.end) return;
  const PackedKeys kk{t.start, t.used};
  const int rep = a.heads / a.kv_heads;
  const int k0 = t.first - t.start;       // first key of the tile, in the sequence
  const int kb0 = k0 + wave * 32;         // of the wave
  const int shift = kk.len - qq.len;      // query x of the sequence sees the keys up to x + shift
  const int q_first = max(k0 - shift, 0);
  const int n_rows = t.seq < a.B && k0 < kk.len ? max(qq.len - q_first, 0) : 0;
  const int per_head = (n_rows + QT - 1) / QT;
  const int nt = per_head * rep;

  const bool loads_g = tid >= 128;
  const uint16_t* src = static_cast<const uint16_t*>(loads_g ? a.g_out : a.q);
  const int64_t row_st = loads_g ? (int64_t)a.heads * HD : a.qs_t, head_st = loads_g ? HD : a.qs_h;
  src += qq.start * row_st + (int64_t)kvh * rep * head_st;
  U32x4 st[PPT];
  float st_l = 0.f;
  auto load = [&](int it) {
    const int hh = it / per_head, q0 = q_first + (it - hh * per_head) * QT;
    const uint16_t* p0 = src + hh * head_st;
#pragma unroll
    for (int p = 0; p < PPT; ++p) {
      const int piece = p * 128 + (tid & 127);
      st[p] = ld16(p0 + min(q0 + piece / (HD / 8), qq.len - 1) * row_st + (piece % (HD / 8)) * 8);
    }
    if (tid < 2 * QT) {
      const int row = q0 + (tid & (QT - 1));
      const float* lp = (tid < QT ? a.lse : a.delta) + (int64_t)(kvh * rep + hh) * a.Tq + qq.start;
      // a row that is not there: its probabilities are 0
      st_l = row < qq.len ? lp[row] : tid < QT ? __builtin_inff() : 0.f;
      st_l = tid < QT ? st_l - kUp : st_l * kDown;
    }
  };
  if (nt > 0) load(0);
  U32x4 kb[2][NC], vb[2][NC];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int64_t row = kk.start + max(min(kb0 + u * 16 + r, kk.len - 1), 0);
    const uint16_t* kp = static_cast<const uint16_t*>(a.k) + row * a.ks_t + kvh * a.ks_h + 8 * g;
    const uint16_t* vp = static_cast<const uint16_t*>(a.v) + row * a.vs_t + kvh * a.vs_h + 8 * g;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      kb[u][c] = ld16(kp + 32 * c);
      vb[u][c] = ld16(vp + 32 * c);
    }
  }
  const float scale = a.scale * kPackedLog2e;
  f32x4_t dk[2][ND], dv[2][ND];
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      dk[u][d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      dv[u][d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
  for (int it = 0; it < nt; ++it) {
    const int buf = it & 1;
#pragma unroll
    for (int p = 0; p < PPT; ++p) {
      const int piece = p * 128 + (tid & 127);
      uint16_t* to = loads_g ? gs[buf] : qs[buf];
      *reinterpret_cast<U32x4*>(&to[piece / (HD / 8) * ST + (piece % (HD / 8)) * 8]) = st[p];
    }
    if (tid < 2 * QT) (tid < QT ? ls[buf] : ds_[buf])[tid & (QT - 1)] = st_l;
    __syncthreads();
    if (it + 1 < nt) load(it + 1);
    const int q0 = q_first + it % per_head * QT;
    if (kb0 >= kk.len || q0 + QT - 1 + shift < kb0) continue;  // no keys, or none that these rows see
    const bool diagonal = q0 + shift < kb0 + 31;
    f32x4_t s[2][2], dp[2][2];  // [16 query rows][16 keys]
#pragma unroll
    for (int q = 0; q < 2; ++q) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        s[q][u] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        dp[q][u] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      }
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const U32x4 qa = *reinterpret_cast<const U32x4*>(&qs[buf][(q * 16 + r) * ST + 32 * c + 8 * g]);
        const U32x4 ga = *reinterpret_cast<const U32x4*>(&gs[buf][(q * 16 + r) * ST + 32 * c + 8 * g]);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          s[q][u] = mfma16<F16>(qa, kb[u][c], s[q][u]);
          dp[q][u] = mfma16<F16>(ga, vb[u][c], dp[q][u]);
        }
      }
    }
    if (diagonal) {
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (kb0 + u * 16 + r > q0 + q * 16 + 4 * g + i + shift) {
              s[q][u][i] = -__builtin_inff();
              dp[q][u][i] = 0.f;
            }
    }
    U32x4 pf[2], df[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const f32x4_t l4 = *reinterpret_cast<const f32x4_t*>(&ls[buf][q * 16 + 4 * g]);
      const f32x4_t d4 = *reinterpret_cast<const f32x4_t*>(&ds_[buf][q * 16 + 4 * g]);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float p[4], ds[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[i] = exp2_f(fmaf(s[q][u][i], scale, -l4[i]));
          ds[i] = p[i] * fmaf(dp[q][u][i], kDown, -d4[i]);
        }
        pf[u].v[2 * q] = pack2<F16>(p[0], p[1]);
        pf[u].v[2 * q + 1] = pack2<F16>(p[2], p[3]);
        df[u].v[2 * q] = pack2<F16>(ds[0], ds[1]);
        df[u].v[2 * q + 1] = pack2<F16>(ds[2], ds[3]);
      }
    }
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      U32x4 ga, qa;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int at = (q * 16 + 4 * g + (r >> 2)) * ST + 16 * d + 4 * (r & 3);
        const u32x2_v w = lds_tr4(&gs[buf][at]);
        const u32x2_v x = lds_tr4(&qs[buf][at]);
        ga.v[2 * q] = w.x;
        ga.v[2 * q + 1] = w.y;
        qa.v[2 * q] = x.x;
        qa.v[2 * q + 1] = x.y;
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        dv[u][d] = mfma16<F16>(ga, pf[u], dv[u][d]);
        dk[u][d] = mfma16<F16>(qa, df[u], dk[u][d]);
      }
    }
  }
  // every row of the slot is written: those behind its length with zeros
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int key = kb0 + u * 16 + r;
    const int row = t.start + key;
    if (row >= t.end) continue;
    const bool used = key < kk.len;
    const int64_t at = ((int64_t)row * a.kv_heads + kvh) * HD + 4 * g;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      uint2 w = make_uint2(0, 0), x = w;
      if (used) {
        w.x = pack2<F16>(dk[u][d][0] * a.scale, dk[u][d][1] * a.scale);
        w.y = pack2<F16>(dk[u][d][2] * a.scale, dk[u][d][3] * a.scale);
        x.x = pack2<F16>(dv[u][d][0] * kDown, dv[u][d][1] * kDown);
        x.y = pack2<F16>(dv[u][d][2] * kDown, dv[u][d][3] * kDown);
      }
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.g_k) + at + 16 * d) = w;
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.g_v) + at + 16 * d) = x;
    }
  }
}

template <bool F16, int HD>
hipError_t packed_bwd_hd(PackedAttnArgs a, hipStream_t s) {
  const int hp = (a.heads / a.kv_heads) % 2 == 0 ? 2 : 1;
  a.qtiles = (int)packed_tiles(a.Tq, a.B, 128 / hp);
  const dim3 grid((unsigned)((int64_t)a.qtiles * (a.heads / hp)));
  if (a.Tq > 0) {
    if (hp == 2)
      packed_dq_kernel<F16, HD, 2><<<grid, 256, 0, s>>>(a);
    else
      packed_dq_kernel<F16, HD, 1><<<grid, 256, 0, s>>>(a);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  if (a.Tk == 0) return hipSuccess;
  packed_dkv_kernel<F16, HD><<<dim3((unsigned)(packed_tiles(a.Tk, a.B, 128) * a.kv_heads)), 256, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_packed_attn_bwd(const PackedAttnArgs& a, hipStream_t s) { MHC_PACKED_HD(packed_bwd_hd, a, s) }

}  // namespace mhc
