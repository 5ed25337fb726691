// Rotary positions, by themselves and on the way of new tokens into a cache of pages.
//   Pair (a, b) of a head's first rd elements, half layout (d, d + rd / 2), interleaved (2 d,
//   2 d + 1):  a' = a c - b s,  b' = b c + a s,  c, s = cos, sin [position, d];  the elements behind
//   rd stay.  The gradient is the transposed map, the same with -s.
//   With gains (append only) x = y rsqrt(mean y^2 + eps) gain comes before.
// Bound by bytes: every element is read once and written once, in fp32 between, rounded once.  The
// turned tensors are stored past the caches' order (non-temporal): by itself 18.4 instead of 19.2 us at 16384 rows, 8 + 4 heads
// of 96, and 8.0 instead of 8.9 at 4096.  Together with the attention that reads them next that is lost again: 59.0
// and 59.4 us (sequences of 512), 100 and 98.5 (of 2048), 27.5 and 28.2 at 4096 rows, 381 and 372 at 65536.
#include "mhc_packed.hpp"

namespace mhc {
namespace {

// V elements from p[i] on: 16 or 8 bytes where V has as many, else one.
template <int DT, int V>
__device__ __forceinline__ void load_v(const void* p, int64_t i, float (&x)[V]) {
  if constexpr (V == 1) {
    x[0] = ld_any(p, i, DT);
  } else if constexpr (DT == kF32) {
    static_assert(V == 4);
    const float4 w = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
    x[0] = w.x; x[1] = w.y; x[2] = w.z; x[3] = w.w;
  } else {
    uint32_t w[V / 2];
    const uint16_t* s = static_cast<const uint16_t*>(p) + i;
    if constexpr (V == 8) *reinterpret_cast<U32x4*>(w) = ld16(s);
    else *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(s);
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
      x[2 * j] = elem_lo<DT == kF16>(w[j]);
      x[2 * j + 1] = elem_hi<DT == kF16>(w[j]);
    }
  }
}
template <int DT, int V, bool NT>
__device__ __forceinline__ void store_v(void* p, int64_t i, const float (&x)[V]) {
  if constexpr (V == 1) {
    st_any(p, i, DT, x[0]);
  } else if constexpr (DT == kF32) {
    const U32x4 w{{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])}};
    if constexpr (NT) st16_nt(static_cast<float*>(p) + i, w);
    else *reinterpret_cast<U32x4*>(static_cast<float*>(p) + i) = w;
  } else {
    uint32_t w[V / 2];
#pragma unroll
    for (int j = 0; j < V / 2; ++j) w[j] = pack2<DT == kF16>(x[2 * j], x[2 * j + 1]);
    uint16_t* d = static_cast<uint16_t*>(p) + i;
    if constexpr (V == 8 && NT) st16_nt(d, *reinterpret_cast<const U32x4*>(w));
    else if constexpr (V == 8) *reinterpret_cast<U32x4*>(d) = *reinterpret_cast<const U32x4*>(w);
    else *reinterpret_cast<uint2*>(d) = *reinterpret_cast<const uint2*>(w);
  }
}

// Where a sequence's row goes: its key's row in the pages (-1: nowhere) and its position
// (kNoSequence: a row behind the last sequence).
constexpr int64_t kNoSequence = INT64_MIN;
struct RowPlace {
  int64_t page, position;
  int row;
};
__device__ __forceinline__ RowPlace row_place(const RotaryArgs& a, int64_t t) {
  const int lane = __lane_id();
  int lo = 0, hi = a.B + 1;  // the last sequence that begins at or before t
  while (hi - lo > 1) {
    const int step = (hi - lo - 1 + 63) / 64;
    const int64_t at = lo + (int64_t)(lane + 1) * step;
    const bool below = at < hi && seq_start(a.cu, (int)(at < hi ? at : lo), (int)a.T) <= t;
    lo += __popcll(__ballot(below)) * step;
    hi = min(hi, lo + step);
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  RowPlace r{-1, kNoSequence, 0};
  if (lo >= a.B) return r;
  const int64_t cap = (int64_t)a.width << a.page_shift;
  const int64_t past = min(max((int64_t)a.lengths[lo], (int64_t)0), cap);
  const int64_t j = max(t - seq_start(a.cu, lo, (int)a.T), (int64_t)0), key = past + j;
  r.position = past + (a.depths ? (int64_t)a.depths[t] : j);
  r.row = (int)(key & ((1 << a.page_shift) - 1));
  if (key < cap) {
    const int p = a.page_table[(int64_t)lo * a.width + (key >> a.page_shift)];
    if ((unsigned)p < (unsigned)a.pages) r.page = p;
  }
  return r;
}

// A unit of a head: V pairs, whose halves begin at e0 and e1 (interleaved: 2 V neighbours, and so
// where nothing turns); with V = 1 what stays is a single element, e1 = e0.
struct UnitAt {
  int e0, e1;
};
template <int V>
__device__ __forceinline__ UnitAt unit_at(const RotaryArgs& a, int u, int turned) {
  if (u < turned && !a.interleaved) return {u * V, a.rd / 2 + u * V};
  if (V > 1 || u < turned) return {u * 2 * V, u * 2 * V + V};
  return {a.rd + u - turned, a.rd + u - turned};
}
// The V angles of unit u in row `angle` of the tables.
template <int V>
__device__ __forceinline__ void unit_angles(const RotaryArgs& a, int64_t angle, int u, bool inside, float (&c)[V], float (&s)[V]) {
  if (!inside) {  // the tables may have no row at all
#pragma unroll
    for (int i = 0; i < V; ++i) c[i] = s[i] = __builtin_nanf("");
  } else if (a.table_dtype == kF32 && a.table_wide) {
    const float* cp = static_cast<const float*>(a.cos) + angle + u * V;
    const float* sp = static_cast<const float*>(a.sin) + angle + u * V;
    if constexpr (V == 1) {
      c[0] = cp[0];
      s[0] = sp[0];
    } else {
#pragma unroll
      for (int i = 0; i < V; i += 4) {
        const float4 cw = *reinterpret_cast<const float4*>(cp + i), sw = *reinterpret_cast<const float4*>(sp + i);
        c[i] = cw.x; c[i + 1] = cw.y; c[i + 2] = cw.z; c[i + 3] = cw.w;
        s[i] = sw.x; s[i + 1] = sw.y; s[i + 2] = sw.z; s[i + 3] = sw.w;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      c[i] = ld_any(a.cos, angle + u * V + i, a.table_dtype);
      s[i] = ld_any(a.sin, angle + u * V + i, a.table_dtype);
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (a.back) s[i] = -s[i];
}
template <int V>
__device__ __forceinline__ void unit_turn(bool interleaved, const float (&c)[V], const float (&s)[V], float (&p)[V], float (&q)[V]) {
  if (!interleaved || V == 1) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float m = p[i], n = q[i];
      p[i] = fmaf(m, c[i], -(n * s[i]));  // the same roundings for every V
      q[i] = fmaf(n, c[i], m * s[i]);
    }
  } else if constexpr (V > 1) {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const float m = p[i], n = p[i + 1], m2 = q[i], n2 = q[i + 1];
      p[i] = fmaf(m, c[i / 2], -(n * s[i / 2]));
      p[i + 1] = fmaf(n, c[i / 2], m * s[i / 2]);
      q[i] = fmaf(m2, c[V / 2 + i / 2], -(n2 * s[V / 2 + i / 2]));
      q[i + 1] = fmaf(n2, c[V / 2 + i / 2], m2 * s[V / 2 + i / 2]);
    }
  }
}

// Eight lanes take HB heads of a row (of q, k and, append, v together), a lane the same V elements
// of both halves of their pairs, so a pair lies in one lane, a head's square sum is one reduction over
// eight lanes, and the row's angles are read once for the HB heads.
template <int DT, int V, int HB, bool APPEND>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
  const int lane8 = threadIdx.x & 7, group = threadIdx.x >> 3;
  const int rotary_heads = a.heads + a.kv_heads, heads = rotary_heads + (APPEND ? a.kv_heads : 0);
  const int parts = (heads + HB - 1) / HB;                // groups of a row
  const int rows = parts < 32 ? 32 / parts : 1;           // of the workgroup
  const int64_t t0 = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * rows;
  __shared__ RowPlace place[APPEND ? 32 : 1];
  if constexpr (APPEND) {
    for (int i = threadIdx.x >> 6; i < rows && t0 + i < a.T; i += 4) {
      const RowPlace r = row_place(a, t0 + i);
      if (__lane_id() == 0) place[i] = r;
    }
    __syncthreads();
  }
  const int row = parts < 32 ? group / parts : 0;
  const int64_t t = t0 + row;
  if (row >= rows || t >= a.T) return;
  const int turned = a.rd / (2 * V);                                // units of pairs
  const int units = turned + (a.hd - a.rd) / (V == 1 ? 1 : 2 * V);  // and of what stays
  int64_t position, key_row = 0;
  bool stored = true;
  if constexpr (APPEND) {
    const RowPlace p = place[row];
    position = p.position;
    stored = p.page >= 0;
    key_row = p.page * a.ys_p + p.row * a.ys_t;
  } else {
    position = a.wide_positions ? static_cast<const int64_t*>(a.positions)[t] : (int64_t) static_cast<const int*>(a.positions)[t];
  }
  const bool none = APPEND && position == kNoSequence;  // behind the last sequence: zeros
  const bool inside = position >= 0 && position < a.table_rows;
  const int64_t angle = (inside ? position : 0) * a.table_stride;

  for (int part = parts < 32 ? group % parts : group; part < parts; part += 32) {
    const char* from[HB];
    char* to[HB];
    int kind[HB];  // 0 q, 1 k, 2 v, -1 none
#pragma unroll
    for (int j = 0; j < HB; ++j) {
      const int head = part * HB + j;
      const int which = head < a.heads ? 0 : head < rotary_heads ? 1 : 2;
      const int h = which == 0 ? head : which == 1 ? head - a.heads : head - rotary_heads;
      kind[j] = head < heads && (which == 0 || stored) ? which : -1;
      constexpr int E = DT == kF32 ? 4 : 2;
      from[j] = static_cast<const char*>(a.x[which]) + (t * a.xs_t[which] + h * a.xs_h[which]) * E;
      const int64_t at = APPEND && which > 0 ? key_row + h * a.ys_h : (t * a.x_heads(which) + h) * a.hd;
      to[j] = static_cast<char*>(a.y[which]) + at * E;
    }
    float p[HB][V], q[HB][V], inv[HB];
    auto load = [&](int u) {
      const UnitAt at = unit_at<V>(a, u, turned);
#pragma unroll
      for (int j = 0; j < HB; ++j) {
        if (kind[j] < 0) continue;
        load_v<DT, V>(from[j], at.e0, p[j]);
        load_v<DT, V>(from[j], at.e1, q[j]);
      }
    };
    const bool once = units <= 8;
#pragma unroll
    for (int j = 0; j < HB; ++j) inv[j] = 1.f;
    if (APPEND && (a.q_gain || a.k_gain)) {
      float ss[HB];
#pragma unroll
      for (int j = 0; j < HB; ++j) ss[j] = 0.f;
      for (int u = lane8; u < units; u += 8) {
        load(u);
        const bool two = V > 1 || u < turned;
#pragma unroll
        for (int j = 0; j < HB; ++j)
#pragma unroll
          for (int i = 0; i < V; ++i) ss[j] += p[j][i] * p[j][i] + (two ? q[j][i] * q[j][i] : 0.f);
      }
#pragma unroll
      for (int j = 0; j < HB; ++j) inv[j] = rsqrtf(row_reduce<8, OpAdd>(ss[j]) / (float)a.hd + a.eps);
    }
    for (int u = lane8; u < units; u += 8) {
      if (!once || !(APPEND && (a.q_gain || a.k_gain))) load(u);
      const UnitAt at = unit_at<V>(a, u, turned);
      float c[V], s[V];
      if (u < turned) unit_angles<V>(a, angle, u, inside, c, s);
#pragma unroll
      for (int j = 0; j < HB; ++j) {
        if (kind[j] < 0) continue;
        const void* gain = !APPEND ? nullptr : kind[j] == 0 ? a.q_gain : kind[j] == 1 ? a.k_gain : nullptr;
        if (gain) {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            p[j][i] *= inv[j] * ld_any(gain, at.e0 + i, a.gain_dtype);
            q[j][i] *= inv[j] * ld_any(gain, at.e1 + i, a.gain_dtype);
          }
        }
        if (kind[j] < 2 && u < turned) unit_turn<V>(a.interleaved, c, s, p[j], q[j]);
        if (none) {
#pragma unroll
          for (int i = 0; i < V; ++i) p[j][i] = q[j][i] = 0.f;
        }
        store_v<DT, V, !APPEND>(to[j], at.e0, p[j]);
        if (V > 1 || u < turned) store_v<DT, V, !APPEND>(to[j], at.e1, q[j]);
      }
    }
  }
}

template <int DT, int V, int HB>
hipError_t launch_heads(const RotaryArgs& a, bool append, hipStream_t s) {
  const int heads = a.heads + (append ? 2 : 1) * a.kv_heads, parts = (heads + HB - 1) / HB;
  const int rows = parts < 32 ? 32 / parts : 1;
  const int64_t blocks = (a.T + rows - 1) / rows;
  constexpr int64_t kLine = 1 << 23;  // a dimension of a launch holds less than 2^32 threads
  const dim3 grid((unsigned)(blocks < kLine ? blocks : kLine), (unsigned)((blocks + kLine - 1) / kLine));
  if constexpr (DT != kF32 && HB != 3) {  // three heads: not appended
    if (append) {
      rotary_kernel<DT, V, HB, true><<<grid, 256, 0, s>>>(a);
      return hipGetLastError();
    }
  }
  rotary_kernel<DT, V, HB, false><<<grid, 256, 0, s>>>(a);
  return hipGetLastError();
}
// Heads a group of lanes: several where that leaves every CU some workgroups.  A 16-bit launch of
// 16384 rows, 8 + 4 heads of 96: 22.1, 20.1, 18.6, 21.0 us with 1 to 4 (4.2 TB/s with 3); 8191 rows appended,
// 16 + 2 + 2 of 128: 34.2, 25.7, 27.8, 26.1; an fp32 one of 4001 rows, 16 + 2 of 128: 16.0, 18.8, 20.2, 18.2.
template <int DT, int V>
hipError_t launch_v(const RotaryArgs& a, bool append, hipStream_t s) {
  if constexpr (V > 1 && DT != kF32) {
    const int heads = a.heads + a.kv_heads;
    if (a.T * heads >= 256 * (int64_t)device_cus())
      return !append && heads % 3 == 0 ? launch_heads<DT, V, 3>(a, append, s) : launch_heads<DT, V, 2>(a, append, s);
  }
  return launch_heads<DT, V, 1>(a, append, s);
}

}  // namespace

// V: as many elements as the sizes, strides and pointers allow; the widest has 16-byte accesses.
hipError_t launch_rotary(RotaryArgs a, bool append, hipStream_t s) {
  auto fits = [&](int v) {
    const int bytes = dtype_bytes(a.dtype) * v;
    if (a.hd % (2 * v) || a.rd % (2 * v)) return false;
    for (int i = 0; i < (append ? 3 : 2); ++i) {
      if (i == 1 && a.kv_heads == 0) continue;
      if (reinterpret_cast<uintptr_t>(a.x[i]) % bytes || reinterpret_cast<uintptr_t>(a.y[i]) % bytes) return false;
      if (a.xs_t[i] % v || a.xs_h[i] % v) return false;
      if (append && i > 0 && (a.ys_p % v || a.ys_t % v || a.ys_h % v)) return false;
    }
    return true;
  };
  auto wide = [&](int v) {  // the tables' rows by 16 bytes
    return v == 1 || (reinterpret_cast<uintptr_t>(a.cos) % 16 == 0 && reinterpret_cast<uintptr_t>(a.sin) % 16 == 0 &&
                      a.table_stride % 4 == 0);
  };
  if (a.dtype == kF32) {
    const bool four = fits(4);
    a.table_wide = wide(four ? 4 : 1);
    return four ? launch_v<kF32, 4>(a, append, s) : launch_v<kF32, 1>(a, append, s);
  }
  const int v = fits(8) ? 8 : fits(4) ? 4 : 1;
  a.table_wide = wide(v);
  if (a.dtype == kBF16)
    return v == 8 ? launch_v<kBF16, 8>(a, append, s) : v == 4 ? launch_v<kBF16, 4>(a, append, s) : launch_v<kBF16, 1>(a, append, s);
  return v == 8 ? launch_v<kF16, 8>(a, append, s) : v == 4 ? launch_v<kF16, 4>(a, append, s) : launch_v<kF16, 1>(a, append, s);
}

}  // namespace mhc
