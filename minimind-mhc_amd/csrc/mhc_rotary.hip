// Rotary positions, by themselves and on the way of new tokens into a cache of pages.
//   Pair (a, b) of a head's first rd elements, half layout (d, d + rd / 2), interleaved (2 d,
//   2 d + 1):  a' = a c - b s,  b' = b c + a s,  c, s = cos, sin [position, d];  the elements behind
//   rd stay.  The gradient is the transposed map, the same with -s.
//   With gains (append only) x = y rsqrt(mean y^2 + eps) gain comes before.
// Bound by bytes: every element is read once and written once, in fp32 between, rounded once.
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
template <int DT, int V>
__device__ __forceinline__ void store_v(void* p, int64_t i, const float (&x)[V]) {
  if constexpr (V == 1) {
    st_any(p, i, DT, x[0]);
  } else if constexpr (DT == kF32) {
    *reinterpret_cast<float4*>(static_cast<float*>(p) + i) = make_float4(x[0], x[1], x[2], x[3]);
  } else {
    uint32_t w[V / 2];
#pragma unroll
    for (int j = 0; j < V / 2; ++j) w[j] = pack2<DT == kF16>(x[2 * j], x[2 * j + 1]);
    uint16_t* d = static_cast<uint16_t*>(p) + i;
    if constexpr (V == 8) *reinterpret_cast<U32x4*>(d) = *reinterpret_cast<const U32x4*>(w);
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

// Eight lanes take a head of a row, a lane the same V elements of both halves of its pairs (or 2 V
// neighbours), so a pair lies in one lane and a head's square sum is one reduction over eight
// lanes.  A workgroup takes `rows` rows, the heads of q, of k and (append) of v in turn.
template <int DT, int V, bool APPEND>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
  const int lane8 = threadIdx.x & 7;
  const int64_t t0 = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * a.rows;
  if (t0 >= a.T) return;
  const int rows = (int)min((int64_t)a.rows, a.T - t0);
  __shared__ RowPlace place[APPEND ? kRotaryRows : 1];
  if constexpr (APPEND) {
    for (int i = threadIdx.x >> 6; i < rows; i += 4) {
      const RowPlace r = row_place(a, t0 + i);
      if (__lane_id() == 0) place[i] = r;
    }
    __syncthreads();
  }
  const int turned = a.rd / (2 * V);                                   // units of pairs
  const int units = turned + (a.hd - a.rd) / (V == 1 ? 1 : 2 * V);     // and of what stays
  const int rotary_heads = a.heads + a.kv_heads;
  const int heads = rotary_heads + (APPEND ? a.kv_heads : 0);
  for (int item = threadIdx.x >> 3; item < rows * heads; item += 32) {
    const int row = item / heads, head = item % heads;
    const int64_t t = t0 + row;
    const int which = head < a.heads ? 0 : head < rotary_heads ? 1 : 2;
    const int h = which == 0 ? head : which == 1 ? head - a.heads : head - rotary_heads;
    const void* x = a.x[which];
    const int64_t from = t * a.xs_t[which] + h * a.xs_h[which];
    void* y = a.y[which];
    int64_t to, position;
    bool none = false;
    if constexpr (APPEND) {
      const RowPlace p = place[row];
      position = p.position;
      none = position == kNoSequence;
      if (which == 0) {
        to = (t * a.heads + h) * a.hd;
      } else {
        if (p.page < 0) continue;
        to = p.page * a.ys_p + p.row * a.ys_t + h * a.ys_h;
      }
    } else {
      position = a.wide_positions ? static_cast<const int64_t*>(a.positions)[t]
                                  : (int64_t) static_cast<const int*>(a.positions)[t];
      to = (t * a.x_heads(which) + h) * a.hd;
    }
    const bool inside = position >= 0 && position < a.table_rows;
    const int64_t angle = (inside ? position : 0) * a.table_stride;

    float p[V], q[V];
    auto load = [&](int u) {
      if (u < turned && !a.interleaved) {
        load_v<DT, V>(x, from + u * V, p);
        load_v<DT, V>(x, from + a.rd / 2 + u * V, q);
      } else if (V > 1 || u < turned) {
        load_v<DT, V>(x, from + u * 2 * V, p);  // what stays begins at rd, two V a unit, too
        load_v<DT, V>(x, from + u * 2 * V + V, q);
      } else {
        load_v<DT, V>(x, from + a.rd + u - turned, p);
        q[0] = 0.f;
      }
    };
    auto store = [&](int u) {
      if (u < turned && !a.interleaved) {
        store_v<DT, V>(y, to + u * V, p);
        store_v<DT, V>(y, to + a.rd / 2 + u * V, q);
      } else if (V > 1 || u < turned) {
        store_v<DT, V>(y, to + u * 2 * V, p);
        store_v<DT, V>(y, to + u * 2 * V + V, q);
      } else {
        store_v<DT, V>(y, to + a.rd + u - turned, p);
      }
    };
    auto turn = [&](int u) {
      if (which == 2 || u >= turned) return;
      float c[V], s[V];
      if (!inside) {  // the tables may have no row at all
#pragma unroll
        for (int i = 0; i < V; ++i) c[i] = s[i] = __builtin_nanf("");
      } else if (a.table_dtype == kF32 && a.table_wide) {
        if constexpr (V == 1) {
          c[0] = static_cast<const float*>(a.cos)[angle + u];
          s[0] = static_cast<const float*>(a.sin)[angle + u];
        } else {
#pragma unroll
          for (int i = 0; i < V; i += 4) {
            const float4 cw = *reinterpret_cast<const float4*>(static_cast<const float*>(a.cos) + angle + u * V + i);
            const float4 sw = *reinterpret_cast<const float4*>(static_cast<const float*>(a.sin) + angle + u * V + i);
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
      if (!a.interleaved || V == 1) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float m = p[i], n = q[i];
          p[i] = fmaf(m, c[i], -(n * s[i]));  // the same roundings for every V
          q[i] = fmaf(n, c[i], m * s[i]);
        }
      } else if constexpr (V > 1) {
#pragma unroll
        for (int i = 0; i < V; i += 2) {
          const float m = p[i], n = p[i + 1];
          p[i] = fmaf(m, c[i / 2], -(n * s[i / 2]));
          p[i + 1] = fmaf(n, c[i / 2], m * s[i / 2]);
          const float m2 = q[i], n2 = q[i + 1];
          q[i] = fmaf(m2, c[V / 2 + i / 2], -(n2 * s[V / 2 + i / 2]));
          q[i + 1] = fmaf(n2, c[V / 2 + i / 2], m2 * s[V / 2 + i / 2]);
        }
      }
    };
    if constexpr (APPEND) {
      const void* gain = which == 0 ? a.q_gain : which == 1 ? a.k_gain : nullptr;
      auto norm = [&](int u, float inv) {
        const bool half = u < turned && !a.interleaved;
        const bool one = V == 1 && u >= turned;
        const int i0 = half ? u * V : one ? a.rd + u - turned : u * 2 * V;
        const int i1 = half ? a.rd / 2 + u * V : one ? i0 : i0 + V;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          p[i] *= inv * ld_any(gain, i0 + i, a.gain_dtype);
          q[i] *= inv * ld_any(gain, i1 + i, a.gain_dtype);
        }
      };
      float inv = 1.f;
      const bool once = units <= 8;
      if (gain || once) {
        float ss = 0.f;
        for (int u = lane8; u < units; u += 8) {
          load(u);
#pragma unroll
          for (int i = 0; i < V; ++i) ss += p[i] * p[i] + q[i] * q[i];
        }
        ss = row_reduce<8, OpAdd>(ss);
        inv = rsqrtf(ss / (float)a.hd + a.eps);
      }
      for (int u = lane8; u < units; u += 8) {
        if (!once) load(u);
        if (gain) norm(u, inv);
        turn(u);
        if (none) {  // behind the last sequence: zeros
#pragma unroll
          for (int i = 0; i < V; ++i) p[i] = q[i] = 0.f;
        }
        store(u);
      }
    } else {
      for (int u = lane8; u < units; u += 8) {
        load(u);
        turn(u);
        store(u);
      }
    }
  }
}

template <int DT, int V>
hipError_t launch_v(const RotaryArgs& a, bool append, hipStream_t s) {
  const int64_t blocks = (a.T + a.rows - 1) / a.rows;
  constexpr int64_t kLine = 1 << 23;  // a dimension of a launch holds less than 2^32 threads
  const dim3 grid((unsigned)(blocks < kLine ? blocks : kLine), (unsigned)((blocks + kLine - 1) / kLine));
  if constexpr (DT != kF32) {
    if (append) {
      rotary_kernel<DT, V, true><<<grid, 256, 0, s>>>(a);
      return hipGetLastError();
    }
  }
  rotary_kernel<DT, V, false><<<grid, 256, 0, s>>>(a);
  return hipGetLastError();
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
  // a few rows a workgroup where there are many, one where there are few
  const int heads = a.heads + (append ? 2 : 1) * a.kv_heads;
  int rows = heads >= 96 ? 1 : 96 / (heads < 1 ? 1 : heads);
  if (rows > kRotaryRows) rows = kRotaryRows;
  while (rows > 1 && (a.T + rows - 1) / rows < 4 * (int64_t)device_cus()) rows = (rows + 1) / 2;
  a.rows = rows;
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
