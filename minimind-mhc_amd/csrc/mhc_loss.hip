// Losses over rows of logits and over a router's scores, with their gradients.
//   log-probability of a label:  lp_t = x_y - l_t,  l_t = max_v x + log sum_v exp(x_v - max),
//     d lp_t / d x_v = [v = y] - exp(x_v - l_t)
//   preference loss of pairs (c, r):  z = beta ((S_c - R_c) - (S_r - R_r)),  S the sequences'
//     sums (or means) of lp,  L = mean -((1 - e) log sig(z) + e log sig(-z)),
//     dL/dz = e sig(z) - (1 - e) sig(-z)
//   balance of E experts over T tokens:  L = coef E sum_e f_e P_e,  f_e = count_e / T,  P_e the
//     mean score;  d score_te = coef E f_e / T
#include "mhc_packed.hpp"

namespace mhc {
namespace {

constexpr float kLowest = -3.40282346638528859812e38f;
constexpr float kLn2 = 0.69314718055994530942f;

template <int DT>
__device__ __forceinline__ float load_elem(const void* p, int64_t i) {
  if constexpr (DT == kF32) return static_cast<const float*>(p)[i];
  else if constexpr (DT == kBF16) return bf16_bits_to_f32(static_cast<const uint16_t*>(p)[i]);
  else return f16_bits_to_f32(static_cast<const uint16_t*>(p)[i]);
}
template <int DT>
__device__ __forceinline__ void store_elem(void* p, int64_t i, float v) {
  if constexpr (DT == kF32) static_cast<float*>(p)[i] = v;
  else if constexpr (DT == kBF16) static_cast<uint16_t*>(p)[i] = f32_to_bf16_bits(v);
  else static_cast<uint16_t*>(p)[i] = f32_to_f16_bits(v);
}
// The elements of 16 bytes, as fp32, and back.
template <int DT>
constexpr int kPer16 = DT == kF32 ? 4 : 8;
template <int DT>
__device__ __forceinline__ void unpack16(const U32x4& w, float (&x)[kPer16<DT>]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (DT == kF32) {
      x[j] = __uint_as_float(w.v[j]);
    } else {
      x[2 * j] = elem_lo<DT == kF16>(w.v[j]);
      x[2 * j + 1] = elem_hi<DT == kF16>(w.v[j]);
    }
  }
}
template <int DT>
__device__ __forceinline__ U32x4 pack16(const float (&x)[kPer16<DT>]) {
  U32x4 w;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (DT == kF32) w.v[j] = __float_as_uint(x[j]);
    else w.v[j] = pack2<DT == kF16>(x[2 * j], x[2 * j + 1]);
  }
  return w;
}

// --------------------------------------------------- log-probabilities of labels
// A workgroup a row, in as many lines of 2^22 of them as it takes: one dimension of a launch holds
// less than 2^32 threads, and wraps without an error.
constexpr int64_t kLaunchLine = 1 << 22;
inline dim3 launch_rows(int64_t rows) {
  return dim3((unsigned)(rows < kLaunchLine ? rows : kLaunchLine), (unsigned)((rows + kLaunchLine - 1) / kLaunchLine));
}
__device__ __forceinline__ int64_t launch_row() { return blockIdx.x + (int64_t)blockIdx.y * kLaunchLine; }

// One workgroup a row, one pass: each thread keeps a running maximum and sum.  A row may
// begin anywhere: the elements before its first 16-byte boundary and behind its last go one
// by one.  Rows whose label does not count are not read.  16384 x 6400 bf16 rows, a quarter of them
// uncounted, 157 MB: 30 us, 5.2 TB/s, the rate of a copy; 2047 x 50257 fp32 55 us, 5.6 TB/s.  (Cached
// instead of non-temporal loads 34 us.)
template <int DT>
__global__ __launch_bounds__(256) void logprob_kernel(LogitArgs a) {
  constexpr int PER = kPer16<DT>;
  __shared__ float sm[4], sl[4];
  const int64_t row = launch_row();
  if (row >= a.T) return;
  const int64_t label = a.labels[row];
  const int tid = threadIdx.x;
  const bool counts = label != a.ignore;
  if (!counts || label < 0 || label >= a.V) {
    if (tid == 0) {
      a.logprobs[row] = counts ? __builtin_nanf("") : 0.f;
      if (a.lse) a.lse[2 * row] = a.lse[2 * row + 1] = counts ? __builtin_nanf("") : 0.f;
    }
    return;
  }
  constexpr int EB = DT == kF32 ? 4 : 2;
  const char* base = static_cast<const char*>(a.logits) + row * a.stride * EB;
  const int head = min((int)((16 - (reinterpret_cast<uintptr_t>(base) & 15)) % 16 / EB), a.V);
  const int n16 = (a.V - head) / PER;
  const char* mid = base + head * EB;
  // the maximum starts at fp32's lowest value, so a row that a mask of that value fills is
  // a uniform one
  float m = kLowest, l = 0.f;
  auto take = [&](float x) {
    if (x > m) {
      l *= exp2_f((m - x) * kPackedLog2e);
      m = x;
    }
    l += exp2_f((x - m) * kPackedLog2e);
  };
  for (int i = tid; i < n16; i += 256) {
    float x[PER];
    unpack16<DT>(ld16_nt(mid + (int64_t)i * 16), x);
    float mx = x[0];
#pragma unroll
    for (int j = 1; j < PER; ++j) mx = fmaxf(mx, x[j]);
    if (mx > m) {
      l *= exp2_f((m - mx) * kPackedLog2e);
      m = mx;
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) l += exp2_f((x[j] - m) * kPackedLog2e);
  }
  const int rest = head + n16 * PER;
  if (tid < head) take(load_elem<DT>(base, tid));
  if (tid < a.V - rest) take(load_elem<DT>(base, rest + tid));
  const float wm = wave_max(m);
  const float wl = wave_sum(l * exp2_f((m - wm) * kPackedLog2e));
  if ((tid & 63) == 0) {
    sm[tid >> 6] = wm;
    sl[tid >> 6] = wl;
  }
  __syncthreads();
  if (tid != 0) return;
  const float mx = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  float sum = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) sum += sl[w] * exp2_f((sm[w] - mx) * kPackedLog2e);
  const float ls = log2f(sum);
  a.logprobs[row] = (load_elem<DT>(base, label) - mx) - ls * kLn2;
  if (a.lse) {  // kept apart: their sum would round at the size of the logits
    a.lse[2 * row] = mx;
    a.lse[2 * row + 1] = ls;
  }
}

// The factor of a row's gradient: its own, or that of its sequence in the preference loss
// (lower bound over the sequences' ends).  False for a row behind the last sequence: zeros then,
// whatever its logits hold.
__device__ __forceinline__ bool row_factor(const LogitArgs& a, int64_t row, float& f) {
  if (!a.cu) {
    f = a.g_row[row];
    return true;
  }
  int lo = 0, hi = a.B;  // the sequence with start <= row < end
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (min(max(a.cu[mid + 1], 0), (int)a.T) <= row) lo = mid + 1;
    else hi = mid;
  }
  if (lo >= a.B) return false;
  f = a.g_seq[lo] * a.g_loss[0];
  return true;
}

// One workgroup a row again: p from the stored maximum and sum, and the gradient, zeros where
// the row does not count.  16384 x 6400 bf16, 367 MB: 54 us, 6.8 TB/s with part of the logits still in
// the memory-side cache; 2047 x 50257 fp32, 720 MB: 138 to 173 us.
template <int DT>
__global__ __launch_bounds__(256) void logprob_bwd_kernel(LogitArgs a) {
  constexpr int PER = kPer16<DT>;
  constexpr int EB = DT == kF32 ? 4 : 2;
  // from the last row back: the forward pass's last rows are still in the memory-side cache
  const int64_t row = a.T - 1 - launch_row();
  if (row < 0) return;
  const int64_t label = a.labels[row];
  const int tid = threadIdx.x;
  float f = 0.f;
  const bool counts = label != a.ignore && row_factor(a, row, f);
  const char* base = static_cast<const char*>(a.logits) + row * a.stride * EB;
  char* out = static_cast<char*>(a.g_logits) + row * a.V * EB;
  const float m = counts ? a.lse[2 * row] : 0.f, ls = counts ? a.lse[2 * row + 1] : 0.f;
  auto one = [&](int i) {
    const float p = counts ? exp2_f(fmaf(load_elem<DT>(base, i) - m, kPackedLog2e, -ls)) : 0.f;
    store_elem<DT>(out, i, counts ? f * ((i == label ? 1.f : 0.f) - p) : 0.f);
  };
  // whole 16-byte pieces only where both rows lie alike
  const int hi_ = (int)((16 - (reinterpret_cast<uintptr_t>(out) & 15)) % 16 / EB);
  const bool alike = ((reinterpret_cast<uintptr_t>(out) ^ reinterpret_cast<uintptr_t>(base)) & 15) == 0;
  const int head = min(hi_, a.V);
  const int n16 = (a.V - head) / PER;
  for (int i = tid; i < n16; i += 256) {
    float x[PER];
    const int at = head + i * PER;
    if (!counts) {
#pragma unroll
      for (int j = 0; j < PER; ++j) x[j] = 0.f;
    } else {
      if (alike) {
        unpack16<DT>(ld16_nt(base + (int64_t)at * EB), x);
      } else {
#pragma unroll
        for (int j = 0; j < PER; ++j) x[j] = load_elem<DT>(base, at + j);
      }
#pragma unroll
      for (int j = 0; j < PER; ++j)
        x[j] = f * ((at + j == label ? 1.f : 0.f) - exp2_f(fmaf(x[j] - m, kPackedLog2e, -ls)));
    }
    *reinterpret_cast<U32x4*>(out + (int64_t)at * EB) = pack16<DT>(x);
  }
  const int rest = head + n16 * PER;
  if (tid < head) one(tid);
  if (tid < a.V - rest) one(rest + tid);
}

// ------------------------------------------------------------- preference loss
__device__ __forceinline__ double softplus(double t) { return fmax(t, 0.0) + log1p(exp(-fabs(t))); }
__device__ __forceinline__ double sigmoid_d(double t) { return 1.0 / (1.0 + exp(-t)); }

// One workgroup a pair: both sequences' sums in 64 bits (a sequence's sum is hundreds of
// units, the rewards' difference less than one), the pair's loss and its rows' factors.  16
// pairs of 16384 rows: 5.4 us, latency.
__global__ __launch_bounds__(256) void preference_kernel(PreferenceArgs a) {
  __shared__ double part[2][4];
  __shared__ int cnt[2][4];
  const int pair = blockIdx.x, tid = threadIdx.x;
  double s[2] = {0.0, 0.0};
  int n[2] = {0, 0};
  for (int side = 0; side < 2; ++side) {
    const int seq = side * a.P + pair;
    const int t0 = seq_start(a.cu, seq, a.T), t1 = max(seq_start(a.cu, seq + 1, a.T), t0);
    for (int t = t0 + tid; t < t1; t += 256) {
      s[side] += (double)a.logprobs[t];
      n[side] += a.labels[t] != a.ignore;
    }
    for (int o = 32; o > 0; o >>= 1) {
      s[side] += __shfl_xor(s[side], o, 64);
      n[side] += __shfl_xor(n[side], o, 64);
    }
    if ((tid & 63) == 0) {
      part[side][tid >> 6] = s[side];
      cnt[side][tid >> 6] = n[side];
    }
  }
  __syncthreads();
  if (tid != 0) return;
  double reward[2], each[2];
  for (int side = 0; side < 2; ++side) {
    const double sum = (part[side][0] + part[side][1]) + (part[side][2] + part[side][3]);
    const int count = cnt[side][0] + cnt[side][1] + cnt[side][2] + cnt[side][3];
    each[side] = a.average ? 1.0 / max(count, 1) : 1.0;
    const int at = side * a.P + pair;
    const double ref = a.reference64 ? static_cast<const double*>(a.reference)[at] : static_cast<const float*>(a.reference)[at];
    reward[side] = a.beta * (sum * each[side] - ref);
  }
  const double z = reward[0] - reward[1], e = a.smoothing;
  a.pair_loss[pair] = (1.0 - e) * softplus(-z) + (e > 0.0 ? e * softplus(z) : 0.0);  // z may be infinite
  const double dz = (e * sigmoid_d(z) - (1.0 - e) * sigmoid_d(-z)) * a.beta / a.P;
  a.chosen[pair] = (float)reward[0];
  a.rejected[pair] = (float)reward[1];
  a.g_seq[pair] = (float)(dz * each[0]);
  a.g_seq[a.P + pair] = (float)(-dz * each[1]);
}

__global__ __launch_bounds__(64) void preference_mean_kernel(PreferenceArgs a) {
  double s = 0.0;
  for (int i = threadIdx.x; i < a.P; i += 64) s += a.pair_loss[i];
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if (threadIdx.x == 0) a.loss[0] = (float)(s / a.P);
}

// -------------------------------------------------------------- balance loss
// Each workgroup sums a range of one sequence's rows into partials; columns of scores in
// registers (thread = column of a row group), counts by LDS integers (their order changes
// nothing).  A second launch adds the ranges in order.  16384 x 8 bf16: 3.7 us, latency.
template <int DT>
__global__ __launch_bounds__(256) void balance_kernel(BalanceArgs a) {
  extern __shared__ float sums[];  // [256] then int counts [E]
  int* counts = reinterpret_cast<int*>(sums + 256);
  const int seq = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
  const int t0 = a.cu ? seq_start(a.cu, seq, a.T) : 0;
  const int t1 = a.cu ? max(seq_start(a.cu, seq + 1, a.T), t0) : a.T;
  const int per = (t1 - t0 + a.parts - 1) / a.parts;
  const int r0 = min(t0 + part * per, t1), r1 = min(r0 + per, t1);
  const int tid = threadIdx.x;
  const int64_t at = ((int64_t)seq * a.parts + part) * a.E;
  for (int e = tid; e < a.E; e += 256) counts[e] = 0;
  __syncthreads();
  for (int64_t i = (int64_t)r0 * a.K + tid; i < (int64_t)r1 * a.K; i += 256) {
    const int64_t e = a.index[i];
    if (e >= 0 && e < a.E) atomicAdd(&counts[e], 1);
  }
  for (int e0 = 0; e0 < a.E; e0 += 256) {
    const int cols = min(a.E - e0, 256), lanes = 256 / cols;  // rows a step
    const int col = tid % cols, sub = tid / cols;
    float s = 0.f;
    if (sub < lanes)
      for (int t = r0 + sub; t < r1; t += lanes) s += load_elem<DT>(a.scores, (int64_t)t * a.stride + e0 + col);
    __syncthreads();
    sums[tid] = s;
    __syncthreads();
    if (tid < cols) {
      for (int j = 1; j < lanes; ++j) s += sums[j * cols + tid];
      a.part_sum[at + e0 + tid] = s;
    }
  }
  for (int e = tid; e < a.E; e += 256) a.part_count[at + e] = counts[e];
}

// One workgroup joins the ranges: LP lanes a (sequence, expert) pair, each every LP-th range
// in order, in 64 bits; then the mean over the sequences with rows.  One launch after the sums
// takes as long as a launch does; with the sequences in turn and a lane an expert 44 us.
__global__ __launch_bounds__(1024) void balance_join_kernel(BalanceArgs a) {
  __shared__ double red[16];
  __shared__ int full[16];
  const int tid = threadIdx.x, pairs = a.B * a.E;
  int lp = 1;
  while (lp < 32 && pairs * lp * 2 <= 2048) lp *= 2;
  double loss = 0.0;
  int filled = 0;
  auto rows = [&](int seq) {
    const int t0 = a.cu ? seq_start(a.cu, seq, a.T) : 0;
    return (a.cu ? max(seq_start(a.cu, seq + 1, a.T), t0) : a.T) - t0;
  };
  for (int i = tid; i < a.B; i += 1024) filled += rows(i) > 0;
  const int sub = tid % lp;
  for (int pair0 = 0; pair0 < pairs; pair0 += 1024 / lp) {  // uniform: every lane takes part in the sums
    const int pair = pair0 + tid / lp;
    const bool live = pair < pairs;
    const int seq = live ? pair / a.E : 0, e = live ? pair % a.E : 0;
    const int64_t at = (int64_t)seq * a.parts * a.E + e;
    double s = 0.0;
    int64_t c = 0;
#pragma unroll 4
    for (int p = live ? sub : a.parts; p < a.parts; p += lp) {
      s += (double)a.part_sum[at + (int64_t)p * a.E];
      c += a.part_count[at + (int64_t)p * a.E];
    }
    for (int o = lp / 2; o > 0; o >>= 1) {
      s += __shfl_xor(s, o, 64);
      c += __shfl_xor(c, o, 64);
    }
    if (!live || sub != 0) continue;
    a.counts[pair] = c;
    const int n = rows(seq);
    if (n > 0) loss += (double)c / n * (s / n);
  }
  for (int o = 32; o > 0; o >>= 1) {
    loss += __shfl_xor(loss, o, 64);
    filled += __shfl_xor(filled, o, 64);
  }
  if ((tid & 63) == 0) {
    red[tid >> 6] = loss;
    full[tid >> 6] = filled;
  }
  __syncthreads();
  if (tid != 0) return;
  double total = 0.0;
  int n = 0;
  for (int w = 0; w < 16; ++w) {
    total += red[w];
    n += full[w];
  }
  a.loss[0] = n ? (float)((double)a.coef * a.E * total / n) : 0.f;
  a.filled[0] = n;
}

// coef E f_e / T for every row: 16384 x 8 bf16 3.0 us, 8191 x 64 fp32 5.0 us, launch and divisions.
template <int DT>
__global__ __launch_bounds__(256) void balance_bwd_kernel(BalanceArgs a) {
  const int64_t i = launch_row() * 256 + threadIdx.x;
  if (i >= (int64_t)a.T * a.E) return;
  const int t = (int)(i / a.E), e = (int)(i % a.E);
  int seq = 0, n = a.T;
  if (a.cu) {
    int lo = 0, hi = a.B;
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (min(max(a.cu[mid + 1], 0), a.T) <= t) lo = mid + 1;
      else hi = mid;
    }
    seq = lo;
    n = seq < a.B ? seq_start(a.cu, seq + 1, a.T) - seq_start(a.cu, seq, a.T) : 0;
  }
  float g = 0.f;
  if (n > 0) {
    const double f = (double)a.counts[(int64_t)seq * a.E + e] / n;
    g = (float)((double)a.coef * a.E * f / ((double)n * a.filled[0]) * (double)a.g_loss[0]);
  }
  store_elem<DT>(a.g_scores, i, g);
}

#define MHC_LOSS_DT(dt, call)                 \
  switch (dt) {                               \
    case kF32: call(kF32); break;             \
    case kBF16: call(kBF16); break;           \
    case kF16: call(kF16); break;             \
    default: return hipErrorInvalidValue;     \
  }

}  // namespace

hipError_t launch_logprobs(const LogitArgs& a, hipStream_t s) {
#define RUN(DT) logprob_kernel<DT><<<launch_rows(a.T), 256, 0, s>>>(a)
  MHC_LOSS_DT(a.dtype, RUN)
#undef RUN
  return hipGetLastError();
}
hipError_t launch_logprobs_bwd(const LogitArgs& a, hipStream_t s) {
#define RUN(DT) logprob_bwd_kernel<DT><<<launch_rows(a.T), 256, 0, s>>>(a)
  MHC_LOSS_DT(a.dtype, RUN)
#undef RUN
  return hipGetLastError();
}
hipError_t launch_preference(const PreferenceArgs& a, hipStream_t s) {
  preference_kernel<<<dim3((unsigned)a.P), 256, 0, s>>>(a);
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  preference_mean_kernel<<<dim3(1), 64, 0, s>>>(a);
  return hipGetLastError();
}

// Ranges a sequence's rows are cut into: two workgroups a CU over all, of 128 rows or more.
int balance_parts(int64_t T, int B) {
  int64_t want = 2 * (int64_t)device_cus() / (B > 0 ? B : 1);
  const int64_t most = T / (128 * (int64_t)(B > 0 ? B : 1)) + 1;
  if (want > most) want = most;
  return want < 1 ? 1 : (int)want;
}
hipError_t launch_balance(const BalanceArgs& a, hipStream_t s) {
  if (a.B > 0) {
    const size_t lds = (256 + a.E) * 4;
#define RUN(DT) balance_kernel<DT><<<dim3((unsigned)((int64_t)a.B * a.parts)), 256, lds, s>>>(a)
    MHC_LOSS_DT(a.dtype, RUN)
#undef RUN
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  balance_join_kernel<<<dim3(1), 1024, 0, s>>>(a);
  return hipGetLastError();
}
hipError_t launch_balance_bwd(const BalanceArgs& a, hipStream_t s) {
  const int64_t blocks = ((int64_t)a.T * a.E + 255) / 256;
#define RUN(DT) balance_bwd_kernel<DT><<<launch_rows(blocks), 256, 0, s>>>(a)
  MHC_LOSS_DT(a.dtype, RUN)
#undef RUN
  return hipGetLastError();
}

}  // namespace mhc
