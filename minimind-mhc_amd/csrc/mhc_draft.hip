// Drafted tokens against the target's probabilities, and the accepted branch moved into place.
//   A sequence's rows are a tree, parents before children: row 0 its last token, the others
//   drafted.  At a node with target p and draft q (what its children were drawn from), with a = 0
//   and c = 1, its children in turn, token x and random u:
//     accepted if  u q(x) c < max(p(x) - a q(x), 0);  else  a += c,  c = sum_v max(p(v) - a q(v), 0)
//   max(p - a q, 0) / c is what a rejected draw leaves of p: after one, (p - q)+ / sum; after
//   another, ((p - q)+ / c - q)+ up to a factor, (p - (1 + c) q)+.  Where no child is left, the next
//   token is the first v whose cumulated max(p - a q, 0) exceeds u_0 times the total.
//   Certain drafts (no q): accepted if  u c < p(x), else c -= p(x) and p(x) = 0.
//   Greedy (no u): accepted if x is the first of the largest p; the next token is that of the last node.
// All in 64 bits: borders between tokens are compared, and a sum in 32 bits would move them.
#include "mhc_packed.hpp"

namespace mhc {
namespace {

constexpr int kDraftNodes = 1024;  // of a sequence, whose numbers are fetched at a time
constexpr int kDraftBlocks = 8;    // 16-byte blocks of a row that a lane keeps
constexpr int kDraftGone = 64;     // rejected siblings that are kept at hand

template <int DT>
struct ProbRow {
  static constexpr int PER = DT == kF32 ? 4 : 8;  // elements of 16 bytes
  // The row's elements lie in the tensor's 16-byte blocks: element e of the row is at e + off.  Blocks
  // are loaded through a descriptor that ends with the row's last word, without a branch, so all of a lane's are in
  // flight together.
  __amdgpu_buffer_rsrc_t rsrc;
  int off, V;
  __device__ void init(const void* p, int64_t row, int V_) {
    V = V_;
    const int64_t at = row * V;
    off = __builtin_amdgcn_readfirstlane((int)(at % PER));
    const int64_t base = wave_uniform(reinterpret_cast<int64_t>(p) + (at - off) * dtype_bytes(DT));
    rsrc = make_rsrc(reinterpret_cast<const void*>(base), ((uint32_t)(off + V) * dtype_bytes(DT) + 3) & ~3u);
  }
  __device__ int blocks() const { return (V + off + PER - 1) / PER; }
  // A block's 16 bytes (none: zeros), and 0 for the elements that are none of the row's.
  __device__ __forceinline__ U32x4 raw(int block, bool there) const {
    return buf_load16(rsrc, oob_unless(there, (uint32_t)block * 16));
  }
  __device__ __forceinline__ void trim(int block, U32x4& w) const {
    const int e0 = block * PER - off;
    if (e0 < 0 || e0 + PER > V) {
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if ((unsigned)(e0 + i) >= (unsigned)V) w.v[DT == kF32 ? i : i / 2] &= DT == kF32 ? 0u : i & 1 ? 0xffffu : 0xffff0000u;
    }
  }
  static __device__ __forceinline__ void open(const U32x4& w, float (&x)[PER]) {
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
};

// A probability: what is no positive finite number counts as 0 (the maximum of NaN and 0 is 0).
__device__ __forceinline__ double prob(float x) {
  x = fmaxf(x, 0.f);
  return (double)(x < __builtin_inff() ? x : 0.f);
}
// The same of the element of 16 bytes' word w (bf16: half `high` of it) where all of them are known to be
// finite and not negative, in two or three integer operations (a conversion takes four times as long): fp32's
// exponent and mantissa moved to their places.  Zero becomes 2^-127 (and the smallest numbers, which have no
// implicit one, up to twice as large): nothing beside a probability that counts.
__device__ __forceinline__ double fast64(uint32_t f) {
  return __builtin_bit_cast(double, (uint64_t)((f >> 3) + 0x38000000u) << 32 | (uint64_t)(f << 29));
}
__device__ __forceinline__ double fast64_bf16(uint32_t w, bool high) {
  const uint32_t b = high ? w >> 16 : w & 0xffffu;
  return __builtin_bit_cast(double, (uint64_t)((b << 13) + 0x38000000u) << 32);
}
__device__ __forceinline__ double left_of(double p, double q, double a) { return fmax(p - a * q, 0.0); }

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
  return v;
}

// A workgroup a sequence: the numbers of all its nodes are fetched side by side (token, then
// p and q at it in the parent's row), every wave walks the tree from LDS, and the whole
// workgroup goes over a vocabulary row only where a draw was rejected (or greedy, at each node)
// and for the next token: a pass of sums over a wave's contiguous part each, then the part that
// holds the border again, over all threads.  Bound by latencies in turn: 64 chains of 8 at a vocabulary of 6400 in fp32 11.9 us.
// Over a wide row one CU works alone, its VALU busy for 47% of its cycles; with sixteen waves a lane has 128 registers, and the
// compiler moves 38 to 43 to scratch memory (four waves: none).  One row of 50257 in bf16 without drafts 12.9 us, the first
// rejected draft 4.7 more, the second, which should read nothing, 6.9 (fp32: 6.7 and 10.8).  What of that is arithmetic and what scratch was not measured.
template <int DT, int W>
__global__ __launch_bounds__(64 * W) void verify_kernel(VerifyArgs a) {
  constexpr int PER = ProbRow<DT>::PER, TH = 64 * W;
  __shared__ float s_p[kDraftNodes], s_q[kDraftNodes], s_u[kDraftNodes];
  __shared__ int s_up[kDraftNodes], s_tok[kDraftNodes];
  __shared__ int s_gone[W][kDraftGone];  // a wave's own: one may be a node ahead
  __shared__ double s_sum[W];
  __shared__ int s_best[W], s_last[W];
  __shared__ float s_max[W];
  const int seq = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int start = seq_start(a.cu, seq, (int)a.T);
  const int end = min(max(a.cu[seq + 1], 0), (int)a.T), n = max(end - start, 0);
  if (seq == a.B - 1)  // rows behind the last sequence
    for (int64_t j = (int64_t)max(end, start) + tid; j < a.T; j += TH) a.path[j] = -1;
  if (n == 0) {
    if (tid == 0) {
      a.kept[seq] = 0;
      a.next[seq] = -1;
    }
    return;
  }
  const bool greedy = a.uniforms == nullptr;
  const int V = a.V;
  ProbRow<DT> P, Q;
  double ratio = 0.0, norm = 1.0;  // a and c
  int cur = 0, kept = 1, best = -1;
  auto enter = [&](int node) {
    P.init(a.probs, start + node, V);
    if (a.draft) Q.init(a.draft, start + node, V);
    ratio = 0.0;
    norm = 1.0;
  };
  // certain drafts: the tokens of cur's children that were rejected (past the list's end: looked
  // up among the rows)
  int rejected = 0, last = 0;  // how many with a probability, and the last node of them
  auto gone = [&](int v) {
    const int listed = min(rejected, kDraftGone);
    for (int k = 0; k < listed; ++k)
      if (s_gone[wave][k] == v) return true;
    if (rejected > kDraftGone)
      for (int j = cur + 1; j <= last; ++j)
        if ((a.parents ? a.parents[start + j] : j - 1) == cur && a.tokens[start + j] == v) return true;
    return false;
  };
  // sum over the row of what is left, by each wave over a contiguous part of the blocks
  const int parts = (P.init(a.probs, start, V), (V + 2 * PER - 2) / PER + W - 1) / W;
  auto weights = [&](int block, const U32x4& pw, const U32x4& qw, double (&w)[PER]) {
    float p[PER], q[PER];
    ProbRow<DT>::open(pw, p);
    ProbRow<DT>::open(qw, q);
#pragma unroll
    for (int i = 0; i < PER; ++i) w[i] = ratio > 0.0 ? left_of(prob(p[i]), prob(q[i]), ratio) : prob(p[i]);
    if (!a.draft && rejected > 0) {
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (w[i] > 0.0 && gone(block * PER + i - P.off)) w[i] = 0.0;
    }
  };
  // The sum of that; also leaves the waves' sums in s_sum.  A row of up to G blocks a lane is
  // kept for the node's next rejections: in registers with four waves, partly in scratch memory with sixteen.
  constexpr int G = kDraftBlocks;
  U32x4 pw[G], qw[G];
  bool have_p = false, have_q = false;  // of the node
  auto total = [&]() {
    const int nb = P.blocks(), b1 = min((wave + 1) * parts, nb);
    const bool held = parts <= 64 * G;
    double s = 0.0;
    for (int b0 = wave * parts; b0 < b1; b0 += 64 * G) {
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const int b = b0 + g * 64 + lane;
        if (!held || !have_p) pw[g] = P.raw(b, b < b1);
        if (ratio > 0.0 && (!held || !have_q)) qw[g] = Q.raw(b, b < b1);
      }
      const bool edge = b0 == 0 || b0 + 64 * G >= nb;  // uniform: the row's first or last block is among them
#pragma unroll
      for (int g = 0; g < G; ++g) {
        if (!edge || b0 + g * 64 >= b1) break;
        P.trim(b0 + g * 64 + lane, pw[g]);
        if (ratio > 0.0) Q.trim(b0 + g * 64 + lane, qw[g]);
      }
      // Rows are finite and not negative: seen from the largest of their bits, taken as whole numbers.
      bool fast = DT != kF16 && ratio > 0.0;
      if (fast) {
        uint32_t top = 0;
        typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if constexpr (DT == kF32)
              top = max(top, max(pw[g].v[j], qw[g].v[j]));
            else
              top = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, top),
                                       __builtin_elementwise_max(__builtin_bit_cast(u16x2, pw[g].v[j]), __builtin_bit_cast(u16x2, qw[g].v[j]))));
          }
        fast = !__any(DT == kF32 ? top >= 0x7f800000u : (top >> 16) >= 0x7f80u || (top & 0xffffu) >= 0x7f80u);
      }
      if (fast) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
          if (b0 + g * 64 >= b1) break;  // uniform
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if constexpr (DT == kF32) {
              s += left_of(fast64(pw[g].v[j]), fast64(qw[g].v[j]), ratio);
            } else {
#pragma unroll
              for (int h = 0; h < 2; ++h) s += left_of(fast64_bf16(pw[g].v[j], h), fast64_bf16(qw[g].v[j], h), ratio);
            }
          }
        }
        continue;
      }
#pragma unroll
      for (int g = 0; g < G; ++g) {
        if (b0 + g * 64 >= b1) break;  // uniform
        double w[PER];
        weights(b0 + g * 64 + lane, pw[g], qw[g], w);
#pragma unroll
        for (int i = 0; i < PER; ++i) s += w[i];
      }
    }
    have_p = true;
    have_q = ratio > 0.0;
    s = wave_sum64(s);
    __syncthreads();
    if (lane == 0) s_sum[wave] = s;
    __syncthreads();
    double t = 0.0;
#pragma unroll
    for (int w = 0; w < W; ++w) t += s_sum[w];
    return t;
  };
  auto largest = [&]() {  // the first of the largest; -1 where all are NaN
    const int nb = P.blocks();
    float m = -__builtin_inff();
    int at = INT32_MAX;
    for (int b0 = tid; b0 < nb; b0 += G * TH) {
      U32x4 pw[G];
#pragma unroll
      for (int g = 0; g < G; ++g) pw[g] = P.raw(b0 + g * TH, b0 + g * TH < nb);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const int b = b0 + g * TH, e0 = b * PER - P.off;
        if (b - tid >= nb) break;  // uniform
        float p[PER], t = -__builtin_inff();
        ProbRow<DT>::open(pw[g], p);
        if (e0 < 0 || e0 + PER > V) {
#pragma unroll
          for (int i = 0; i < PER; ++i)
            if ((unsigned)(e0 + i) >= (unsigned)V) p[i] = __builtin_nanf("");
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) t = fmaxf(t, p[i]);
        if (t > m || at == INT32_MAX) {  // seldom: the place of the block's first largest
          int first = INT32_MAX;
#pragma unroll
          for (int i = PER - 1; i >= 0; --i)
            if (p[i] == t) first = e0 + i;
          if (first != INT32_MAX) {
            m = t;
            at = first;
          }
        }
      }
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const float om = __shfl_xor(m, d);
      const int oa = __shfl_xor(at, d);
      if (om > m || (om == m && oa < at)) {
        m = om;
        at = oa;
      }
    }
    __syncthreads();
    if (lane == 0) {
      s_max[wave] = m;
      s_best[wave] = at;
    }
    __syncthreads();
    m = s_max[0];
    at = s_best[0];
#pragma unroll
    for (int w = 1; w < W; ++w)
      if (s_max[w] > m || (s_max[w] == m && s_best[w] < at)) {
        m = s_max[w];
        at = s_best[w];
      }
    return at == INT32_MAX ? -1 : at;
  };

  enter(0);
  if (greedy) best = largest();
  if (tid == 0) a.path[start] = 0;
  for (int c0 = 0; c0 < n; c0 += kDraftNodes) {
    const int m = min(n - c0, kDraftNodes);
    __syncthreads();
    for (int i = tid; i < m; i += TH) {
      const int j = c0 + i, row = start + j;
      int up = a.parents ? a.parents[row] : j - 1;
      if (j == 0 || up < 0 || up >= j) up = -1;
      const int64_t x = a.tokens[row];
      const bool in = up >= 0 && x >= 0 && x < V;
      s_up[i] = up;
      s_tok[i] = in ? (int)x : -1;
      if (!greedy) {
        const int64_t at = (int64_t)(start + max(up, 0)) * V + (in ? x : 0);
        s_p[i] = in ? ld_any(a.probs, at, DT) : 0.f;
        s_q[i] = !a.draft ? 1.f : in ? ld_any(a.draft, at, DT) : 0.f;
        s_u[i] = a.uniforms[row];
      }
    }
    __syncthreads();
    // the children of the node that the walk is at come after it, in order
    for (int i = 0; i < m;) {
      const int look = min(m - i, 64);
      const uint64_t mine = __ballot(lane < look && s_up[i + (lane < look ? lane : 0)] == cur);
      if (mine == 0) {
        i += look;
        continue;
      }
      i += __ffsll((unsigned long long)mine) - 1;
      const int j = c0 + i;
      bool yes;
      if (greedy) {
        yes = s_tok[i] == best && best >= 0;
      } else if (a.draft) {
        const double q = prob(s_q[i]);
        yes = (double)s_u[i] * q * norm < left_of(prob(s_p[i]), q, ratio);
      } else {
        double p = prob(s_p[i]);
        if (rejected > 0 && p > 0.0 && gone(s_tok[i])) p = 0.0;
        yes = (double)s_u[i] * norm < p;
        if (!yes && p > 0.0) {
          norm = fmax(norm - p, 0.0);
          last = j;
          if (rejected < kDraftGone) s_gone[wave][rejected] = s_tok[i];
          ++rejected;
        }
      }
      if (yes) {
        cur = j;
        rejected = 0;
        have_p = have_q = false;
        if (tid == 0) a.path[start + kept] = j;
        ++kept;
        enter(j);
        if (greedy) best = largest();
      } else if (a.draft && !greedy) {
        ratio += norm;
        norm = total();
      }
      ++i;
    }
  }
  for (int j = kept + tid; j < n; j += TH) a.path[start + j] = -1;
  if (greedy) {
    if (tid == 0) {
      a.kept[seq] = kept;
      a.next[seq] = best;
    }
    return;
  }
  double all = ratio > 0.0 ? norm : total();  // the last rejection's sum, and the waves' parts of it
  if (!(all > 0.0)) {  // nothing left: the target itself
    ratio = 0.0;
    rejected = 0;
    all = total();
  }
  const double border = (double)a.uniforms[start] * all;
  // the part that holds the border: the first whose cumulated sum exceeds it, else the last with any
  double before = 0.0, run = 0.0;
  int part = -1;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    if (s_sum[w] > 0.0 && !(part >= 0 && run > border)) {
      part = w;
      before = run;
      run += s_sum[w];
    }
  }
  int token = -1;
  __syncthreads();
  if (part >= 0) {
    // that part's blocks over all threads, neighbouring ones to a thread
    const int nb = P.blocks(), b0 = part * parts, b1 = min(b0 + parts, nb);
    const int each = (b1 - b0 + TH - 1) / TH;
    const int t0 = b0 + tid * each, t1 = min(t0 + each, b1);
    double s = 0.0;
    for (int b = t0; b < t1; ++b) {
      double w[PER];
      U32x4 pw = P.raw(b, true), qw{};
      if (ratio > 0.0) {
        qw = Q.raw(b, true);
        Q.trim(b, qw);
      }
      P.trim(b, pw);
      weights(b, pw, qw, w);
#pragma unroll
      for (int i = 0; i < PER; ++i) s += w[i];
    }
    double inc = s;  // over the lanes up to this one
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const double o = __shfl_up(inc, d);
      if (lane >= d) inc += o;
    }
    if (lane == 63) s_sum[wave] = inc;
    __syncthreads();
    double at = before;
    for (int w = 0; w < wave; ++w) at += s_sum[w];
    double cum = at + inc - s;
    int first = INT32_MAX, most = -1;  // the first past the border, the last with a weight
    for (int b = t0; b < t1; ++b) {
      double w[PER];
      U32x4 pw = P.raw(b, true), qw{};
      if (ratio > 0.0) {
        qw = Q.raw(b, true);
        Q.trim(b, qw);
      }
      P.trim(b, pw);
      weights(b, pw, qw, w);
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        cum += w[i];
        if (w[i] > 0.0) {
          const int v = b * PER + i - P.off;
          most = v;
          if (cum > border && first == INT32_MAX) first = v;
        }
      }
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      first = min(first, __shfl_xor(first, d));
      most = max(most, __shfl_xor(most, d));
    }
    if (lane == 0) {
      s_best[wave] = first;
      s_last[wave] = most;
    }
    __syncthreads();
    first = INT32_MAX;
    for (int w = 0; w < W; ++w) {
      first = min(first, s_best[w]);
      most = max(most, s_last[w]);
    }
    token = first == INT32_MAX ? most : first;
  }
  if (tid == 0) {
    a.kept[seq] = kept;
    a.next[seq] = token;
  }
}

// The keys of the accepted rows, lengths + path[j] to lengths + j, in every plane.  A thread
// takes 16 bytes of a row in one plane and 8 rows at a time: all read before one is written.
// A row is moved to a place before it or its own (path[j] >= j), so a later group of rows is
// read after nothing of it was overwritten.  Latencies in turn: 64 sequences, 8 layers, 2 MB in 6.3 us.
__global__ __launch_bounds__(256) void keep_kernel(KeepArgs a) {
  const int seq = blockIdx.y * a.seqs_line + blockIdx.z;
  if (seq >= a.B) return;
  const int start = seq_start(a.cu, seq, a.T);
  const int n = max(min(max(a.cu[seq + 1], 0), a.T) - start, 0);
  const int64_t cap = (int64_t)a.width << a.page_shift;
  const int64_t past = min(max((int64_t)a.lengths[seq], (int64_t)0), cap);
  const int kept = min(max(a.kept[seq], 0), n);
  if (blockIdx.x == 0 && threadIdx.x == 0) a.new_lengths[seq] = (int)min(past + kept, cap);
  const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (item >= (int64_t)a.planes * a.row16) return;
  char* plane = static_cast<char*>(a.pages_at) + item / a.row16 * a.plane_bytes + item % a.row16 * 16;
  const int* table = a.page_table + (int64_t)seq * a.width;
  auto place = [&](int64_t key) -> int64_t {  // its row in the pages, or -1
    if (key >= cap) return -1;
    const int p = table[key >> a.page_shift];
    return (unsigned)p < (unsigned)a.pages ? ((int64_t)p << a.page_shift) + (key & ((1 << a.page_shift) - 1)) : -1;
  };
  constexpr int G = 8;
  for (int j0 = 0; j0 < kept; j0 += G) {
    U32x4 w[G];
    int64_t to[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      to[g] = -1;
      const int j = j0 + g;
      if (j >= kept) continue;
      const int from = a.path[start + j];
      if (from <= j || from >= n) continue;  // in its place, or no row of the sequence
      const int64_t src = place(past + from), dst = place(past + j);
      if (src < 0 || dst < 0) continue;
      w[g] = ld16(plane + src * a.row_bytes);
      to[g] = dst;
    }
#pragma unroll
    for (int g = 0; g < G; ++g)
      if (to[g] >= 0) *reinterpret_cast<U32x4*>(plane + to[g] * a.row_bytes) = w[g];
  }
}

template <int DT>
hipError_t launch_verify_dt(const VerifyArgs& a, hipStream_t s) {
  // four waves keep a row of up to 2048 blocks (in registers), sixteen one of 8192
  if (a.V > 2048 * ProbRow<DT>::PER - 2 * ProbRow<DT>::PER) verify_kernel<DT, 16><<<dim3((unsigned)a.B), 1024, 0, s>>>(a);
  else verify_kernel<DT, 4><<<dim3((unsigned)a.B), 256, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_verify(const VerifyArgs& a, hipStream_t s) {
  if (a.dtype == kF32) return launch_verify_dt<kF32>(a, s);
  return a.dtype == kBF16 ? launch_verify_dt<kBF16>(a, s) : launch_verify_dt<kF16>(a, s);
}

hipError_t launch_keep(KeepArgs a, hipStream_t s) {
  const int64_t items = (int64_t)a.planes * a.row16, blocks = items > 0 ? (items + 255) / 256 : 1;
  a.seqs_line = a.B < 32768 ? a.B : 32768;
  keep_kernel<<<dim3((unsigned)blocks, (unsigned)((a.B + a.seqs_line - 1) / a.seqs_line), (unsigned)a.seqs_line), 256, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace mhc
