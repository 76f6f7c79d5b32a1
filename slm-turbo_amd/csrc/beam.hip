// The best continuations of a request's beams, over all beams and the vocabulary.  (The
// reference has no beam search.)
//
//   total[w, v] = score_w + x[w, v] - log sum_u e^{x[w, u]},   rank = total / length^penalty,
// the K largest ranks, equal ones by (w, x, v); a beam that has ended offers its score as it is.
//
// Two launches.  rows_kernel takes a part of a row per workgroup: every wave its largest logit
// m, the sum of e^{x - m}, and its best logits, of which the workgroup keeps K in order.  Within
// a beam the order of ranks is that of the logits, so no more of a part can be among a
// request's best.  request_kernel, one workgroup a request, adds up the parts' sums, ranks what
// the parts kept, and writes the K best.
//
// How a wave finds its best without a sort: the K-th largest of its lanes' largest is at most
// its K-th largest element, and little more than K elements reach it.  It is searched bit by
// bit, with ballots, in the upper bits of the values' order; what reaches it is listed, and the
// lists are ordered by counting.  Where too many reach it (equal logits) it is searched among
// all elements, and if still too many tie the best are taken out one after another.
//
// Ranks are in 64 bits, and so are the sums and the exponentials in them (a Taylor sum): which
// of two beams' candidates goes first hangs on their difference, and fp32 sums of a vocabulary
// would leave it to rounding.
#include "slmt_internal.h"

#include <algorithm>
#include <type_traits>

namespace slmt {
namespace beam {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMost = 64;            // beams and candidates of a request
constexpr int kList = 256;           // entries that a wave lists
constexpr float kLargest = 3.4028234663852886e38f;

typedef _Float16 f16;

// Order of fp32 values as unsigned numbers; every number above -infinity is above kNone.
constexpr uint32_t kNone = 0x007FFFFFu;
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}
__device__ __forceinline__ uint64_t order_of(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  return u >> 63 ? ~u : u | (uint64_t(1) << 63);
}

__device__ __forceinline__ int popcount(uint64_t m) { return __builtin_popcountll(m); }
__device__ __forceinline__ int below(uint64_t m) {   // set lanes below this one
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
}

// e^d of d <= 0, to 2^-42: 2^n of the whole part of d log2(e), a Taylor sum of the rest.
__device__ __forceinline__ double exp64(double d) {
  const double y = d * 1.4426950408889634074, n = __builtin_rint(y), f = y - n;
  double s = 7.0549116208011233299e-9;      // ln(2)^k / k!
  s = __builtin_fma(s, f, 1.0178086009239699728e-7);
  s = __builtin_fma(s, f, 1.3215486790144309488e-6);
  s = __builtin_fma(s, f, 1.5252733804059840280e-5);
  s = __builtin_fma(s, f, 1.5403530393381609954e-4);
  s = __builtin_fma(s, f, 1.3333558146428443423e-3);
  s = __builtin_fma(s, f, 9.6181291076284771620e-3);
  s = __builtin_fma(s, f, 5.5504108664821579953e-2);
  s = __builtin_fma(s, f, 2.4022650695910071233e-1);
  s = __builtin_fma(s, f, 6.9314718055994530942e-1);
  s = __builtin_fma(s, f, 1.0);
  return __builtin_ldexp(s, (int)n);
}

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) x += __shfl_xor(x, o, 64);
  return x;
}
__device__ __forceinline__ uint64_t wave_most(uint64_t x) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint64_t y = __shfl_xor(x, o, 64);
    x = y > x ? y : x;
  }
  return x;
}

template <typename T>
__device__ __forceinline__ float to_float(T x) { return (float)x; }
struct bf16 { uint16_t u; };
template <>
__device__ __forceinline__ float to_float<bf16>(bf16 x) { return __builtin_bit_cast(float, (uint32_t)x.u << 16); }

__device__ __forceinline__ bool alive(const BeamParams& p, int row) {
  return p.scores[row] > -INFINITY && !(p.finished && p.finished[row]);
}

// What a part of a row leaves: its largest logit, the sum of e^{x - that}, its K best.
struct Parts {
  int n;                       // parts of a row
  float* top;                  // [rows][n]
  double* sum;                 // [rows][n]
  uint64_t* best;              // [rows][n][K]: order of the value, then ~index; 0: none
};

// E elements a thread, in units of 16 bytes or less.
template <typename T, int E>
__global__ void __launch_bounds__(kThreads) rows_kernel(const BeamParams p, const Parts parts) {
  constexpr int UN = 16 / (int)sizeof(T) < E ? 16 / (int)sizeof(T) : E, U = E / UN;
  __shared__ uint64_t list[kWaves][kList];
  __shared__ int counts[kWaves];
  __shared__ float tops[kWaves];
  __shared__ double sums[kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row = blockIdx.x / parts.n, part = blockIdx.x - row * parts.n;
  if (!alive(p, row)) return;          // (request_kernel reads nothing of it)
  const T* const x0 = reinterpret_cast<const T*>(p.logits) + (int64_t)row * p.row_stride;
  const int shift = (int)((reinterpret_cast<uintptr_t>(x0) / sizeof(T)) % UN);   // units lie at multiples of their size
  const int from = part * (kThreads * E) - shift;

  float x[E];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = from + (u * kThreads + tid) * UN;
    if (i >= 0 && i + UN <= p.V) {
      struct alignas(UN * sizeof(T)) Unit { T t[UN]; };
      const Unit v = *reinterpret_cast<const Unit*>(x0 + i);
#pragma unroll
      for (int e = 0; e < UN; ++e) x[u * UN + e] = to_float(v.t[e]);
    } else {
#pragma unroll
      for (int e = 0; e < UN; ++e) x[u * UN + e] = i + e >= 0 && i + e < p.V ? to_float(x0[i + e]) : -INFINITY;
    }
  }
  float most = -INFINITY;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    x[e] = fminf(fmaxf(x[e], -INFINITY), kLargest) + 0.0f;      // (NaN: -infinity; -0: 0)
    most = fmaxf(most, x[e]);
  }
  const float m = wave_max(most);
  double sum = 0.0;
  if (m > -INFINITY) {
#pragma unroll
    for (int e = 0; e < E; ++e) sum += exp64(fmax((double)x[e] - (double)m, -1400.0));   // (e^-1400 is 0 in 64 bits)
    sum = wave_sum(sum);
  }

  // ---- the wave's best
  auto index_of = [&](int e) { return from + ((e / UN) * kThreads + tid) * UN + e % UN; };
  auto entry = [&](int e) -> uint64_t { return ((uint64_t)order_of(x[e]) << 32) | (uint32_t)~index_of(e); };
  uint32_t key[E];
#pragma unroll
  for (int e = 0; e < E; ++e) key[e] = order_of(x[e]);
  uint32_t least = 0;                                    // of the upper 16 bits of the order
  const uint32_t mine = order_of(most) >> 16;
#pragma unroll
  for (int b = 15; b >= 0; --b) {
    const uint32_t t = least | (1u << b);
    if (popcount(__builtin_amdgcn_ballot_w64(mine >= t)) >= p.K) least = t;
  }
  auto reach = [&](int e, uint32_t t) { return key[e] > kNone && (key[e] >> 16) >= t; };
  auto count = [&](uint32_t t) {
    int n = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) n += popcount(__builtin_amdgcn_ballot_w64(reach(e, t)));
    return n;
  };
  int n = count(least);
  if (n > 2 * p.K + 16) {              // many above it: the K-th largest of all elements
    least = 0;
    for (int b = 15; b >= 0; --b) {
      const uint32_t t = least | (1u << b);
      if (count(t) >= p.K) least = t;
    }
    n = count(least);
  }
  if (n <= kList) {
    int at = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const bool in = reach(e, least);
      const uint64_t who = __builtin_amdgcn_ballot_w64(in);
      if (who) {
        if (in) list[wave][at + below(who)] = entry(e);
        at += popcount(who);
      }
    }
  } else {                             // ties: one after another
    uint64_t last = ~uint64_t(0);
    n = 0;
    for (; n < p.K; ++n) {
      uint64_t best = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const uint64_t c = key[e] > kNone ? entry(e) : 0;
        if (c < last && c > best) best = c;
      }
      best = wave_most(best);
      if (best == 0) break;
      if (lane == 0) list[wave][n] = best;
      last = best;
    }
  }
  if (lane == 0) {
    counts[wave] = n;
    tops[wave] = m;
    sums[wave] = sum;
  }
  __syncthreads();
  const int64_t out = (int64_t)row * parts.n + part;
  if (tid == 0) {
    float top = -INFINITY;
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, tops[w]);
    double s = 0.0;
    for (int w = 0; w < kWaves; ++w)
      if (tops[w] > -INFINITY) s += sums[w] * exp64(fmax((double)tops[w] - (double)top, -1400.0));
    parts.top[out] = top;
    parts.sum[out] = s;
  }
  // ---- the workgroup's K best, in order: a candidate's place is the number of those before it
  int all = 0;
  for (int w = 0; w < kWaves; ++w) all += counts[w];
  uint64_t* const best = parts.best + out * p.K;
  for (int i = tid; i < all; i += kThreads) {
    int w = 0, k = i;
    while (k >= counts[w]) k -= counts[w++];
    const uint64_t c = list[w][k];
    int rank = 0;
    for (int v = 0; v < kWaves; ++v)
      for (int j = 0; j < counts[v]; ++j) rank += list[v][j] > c;
    if (rank < p.K) best[rank] = c;
  }
  for (int i = all + tid; i < p.K; i += kThreads) best[i] = 0;
}

struct Candidate {
  uint64_t rank;               // order of the rank; 0: none
  uint32_t flat;               // beam * V + token
  float x;                     // its logit
};
// (Equal ranks of a beam are equal logits, or ones that far below the largest lose their difference.)
__device__ __forceinline__ bool before(const Candidate& a, const Candidate& b, int V) {
  if (a.rank != b.rank) return a.rank > b.rank;
  return a.x != b.x && a.flat / (uint32_t)V == b.flat / (uint32_t)V ? a.x > b.x : a.flat < b.flat;
}

// One workgroup a request.
template <int THREADS>
__global__ void __launch_bounds__(THREADS) request_kernel(const BeamParams p, const Parts parts) {
  constexpr int WAVES = THREADS / 64;
  __shared__ Candidate list[WAVES][kList / 2];
  __shared__ int counts[WAVES];
  __shared__ double offs[kMost], tops[kMost], divs[kMost];
  __shared__ int states[kMost];        // 0: no candidates, 1: its logits, 2: ended
  __shared__ Candidate best[kMost];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = blockIdx.x;
  constexpr int kCap = kList / 2;

  // ---- the beams' sums
  for (int w = wave; w < p.W; w += WAVES) {
    const int row = r * p.W + w;
    const bool ended = p.finished && p.finished[row];
    const float score = p.scores[row];
    int state = 0;
    double top = 0.0, off = (double)score;
    if (score > -INFINITY && ended) state = 2;
    else if (score > -INFINITY) {
      const float* const tp = parts.top + (int64_t)row * parts.n;
      const double* const sp = parts.sum + (int64_t)row * parts.n;
      float t = -INFINITY;
      for (int i = lane; i < parts.n; i += 64) t = fmaxf(t, tp[i]);
      t = wave_max(t);
      double sum = 0.0;
      if (t > -INFINITY) {
        for (int i = lane; i < parts.n; i += 64) sum += sp[i] * exp64(fmax((double)tp[i] - (double)t, -1400.0));
        sum = wave_sum(sum);
        state = 1;
        top = (double)t;
        off -= log(sum);
      }
    }
    if (lane == 0) {
      states[w] = state;
      tops[w] = top;
      offs[w] = off;
      const int len = p.lengths ? p.lengths[row] + (ended ? 0 : 1) : 1;
      divs[w] = p.penalty == 0.0 ? 1.0 : pow((double)max(len, 1), p.penalty);
    }
  }
  if (tid < kMost) best[tid] = Candidate{0, 0, 0.f};
  __syncthreads();

  // ---- candidates
  const int each = parts.n * p.K, all = p.W * each;
  auto total_of = [&](int w, float x) { return states[w] == 2 ? offs[w] : ((double)x - tops[w]) + offs[w]; };
  auto candidate = [&](int i) -> Candidate {
    const int w = i / each, k = i - w * each;
    Candidate c{0, 0, 0.f};
    if (states[w] == 0 || (states[w] == 2 && k > 0)) return c;
    if (states[w] == 1) {
      const uint64_t e = parts.best[(int64_t)(r * p.W + w) * each + k];
      if (e == 0) return c;
      c.x = value_of((uint32_t)(e >> 32));
      c.flat = (uint32_t)w * (uint32_t)p.V + ~(uint32_t)e;
    } else {
      c.flat = (uint32_t)w * (uint32_t)p.V + (uint32_t)p.pad;
    }
    const double rank = total_of(w, c.x) / divs[w] + 0.0;
    if (rank > -INFINITY) c.rank = order_of(rank);
    return c;
  };
  uint64_t mine = 0;
  for (int i = tid; i < all; i += THREADS) {
    const uint64_t k = candidate(i).rank;
    mine = k > mine ? k : mine;
  }
  uint32_t least = 0;                                    // of the upper 20 bits of the order
  for (int b = 19; b >= 0; --b) {
    const uint32_t t = least | (1u << b);
    if (popcount(__builtin_amdgcn_ballot_w64((uint32_t)(mine >> 44) >= t)) >= p.K) least = t;
  }
  int n = 0;
  bool full = false;
  for (int i0 = wave * 64; i0 < all; i0 += THREADS) {
    const Candidate c = i0 + lane < all ? candidate(i0 + lane) : Candidate{0, 0, 0.f};
    const bool in = c.rank != 0 && (uint32_t)(c.rank >> 44) >= least;
    const uint64_t who = __builtin_amdgcn_ballot_w64(in);
    if (n + popcount(who) > kCap) {
      full = true;
      break;
    }
    if (in) list[wave][n + below(who)] = c;
    n += popcount(who);
  }
  if (full) {                          // one after another
    Candidate last{~uint64_t(0), 0, 0.f};
    bool any = false;
    for (n = 0; n < p.K; ++n) {
      Candidate b{0, 0xFFFFFFFFu, 0.f};
      for (int i0 = wave * 64; i0 < all; i0 += THREADS) {
        const Candidate c = i0 + lane < all ? candidate(i0 + lane) : Candidate{0, 0, 0.f};
        if (c.rank != 0 && (!any || before(last, c, p.V)) && before(c, b, p.V)) b = c;
      }
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const Candidate c{(uint64_t)__shfl_xor(b.rank, o, 64), (uint32_t)__shfl_xor((int)b.flat, o, 64), __shfl_xor(b.x, o, 64)};
        if (before(c, b, p.V)) b = c;
      }
      if (b.rank == 0) break;
      if (lane == 0) list[wave][n] = b;
      last = b;
      any = true;
    }
  }
  if (lane == 0) counts[wave] = n;
  __syncthreads();
  int listed = 0;
  for (int w = 0; w < WAVES; ++w) listed += counts[w];
  for (int i = tid; i < listed; i += THREADS) {
    int w = 0, k = i;
    while (k >= counts[w]) k -= counts[w++];
    const Candidate c = list[w][k];
    int rank = 0;
    for (int v = 0; v < WAVES; ++v)
      for (int j = 0; j < counts[v]; ++j) rank += before(list[v][j], c, p.V);
    if (rank < p.K) best[rank] = c;
  }
  __syncthreads();
  if (wave != 0) return;

  // ---- the K best, a lane each
  const Candidate c = best[lane];
  const bool have = c.rank != 0;
  const int parent = have ? (int)(c.flat / (uint32_t)p.V) : 0;
  const int64_t token = have ? (int64_t)(c.flat - (uint32_t)parent * (uint32_t)p.V) : 0;
  const float score = have ? (float)total_of(parent, c.x) : -INFINITY;
  int at = lane;
  if (p.keep_rows) {                   // a beam's best child takes its row, the others the rows left, in order
    bool again = false;
    uint64_t taken = 0;
    for (int j = 0; j < p.K; ++j) {
      const int other = __builtin_amdgcn_readlane(parent, j);
      if (j < lane && other == parent) again = true;
      taken |= uint64_t(1) << other;
    }
    const uint64_t rest = __builtin_amdgcn_ballot_w64(again && lane < p.K);
    int skip = below(rest);
    if (again) {
      for (int row = 0; row < p.W; ++row) {
        if (taken >> row & 1) continue;
        if (skip-- == 0) {
          at = row;
          break;
        }
      }
    } else {
      at = parent;
    }
  }
  if (lane >= p.K) return;
  const int row = r * p.W + parent;
  const int64_t to = (int64_t)r * p.K + at;
  const bool ended = p.finished && p.finished[row];
  p.tokens[to] = token;
  p.parents[to] = parent;
  p.out_scores[to] = score;
  if (p.out_finished) p.out_finished[to] = ended || token == p.eos;
  if (p.out_lengths) p.out_lengths[to] = p.lengths[row] + (ended ? 0 : 1);
}

// Elements a thread: 16, or 4 where that leaves the chip empty.
int elements(int rows, int V) { return (int64_t)rows * V > (int64_t)256 * kThreads * 16 ? 16 : 4; }
int parts_of(int rows, int V) {
  const int part = kThreads * elements(rows, V);
  return (V + 7 + part - 1) / part;      // (a row may start up to 7 elements into a unit)
}

template <typename T>
int launch(const BeamParams& p, const Parts& parts, hipStream_t stream) {
  const int rows = p.R * p.W;
  const int64_t grid = (int64_t)rows * parts.n;
  if (int rc = check_grid("beam select", grid, kThreads)) return rc;
  if (elements(rows, p.V) == 16) hipLaunchKernelGGL((rows_kernel<T, 16>), dim3((unsigned)grid), dim3(kThreads), 0, stream, p, parts);
  else hipLaunchKernelGGL((rows_kernel<T, 4>), dim3((unsigned)grid), dim3(kThreads), 0, stream, p, parts);
  if (int rc = check_launch("beam select")) return rc;
  if ((int64_t)p.W * parts.n * p.K <= 4096) hipLaunchKernelGGL((request_kernel<256>), dim3(p.R), dim3(256), 0, stream, p, parts);
  else hipLaunchKernelGGL((request_kernel<1024>), dim3(p.R), dim3(1024), 0, stream, p, parts);
  return check_launch("beam select");
}

}  // namespace beam

// Sums first, then the lists, then the largest logits.
int64_t beam_workspace_bytes(int R, int W, int V, int K) {
  const int64_t n = (int64_t)R * W * beam::parts_of(R * W, V);
  return n * (8 + 8 * (int64_t)K + 4);
}

int launch_beam(int dtype, const BeamParams& p, void* workspace, hipStream_t stream) {
  const int n = beam::parts_of(p.R * p.W, p.V);
  const int64_t all = (int64_t)p.R * p.W * n;
  double* const sum = reinterpret_cast<double*>(workspace);
  uint64_t* const best = reinterpret_cast<uint64_t*>(sum + all);
  const beam::Parts parts{n, reinterpret_cast<float*>(best + all * p.K), sum, best};
  if (dtype == SLMT_F32) return beam::launch<float>(p, parts, stream);
  if (dtype == SLMT_F16) return beam::launch<beam::f16>(p, parts, stream);
  return beam::launch<beam::bf16>(p, parts, stream);
}

}  // namespace slmt
