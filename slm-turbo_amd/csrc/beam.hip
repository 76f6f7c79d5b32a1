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
// Ranks, sums and the exponentials in them are held in 64 bits: which of two beams' candidates
// goes first hangs on their difference, and fp32 sums of a vocabulary would leave it to rounding.
// The exponentials are a polynomial's, right to 5e-11 of each (34 bits), and so is a row's sum.
// Equal rows have equal sums: the order of operations goes by the elements' indices alone.
//
// What bounds it: 128 rows of 151936 bf16 logits, 28.8 us a call (7.5 by bytes at the rate of a
// large copy): rows_kernel 22, by instructions, 14 of an element's some 20 in 64 bits (vector
// units 41 % busy over the launch); request_kernel 9.0, a chain of loads, logarithms and
// barriers in 16 workgroups.  4 rows of 32000: 14.3, the host's (4.4 + 5.5 in the kernels).
#include "slmt_internal.h"

#include <algorithm>
#include <type_traits>

namespace slmt {
namespace beam {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kRequestThreads = 1024;   // of a request's workgroup
static_assert(kWaves == 4, "a candidate's threads are a quad");
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

// 2^y of -2^31 < y <= 0, to 5e-11: the power of y's whole part, and of the rest a polynomial (the coefficients of the least relative
// error over -1/2 .. 1/2 with a constant of 1).
// (The constants stay in scalar registers: left alone, each is copied to two vector registers, to be added to in place.)
struct Power2 {
  static constexpr double kWhole = 0x1.8p52;
  double c7 = 0x1.fde5fdb37b06cp-17, c6 = 0x1.445c84056ad21p-13, c5 = 0x1.5d8a85fef3d02p-10, c4 = 0x1.3b29f39d4ae1ep-7,
         c3 = 0x1.c6b08ac06baddp-5, c2 = 0x1.ebfbe0778728fp-3, c1 = 0x1.62e42ff0e191cp-1;
  __device__ __forceinline__ Power2() {
    asm("" : "+s"(c7));
    asm("" : "+s"(c6));
    asm("" : "+s"(c5));
    asm("" : "+s"(c4));
    asm("" : "+s"(c3));
    asm("" : "+s"(c2));
    asm("" : "+s"(c1));
  }
  __device__ __forceinline__ double operator()(double y) const {
    const double n = y + kWhole, f = y - (n - kWhole);       // the nearest whole number, in the low dword too
    double s = __builtin_fma(f, c7, c6);
    s = __builtin_fma(s, f, c5);
    s = __builtin_fma(s, f, c4);
    s = __builtin_fma(s, f, c3);
    s = __builtin_fma(s, f, c2);
    s = __builtin_fma(s, f, c1);
    s = __builtin_fma(s, f, 1.0);
    return __builtin_ldexp(s, (int)(uint32_t)__builtin_bit_cast(uint64_t, n));
  }
};
constexpr double kLog2e = 1.4426950408889634074;

// Sums over the wave's lanes, without LDS.
template <int CTRL>
__device__ __forceinline__ double dpp_d(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  return __builtin_bit_cast(double, ((uint64_t)dpp_u<CTRL>((uint32_t)(u >> 32)) << 32) | dpp_u<CTRL>((uint32_t)u));
}
__device__ __forceinline__ double wave_sum(double x) {
  x += dpp_d<DPP_QUAD_XOR1>(x);
  x += dpp_d<DPP_QUAD_XOR2>(x);
  x += dpp_d<DPP_ROW_ROR4>(x);
  x += dpp_d<DPP_ROW_ROR8>(x);
  const uint64_t u = __builtin_bit_cast(uint64_t, x);      // (the same in all lanes of a row of 16)
  double y = 0.0;
#pragma unroll
  for (int r = 0; r < 4; ++r)
    y += __builtin_bit_cast(double, ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(u >> 32), 16 * r) << 32) |
                                        (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, 16 * r));
  return y;
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
  uint32_t each_inverse;       // 2^32 / (n K), rounded up
  float* top;                  // [rows][n]
  double* sum;                 // [rows][n]
  uint64_t* best;              // [rows][n][K]: order of the value, then ~index; 0: none
};

// E elements a thread, in units of 16 bytes or less.  Parts, waves and units go by an element's index and not by its address, so
// that equal rows have equal sums, to the last bit, wherever they lie: the loads of a row that is not a multiple of 16 bytes away
// are unaligned ones.  (128 rows of 151936 / 151935 bf16 28.4 / 28.9 us a call; by units at multiples of 16 bytes 28.5 / 29.2.)
template <typename T, int E>
__global__ void __launch_bounds__(kThreads) rows_kernel(const BeamParams p, const Parts parts) {
  constexpr int UN = 16 / (int)sizeof(T) < E ? 16 / (int)sizeof(T) : E, U = E / UN;
  __shared__ uint64_t list[kWaves][kList + 1];   // (read at one place of all four at a time: of different banks)
  __shared__ int counts[kWaves];
  __shared__ float tops[kWaves];
  __shared__ double sums[kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row = blockIdx.x / parts.n, part = blockIdx.x - row * parts.n;
  const bool live = alive(p, row);
  const T* const x0 = reinterpret_cast<const T*>(p.logits) + (int64_t)row * p.row_stride;
  const int from = part * (kThreads * E);

  float x[E];
  struct Unit { T t[UN]; };
  if (from + kThreads * E <= p.V) {    // all loads are under way before the first is waited for
    Unit v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) __builtin_memcpy(&v[u], x0 + from + (u * kThreads + tid) * UN, sizeof(Unit));
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = to_float(v[e / UN].t[e % UN]);
  } else {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = from + (u * kThreads + tid) * UN;
      if (i + UN <= p.V) {
        Unit v;
        __builtin_memcpy(&v, x0 + i, sizeof(Unit));
#pragma unroll
        for (int e = 0; e < UN; ++e) x[u * UN + e] = to_float(v.t[e]);
      } else {
#pragma unroll
        for (int e = 0; e < UN; ++e) x[u * UN + e] = i + e < p.V ? to_float(x0[i + e]) : -INFINITY;
      }
    }
  }
  if (!live) return;                   // (request_kernel reads nothing of it; asked before the loads it would hold them up)
  const Power2 pow2;
  float most = -INFINITY;
#pragma unroll
  for (int e = 0; e < E; ++e) most = fmaxf(most, x[e]);  // (a NaN never is the larger)
  float m = wave_max(most);
  double sum = 0.0;
  if (__builtin_fabsf(m) < 1048576.0f) {
    const double scale = kLog2e, from = -(double)m * kLog2e;
    const float least = m - 1000.0f;   // (-infinity and NaN too: 0)
#pragma unroll
    for (int e = 0; e < E; ++e) sum += pow2(__builtin_fma((double)fmaxf(x[e], least), scale, from));
    sum = wave_sum(sum);
  } else if (m > -INFINITY) {          // infinities, masks of a type's lowest number
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (x[e] > kLargest) x[e] = kLargest;
      if (x[e] > -INFINITY) sum += pow2(fmax(((double)x[e] - (double)fminf(m, kLargest)) * kLog2e, -2000.0));
    }
    m = fminf(m, kLargest);
    most = fminf(most, kLargest);
    sum = wave_sum(sum);
  }

  // ---- the wave's best: what reaches the value that has `t` as the upper 16 bits of its order
  auto index_of = [&](int e) { return from + ((e / UN) * kThreads + tid) * UN + e % UN; };
  auto entry = [&](int e) -> uint64_t { return ((uint64_t)order_of(x[e] + 0.0f) << 32) | (uint32_t)~index_of(e); };   // (-0: 0)
  auto value = [&](uint32_t t) { return t <= (kNone >> 16) ? -kLargest : value_of(t << 16); };
  uint32_t least = 0;
  const uint32_t mine = order_of(most) >> 16;
#pragma unroll
  for (int b = 15; b >= 0; --b) {
    const uint32_t t = least | (1u << b);
    if (popcount(__builtin_amdgcn_ballot_w64(mine >= t)) >= p.K) least = t;
  }
  auto write = [&](float from) {       // what reaches it, as far as the list holds
    int at = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const bool in = x[e] >= from;
      const uint64_t who = __builtin_amdgcn_ballot_w64(in);
      if (who) {
        const int to = at + below(who);
        if (in && to < kList) list[wave][to] = entry(e);
        at += popcount(who);
      }
    }
    return at;
  };
  int n = write(value(least));
  if (n > 2 * p.K + 32) {              // many above it: the K-th largest of all elements
    least = 0;
#pragma unroll 1
    for (int b = 15; b >= 0; --b) {
      const float from = value(least | (1u << b));
      int reach = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) reach += popcount(__builtin_amdgcn_ballot_w64(x[e] >= from));
      if (reach >= p.K) least |= 1u << b;
    }
    n = write(value(least));
  }
  if (n > kList) {                     // ties: one after another
    uint64_t last = ~uint64_t(0);
#pragma unroll 1
    for (n = 0; n < p.K; ++n) {
      uint64_t best = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const uint64_t c = x[e] > -INFINITY ? entry(e) : 0;
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
      if (tops[w] > -INFINITY) s += sums[w] * pow2(fmax(((double)tops[w] - (double)top) * kLog2e, -2000.0));
    parts.top[out] = top;
    parts.sum[out] = s;
  }
  // ---- the workgroup's K best, in order: a candidate's place is the number of those before it
  int all = 0;
  for (int w = 0; w < kWaves; ++w) all += counts[w];
  uint64_t* const best = parts.best + out * p.K;
  // (four threads a candidate, each with one wave's list)
  for (int i = tid / kWaves; i < all; i += kThreads / kWaves) {
    int w = 0, k = i;
    while (k >= counts[w]) k -= counts[w++];
    const uint64_t c = list[w][k];
    const uint64_t* const other = list[tid % kWaves];
    const int m = counts[tid % kWaves];
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < m; ++j) rank += other[j] > c;
    rank += (int)dpp_u<DPP_QUAD_XOR1>((uint32_t)rank);
    rank += (int)dpp_u<DPP_QUAD_XOR2>((uint32_t)rank);
    if (rank < p.K && tid % kWaves == 0) best[rank] = c;
  }
  for (int i = all + tid; i < p.K; i += kThreads) best[i] = 0;
}

constexpr int kTokenBits = 22;       // vocabularies go up to 2^22, beams to 2^6
struct Candidate {
  uint64_t rank;               // order of the rank; 0: none
  uint32_t flat;               // beam and token (kTokenBits)
  float x;                     // its logit
};
// (Equal ranks of a beam are equal logits, or ones that far below the largest lose their difference.)
__device__ __forceinline__ bool before(const Candidate& a, const Candidate& b) {
  if (a.rank != b.rank) return a.rank > b.rank;
  return a.x != b.x && a.flat >> kTokenBits == b.flat >> kTokenBits ? a.x > b.x : a.flat < b.flat;
}

// One workgroup a request.  C: candidates a thread, in registers; 0: any number, read again at each use.
template <int C>
__global__ void __launch_bounds__(kRequestThreads) request_kernel(const BeamParams p, const Parts parts) {
  constexpr int THREADS = kRequestThreads, WAVES = THREADS / 64;
  constexpr int kCap = 2048;           // that are listed
  constexpr int kWide = 16;
  static_assert(WAVES * kMost <= kCap, "every wave's best, where more tie");
  __shared__ Candidate list[kCap], best[kMost], near[64];
  __shared__ int listed, many, tally[30];
  __shared__ double offs[kMost], tops[kMost], divs[kMost];
  __shared__ int states[kMost];        // 0: no candidates, 1: its logits, 2: ended
  __shared__ int lens[kMost], ends[kMost];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = blockIdx.x;
  const int each = parts.n * p.K, all = p.W * each;
  const uint64_t* const entries = parts.best + (int64_t)r * all;
  uint64_t held[C ? C : 1];
  const Power2 pow2;
#pragma unroll
  for (int c = 0; c < C; ++c) held[c] = c * THREADS + tid < all ? entries[c * THREADS + tid] : 0;

  // ---- the beams' sums
  for (int w = wave; w < p.W; w += WAVES) {
    const int row = r * p.W + w;
    // (all loads at once; of a beam without candidates the parts are whatever the workspace held)
    const float* const tp = parts.top + (int64_t)row * parts.n;
    const double* const sp = parts.sum + (int64_t)row * parts.n;
    const float t0 = lane < parts.n ? tp[lane] : -INFINITY;
    const double s0 = lane < parts.n ? sp[lane] : 0.0;
    const bool ended = p.finished && p.finished[row];
    const float score = p.scores[row];
    const int grown = p.lengths ? p.lengths[row] + (ended ? 0 : 1) : 1;
    int state = 0;
    double top = 0.0, off = (double)score;
    if (score > -INFINITY && ended) state = 2;
    else if (score > -INFINITY) {
      float t = t0;
      for (int i = lane + 64; i < parts.n; i += 64) t = fmaxf(t, tp[i]);
      t = wave_max(t);
      if (t > -INFINITY) {
        double sum = lane < parts.n ? s0 * pow2(fmax(((double)t0 - (double)t) * kLog2e, -2000.0)) : 0.0;
        for (int i = lane + 64; i < parts.n; i += 64) sum += sp[i] * pow2(fmax(((double)tp[i] - (double)t) * kLog2e, -2000.0));
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
      ends[w] = ended;
      lens[w] = grown;
      divs[w] = p.penalty == 0.0 ? 1.0 : p.penalty == 1.0 ? (double)max(grown, 1) : exp2(p.penalty * log2((double)max(grown, 1)));
    }
  }
  if (tid == 0) listed = many = 0;
  if (tid < 30) tally[tid] = 0;
  if (tid < kMost) best[tid] = Candidate{0, 0, 0.f};
  __syncthreads();

  // ---- candidates
  auto total_of = [&](int w, float x) { return states[w] == 2 ? offs[w] : ((double)x - tops[w]) + offs[w]; };
  auto rated = [&](int i, uint64_t e) -> Candidate {
    int w = (int)__umulhi((uint32_t)i, parts.each_inverse);
    w -= w * each > i;
    w += (w + 1) * each <= i;          // (each = 1)
    const int k = i - w * each;
    Candidate c{0, 0, 0.f};
    const int state = states[w];
    if (state == 0 || (state == 2 && k > 0) || (state == 1 && e == 0)) return c;
    c.flat = ((uint32_t)w << kTokenBits) | (state == 1 ? ~(uint32_t)e : (uint32_t)p.pad);
    c.x = state == 1 ? value_of((uint32_t)(e >> 32)) : 0.f;
    double rank = total_of(w, c.x);
    if (p.penalty != 0.0) rank /= divs[w];
    if (rank > -INFINITY) c.rank = order_of(rank + 0.0);
    return c;
  };
  auto candidate = [&](int i) { return i < all ? rated(i, entries[i]) : Candidate{0, 0, 0.f}; };
  // the lane's one of the 64 from i0 on: turned by one each time, or a lane had the same place of every ordered list
  auto turned = [&](int i0) { return candidate(i0 + ((lane + i0 / THREADS) & 63)); };
  Candidate own[C ? C : 1];
  uint64_t mine = 0;
  if constexpr (C > 0) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      own[c] = c * THREADS + tid < all ? rated(c * THREADS + tid, held[c]) : Candidate{0, 0, 0.f};
      mine = own[c].rank > mine ? own[c].rank : mine;
    }
  } else {
    for (int i0 = wave * 64; i0 < all; i0 += THREADS) {
      const uint64_t k = turned(i0).rank;
      mine = k > mine ? k : mine;
    }
  }
  // the K-th largest of the lanes' largest, by the upper 20 bits of the ranks' order
  auto threshold = [&](uint64_t largest) {
    uint32_t t = 0;
    for (int b = 19; b >= 0; --b)
      if (popcount(__builtin_amdgcn_ballot_w64((uint32_t)(largest >> 44) >= (t | (1u << b)))) >= p.K) t |= 1u << b;
    return t;
  };
  // The same over the workgroup, two bits at a time.  For many: of 64 lanes' largest the last ones are far below the K-th of
  // all.  A row of 151936, us a call by waves and so: its best 64 580 and 61, its best 32 29.7 and 23.6, its best 16 13.5 and 15.7.
  auto common_threshold = [&](uint64_t largest) {
    uint32_t t = 0;
    for (int b = 18; b >= 0; b -= 2) {
      const uint32_t x = (uint32_t)(largest >> 44);
      int n[3];
#pragma unroll
      for (int i = 0; i < 3; ++i) n[i] = popcount(__builtin_amdgcn_ballot_w64(x >= (t | ((uint32_t)(i + 1) << b))));
      int* const total = tally + 3 * (b >> 1);
      if (lane < 3) atomicAdd(total + lane, lane == 0 ? n[0] : lane == 1 ? n[1] : n[2]);
      __syncthreads();
      t |= (uint32_t)(total[2] >= p.K ? 3 : total[1] >= p.K ? 2 : total[0] >= p.K ? 1 : 0) << b;
    }
    return t;
  };
  const bool wide = p.K > kWide;
  uint32_t least = wide ? common_threshold(mine) : threshold(mine);
  auto reaches = [&](const Candidate& c) { return c.rank != 0 && (uint32_t)(c.rank >> 44) >= least; };
  // a wave's entries stand together in the list, the waves' in any order
  auto reserve = [&](int n) {
    int from = 0;
    if (lane == 0) from = atomicAdd(&listed, n);
    return __builtin_amdgcn_readfirstlane(from);
  };
  int n = 0;
  if constexpr (C > 0) {
#pragma unroll
    for (int c = 0; c < C; ++c) n += popcount(__builtin_amdgcn_ballot_w64(reaches(own[c])));
    int at = reserve(n);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const bool in = reaches(own[c]);
      const uint64_t who = __builtin_amdgcn_ballot_w64(in);
      const int to = at + below(who);
      if (in && to < kCap) list[to] = own[c];
      at += popcount(who);
    }
  } else {
#pragma unroll 1
    for (int i0 = wave * 64; i0 < all; i0 += THREADS) {
      const Candidate c = turned(i0);
      const bool in = reaches(c);
      const uint64_t who = __builtin_amdgcn_ballot_w64(in);
      if (who) {
        const int to = reserve(popcount(who)) + below(who);
        if (in && to < kCap) list[to] = c;
      }
    }
  }
  __syncthreads();
  if (listed > kCap) {                 // ties: every wave's best, one after another
    __syncthreads();
    if (tid == 0) listed = 0;
    __syncthreads();
    Candidate last{~uint64_t(0), 0, 0.f};
    bool any = false;
#pragma unroll 1
    for (n = 0; n < p.K; ++n) {
      Candidate b{0, 0xFFFFFFFFu, 0.f};
#pragma unroll 1
      for (int i0 = wave * 64; i0 < all; i0 += THREADS) {
        const Candidate c = candidate(i0 + lane);
        if (c.rank != 0 && (!any || before(last, c)) && before(c, b)) b = c;
      }
#pragma unroll 1
      for (int o = 1; o < 64; o <<= 1) {
        const Candidate c{(uint64_t)__shfl_xor(b.rank, o, 64), (uint32_t)__shfl_xor((int)b.flat, o, 64), __shfl_xor(b.x, o, 64)};
        if (before(c, b)) b = c;
      }
      if (b.rank == 0) break;
      const int at = reserve(1);
      if (lane == 0) list[at] = b;
      last = b;
      any = true;
    }
    __syncthreads();
  }
  // ---- what the waves listed, once more: one wave finds the K-th among it, and orders what reaches that
  const int count = listed;
  if (wave == 0 && !wide) {
    mine = 0;
#pragma unroll 1
    for (int i = lane; i < count; i += 64) mine = list[i].rank > mine ? list[i].rank : mine;
    least = threshold(mine);
    int m = 0;
#pragma unroll 1
    for (int i0 = 0; i0 < count; i0 += 64) {
      const Candidate c = i0 + lane < count ? list[i0 + lane] : Candidate{0, 0, 0.f};
      const bool in = reaches(c);
      const uint64_t who = __builtin_amdgcn_ballot_w64(in);
      const int to = m + below(who);
      if (in && to < 64) near[to] = c;
      m += popcount(who);
    }
    if (m <= 64) {
      __builtin_amdgcn_wave_barrier();
      const Candidate c = lane < m ? near[lane] : Candidate{0, 0, 0.f};
      int rank = 0, equal = 0;
#pragma unroll 1
      for (int j = 0; j < m; ++j) {
        const uint64_t other = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(c.rank >> 32), j) << 32) |
                               (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)c.rank, j);
        rank += other > c.rank;
        equal += other == c.rank;
      }
      if (__builtin_amdgcn_ballot_w64(lane < m && equal > 1)) {
        rank = 0;
#pragma unroll 1
        for (int j = 0; j < m; ++j) rank += before(near[j], c);
      }
      if (lane < m && rank < p.K) best[rank] = c;
      __builtin_amdgcn_wave_barrier();
    } else if (lane == 0) {
      many = 1;
    }
  }
  __syncthreads();
  if (wide || many) {                  // (more than a lane each: every one's place by counting)
#pragma unroll 1
    for (int i = tid; i < count; i += THREADS) {
      const Candidate c = list[i];
      int rank = 0;
#pragma unroll 4
      for (int j = 0; j < count; ++j) rank += before(list[j], c);
      if (rank < p.K) best[rank] = c;
    }
    __syncthreads();
  }
  if (wave != 0) return;

  // ---- the K best, a lane each
  const Candidate c = best[lane];
  const bool have = c.rank != 0;
  const int parent = have ? (int)(c.flat >> kTokenBits) : 0;
  const int64_t token = have ? (int64_t)(c.flat & ((1u << kTokenBits) - 1)) : 0;
  const float score = have ? (float)total_of(parent, c.x) : -INFINITY;
  int at = lane;
  if (p.keep_rows) {                   // a beam's best child takes its row, the others the rows left, in order
    bool again = false;
    uint64_t taken = 0;
#pragma unroll 1
    for (int j = 0; j < p.K; ++j) {
      const int other = __builtin_amdgcn_readlane(parent, j);
      if (j < lane && other == parent) again = true;
      taken |= uint64_t(1) << other;
    }
    const uint64_t rest = __builtin_amdgcn_ballot_w64(again && lane < p.K);
    uint64_t left = ~taken;
    for (int skip = again ? below(rest) : 0; skip > 0; --skip) left &= left - 1;
    at = again ? (int)__builtin_ctzll(left | (uint64_t(1) << 63)) : parent;
  }
  if (lane >= p.K) return;
  const int64_t to = (int64_t)r * p.K + at;
  const bool ended = ends[parent];
  p.tokens[to] = token;
  p.parents[to] = parent;
  p.out_scores[to] = score;
  if (p.out_finished) p.out_finished[to] = ended || token == p.eos;
  if (p.out_lengths) p.out_lengths[to] = lens[parent];
}

// Elements a thread: many, for less of what each wave does once; fewer where that leaves the chip empty.  With 4 / 16 / 32,
// us: 128 rows of 151936 64.2 / 32.0 / 31.0 a call; 4 rows of 32000 4.4 / 5.2 / 6.2 in rows_kernel and 6.3 / 6.0 / 6.0 in
// request_kernel; 40 rows of 50001, of which 8 have a score, 6.5 / 6.5 / 7.2 and 8.2 / 7.4 / 7.4.
int elements(int rows, int V) {
  const int64_t n = (int64_t)rows * V / kThreads;
  return n > 512 * 32 ? 32 : n > 256 * 16 ? 16 : 4;
}
int parts_of(int rows, int V) {
  const int part = kThreads * elements(rows, V);
  return (V + part - 1) / part;
}

template <typename T>
int launch(const BeamParams& p, const Parts& parts, hipStream_t stream) {
  const int rows = p.R * p.W;
  const int64_t grid = (int64_t)rows * parts.n;
  if (int rc = check_grid("beam select", grid, kThreads)) return rc;
  if (int rc = check_grid("beam select", p.R, kRequestThreads)) return rc;
  const int each = elements(rows, p.V);
  const dim3 g((unsigned)grid), t(kThreads);
  if (each == 32) hipLaunchKernelGGL((rows_kernel<T, 32>), g, t, 0, stream, p, parts);
  else if (each == 16) hipLaunchKernelGGL((rows_kernel<T, 16>), g, t, 0, stream, p, parts);
  else hipLaunchKernelGGL((rows_kernel<T, 4>), g, t, 0, stream, p, parts);
  if (int rc = check_launch("beam select")) return rc;
  const int64_t all = (int64_t)p.W * parts.n * p.K;
  // Candidates in registers where they fit: 1216 of 16 requests 9.0 us in the kernel, read again at each use 10.4; 512 of one
  // 5.5 and 6.0.
  if (all <= 4 * kRequestThreads) hipLaunchKernelGGL((request_kernel<4>), dim3(p.R), dim3(kRequestThreads), 0, stream, p, parts);
  else hipLaunchKernelGGL((request_kernel<0>), dim3(p.R), dim3(kRequestThreads), 0, stream, p, parts);
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
  const uint64_t each = (uint64_t)n * p.K;
  const beam::Parts parts{n, (uint32_t)std::min<uint64_t>(((uint64_t(1) << 32) + each - 1) / each, 0xffffffffu), reinterpret_cast<float*>(best + all * p.K), sum, best};
  if (dtype == SLMT_F32) return beam::launch<float>(p, parts, stream);
  if (dtype == SLMT_F16) return beam::launch<beam::f16>(p, parts, stream);
  return beam::launch<beam::bf16>(p, parts, stream);
}

}  // namespace slmt
