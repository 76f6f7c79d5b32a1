// Sampling of the next token of every row of logits from given uniforms: temperature, top-k, top-p and
// min-p, without sorting the row.
//
// Order a row by logit, largest first, equal ones by index.  With w = exp((l - max l) / T) each cut keeps
// a prefix of that order: the first k; the elements before which lies less than top_p of the first k's
// mass; those with w >= min_p.  The token is the first in index order whose running sum of the kept w
// passes u times the kept mass.
//
// Sums are 64-bit integers, w in units of 2^-(62 - ceil(log2 V)), 2^-51 at most: they hold the whole vocabulary, are
// the same in whatever order they are formed, and an element below half a unit, which no uniform could reach, is
// nothing.  w itself has the precision of fp64: over 10^5 elements the errors of fp32 sums move the token in one row
// of a hundred.  w = 2^-y is a table entry for the first six bits of y's fraction times a Taylor sum over the rest,
// half of what the library's exponential takes here.
//
// The cuts are found in a histogram over bins of 1/64 in y.  A small k (kCounted) needs the bins' counts alone, and
// no weight but those of the elements up to the k-th one's bin, which are listed, ordered and drawn from directly.
// Otherwise the bins hold masses too; they tell which elements are kept whatever happens within a bin, and which lie
// in the bins where a cut falls: only these are listed and ordered.  A list that overflows (more than kList elements
// about a cut, as in a row of equal logits) is not used: the cuts are then found digit by digit of the logits' bits,
// reading the row again.
//
// Rows of up to kRowMax elements take one launch, a workgroup per row (us, one row of 32000 / 64 rows: top-k 50 and top-p
// 13.4 / 14.5, top-p alone 35.4 / 37.5, min-p 21.5 / 22.6; as longer ones 22.9 / 27.1, 28.9 / 38.7, 18.4 / 22).  Longer ones take
// four, each reading the row once at most (the first from memory, the others from the caches):
//   top        the largest logit of every workgroup's part, and its index
//   histogram  the bins (not where no cut needs them)
//   masses     the cuts' bins, the mass of what is kept for sure in each part, the list of the others
//   draw       one workgroup per row: the cuts, the part, the token
// (The last of a row's workgroups to finish a launch could go on with the next one's work; the fences that this needs
// between the XCDs' caches took longer, 241 us instead of 103 for 64 rows of 151936.)
//
// The logits are read once from memory, 4 us for 64 rows of 151936 in fp16.  The calls take longer for their arithmetic and
// latency: in a kernel trace top 7 us, histogram 18, masses 24 (both some forty instructions an element for its weight), draw
// 17 (a workgroup's chain of some twenty barriers and dependent reads), of which a call in a row of them takes 63, as a launch
// begins before the one ahead has drained; 16 fp32 rows of 128001 with min-p alone 20 us.
#include "slmt_internal.h"

#include <type_traits>

namespace slmt {
namespace {

constexpr int kPer = 8;                      // elements of a thread at a time
constexpr int kThreads = 512, kPart = kThreads * kPer;
constexpr int kBins = 4096;                  // (y < 52: at most 3329 are used; also: no bin)
constexpr int kLongBins = 48 * 64;           // of longer rows, y < 47 there
constexpr int kList = 2048, kCounted = 1024, kPlain = 512;
constexpr int kMaxVocab = 1 << 22, kMaxSplits = 256;
// A split has a part more at most than its share of the row's full ones, and the splits' rounding up to eights adds one in all.
constexpr int kMaxParts = 1536;
static_assert(kMaxVocab / kPart + kMaxSplits + kMaxSplits * kPer / kPart + 1 <= kMaxParts && kMaxParts % kThreads == 0);
constexpr int kRowThreads = 1024, kRowChunk = kRowThreads * kPer, kRowChunks = 4, kRowMax = kRowChunks * kRowChunk;
template <int NT>
constexpr int kBinsOf = NT == kRowThreads ? kBins : kLongBins;         // by the threads of a workgroup

typedef unsigned long long u64;
typedef __bf16 Bf16;
typedef _Float16 Fp16;

struct Cut {               // what the bins say of a row's cuts
  int low, high;           // bins of the top-p cut (kBins: no such cut); every element of a bin before `low` passes it
  int kbin;                // bin of the k-th element (kBins: no such cut)
  uint32_t kcount;         // elements before kbin
  u64 kmass, lowmass;      // masses before kbin and before low
  u64 total;               // of the row
  // With counts alone: low is 0, high the k-th element's bin, and there are no masses.
};

// A longer row's split: `splits` workgroups take `length` elements each (a multiple of kPer), in `steps` parts.
struct Split {
  int splits, length, steps;
  __host__ __device__ int parts() const { return splits * steps; }
  __device__ __forceinline__ int part_of(uint32_t i) const { return (int)(i / length) * steps + (int)(i % length) / kPart; }
};

// A row's place in the workspace.
struct Row {
  u64* mass;               // [kLongBins]
  u64* part_mass;          // [parts]
  u64* list;               // [kList]: order key, index
  Cut* cut;
  float* top;              // [splits]
  uint32_t* top_at;        // [splits]
  uint32_t* count;         // [kLongBins]
  uint32_t* listed;
};
__host__ __device__ __forceinline__ int64_t row_bytes(const Split& sp) {
  return ((kLongBins + sp.parts() + kList) * 8ll + sizeof(Cut) + sp.splits * 8ll + kLongBins * 4ll + 8 + 15) & ~15ll;
}
__device__ __forceinline__ Row row_at(uint8_t* ws, int64_t row, const Split& sp) {
  Row r;
  uint8_t* p = ws + row * row_bytes(sp);
  r.mass = reinterpret_cast<u64*>(p);
  r.part_mass = r.mass + kLongBins;
  r.list = r.part_mass + sp.parts();
  r.cut = reinterpret_cast<Cut*>(r.list + kList);
  r.top = reinterpret_cast<float*>(r.cut + 1);
  r.top_at = reinterpret_cast<uint32_t*>(r.top + sp.splits);
  r.count = r.top_at + sp.splits;
  r.listed = r.count + kLongBins;
  return r;
}

struct Params {
  SampleParams s;
  Split sp;
  uint8_t* ws;
};

// Logits i .. i + 7 of a row (those past its end -infinity).  What is no number is never drawn: -infinity too.
template <typename T>
__device__ __forceinline__ void load(const T* row, int i, int V, float* x) {
  T raw[kPer];
  if (i + kPer <= V) {
    __builtin_memcpy(raw, row + i, sizeof(raw));
#pragma unroll
    for (int e = 0; e < kPer; ++e) x[e] = fmaxf((float)raw[e], -INFINITY);
  } else {
#pragma unroll
    for (int e = 0; e < kPer; ++e) x[e] = i + e < V ? fmaxf((float)row[min(i + e, V - 1)], -INFINITY) : -INFINITY;
  }
}

// Place of a logit in the order: smaller for larger logits, the same for +0 and -0.
__device__ __forceinline__ uint32_t order_key(float l) {
  const uint32_t u = __builtin_bit_cast(uint32_t, l + 0.0f);
  return u >> 31 ? u : 0x7fffffffu - u;
}
__device__ __forceinline__ float logit_of(uint32_t key) {
  return __builtin_bit_cast(float, key >> 31 ? key : 0x7fffffffu - key);
}
__device__ __forceinline__ u64 place_of(float l, int i) { return ((u64)order_key(l) << 32) | (uint32_t)i; }

// What a row's call asks for.
struct Ask {
  double inv_t, min_p, top_p;
  int k;                   // 0: no cut
  bool greedy, cuts, counted;
};
__device__ __forceinline__ Ask ask_of(const SampleParams& s, int row) {
  Ask a;
  const float t = s.temperatures ? s.temperatures[row] : s.temperature;
  const float p = s.top_ps ? s.top_ps[row] : s.top_p, m = s.min_ps ? s.min_ps[row] : s.min_p;
  const int k = s.top_ks ? s.top_ks[row] : s.top_k;
  a.greedy = !(t > 0.0f);
  a.inv_t = 1.0 / (double)t;
  a.top_p = p < 1.0f ? fmax((double)p, 0.0) : 1.0;          // (1, more, or no number: no cut)
  a.min_p = m > 0.0f ? fmin((double)m, 1.0) : 0.0;
  a.k = k > 0 && k < s.V ? k : 0;
  a.counted = a.k > 0 && a.k <= kCounted;
  a.cuts = a.k > 0 || a.top_p < 1.0;
  return a;
}

// 2^(-j / 64), rounded to the nearest.
__device__ const double kPowers[64] = {
    0x1.0000000000000p+0, 0x1.fa7c1819e90d8p-1, 0x1.f50765b6e4540p-1, 0x1.efa1bee615a27p-1,
    0x1.ea4afa2a490dap-1, 0x1.e502ee78b3ff6p-1, 0x1.dfc97337b9b5fp-1, 0x1.da9e603db3285p-1,
    0x1.d5818dcfba487p-1, 0x1.d072d4a07897cp-1, 0x1.cb720dcef9069p-1, 0x1.c67f12e57d14bp-1,
    0x1.c199bdd85529cp-1, 0x1.bcc1e904bc1d2p-1, 0x1.b7f76f2fb5e47p-1, 0x1.b33a2b84f15fbp-1,
    0x1.ae89f995ad3adp-1, 0x1.a9e6b5579fdbfp-1, 0x1.a5503b23e255dp-1, 0x1.a0c667b5de565p-1,
    0x1.9c49182a3f090p-1, 0x1.97d829fde4e50p-1, 0x1.93737b0cdc5e5p-1, 0x1.8f1ae99157736p-1,
    0x1.8ace5422aa0dbp-1, 0x1.868d99b4492edp-1, 0x1.82589994cce13p-1, 0x1.7e2f336cf4e62p-1,
    0x1.7a11473eb0187p-1, 0x1.75feb564267c9p-1, 0x1.71f75e8ec5f74p-1, 0x1.6dfb23c651a2fp-1,
    0x1.6a09e667f3bcdp-1, 0x1.6623882552225p-1, 0x1.6247eb03a5585p-1, 0x1.5e76f15ad2148p-1,
    0x1.5ab07dd485429p-1, 0x1.56f4736b527dap-1, 0x1.5342b569d4f82p-1, 0x1.4f9b2769d2ca7p-1,
    0x1.4bfdad5362a27p-1, 0x1.486a2b5c13cd0p-1, 0x1.44e086061892dp-1, 0x1.4160a21f72e2ap-1,
    0x1.3dea64c123422p-1, 0x1.3a7db34e59ff7p-1, 0x1.371a7373aa9cbp-1, 0x1.33c08b26416ffp-1,
    0x1.306fe0a31b715p-1, 0x1.2d285a6e4030bp-1, 0x1.29e9df51fdee1p-1, 0x1.26b4565e27cddp-1,
    0x1.2387a6e756238p-1, 0x1.2063b88628cd6p-1, 0x1.1d4873168b9aap-1, 0x1.1a35beb6fcb75p-1,
    0x1.172b83c7d517bp-1, 0x1.1429aaea92de0p-1, 0x1.11301d0125b51p-1, 0x1.0e3ec32d3d1a2p-1,
    0x1.0b5586cf9890fp-1, 0x1.0874518759bc8p-1, 0x1.059b0d3158574p-1, 0x1.02c9a3e778061p-1,
};

// The weights of a row's elements.
constexpr double kRound = 6755399441055744.0;      // 1.5 2^52: adding it leaves the nearest whole number in the low bits
constexpr double kTop = 1e300;                     // stands for a logit of infinity
struct Scale {
  double top;
  double per;              // 64 y of a distance: 64 log2(e) / T
  double past;             // 64 y from which a weight is nothing
  double least;            // min_p in units of a weight
  float ftop, bins_per;    // top and `per`, for bins that hold counts alone
  int bits;                // units of w = 1: 2^bits
  const double* table;     // kPowers, in LDS
};
// (every thread of the workgroup calls it, early: a barrier has to follow before the first weight)
__device__ __forceinline__ void fill_table(double* table) {
  if (threadIdx.x < 64) table[threadIdx.x] = kPowers[threadIdx.x];
}
__device__ __forceinline__ Scale scale_of(float top, const Ask& a, int V, const double* table) {
  Scale s;
  s.bits = min(62 - (32 - __builtin_clz((unsigned)max(V - 1, 1))), 51);
  s.ftop = top;
  s.top = fmin((double)top, kTop);
  s.per = a.inv_t * (64.0 * 1.4426950408889634074);
  s.past = 64.0 * (s.bits + 1);
  s.least = __builtin_ldexp(a.min_p, s.bits);
  s.bins_per = (float)s.per;
  s.table = table;
  return s;
}
// 64 y of a logit, never less than 0; past + 64 for all that lie further, or are no number.
__device__ __forceinline__ double place(const Scale& s, float l) {
  return fmin((s.top - fmin((double)l, kTop)) * s.per, s.past + 64.0);
}
struct Weight {
  u64 mass;                // 0: never drawn
  int bin;                 // (of a mass of 0: past those that are used)
  bool over;               // w >= min_p
};
// (no branch: eight of them run side by side)
__device__ __forceinline__ Weight weight_of(const Scale& s, float l) {
  Weight w;
  const double y = place(s, l), near = y + kRound;
  const int k = (int)(uint32_t)__builtin_bit_cast(u64, near);
  const double z = (y - (near - kRound)) * (-0.69314718055994530942 / 64.0);     // -0.0055 .. 0.0055
  double e = 1.0 / 120.0;
  e = __builtin_fma(e, z, 1.0 / 24.0);
  e = __builtin_fma(e, z, 1.0 / 6.0);
  e = __builtin_fma(e, z, 0.5);
  e = __builtin_fma(e, z, 1.0);
  const double t = s.table[k & 63];
  e = __builtin_ldexp(__builtin_fma(t * z, e, t), s.bits - (k >> 6));
  w.mass = __builtin_bit_cast(u64, e + 4503599627370496.0) & 0xfffffffffffffull;  // 2^52 leaves the nearest whole number
  w.bin = k;
  w.over = e >= s.least;
  return w;
}
// The mass of an element that min-p lets pass, else 0.
__device__ __forceinline__ u64 mass_over(const Scale& s, float l) {
  const Weight w = weight_of(s, l);
  return w.over ? w.mass : 0;
}
// An element's bin; kBins: never drawn.  Bins that hold counts alone need no more than that they follow the order: fp32's
// roundings do.  (They take elements of no weight too, which are the order's last and never drawn.)
template <int NT>
__device__ __forceinline__ int bin_at(const Scale& s, bool counted, float l) {
  if (counted) {
    const float y = l == s.ftop ? 0.0f : (s.ftop - l) * s.bins_per;
    return y < (float)(kBinsOf<NT> - 1) ? (int)y : kBins;
  }
  const Weight w = weight_of(s, l);
  return w.mass ? w.bin : kBins;
}

// v plus the value of a lane before, by a DPP control (lanes without one add 0).
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 add_dpp(u64 v) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xf, false);
  return v + (((u64)hi << 32) | lo);
}
__device__ __forceinline__ u64 wave_scan(u64 v) {
  v = add_dpp<0x111, 0xf>(v);     // row_shr 1, 2, 4, 8 within 16 lanes
  v = add_dpp<0x112, 0xf>(v);
  v = add_dpp<0x114, 0xf>(v);
  v = add_dpp<0x118, 0xf>(v);
  v = add_dpp<0x142, 0xa>(v);     // row_bcast 15: lane 15 (47) to the next 16
  return add_dpp<0x143, 0xc>(v);  // row_bcast 31: lane 31 to the upper 32
}
// A barrier of NT threads; of one wave, which needs none, the order of its own LDS accesses.
template <int NT>
__device__ __forceinline__ void sync() {
  if constexpr (NT > 64) {
    __syncthreads();
  } else {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}
// Inclusive scan over NT threads; `sums`: an entry per wave.  Two barriers.
template <int NT>
__device__ __forceinline__ u64 scan64(u64 v, u64* sums, u64& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  v = wave_scan(v);
  if (lane == 63) sums[wave] = v;
  sync<NT>();
  u64 before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    if (w == wave) before = total;
    total += sums[w];
  }
  sync<NT>();
  return v + before;
}

// The largest of the wave's values, in lane 63.
__device__ __forceinline__ float wave_largest(float m) {
  auto step = [&](auto ctrl, auto rows) {
    const int o = __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, -INFINITY), __builtin_bit_cast(int, m), ctrl.value, rows.value, 0xf, false);
    m = fmaxf(m, __builtin_bit_cast(float, o));
  };
  using std::integral_constant;
  step(integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{});
  step(integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{});
  step(integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{});
  step(integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{});
  step(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});
  step(integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});
  return m;
}
// The larger logit of two, the lower index of equal ones.
__device__ __forceinline__ void larger(float& m, uint32_t& at, float v, uint32_t a) {
  if (v > m || (v == m && a < at)) m = v, at = a;
}
__device__ __forceinline__ void wave_top(float& m, uint32_t& at) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) larger(m, at, __shfl_xor(m, o, 64), __shfl_xor(at, o, 64));
}
// The row's largest logit and its first index, from the splits.  Every thread of a wave gets it.
__device__ __forceinline__ float top_of(const Row& r, int n, uint32_t* at = nullptr) {
  float m = -INFINITY;
  uint32_t i = 0xffffffffu;
  for (int c = threadIdx.x & 63; c < n; c += 64) larger(m, i, r.top[c], r.top_at[c]);
  wave_top(m, i);
  if (at) *at = i;
  return m;
}

// Adds a thread's eight elements to the bins.  Of counts alone the largest of the eight is enough: the k-th largest of
// these lies at or below the k-th largest element, and few others at or above it, so that its bin ends the list as well.
// (Where there are fewer eights than that, no bin is found, and every element is listed or the row read again; a row of
// fewer than two eights for each of the k has its elements counted one by one.)
template <int NT>
__device__ __forceinline__ void count_one(const Scale& s, float l, uint32_t* count) {
  const int bin = bin_at<NT>(s, true, l);
  if (bin < kBins) atomicAdd(&count[bin], 1u);
}
template <int NT>
__device__ __forceinline__ void add_to_bins(const Scale& s, const Ask& a, const float* x, u64* mass, uint32_t* count) {
  if (a.counted) {
    float m = x[0];
#pragma unroll
    for (int e = 1; e < kPer; ++e) m = fmaxf(m, x[e]);
    count_one<NT>(s, m, count);
    return;
  }
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    const Weight w = weight_of(s, x[e]);
    if (w.mass) {
      atomicAdd(&mass[w.bin], w.mass);
      if (a.k) atomicAdd(&count[w.bin], 1u);
    }
  }
}

// The cuts' bins.  `out`: shared; complete after the call.
template <int NT, int NB>
__device__ __forceinline__ void find_cut(const u64* mass, const uint32_t* counts, const Ask& a, u64* sums, Cut* out) {
  constexpr int kEach = NB / NT;
  const int tid = threadIdx.x, b0 = tid * kEach;
  u64 m[kEach];
  uint32_t n[kEach];
  u64 mine = 0, count = 0, total = 0, counted = 0, before = 0, nbefore = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    m[i] = a.counted ? 0 : mass[b0 + i];
    n[i] = a.k ? counts[b0 + i] : 0;
    mine += m[i];
    count += n[i];
  }
  if (!a.counted) before = scan64<NT>(mine, sums, total) - mine;
  if (a.k) nbefore = scan64<NT>(count, sums, counted) - count;
  if (tid == 0) *out = a.counted ? Cut{0, kBins - 1, kBins - 1, 0, 0, 0, 0} : Cut{kBins, kBins, kBins, 0, total, 0, total};
  __syncthreads();
  // the bin of the k-th element (none where fewer than k can be drawn)
  if (a.k && nbefore < (u64)a.k && nbefore + count >= (u64)a.k) {
    u64 mm = before, nn = nbefore;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if (nn < (u64)a.k && nn + n[i] >= (u64)a.k) {
        out->kbin = b0 + i;
        out->kcount = (uint32_t)nn;
        out->kmass = mm;
        if (a.counted) out->high = b0 + i;
        else out->lowmass = mm + m[i];       // (for the next step: the mass up to its end)
      }
      nn += n[i];
      mm += m[i];
    }
  }
  __syncthreads();
  if (a.counted || a.top_p >= 1.0) return;
  // the mass that top_p is a part of lies between these
  const bool cut = out->kbin < kBins;
  const double least = a.top_p * (double)(cut ? out->kmass : total), most = a.top_p * (double)(cut ? out->lowmass : total);
  __syncthreads();
  u64 mm = before;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const u64 end = mm + m[i];
    const bool first = tid == 0 && i == 0;
    if ((double)end >= least && (first || (double)mm < least)) {
      out->low = b0 + i;
      out->lowmass = mm;
    }
    if ((double)end >= most && (first || (double)mm < most)) out->high = b0 + i;
    mm = end;
  }
  __syncthreads();
}

// Whether an element of this bin may or may not be kept, as the cuts fall within the bin.
__device__ __forceinline__ bool in_doubt(const Cut& c, int bin) { return (bin >= c.low && bin <= c.high) || bin == c.kbin; }
// The bins before which every element passes the cuts.
__device__ __forceinline__ int sure_bins(const Cut& c) { return min(c.low, c.kbin); }

// Of a thread's eight elements from index i on: the mass of those kept for sure; those in doubt go on the list (in LDS).
template <int NT>
__device__ __forceinline__ u64 sort_out(const Scale& s, const Ask& a, const Cut& cut, const float* x, int i, u64* list,
                                        uint32_t* listed) {
  u64 mass = 0;
  uint32_t doubt = 0;
  if (a.counted) {
    float m = x[0];
#pragma unroll
    for (int e = 1; e < kPer; ++e) m = fmaxf(m, x[e]);
    if (bin_at<NT>(s, true, m) <= cut.high) {    // (no bin is past every one)
#pragma unroll
      for (int e = 0; e < kPer; ++e) doubt |= (uint32_t)(bin_at<NT>(s, true, x[e]) <= cut.high) << e;
    }
  } else {
    const int sure = sure_bins(cut);
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const Weight w = weight_of(s, x[e]);
      mass += w.bin < sure && w.over ? w.mass : 0;
      doubt |= (uint32_t)(w.mass && w.bin >= sure && in_doubt(cut, w.bin)) << e;
    }
  }
  if (doubt) {
#pragma unroll
    for (int e = 0; e < kPer; ++e)
      if (doubt >> e & 1) {
        const uint32_t at = atomicAdd(listed, 1u);
        if (at < (uint32_t)kList) list[at] = place_of(x[e], i + e);
      }
  }
  return mass;
}

// The last kept element in the order; none where `some` is false.
struct Last {
  u64 at;
  bool some;
};

struct __attribute__((aligned(16))) Lists {
  u64 list[kList], sorted[kList];
  u64 digit_mass[256];
  uint32_t digit_count[256];
};

// Orders the list.  A short one: every entry to the place that is the number of those before it (no two are the same), by
// comparing it with all.  A long one goes into buckets of equal parts of its range first, and an entry is compared with
// its bucket's.  (us for a row of 16000 with top_k 1000, this and the parts that the draw from a list goes by: 70 without,
// 24.5 with; of 4000 with top_k 200, whose list is between 256 and 512 long, 16.9 plain, 19.0 in buckets.)
template <int NT>
__device__ __forceinline__ void order(Lists& ls, int n, u64* sums) {
  const int tid = threadIdx.x;
  sync<NT>();
  if (NT == 64 || n <= kPlain) {
    for (int i = tid; i < n; i += NT) {
      const u64 mine = ls.list[i];
      int before = 0;
      for (int j = 0; j + 8 <= n; j += 8) {  // (two entries a read, eight in flight)
        ulonglong2 two[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) two[q] = *reinterpret_cast<const ulonglong2*>(&ls.list[j + 2 * q]);
#pragma unroll
        for (int q = 0; q < 4; ++q) before += (two[q].x < mine) + (two[q].y < mine);
      }
      for (int j = n & ~7; j < n; ++j) before += ls.list[j] < mine;
      ls.sorted[before] = mine;
    }
    sync<NT>();
    return;
  }
  if constexpr (NT > 64) {
    constexpr int kWaves = NT / 64, kBuckets = 512;
    uint32_t* const bucket = reinterpret_cast<uint32_t*>(ls.digit_mass);
    static_assert(sizeof(ls.digit_mass) == kBuckets * 4 && kBuckets / 2 <= NT && 2 * kWaves <= 256);
    u64 lo = ~0ull, hi = 0;
    for (int i = tid; i < n; i += NT) lo = min(lo, ls.list[i]), hi = max(hi, ls.list[i]);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) lo = min(lo, (u64)__shfl_xor(lo, o, 64)), hi = max(hi, (u64)__shfl_xor(hi, o, 64));
    if ((tid & 63) == 0) ls.digit_mass[tid >> 6] = lo, ls.digit_mass[kWaves + (tid >> 6)] = hi;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) lo = min(lo, ls.digit_mass[w]), hi = max(hi, ls.digit_mass[kWaves + w]);
    const int shift = max(64 - 9 - __builtin_clzll((hi - lo) | 1), 0);   // (n > 1)
    auto of = [&](u64 v) { return (uint32_t)((v - lo) >> shift); };
    __syncthreads();
    for (int c = tid; c < kBuckets; c += NT) bucket[c] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += NT) atomicAdd(&bucket[of(ls.list[i])], 1u);
    __syncthreads();
    const bool two = tid < kBuckets / 2;
    const uint32_t c0 = two ? bucket[2 * tid] : 0, c1 = two ? bucket[2 * tid + 1] : 0;
    u64 all;
    const uint32_t start = (uint32_t)scan64<NT>(c0 + c1, sums, all) - c0 - c1;
    if (two) bucket[2 * tid] = start, bucket[2 * tid + 1] = start + c0;
    __syncthreads();
    for (int i = tid; i < n; i += NT) {
      const u64 mine = ls.list[i];
      ls.sorted[atomicAdd(&bucket[of(mine)], 1u)] = mine;              // (leaves every bucket's end in its place)
    }
    __syncthreads();
    for (int i = tid; i < n; i += NT) {
      const u64 mine = ls.sorted[i];
      const uint32_t b = of(mine), end = bucket[b];
      uint32_t before = b ? bucket[b - 1] : 0;
      for (uint32_t j = before; j < end; ++j) before += ls.sorted[j] < mine;
      ls.list[before] = mine;
    }
    __syncthreads();
    for (int i = tid; i < n; i += NT) ls.sorted[i] = ls.list[i];
    __syncthreads();
  }
}

// The last kept element, from a list of all that are in doubt.
template <int NT>
__device__ __forceinline__ Last last_of_list(Lists& ls, int n, const Cut& cut, const Ask& a, const Scale& s, u64* sums) {
  const int tid = threadIdx.x;
  order<NT>(ls, n, sums);
  // a few entries a thread: their bins and masses
  constexpr int kEach = kList / NT;
  u64 m[kEach];
  int bin[kEach];
  u64 mine = 0, kmine = 0;
  uint32_t earlier = 0;                      // entries of bins before kbin
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int j = tid * kEach + i;
    Weight w{0, kBins, false};
    if (j < n) w = weight_of(s, logit_of((uint32_t)(ls.sorted[j] >> 32)));
    m[i] = w.mass;
    bin[i] = w.bin;
    mine += w.mass;
    earlier += j < n && w.bin < cut.kbin;
  }
  u64 total, first_k = 0, chosen = 0;
  if (cut.kbin < kBins) {
    scan64<NT>(earlier, sums, first_k);      // where kbin's entries start
    const u64 end = first_k + (u64)(a.k - cut.kcount);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const u64 j = tid * kEach + i;
      if (j >= first_k && j < end) kmine += m[i];
    }
    scan64<NT>(kmine, sums, chosen);
  }
  const u64 kmass = cut.kbin < kBins ? cut.kmass + chosen : cut.total;
  const double limit = a.top_p * (double)kmass;
  u64 before = scan64<NT>(mine, sums, total) - mine + cut.lowmass;
  uint32_t kept = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const u64 j = tid * kEach + i;
    bool keep = j < (u64)n;
    if (cut.kbin < kBins) keep = keep && (bin[i] < cut.kbin || j < first_k + (u64)(a.k - cut.kcount));
    if (cut.low < kBins) keep = keep && bin[i] <= cut.high && ((double)before < limit || (cut.low == 0 && j == 0));
    kept += keep;
    before += m[i];
  }
  u64 all;
  scan64<NT>(kept, sums, all);
  Last last{0, all > 0};
  if (all) last.at = ls.sorted[all - 1];
  return last;
}

// A row's token and its probability.
__device__ __forceinline__ void answer(const SampleParams& s, int row, int64_t token, float prob) {
  s.tokens[row] = token;
  if (s.probs) s.probs[row] = prob;
}
// The mass at which a row's uniform lies.
__device__ __forceinline__ u64 target_of(const SampleParams& s, int row, u64 total) {
  const double at = (double)s.uniforms[row] * (double)total;
  return at > 0.0 ? min((u64)fmin(at, 0x1p62), total - 1) : 0;
}

// Draws from a list of all the elements up to the k-th one's bin (counts alone): the first k in the order, cut by top-p
// and min-p, and of those kept the one whose masses before it, by index, the target falls behind.  n <= MOST.
template <int NT, int MOST>
__device__ __forceinline__ void draw_of_list(Lists& ls, int n, const Ask& a, const Scale& s, const SampleParams& sp, int row,
                                             u64* sums) {
  const int tid = threadIdx.x;
  order<NT>(ls, n, sums);
  constexpr int kEach = MOST / NT;
  u64 m[kEach], mine = 0, total, before;
  bool over[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int j = tid * kEach + i;
    Weight w{0, kBins, false};
    if (j < n && j < a.k) w = weight_of(s, logit_of((uint32_t)(ls.sorted[j] >> 32)));
    m[i] = w.mass;
    over[i] = w.mass && w.over;
    mine += w.mass;
  }
  before = scan64<NT>(mine, sums, total) - mine;
  const double limit = a.top_p * (double)total;
  mine = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int j = tid * kEach + i;
    const bool keep = over[i] && (a.top_p >= 1.0 || (double)before < limit || j == 0);
    before += m[i];
    if (!keep) m[i] = 0;
    mine += m[i];
  }
  scan64<NT>(mine, sums, total);
  const u64 target = target_of(sp, row, total);
  if constexpr (NT == 64) {
    // (the kept ones are the first of the order: their masses take the unordered list's place)
    static_assert(kEach == 1);
    const int some = __builtin_popcountll(__builtin_amdgcn_ballot_w64(m[0] != 0));
    ls.list[tid] = m[0];
    sync<NT>();
    const uint32_t at = (uint32_t)ls.sorted[tid];
    u64 sum = 0;
#pragma unroll 4
    for (int j = 0; j < some; ++j) sum += (uint32_t)ls.sorted[j] < at ? ls.list[j] : 0;
    if (tid < some && target >= sum && target < sum + m[0]) answer(sp, row, at, (float)((double)m[0] / (double)total));
  } else {
    // The masses of 256 parts of the indices; then, of the part that the target falls into, its kept elements alone.
    constexpr int kParts = 256;
    const uint32_t width = (uint32_t)(sp.V + kParts - 1) / kParts;
    uint32_t at[kEach], part[kEach];
    if (tid < kParts) ls.digit_mass[tid] = 0;
    if (tid == 0) ls.digit_count[0] = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int j = tid * kEach + i;
      at[i] = j < n ? (uint32_t)ls.sorted[j] : 0;
      part[i] = at[i] / width;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (m[i]) atomicAdd(&ls.digit_mass[part[i]], m[i]);
    __syncthreads();
    u64 all;
    const u64 own = tid < kParts ? ls.digit_mass[tid] : 0, end = scan64<NT>(own, sums, all);
    if (target >= end - own && target < end) ls.digit_count[1] = (uint32_t)tid, ls.digit_mass[0] = end - own;
    __syncthreads();
    const uint32_t drawn = ls.digit_count[1];
    const u64 rest = target - ls.digit_mass[0];
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (m[i] && part[i] == drawn) {
        const uint32_t c = atomicAdd(&ls.digit_count[0], 1u);
        ls.list[c] = m[i];
        ls.sorted[c] = at[i];
      }
    __syncthreads();
    const int members = (int)ls.digit_count[0];
    for (int i = tid; i < members; i += NT) {
      const u64 mass = ls.list[i], index = ls.sorted[i];
      u64 sum = 0;
#pragma unroll 4
      for (int j = 0; j < members; ++j) sum += ls.sorted[j] < index ? ls.list[j] : 0;
      if (rest >= sum && rest < sum + mass) answer(sp, row, (int64_t)index, (float)((double)mass / (double)total));
    }
  }
}

// The cuts from the row itself, digit by digit of the order key.  Finds the key at which the running count
// (by_count) or mass of the elements in bins first .. last reaches `want`, and what lies before that key.
struct Digits {
  uint32_t key;
  uint32_t ties;           // elements of that key
  u64 count, mass;         // before it, from the given start on
};
template <int NT, typename T>
__device__ __forceinline__ Digits descend(Lists& ls, u64* sums, u64* found, const T* logits, int V, const Scale& s, bool counted,
                                          int first, int last, bool by_count, u64 count0, u64 mass0, u64 want_count, double want_mass) {
  const int tid = threadIdx.x;
  Digits d{0, 0, count0, mass0};
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    for (int b = tid; b < 256; b += NT) ls.digit_mass[b] = 0, ls.digit_count[b] = 0;
    __syncthreads();
    for (int i0 = tid * kPer; i0 < V; i0 += NT * kPer) {
      float x[kPer];
      load(logits, i0, V, x);
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const uint32_t key = order_key(x[e]);
        if (shift < 24 && (key >> (shift + 8)) != (d.key >> (shift + 8))) continue;
        const int bin = bin_at<NT>(s, counted, x[e]);
        if (bin == kBins || bin < first || bin > last) continue;
        atomicAdd(&ls.digit_count[(key >> shift) & 255], 1u);
        atomicAdd(&ls.digit_mass[(key >> shift) & 255], weight_of(s, x[e]).mass);
      }
    }
    __syncthreads();
    u64 all;
    const u64 m = tid < 256 ? ls.digit_mass[tid] : 0, c = tid < 256 ? ls.digit_count[tid] : 0;
    const u64 mend = scan64<NT>(m, sums, all) + d.mass, cend = scan64<NT>(c, sums, all) + d.count;
    // the first digit that reaches it; where rounding leaves none, the last that has elements
    const bool reaches = c && (by_count ? cend >= want_count : (double)mend >= want_mass);
    const bool before = by_count ? cend - c >= want_count : (double)(mend - m) >= want_mass;
    if (tid == 0) found[0] = 0xffffffffull, found[1] = 0;
    __syncthreads();
    if (reaches && (!before || cend - c == d.count)) atomicMin(&found[0], (u64)tid);
    if (c) atomicMax(&found[1], (u64)tid);
    __syncthreads();
    const uint32_t digit = (uint32_t)(found[0] == 0xffffffffull ? found[1] : found[0]);
    __syncthreads();
    if ((uint32_t)tid == digit) found[0] = cend - c, found[1] = mend - m, found[2] = c;
    __syncthreads();
    d.key |= digit << shift;
    d.count = found[0];
    d.mass = found[1];
    d.ties = (uint32_t)found[2];
    __syncthreads();
  }
  return d;
}

template <int NT, typename T>
__device__ __noinline__ Last last_of_row(Lists& ls, u64* sums, u64* found, const T* logits, int V, Cut cut, const Ask& a,
                                         const Scale& s) {
  const int tid = threadIdx.x;
  uint32_t key = 0xffffffffu, ties = 0;
  bool some = false;
  u64 kmass = cut.total;
  if (a.counted) {                           // (the bins have no masses: from the first to the list's last)
    u64 mine = 0, more = 0, listed;
    for (int i0 = tid * kPer; i0 < V; i0 += NT * kPer) {
      float x[kPer];
      load(logits, i0, V, x);
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        if (bin_at<NT>(s, true, x[e]) <= cut.high) {
          mine += weight_of(s, x[e]).mass;
          ++more;
        }
    }
    scan64<NT>(mine, sums, kmass);
    scan64<NT>(more, sums, listed);
    if (listed > (u64)a.k) {
      const Digits d = descend<NT>(ls, sums, found, logits, V, s, true, 0, cut.high, true, 0, 0, (u64)a.k, 0.0);
      key = d.key;
      ties = (uint32_t)((u64)a.k - d.count);
      some = true;
      kmass = d.mass + ties * weight_of(s, logit_of(key)).mass;
    }
    cut.kbin = kBins;
    if (a.top_p >= 1.0) cut.low = kBins;
  }
  if (cut.kbin < kBins) {
    const Digits d = descend<NT>(ls, sums, found, logits, V, s, a.counted, cut.kbin, cut.kbin, true, cut.kcount, cut.kmass, (u64)a.k, 0.0);
    key = d.key;
    ties = (uint32_t)((u64)a.k - d.count);
    some = true;
    kmass = d.mass + ties * weight_of(s, logit_of(key)).mass;
  }
  if (cut.low < kBins) {
    const double limit = a.top_p * (double)kmass;
    const Digits d = descend<NT>(ls, sums, found, logits, V, s, a.counted, cut.low, cut.high, false, 0, cut.lowmass, 0, limit);
    // of its ties, those before which lies less than the limit (the row's first element in any case)
    const u64 each = weight_of(s, logit_of(d.key)).mass;
    uint32_t lo = cut.low == 0 && d.count == 0 ? 1 : 0, hi = d.ties;
    while (lo < hi) {
      const uint32_t mid = (lo + hi + 1) / 2;
      if ((double)(d.mass + (mid - 1) * each) < limit) lo = mid;
      else hi = mid - 1;
    }
    if (!some || d.key < key || (d.key == key && lo < ties)) key = d.key, ties = lo;
    some = true;
  }
  if (!some) return Last{~0ull, true};       // (no cut after all)
  // the index of the last of its ties
  Last last{(u64)key << 32, true};
  if (ties == 0) {
    // (no tie of this key: every index of a smaller key passes)
    last.at = ((u64)key << 32) - 1;
    return last;
  }
  u64 seen = 0;
  for (int c = 0; c < V; c += NT * kPer) {
    float x[kPer];
    load(logits, c + tid * kPer, V, x);
    u64 mine = 0, all;
#pragma unroll
    for (int e = 0; e < kPer; ++e) mine += order_key(x[e]) == key && c + tid * kPer + e < V;
    u64 at = seen + scan64<NT>(mine, sums, all) - mine;
    if (seen < ties && seen + all >= ties) {
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        if (order_key(x[e]) == key && c + tid * kPer + e < V && ++at == ties) found[3] = c + tid * kPer + e;
    }
    seen += all;
    __syncthreads();
    if (seen >= ties) break;
  }
  last.at |= found[3];
  return last;
}

// ------------------------------------------------------------------ rows of up to kRowMax elements
struct RowShared {
  union {
    struct {
      u64 mass[kBins];
      uint32_t count[kBins];
    } bins;
    Lists lists;
  };
  double table[64];
  u64 part[kRowChunks * kRowThreads / 64];   // masses of 512 elements each, a wave's of one chunk
  u64 sums[kRowThreads / 64];
  u64 found[4];
  float ms[kRowThreads / 64];
  uint32_t is[kRowThreads / 64];
  uint32_t listed;
  Cut cut;
};

// One pass over the row after another, each a loop over its chunks with the next one's loads in flight: what a workgroup
// alone on its CU waits for is as much its own code as its data (with the chunks unrolled and the row in registers the
// passes took 3 us each, 20 in all, for 32000 elements).
template <typename T>
__global__ void __launch_bounds__(kRowThreads) row_kernel(const SampleParams sp) {
  constexpr int NT = kRowThreads, kWaves = NT / 64;
  __shared__ RowShared sh;
  const int row = blockIdx.x, tid = threadIdx.x, wave = tid >> 6, V = sp.V;
  const Ask a = ask_of(sp, row);
  const T* const logits = reinterpret_cast<const T*>(sp.logits) + row * sp.row_stride;
  // element e of chunk c: index c * kRowChunk + tid * kPer + e
  const int chunks = (V + kRowChunk - 1) / kRowChunk;
  auto each = [&](auto f) {
    float x[kPer], next[kPer];
    load(logits, tid * kPer, V, x);
#pragma unroll 1
    for (int c = 0; c < chunks; ++c) {
      load(logits, (c + 1) * kRowChunk + tid * kPer, V, next);
      f(c, c * kRowChunk + tid * kPer, x);
#pragma unroll
      for (int e = 0; e < kPer; ++e) x[e] = next[e];
    }
  };
  if (a.cuts && !a.greedy)
    for (int b = tid; b < kBins; b += NT) sh.bins.mass[b] = 0, sh.bins.count[b] = 0;
  if (tid == 0) sh.listed = 0;
  fill_table(sh.table);
  float m = -INFINITY;
  uint32_t at = min(tid * kPer, V - 1);
  if (a.greedy) {
    each([&](int, int i, const float* x) {
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        if (x[e] > m) m = x[e], at = i + e;
    });
    wave_top(m, at);
    if ((tid & 63) == 0) sh.ms[wave] = m, sh.is[wave] = at;
    __syncthreads();
    if (tid != 0) return;
    for (int w = 1; w < kWaves; ++w) larger(m, at, sh.ms[w], sh.is[w]);
    answer(sp, row, at, m == -INFINITY ? 0.0f : 1.0f);
    return;
  }
  float eights[kRowChunks];                  // the largest of each chunk's eight
#pragma unroll
  for (int q = 0; q < kRowChunks; ++q) eights[q] = -INFINITY;
  each([&](int c, int, const float* x) {
    float l = x[0];
#pragma unroll
    for (int e = 1; e < kPer; ++e) l = fmaxf(l, x[e]);
#pragma unroll
    for (int q = 0; q < kRowChunks; ++q) eights[q] = q == c ? l : eights[q];
    m = fmaxf(m, l);
  });
  m = wave_largest(m);
  if ((tid & 63) == 63) sh.ms[wave] = m;
  __syncthreads();
  m = wave_largest(sh.ms[tid & (kWaves - 1)]);
  m = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, m), 63));
  if (m == -INFINITY) {
    if (tid == 0) answer(sp, row, 0, 0.0f);
    return;
  }
  const Scale s = scale_of(m, a, V, sh.table);
  Cut cut{kBins, kBins, kBins, 0, 0, 0, 0};
  if (a.cuts) {
    if (a.counted) {
      if (V >= 2 * kPer * a.k) {
#pragma unroll
        for (int q = 0; q < kRowChunks; ++q) count_one<NT>(s, eights[q], sh.bins.count);
      } else {
        each([&](int, int, const float* x) {
#pragma unroll
          for (int e = 0; e < kPer; ++e) count_one<NT>(s, x[e], sh.bins.count);
        });
      }
    } else {
      each([&](int, int, const float* x) { add_to_bins<NT>(s, a, x, sh.bins.mass, sh.bins.count); });
    }
    __syncthreads();
    find_cut<NT, kBins>(sh.bins.mass, sh.bins.count, a, sh.sums, &sh.cut);
    cut = sh.cut;
    __syncthreads();                         // (the lists take the bins' place)
  }
  if (a.counted) {                           // (only the eights whose largest is that large are read again)
    uint32_t some = 0;
#pragma unroll
    for (int q = 0; q < kRowChunks; ++q) some |= (uint32_t)(bin_at<NT>(s, true, eights[q]) <= cut.high) << q;
#pragma unroll 1
    while (some) {
      const int i = __builtin_ctz(some) * kRowChunk + tid * kPer;
      some &= some - 1;
      float x[kPer];
      load(logits, i, V, x);
      sort_out<NT>(s, a, cut, x, i, sh.lists.list, &sh.listed);
    }
  } else {
    each([&](int c, int i, const float* x) {
      const u64 sum = wave_scan(sort_out<NT>(s, a, cut, x, i, sh.lists.list, &sh.listed));
      if ((tid & 63) == 63) sh.part[c * kWaves + wave] = sum;
    });
  }
  __syncthreads();
  const uint32_t n = sh.listed;
  if (a.counted && n <= (uint32_t)kList) {
    if (n > 64) draw_of_list<NT, kList>(sh.lists, (int)n, a, s, sp, row, sh.sums);
    else if (wave == 0) draw_of_list<64, 64>(sh.lists, (int)n, a, s, sp, row, sh.sums);
    return;
  }
  // what of those in doubt is kept, beside the sure ones' masses
  Last last{0, false};
  auto kept = [&](float l, int i, bool sure) {           // (of those in doubt, and with `sure` of the others)
    const int bin = bin_at<NT>(s, a.counted, l);
    const bool keep = bin < sure_bins(cut) ? sure : bin < kBins && last.some && in_doubt(cut, bin) && place_of(l, i) <= last.at;
    return keep ? mass_over(s, l) : 0ull;
  };
  if (n > (uint32_t)kList) {
    last = last_of_row<NT>(sh.lists, sh.sums, sh.found, logits, V, cut, a, s);
    each([&](int c, int i, const float* x) {
      u64 mass = 0;
#pragma unroll
      for (int e = 0; e < kPer; ++e) mass += kept(x[e], i + e, false);
      const u64 sum = wave_scan(mass);
      if ((tid & 63) == 63) sh.part[c * kWaves + wave] = (a.counted ? 0 : sh.part[c * kWaves + wave]) + sum;
    });
  } else if (n) {
    last = last_of_list<NT>(sh.lists, (int)n, cut, a, s, sh.sums);
    for (uint32_t i = tid; i < n; i += NT) {
      const u64 at = sh.lists.sorted[i];
      if (last.some && at <= last.at) atomicAdd(&sh.part[(uint32_t)at / (64 * kPer)], mass_over(s, logit_of((uint32_t)(at >> 32))));
    }
  }
  __syncthreads();
  if (tid == 0) sh.found[0] = 0, sh.found[1] = 0;      // (the first element has mass, so one is found; the row's start in any case)
  u64 total;
  const u64 own = tid < chunks * kWaves ? sh.part[tid] : 0;
  const u64 end = scan64<NT>(own, sh.sums, total);
  const u64 target = target_of(sp, row, total);
  if (target >= end - own && target < end) sh.found[0] = tid, sh.found[1] = end - own;
  __syncthreads();
  if (wave != (int)sh.found[0] % kWaves) return;
  // the wave that holds it
  const int i = (int)sh.found[0] / kWaves * kRowChunk + tid * kPer;
  float x[kPer];
  u64 w[kPer], mine = 0;
  load(logits, i, V, x);
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    w[e] = kept(x[e], i + e, true);
    mine += w[e];
  }
  u64 before = sh.found[1] + wave_scan(mine) - mine;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    if (target >= before && target < before + w[e]) answer(sp, row, i + e, (float)((double)w[e] / (double)total));
    before += w[e];
  }
}

// ------------------------------------------------------------------ longer rows
// Calls f(x, i, step) with the eights of this workgroup's part of the row, the next ones' loads in flight.
template <typename T, typename F>
__device__ __forceinline__ void each_eight(const Params& p, const T* logits, int split, F f) {
  const int first = split * p.sp.length, end = min(first + p.sp.length, p.s.V);
  int i = first + threadIdx.x * kPer;
  float x[kPer], next[kPer];
  load(logits, i, end, x);
#pragma unroll 1
  for (int step = 0; first + step * kPart < end; ++step, i += kPart) {   // (the same for all threads)
    load(logits, i + kPart, end, next);
    f(x, i, step);
#pragma unroll
    for (int e = 0; e < kPer; ++e) x[e] = next[e];
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) top_kernel(const Params p) {
  constexpr int kWaves = kThreads / 64;
  __shared__ float ms[kWaves];
  __shared__ uint32_t is[kWaves];
  const int row = blockIdx.x / p.sp.splits, split = blockIdx.x - row * p.sp.splits, tid = threadIdx.x;
  const Row r = row_at(p.ws, row, p.sp);
  const T* const logits = reinterpret_cast<const T*>(p.s.logits) + row * p.s.row_stride;
  float m = -INFINITY;
  uint32_t at = min(split * p.sp.length, p.s.V - 1);
  const bool greedy = ask_of(p.s, row).greedy;           // (only these rows need the index)
  each_eight(p, logits, split, [&](const float* x, int i, int) {
    if (greedy) {
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        if (x[e] > m) m = x[e], at = i + e;
    } else {
#pragma unroll
      for (int e = 0; e < kPer; ++e) m = fmaxf(m, x[e]);
    }
  });
  // (the bins and the list start empty; this is the first launch of the call)
  for (int b = split * kThreads + tid; b < kLongBins; b += p.sp.splits * kThreads) r.mass[b] = 0, r.count[b] = 0;
  if (split == 0 && tid == 0) *r.listed = 0;
  wave_top(m, at);
  if ((tid & 63) == 0) ms[tid >> 6] = m, is[tid >> 6] = at;
  __syncthreads();
  if (tid == 0) {
#pragma unroll
    for (int w = 1; w < kWaves; ++w) larger(m, at, ms[w], is[w]);
    r.top[split] = m;
    r.top_at[split] = at;
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) histogram_kernel(const Params p) {
  __shared__ u64 mass[kLongBins];
  __shared__ uint32_t count[kLongBins];
  __shared__ double table[64];
  const int row = blockIdx.x / p.sp.splits, split = blockIdx.x - row * p.sp.splits, tid = threadIdx.x;
  const Ask a = ask_of(p.s, row);
  if (a.greedy || !a.cuts) return;
  const Row r = row_at(p.ws, row, p.sp);
  const T* const logits = reinterpret_cast<const T*>(p.s.logits) + row * p.s.row_stride;
  fill_table(table);
  const Scale s = scale_of(top_of(r, p.sp.splits), a, p.s.V, table);
  if (s.ftop == -INFINITY) return;
  for (int b = tid; b < kLongBins; b += kThreads) mass[b] = 0, count[b] = 0;
  __syncthreads();
  each_eight(p, logits, split, [&](const float* x, int, int) { add_to_bins<kThreads>(s, a, x, mass, count); });
  __syncthreads();
  for (int b = tid; b < kLongBins; b += kThreads) {
    if (!a.counted && mass[b]) atomicAdd(&r.mass[b], mass[b]);
    if (a.k && count[b]) atomicAdd(&r.count[b], count[b]);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) masses_kernel(const Params p) {
  __shared__ u64 sums[kThreads / 64];
  __shared__ u64 part[kMaxParts], list[kList];
  __shared__ double table[64];
  __shared__ Cut shared_cut;
  __shared__ uint32_t listed, to;
  const int row = blockIdx.x / p.sp.splits, split = blockIdx.x - row * p.sp.splits, tid = threadIdx.x;
  const Ask a = ask_of(p.s, row);
  if (a.greedy) return;
  const Row r = row_at(p.ws, row, p.sp);
  const T* const logits = reinterpret_cast<const T*>(p.s.logits) + row * p.s.row_stride;
  fill_table(table);
  const Scale s = scale_of(top_of(r, p.sp.splits), a, p.s.V, table);
  if (s.ftop == -INFINITY) return;
  for (int c = tid; c < p.sp.steps; c += kThreads) part[c] = 0;
  if (tid == 0) listed = 0;
  Cut cut{kBins, kBins, kBins, 0, 0, 0, 0};
  if (a.cuts) {
    find_cut<kThreads, kLongBins>(r.mass, r.count, a, sums, &shared_cut);
    cut = shared_cut;
    if (split == 0 && tid == 0) *r.cut = cut;
  }
  __syncthreads();
  each_eight(p, logits, split, [&](const float* x, int i, int step) {
    const u64 mass = sort_out<kThreads>(s, a, cut, x, i, list, &listed);
    if (a.counted) return;
    const u64 sum = wave_scan(mass);
    if ((tid & 63) == 63 && sum) atomicAdd(&part[step], sum);
  });
  __syncthreads();
  for (int c = tid; c < p.sp.steps; c += kThreads) r.part_mass[split * p.sp.steps + c] = part[c];
  // (one request to memory for the workgroup's place in the row's list, not one for every element)
  const uint32_t n = listed;
  if (n == 0) return;
  if (tid == 0) to = atomicAdd(r.listed, n);
  __syncthreads();
  for (uint32_t e = tid; e < min(n, (uint32_t)kList) && to + e < (uint32_t)kList; e += kThreads) r.list[to + e] = list[e];
}

template <typename T>
__global__ void __launch_bounds__(kThreads) draw_kernel(const Params p) {
  constexpr int NT = kThreads;
  __shared__ Lists ls;
  __shared__ u64 part[kMaxParts];
  __shared__ u64 sums[NT / 64], found[4];
  __shared__ double table[64];
  const int row = blockIdx.x, tid = threadIdx.x, V = p.s.V;
  const Ask a = ask_of(p.s, row);
  const Row r = row_at(p.ws, row, p.sp);
  const int parts = p.sp.parts();
  uint32_t top_at;
  fill_table(table);
  const float top = top_of(r, p.sp.splits, &top_at);
  if (a.greedy || top == -INFINITY) {
    // (the splits' first indices: 0 for a row that leaves nothing)
    if (tid == 0) answer(p.s, row, top_at, top == -INFINITY ? 0.0f : 1.0f);
    return;
  }
  const Scale s = scale_of(top, a, V, table);
  const T* const logits = reinterpret_cast<const T*>(p.s.logits) + row * p.s.row_stride;
  Cut cut{kBins, kBins, kBins, 0, 0, 0, 0};
  Last last{0, false};
  if (a.cuts) {
    cut = *r.cut;
    const uint32_t n = *r.listed;
    if (n <= (uint32_t)kList) {
      for (int i = tid; i < (int)n; i += NT) ls.list[i] = r.list[i];
      if (a.counted) {
        __syncthreads();
        if (n > 64) draw_of_list<NT, kList>(ls, (int)n, a, s, p.s, row, sums);
        else if (tid < 64) draw_of_list<64, 64>(ls, (int)n, a, s, p.s, row, sums);
        return;
      }
    }
    for (int c = tid; c < parts; c += NT) part[c] = r.part_mass[c];
    __syncthreads();
    if (n > (uint32_t)kList) {
      last = last_of_row<NT>(ls, sums, found, logits, V, cut, a, s);
      __syncthreads();
      for (int c = 0; c < parts; ++c) {    // the kept ones among those in doubt, part by part
        float x[kPer];
        const int split = c / p.sp.steps, i0 = split * p.sp.length + (c - split * p.sp.steps) * kPart + tid * kPer;
        load(logits, i0, min((split + 1) * p.sp.length, V), x);
        u64 mass = 0, all;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          const int bin = bin_at<kThreads>(s, a.counted, x[e]);
          if (bin < kBins && bin >= sure_bins(cut) && in_doubt(cut, bin) && place_of(x[e], i0 + e) <= last.at)
            mass += mass_over(s, x[e]);
        }
        scan64<NT>(mass, sums, all);
        if (tid == 0) part[c] += all;
      }
    } else if (n) {
      last = last_of_list<NT>(ls, (int)n, cut, a, s, sums);
      for (uint32_t i = tid; i < n; i += NT) {
        const u64 at = ls.sorted[i];
        if (last.some && at <= last.at) atomicAdd(&part[p.sp.part_of((uint32_t)at)], mass_over(s, logit_of((uint32_t)(at >> 32))));
      }
    }
  } else {
    for (int c = tid; c < parts; c += NT) part[c] = r.part_mass[c];
  }
  __syncthreads();
  // the part that holds the drawn mass
  if (tid == 0) found[0] = 0, found[1] = 0;            // (as above)
  constexpr int kEach = kMaxParts / NT;
  u64 mine = 0, total;
#pragma unroll
  for (int i = 0; i < kEach; ++i) mine += tid * kEach + i < parts ? part[tid * kEach + i] : 0;
  u64 before = scan64<NT>(mine, sums, total) - mine;
  const u64 target = target_of(p.s, row, total);
  if (target >= before && target < before + mine) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const u64 m = tid * kEach + i < parts ? part[tid * kEach + i] : 0;
      if (target >= before && target < before + m) found[0] = tid * kEach + i, found[1] = before;
      before += m;
    }
  }
  __syncthreads();
  const int split = (int)found[0] / p.sp.steps;
  const int i0 = split * p.sp.length + ((int)found[0] - split * p.sp.steps) * kPart + tid * kPer;
  before = found[1];
  float x[kPer];
  u64 m[kPer];
  load(logits, i0, min((split + 1) * p.sp.length, V), x);
  mine = 0;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    const int bin = bin_at<kThreads>(s, a.counted, x[e]);
    const bool keep = bin < kBins && (bin < sure_bins(cut) || (last.some && in_doubt(cut, bin) && place_of(x[e], i0 + e) <= last.at));
    m[e] = keep ? mass_over(s, x[e]) : 0;
    mine += m[e];
  }
  u64 all;
  before += scan64<NT>(mine, sums, all) - mine;
  if (target >= before && target < before + mine) {
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      if (target >= before && target < before + m[e]) answer(p.s, row, i0 + e, (float)((double)m[e] / (double)total));
      before += m[e];
    }
  }
}

// Workgroups of a row of V elements, of `rows`: two for each of the 256 CUs and 2048
// elements for each at least.
Split split_of(int rows, int V) {
  Split sp;
  const int most = (V + kPart / 2 - 1) / (kPart / 2), even = rows >= 512 ? 1 : 512 / rows;
  sp.splits = even < most ? even : most;
  if (sp.splits > kMaxSplits) sp.splits = kMaxSplits;
  sp.length = ((V + sp.splits - 1) / sp.splits + kPer - 1) / kPer * kPer;
  sp.splits = (V + sp.length - 1) / sp.length;
  sp.steps = (sp.length + kPart - 1) / kPart;
  return sp;
}

template <typename T>
int launch(const Params& p, hipStream_t stream) {
  const SampleParams& s = p.s;
  const bool greedy = !s.temperatures && !(s.temperature > 0.0f);
  const bool cuts = s.top_ks || s.top_ps || (s.top_k > 0 && s.top_k < s.V) || s.top_p < 1.0f;
  if (s.V <= kRowMax) {
    if (const int rc = check_grid("sample", s.rows, kRowThreads)) return rc;
    hipLaunchKernelGGL(row_kernel<T>, dim3(s.rows), dim3(kRowThreads), 0, stream, s);
    return check_launch("sample");
  }
  if (const int rc = check_grid("sample", (int64_t)p.sp.splits * s.rows, kThreads)) return rc;
  const dim3 grid((unsigned)p.sp.splits * s.rows), block(kThreads);
  hipLaunchKernelGGL(top_kernel<T>, grid, block, 0, stream, p);
  if (!greedy) {
    if (cuts) hipLaunchKernelGGL(histogram_kernel<T>, grid, block, 0, stream, p);
    hipLaunchKernelGGL(masses_kernel<T>, grid, block, 0, stream, p);
  }
  hipLaunchKernelGGL(draw_kernel<T>, dim3(s.rows), block, 0, stream, p);
  return check_launch("sample");
}

}  // namespace

int64_t sample_workspace_bytes(int rows, int V) {
  if (V > kMaxVocab)
    return fail(SLMT_ERR_UNSUPPORTED, "sample: vocabularies of up to 4194304 entries, got " + std::to_string(V)), -1;
  return V <= kRowMax || rows == 0 ? 0 : rows * row_bytes(split_of(rows, V));
}

int launch_sample(int dtype, const SampleParams& s, void* workspace, hipStream_t stream) {
  const Params p{s, split_of(s.rows, s.V), reinterpret_cast<uint8_t*>(workspace)};
  if (dtype == SLMT_F16) return launch<Fp16>(p, stream);
  if (dtype == SLMT_BF16) return launch<Bf16>(p, stream);
  return launch<float>(p, stream);
}

}  // namespace slmt
