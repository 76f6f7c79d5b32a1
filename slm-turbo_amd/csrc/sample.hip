// Sampling of the next token of every row of logits from given uniforms: temperature, top-k, top-p and
// min-p, without sorting the row.
//
// Order a row by logit, largest first, equal ones by index.  With w = exp((l - max l) / T) each cut keeps
// a prefix of that order: the first k; the elements before which lies less than top_p of the first k's
// mass; those with w >= min_p.  The token is the first in index order whose running sum of the kept w
// passes u times the kept mass.
//
// Sums are 64-bit integers, w in units of 2^-(62 - ceil(log2 V)), 2^-52 at most: they hold the whole vocabulary, are
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
// Rows of up to kRowMax elements take one launch, a workgroup per row that holds it in registers.  Longer ones take
// four, each reading the row once at most (the first from memory, the others from the caches):
//   top        the largest logit of every part of kPart elements, and its index
//   histogram  the bins (not where no cut needs them)
//   masses     the cuts' bins, the mass of what is kept for sure in each part, the list of the others
//   draw       one workgroup per row: the cuts, the part, the token
// (The last of a row's workgroups to finish a launch could go on with the next one's work; the fences that this needs
// between the XCDs' caches took longer, 241 us instead of 103 for 64 rows of 151936.)
#include "slmt_internal.h"

namespace slmt {
namespace {

constexpr int kPer = 8;                      // elements of a thread at a time
constexpr int kThreads = 512, kPart = kThreads * kPer;
constexpr int kBins = 4096;                  // (y < 54: at most 3456 are used)
constexpr int kList = 2048, kCounted = 1024;
constexpr int kMaxParts = 1024;              // vocabularies of 2^22 elements
constexpr int kRowThreads = 1024, kRowChunk = kRowThreads * kPer, kRowChunks = 4, kRowMax = kRowChunks * kRowChunk;

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

// A row's place in the workspace.
struct Row {
  u64* mass;               // [kBins]
  u64* part_mass;          // [parts]
  u64* list;               // [kList]: order key, index
  Cut* cut;
  float* top;              // [parts]
  uint32_t* top_at;        // [parts]
  uint32_t* count;         // [kBins]
  uint32_t* listed;
};
__host__ __device__ constexpr int64_t row_bytes(int parts) {
  return (kBins + parts + kList) * 8ll + sizeof(Cut) + parts * 8ll + kBins * 4ll + 8;
}
__device__ __forceinline__ Row row_at(uint8_t* ws, int64_t row, int parts) {
  Row r;
  uint8_t* p = ws + row * ((row_bytes(parts) + 15) & ~15ll);
  r.mass = reinterpret_cast<u64*>(p);
  r.part_mass = r.mass + kBins;
  r.list = r.part_mass + parts;
  r.cut = reinterpret_cast<Cut*>(r.list + kList);
  r.top = reinterpret_cast<float*>(r.cut + 1);
  r.top_at = reinterpret_cast<uint32_t*>(r.top + parts);
  r.count = r.top_at + parts;
  r.listed = r.count + kBins;
  return r;
}

struct Params {
  SampleParams s;
  int parts, splits;       // of a row, and its workgroups
  uint8_t* ws;
};

// Logits i .. i + 7 of a row (those past its end -infinity).  What is no number is never drawn.
template <typename T>
__device__ __forceinline__ void load(const T* row, int i, int V, float* x) {
  T raw[kPer];
  if (i + kPer <= V) {
    __builtin_memcpy(raw, row + i, sizeof(raw));
#pragma unroll
    for (int e = 0; e < kPer; ++e) x[e] = (float)raw[e];
  } else {
#pragma unroll
    for (int e = 0; e < kPer; ++e) x[e] = i + e < V ? (float)row[min(i + e, V - 1)] : -INFINITY;
  }
#pragma unroll
  for (int e = 0; e < kPer; ++e) x[e] = x[e] == x[e] ? x[e] : -INFINITY;
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

// The weights of a row's elements.
struct Scale {
  float top;
  double per;              // 64 y of a distance: 64 log2(e) / T
  double past;             // 64 y from which a weight is nothing
  float bins_per;          // the same as `per`, for bins that hold counts alone
  int shift;               // of w = 1's 53 bits
  const double* table;     // 2^(-j / 64), in LDS
};
// (every thread of the workgroup calls this; a barrier has to follow before the first weight)
__device__ __forceinline__ Scale scale_of(float top, double inv_t, int V, double* table) {
  Scale s;
  const int bits = min(62 - (32 - __builtin_clz((unsigned)max(V - 1, 1))), 52);
  s.top = top;
  s.per = inv_t * (64.0 * 1.4426950408889634074);
  s.past = 64.0 * (bits + 1);
  s.bins_per = (float)s.per;
  s.shift = 53 - bits;
  s.table = table;
  if (threadIdx.x < 64) table[threadIdx.x] = exp2(-(double)threadIdx.x / 64.0);
  return s;
}
constexpr double kRound = 6755399441055744.0;      // 1.5 2^52: adding it leaves the nearest whole number in the low bits
// 64 y of a logit; s.past or more, or no number, where its weight is nothing.
__device__ __forceinline__ double place(const Scale& s, float l) {
  return l == s.top ? 0.0 : ((double)s.top - (double)l) * s.per;
}
struct Weight {
  u64 mass;                // 0: never drawn
  int bin;
  double w;                // to compare with min_p; set where that is wanted
};
__device__ __forceinline__ Weight weight_of(const Scale& s, float l, bool want_w = false) {
  Weight w{0, kBins, 0.0};
  const double y = place(s, l);
  if (y < s.past) {
    const double near = y + kRound;
    const int k = (int)(uint32_t)__builtin_bit_cast(u64, near);
    const double z = (y - (near - kRound)) * (-0.69314718055994530942 / 64.0);     // -0.0055 .. 0.0055
    double e = 1.0 / 120.0;
    e = __builtin_fma(e, z, 1.0 / 24.0);
    e = __builtin_fma(e, z, 1.0 / 6.0);
    e = __builtin_fma(e, z, 0.5);
    e = __builtin_fma(e, z, 1.0);
    const double t = s.table[k & 63];
    e = __builtin_fma(t * z, e, t);                                                // 1/2 .. 1.006
    const u64 u = __builtin_bit_cast(u64, e);
    const int one = (int)(u >> 52) - 1022;                                         // 1 where e is 1 or more
    const int shift = s.shift + (k >> 6) - one;                                    // 0 .. 55
    const u64 m = (u & 0xfffffffffffffull) | 0x10000000000000ull;
    w.mass = ((m << 1 >> shift) + 1) >> 1;
    w.bin = k;
    if (want_w) w.w = __builtin_ldexp(e, -(k >> 6));
  }
  return w;
}
// The mass of an element that min-p lets pass, else 0.
__device__ __forceinline__ u64 mass_over(const Scale& s, float l, double min_p) {
  const Weight w = weight_of(s, l, true);
  return w.w >= min_p ? w.mass : 0;
}
// An element's bin; kBins: never drawn.  Bins that hold counts alone need no more than that they follow the order: fp32's
// roundings do.  (They take elements of no weight too, which are the order's last and never drawn.)
__device__ __forceinline__ int bin_at(const Scale& s, bool counted, float l) {
  if (counted) {
    const float y = l == s.top ? 0.0f : (s.top - l) * s.bins_per;
    return y < (float)(kBins - 1) ? (int)y : kBins;
  }
  const double y = place(s, l);
  return y < s.past ? (int)(uint32_t)__builtin_bit_cast(u64, y + kRound) : kBins;
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
// Inclusive scan over the workgroup of NT threads; `sums`: an entry per wave.  Two barriers.
template <int NT>
__device__ __forceinline__ u64 scan64(u64 v, u64* sums, u64& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  v = wave_scan(v);
  if (lane == 63) sums[wave] = v;
  __syncthreads();
  u64 before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    if (w == wave) before = total;
    total += sums[w];
  }
  __syncthreads();
  return v + before;
}

// The larger logit of two, the lower index of equal ones.
__device__ __forceinline__ void larger(float& m, uint32_t& at, float v, uint32_t a) {
  if (v > m || (v == m && a < at)) m = v, at = a;
}
__device__ __forceinline__ void wave_top(float& m, uint32_t& at) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) larger(m, at, __shfl_xor(m, o, 64), __shfl_xor(at, o, 64));
}
// The row's largest logit and its first index, from the parts.  Every thread of a wave gets it.
__device__ __forceinline__ float top_of(const Row& r, int parts, uint32_t* at = nullptr) {
  float m = -INFINITY;
  uint32_t i = 0xffffffffu;
  for (int c = threadIdx.x & 63; c < parts; c += 64) larger(m, i, r.top[c], r.top_at[c]);
  wave_top(m, i);
  if (at) *at = i;
  return m;
}

// Adds an element to the bins.
__device__ __forceinline__ void add_to_bins(const Scale& s, const Ask& a, float l, u64* mass, uint32_t* count) {
  if (a.counted) {
    const int bin = bin_at(s, true, l);
    if (bin < kBins) atomicAdd(&count[bin], 1u);
    return;
  }
  const Weight w = weight_of(s, l);
  if (w.mass) {
    atomicAdd(&mass[w.bin], w.mass);
    if (a.k) atomicAdd(&count[w.bin], 1u);
  }
}

// The cuts' bins.  `out`: shared; complete after the call.
template <int NT>
__device__ __forceinline__ void find_cut(const u64* mass, const uint32_t* counts, const Ask& a, u64* sums, Cut* out) {
  constexpr int kEach = kBins / NT;
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

// Puts an element that is kept for sure into `mass`, one in doubt on the list.
__device__ __forceinline__ void sort_out(const Scale& s, const Ask& a, const Cut& cut, float l, int i, u64& mass, u64* list,
                                         uint32_t* listed) {
  const int bin = bin_at(s, a.counted, l);
  if (bin < sure_bins(cut)) {
    mass += a.min_p > 0.0 ? mass_over(s, l, a.min_p) : weight_of(s, l).mass;
  } else if (bin < kBins && in_doubt(cut, bin)) {
    const uint32_t at = atomicAdd(listed, 1u);
    if (at < (uint32_t)kList) list[at] = place_of(l, i);
  }
}

// The last kept element in the order; none where `some` is false.
struct Last {
  u64 at;
  bool some;
};

struct Lists {
  u64 list[kList], sorted[kList];
  u64 digit_mass[256];
  uint32_t digit_count[256];
};

// Orders the list: every entry to the place that is the number of those before it (no two are the same).
template <int NT>
__device__ __forceinline__ void order(Lists& ls, int n) {
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += NT) {
    const u64 mine = ls.list[i];
    int before = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) before += ls.list[j] < mine;
    ls.sorted[before] = mine;
  }
  __syncthreads();
}

// The last kept element, from a list of all that are in doubt.
template <int NT>
__device__ __forceinline__ Last last_of_list(Lists& ls, int n, const Cut& cut, const Ask& a, const Scale& s, u64* sums) {
  const int tid = threadIdx.x;
  order<NT>(ls, n);
  // a few entries a thread: their bins and masses
  constexpr int kEach = kList / NT;
  u64 m[kEach];
  int bin[kEach];
  u64 mine = 0, kmine = 0;
  uint32_t earlier = 0;                      // entries of bins before kbin
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int j = tid * kEach + i;
    Weight w{0, kBins, 0.0};
    if (j < n) w = weight_of(s, logit_of((uint32_t)(ls.sorted[j] >> 32)));
    m[i] = w.mass;
    bin[i] = w.bin;
    mine += w.mass;
    earlier += j < n && w.bin < cut.kbin;
  }
  u64 total, first_k = 0;
  if (cut.kbin < kBins) {
    scan64<NT>(earlier, sums, first_k);      // where kbin's entries start
    const u64 end = first_k + (u64)(a.k - cut.kcount);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const u64 j = tid * kEach + i;
      if (j >= first_k && j < end) kmine += m[i];
    }
  }
  u64 chosen;
  scan64<NT>(kmine, sums, chosen);
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
// and min-p, and of those kept the one whose masses before it, by index, the target falls behind.
template <int NT>
__device__ __forceinline__ void draw_of_list(Lists& ls, int n, const Ask& a, const Scale& s, const SampleParams& sp, int row,
                                             u64* sums) {
  const int tid = threadIdx.x;
  order<NT>(ls, n);
  constexpr int kEach = kList / NT;
  u64 m[kEach], mine = 0, total, before;
  bool over[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int j = tid * kEach + i;
    Weight w{0, kBins, 0.0};
    if (j < n && j < a.k) w = weight_of(s, logit_of((uint32_t)(ls.sorted[j] >> 32)), true);
    m[i] = w.mass;
    over[i] = w.mass && w.w >= a.min_p;
    mine += w.mass;
  }
  before = scan64<NT>(mine, sums, total) - mine;
  const double limit = a.top_p * (double)total;
  mine = 0;
  uint32_t kept = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int j = tid * kEach + i;
    const bool keep = over[i] && (a.top_p >= 1.0 || (double)before < limit || j == 0);
    before += m[i];
    if (!keep) m[i] = 0;
    mine += m[i];
    kept += keep;
  }
  u64 some;
  scan64<NT>(kept, sums, some);
  scan64<NT>(mine, sums, total);
  // (the kept ones are the first of the order: their masses and indices take the unordered list's place)
#pragma unroll
  for (int i = 0; i < kEach; ++i) ls.list[tid * kEach + i] = m[i];
  __syncthreads();
  const u64 target = target_of(sp, row, total);
  for (int i = tid; i < (int)some; i += NT) {
    const uint32_t at = (uint32_t)ls.sorted[i];
    const u64 own = ls.list[i];
    u64 sum = 0;
#pragma unroll 4
    for (int j = 0; j < (int)some; ++j) sum += (uint32_t)ls.sorted[j] < at ? ls.list[j] : 0;
    if (target >= sum && target < sum + own) answer(sp, row, at, (float)((double)own / (double)total));
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
        const int bin = bin_at(s, counted, x[e]);
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
  if (a.counted) {                           // (the masses that the counts left out)
    u64 mine = 0, more = 0;
    for (int i0 = tid * kPer; i0 < V; i0 += NT * kPer) {
      float x[kPer];
      load(logits, i0, V, x);
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const int bin = bin_at(s, true, x[e]);
        if (bin < cut.kbin) mine += weight_of(s, x[e]).mass;
        more += bin <= cut.kbin;
      }
    }
    u64 drawable;
    scan64<NT>(mine, sums, cut.kmass);
    scan64<NT>(more, sums, drawable);
    if (drawable < (u64)a.k) cut.kbin = kBins;           // (fewer than k: no such cut)
    if (cut.kbin == kBins) {
      u64 rest = 0;
      for (int i0 = tid * kPer; i0 < V; i0 += NT * kPer) {
        float x[kPer];
        load(logits, i0, V, x);
#pragma unroll
        for (int e = 0; e < kPer; ++e) rest += weight_of(s, x[e]).mass;
      }
      scan64<NT>(rest, sums, kmass);
    }
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

template <typename T>
__global__ void __launch_bounds__(kRowThreads) row_kernel(const SampleParams sp) {
  constexpr int NT = kRowThreads, kWaves = NT / 64;
  __shared__ RowShared sh;
  const int row = blockIdx.x, tid = threadIdx.x, wave = tid >> 6, V = sp.V;
  const Ask a = ask_of(sp, row);
  const T* const logits = reinterpret_cast<const T*>(sp.logits) + row * sp.row_stride;
  // element e of chunk c: index c * kRowChunk + tid * kPer + e
  const int chunks = (V + kRowChunk - 1) / kRowChunk;
  float x[kRowChunks][kPer];
#pragma unroll
  for (int c = 0; c < kRowChunks; ++c)
    if (c < chunks) load(logits, c * kRowChunk + tid * kPer, V, x[c]);
  if (a.cuts && !a.greedy)
    for (int b = tid; b < kBins; b += NT) sh.bins.mass[b] = 0, sh.bins.count[b] = 0;
  float m = -INFINITY;
  uint32_t at = min(tid * kPer, V - 1);
#pragma unroll
  for (int c = 0; c < kRowChunks; ++c)
    if (c < chunks) {
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        if (x[c][e] > m) m = x[c][e], at = c * kRowChunk + tid * kPer + e;
    }
  wave_top(m, at);
  if ((tid & 63) == 0) sh.ms[wave] = m, sh.is[wave] = at;
  if (tid == 0) sh.listed = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) larger(m, at, sh.ms[w], sh.is[w]);
  if (a.greedy || m == -INFINITY) {
    if (tid == 0) answer(sp, row, at, m == -INFINITY ? 0.0f : 1.0f);
    return;
  }
  const Scale s = scale_of(m, a.inv_t, V, sh.table);
  __syncthreads();
  Cut cut{kBins, kBins, kBins, 0, 0, 0, 0};
  if (a.cuts) {
#pragma unroll
    for (int c = 0; c < kRowChunks; ++c)
      if (c < chunks) {
#pragma unroll
        for (int e = 0; e < kPer; ++e) add_to_bins(s, a, x[c][e], sh.bins.mass, sh.bins.count);
      }
    __syncthreads();
    find_cut<NT>(sh.bins.mass, sh.bins.count, a, sh.sums, &sh.cut);
    cut = sh.cut;
    __syncthreads();                         // (the lists take the bins' place)
  }
  u64 mass[kRowChunks] = {};
#pragma unroll
  for (int c = 0; c < kRowChunks; ++c)
    if (c < chunks) {
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        sort_out(s, a, cut, x[c][e], c * kRowChunk + tid * kPer + e, mass[c], sh.lists.list, &sh.listed);
    }
  __syncthreads();
  const uint32_t n = sh.listed;
  if (a.counted && n <= (uint32_t)kList) {
    draw_of_list<NT>(sh.lists, (int)n, a, s, sp, row, sh.sums);
    return;
  }
  Last last{0, false};
  if (n > (uint32_t)kList) last = last_of_row<NT>(sh.lists, sh.sums, sh.found, logits, V, cut, a, s);
  else if (n) last = last_of_list<NT>(sh.lists, (int)n, cut, a, s, sh.sums);
  // every thread's kept mass of each chunk, and its waves' sums
  auto kept = [&](float l, int i, bool sure) {           // (of those in doubt, and with `sure` of the others)
    const int bin = bin_at(s, a.counted, l);
    const bool keep = bin < sure_bins(cut) ? sure : bin < kBins && last.some && in_doubt(cut, bin) && place_of(l, i) <= last.at;
    return keep ? mass_over(s, l, a.min_p) : 0ull;
  };
#pragma unroll
  for (int c = 0; c < kRowChunks; ++c) {
    if (c < chunks && last.some) {
#pragma unroll
      for (int e = 0; e < kPer; ++e) mass[c] += kept(x[c][e], c * kRowChunk + tid * kPer + e, false);
    }
    const u64 sum = wave_scan(mass[c]);
    if ((tid & 63) == 63) sh.part[c * kWaves + wave] = sum;
  }
  __syncthreads();
  u64 total;
  const u64 own = tid < kRowChunks * kWaves ? sh.part[tid] : 0;
  const u64 end = scan64<NT>(own, sh.sums, total);
  const u64 target = target_of(sp, row, total);
  if (target >= end - own && target < end) sh.found[0] = tid, sh.found[1] = end - own;
  __syncthreads();
  if (wave != (int)sh.found[0] % kWaves) return;
  // the wave that holds it
  const int chunk = (int)sh.found[0] / kWaves;
#pragma unroll
  for (int c = 0; c < kRowChunks; ++c)
    if (c == chunk) {
      u64 before = sh.found[1] + wave_scan(mass[c]) - mass[c];
      if (target >= before && target < before + mass[c]) {
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          const int i = c * kRowChunk + tid * kPer + e;
          const u64 w = kept(x[c][e], i, true);
          if (target >= before && target < before + w) answer(sp, row, i, (float)((double)w / (double)total));
          before += w;
        }
      }
    }
}

// ------------------------------------------------------------------ longer rows
template <typename T>
__global__ void __launch_bounds__(kThreads) top_kernel(const Params p) {
  constexpr int kWaves = kThreads / 64;
  __shared__ float ms[kWaves];
  __shared__ uint32_t is[kWaves];
  const int row = blockIdx.x / p.splits, split = blockIdx.x - row * p.splits, tid = threadIdx.x;
  const Row r = row_at(p.ws, row, p.parts);
  // (the bins and the list start empty; this is the first launch of the call)
  for (int b = split * kThreads + tid; b < kBins; b += p.splits * kThreads) r.mass[b] = 0, r.count[b] = 0;
  if (split == 0 && tid == 0) *r.listed = 0;
  const T* const logits = reinterpret_cast<const T*>(p.s.logits) + row * p.s.row_stride;
  float x[kPer];
  load(logits, split * kPart + tid * kPer, p.s.V, x);
  for (int c = split; c < p.parts; c += p.splits) {
    float next[kPer];
    if (c + p.splits < p.parts) load(logits, (c + p.splits) * kPart + tid * kPer, p.s.V, next);
    float m = -INFINITY;
    uint32_t at = min(c * kPart + tid * kPer, p.s.V - 1);
#pragma unroll
    for (int e = 0; e < kPer; ++e)
      if (x[e] > m) m = x[e], at = c * kPart + tid * kPer + e;
    wave_top(m, at);
    if ((tid & 63) == 0) ms[tid >> 6] = m, is[tid >> 6] = at;
    __syncthreads();
    if (tid == 0) {
#pragma unroll
      for (int w = 1; w < kWaves; ++w) larger(m, at, ms[w], is[w]);
      r.top[c] = m;
      r.top_at[c] = at;
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kPer; ++e) x[e] = next[e];
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) histogram_kernel(const Params p) {
  __shared__ u64 mass[kBins];
  __shared__ uint32_t count[kBins];
  __shared__ double table[64];
  const int row = blockIdx.x / p.splits, split = blockIdx.x - row * p.splits, tid = threadIdx.x;
  const Ask a = ask_of(p.s, row);
  if (a.greedy || !a.cuts) return;
  const Row r = row_at(p.ws, row, p.parts);
  const T* const logits = reinterpret_cast<const T*>(p.s.logits) + row * p.s.row_stride;
  float x[kPer];
  load(logits, split * kPart + tid * kPer, p.s.V, x);
  const Scale s = scale_of(top_of(r, p.parts), a.inv_t, p.s.V, table);
  if (s.top == -INFINITY) return;
  for (int b = tid; b < kBins; b += kThreads) mass[b] = 0, count[b] = 0;
  __syncthreads();
  for (int c = split; c < p.parts; c += p.splits) {
    float next[kPer];
    if (c + p.splits < p.parts) load(logits, (c + p.splits) * kPart + tid * kPer, p.s.V, next);
#pragma unroll
    for (int e = 0; e < kPer; ++e) add_to_bins(s, a, x[e], mass, count);
#pragma unroll
    for (int e = 0; e < kPer; ++e) x[e] = next[e];
  }
  __syncthreads();
  for (int b = tid; b < kBins; b += kThreads) {
    if (!a.counted && mass[b]) atomicAdd(&r.mass[b], mass[b]);
    if (a.k && count[b]) atomicAdd(&r.count[b], count[b]);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) masses_kernel(const Params p) {
  __shared__ u64 sums[kThreads / 64];
  __shared__ double table[64];
  __shared__ Cut shared_cut;
  const int row = blockIdx.x / p.splits, split = blockIdx.x - row * p.splits, tid = threadIdx.x;
  const Ask a = ask_of(p.s, row);
  if (a.greedy) return;
  const Row r = row_at(p.ws, row, p.parts);
  const T* const logits = reinterpret_cast<const T*>(p.s.logits) + row * p.s.row_stride;
  float x[kPer];
  load(logits, split * kPart + tid * kPer, p.s.V, x);
  const Scale s = scale_of(top_of(r, p.parts), a.inv_t, p.s.V, table);
  if (s.top == -INFINITY) return;
  Cut cut{kBins, kBins, kBins, 0, 0, 0, 0};
  if (a.cuts) {
    find_cut<kThreads>(r.mass, r.count, a, sums, &shared_cut);
    cut = shared_cut;
    if (split == 0 && tid == 0) *r.cut = cut;
  }
  __syncthreads();
  for (int c = split; c < p.parts; c += p.splits) {
    float next[kPer];
    if (c + p.splits < p.parts) load(logits, (c + p.splits) * kPart + tid * kPer, p.s.V, next);
    u64 mass = 0, total;
#pragma unroll
    for (int e = 0; e < kPer; ++e) sort_out(s, a, cut, x[e], c * kPart + tid * kPer + e, mass, r.list, r.listed);
    if (sure_bins(cut) > 0) {
      scan64<kThreads>(mass, sums, total);
      if (tid == 0) r.part_mass[c] = total;
    } else if (tid == 0) {
      r.part_mass[c] = 0;
    }
#pragma unroll
    for (int e = 0; e < kPer; ++e) x[e] = next[e];
  }
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
  const Row r = row_at(p.ws, row, p.parts);
  uint32_t top_at;
  const float top = top_of(r, p.parts, &top_at);
  if (a.greedy || top == -INFINITY) {
    // (the parts' first indices: 0 for a row that leaves nothing)
    if (tid == 0) answer(p.s, row, top_at, top == -INFINITY ? 0.0f : 1.0f);
    return;
  }
  const Scale s = scale_of(top, a.inv_t, V, table);
  const T* const logits = reinterpret_cast<const T*>(p.s.logits) + row * p.s.row_stride;
  Cut cut{kBins, kBins, kBins, 0, 0, 0, 0};
  Last last{0, false};
  if (a.cuts) {
    cut = *r.cut;
    const uint32_t n = *r.listed;
    if (n <= (uint32_t)kList) {
      for (int i = tid; i < (int)n; i += NT) ls.list[i] = r.list[i];
      if (a.counted) {
        draw_of_list<NT>(ls, (int)n, a, s, p.s, row, sums);
        return;
      }
    }
    for (int c = tid; c < p.parts; c += NT) part[c] = r.part_mass[c];
    __syncthreads();
    if (n > (uint32_t)kList) {
      last = last_of_row<NT>(ls, sums, found, logits, V, cut, a, s);
      __syncthreads();
      for (int c = 0; c < p.parts; ++c) {    // the kept ones among those in doubt, part by part
        float x[kPer];
        const int i0 = c * kPart + tid * kPer;
        load(logits, i0, V, x);
        u64 mass = 0, all;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          const int bin = bin_at(s, a.counted, x[e]);
          if (bin < kBins && bin >= sure_bins(cut) && in_doubt(cut, bin) && place_of(x[e], i0 + e) <= last.at)
            mass += mass_over(s, x[e], a.min_p);
        }
        scan64<NT>(mass, sums, all);
        if (tid == 0) part[c] += all;
      }
    } else if (n) {
      last = last_of_list<NT>(ls, (int)n, cut, a, s, sums);
      for (uint32_t i = tid; i < n; i += NT) {
        const u64 at = ls.sorted[i];
        if (last.some && at <= last.at) atomicAdd(&part[(uint32_t)at / kPart], mass_over(s, logit_of((uint32_t)(at >> 32)), a.min_p));
      }
    }
  } else {
    for (int c = tid; c < p.parts; c += NT) part[c] = r.part_mass[c];
  }
  __syncthreads();
  // the part that holds the drawn mass
  constexpr int kEach = kMaxParts / NT;
  u64 mine = 0, total;
#pragma unroll
  for (int i = 0; i < kEach; ++i) mine += tid * kEach + i < p.parts ? part[tid * kEach + i] : 0;
  u64 before = scan64<NT>(mine, sums, total) - mine;
  const u64 target = target_of(p.s, row, total);
  if (target >= before && target < before + mine) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const u64 m = tid * kEach + i < p.parts ? part[tid * kEach + i] : 0;
      if (target >= before && target < before + m) found[0] = tid * kEach + i, found[1] = before;
      before += m;
    }
  }
  __syncthreads();
  const int i0 = (int)found[0] * kPart + tid * kPer;
  before = found[1];
  float x[kPer];
  u64 m[kPer];
  load(logits, i0, V, x);
  mine = 0;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    const int bin = bin_at(s, a.counted, x[e]);
    const bool keep = bin < kBins && (bin < sure_bins(cut) || (last.some && in_doubt(cut, bin) && place_of(x[e], i0 + e) <= last.at));
    m[e] = keep ? mass_over(s, x[e], a.min_p) : 0;
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

template <typename T>
int launch(Params p, hipStream_t stream) {
  const SampleParams& s = p.s;
  const bool greedy = !s.temperatures && !(s.temperature > 0.0f);
  const bool cuts = s.top_ks || s.top_ps || (s.top_k > 0 && s.top_k < s.V) || s.top_p < 1.0f;
  if (s.V <= kRowMax) {
    hipLaunchKernelGGL(row_kernel<T>, dim3(s.rows), dim3(kRowThreads), 0, stream, s);
    return check_launch("sample");
  }
  // about four workgroups for each of the 256 CUs, a part for each at least
  p.splits = s.rows >= 1024 ? 1 : min(p.parts, (1024 + s.rows - 1) / s.rows);
  const dim3 grid((unsigned)p.splits * s.rows), block(kThreads);
  hipLaunchKernelGGL(top_kernel<T>, grid, block, 0, stream, p);
  if (!greedy) {
    if (cuts) hipLaunchKernelGGL(histogram_kernel<T>, grid, block, 0, stream, p);
    hipLaunchKernelGGL(masses_kernel<T>, grid, block, 0, stream, p);
  }
  hipLaunchKernelGGL(draw_kernel<T>, dim3(s.rows), block, 0, stream, p);
  return check_launch("sample");
}

int parts_of(int V) { return (V + kPart - 1) / kPart; }

}  // namespace

int64_t sample_workspace_bytes(int rows, int V) {
  if (V > kMaxParts * kPart)
    return fail(SLMT_ERR_UNSUPPORTED, "sample: vocabularies of up to 4194304 entries, got " + std::to_string(V)), -1;
  return V <= kRowMax ? 0 : rows * ((row_bytes(parts_of(V)) + 15) & ~15ll);
}

int launch_sample(int dtype, const SampleParams& s, void* workspace, hipStream_t stream) {
  Params p{s, parts_of(s.V), 1, reinterpret_cast<uint8_t*>(workspace)};
  if (dtype == SLMT_F16) return launch<Fp16>(p, stream);
  if (dtype == SLMT_BF16) return launch<Bf16>(p, stream);
  return launch<float>(p, stream);
}

}  // namespace slmt
