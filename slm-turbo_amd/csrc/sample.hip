// Sampling of the next token of every row of logits from given uniforms: temperature, top-k, top-p and
// min-p, without sorting the row.
//
// Order a row by logit, largest first, equal ones by index.  With w = exp((l - max l) / T) each cut keeps
// a prefix of that order: the first k; the elements before which lies less than top_p of the first k's
// mass; those with w >= min_p.  The token is the first in index order whose running sum of the kept w
// passes u times the kept mass.
//
// Sums are 64-bit integers, w in units of 2^-(62 - ceil(log2 V)): they hold the whole vocabulary, are
// the same in whatever order they are formed, and an element below half a unit, which no uniform could
// reach, is nothing.  w itself is formed in fp64: over 10^5 elements the fp32 sums' errors move the token
// in one row of a hundred.
//
// Four launches, each reading the row once at most (the first from memory, the others from the caches):
//   top        the largest logit of every part of kPart elements, and its index
//   histogram  counts and masses of kBins bins of equal width in (max l - l) / T
//   masses     from the bins: which elements are kept whatever happens within a bin, and which are in
//              the bins where a cut falls; the mass of the former for each part, a list of the latter
//   draw       one workgroup per row sorts that list, finds the cuts, then the part and the token
// A list that overflows (more than kList elements in the cuts' bins, as in a row of equal logits) is not
// used: the row's workgroup then finds the cuts digit by digit of the logits' bits, reading the row again.
// A call without top-k and top-p takes no histogram; T = 0 alone takes the first and the last.
#include "slmt_internal.h"

namespace slmt {
namespace {

constexpr int kThreads = 512, kPer = 8, kPart = kThreads * kPer;
constexpr int kBins = 4096, kList = 2048, kWaves = kThreads / 64;
constexpr int kMaxParts = 1024;              // vocabularies of 2^22 elements

typedef unsigned long long u64;
typedef __bf16 Bf16;
typedef _Float16 Fp16;

struct Cut {               // what the bins say of a row's cuts
  int low, high;           // bins of the top-p cut (kBins: no such cut); every element of a bin before `low` passes it
  int kbin;                // bin of the k-th element (kBins: no such cut)
  uint32_t kcount;         // elements before kbin
  u64 kmass, lowmass;      // masses before kbin and before low
  u64 total;               // of the row
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
  int parts, splits;       // workgroups of a row (but in the last launch)
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

// What a row's call asks for.
struct Ask {
  double inv_t, min_p, top_p;
  int k;                   // 0: no cut
  bool greedy;
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
  return a;
}

// The weights of a row's elements.
struct Scale {
  float top;
  double inv_t, unit, past, per;   // units of 1; distance from which a weight is nothing; bins per distance
};
__device__ __forceinline__ Scale scale_of(float top, double inv_t, int V) {
  Scale s;
  const int bits = 62 - (32 - __builtin_clz((unsigned)max(V - 1, 1)));
  s.top = top;
  s.inv_t = inv_t;
  s.unit = __builtin_ldexp(1.0, bits);
  s.past = (bits + 1) * 0.69314718055994530942;
  s.per = kBins / s.past;
  return s;
}
struct Weight {
  u64 mass;                // 0: never drawn
  int bin;
  bool over;               // w >= min_p
};
__device__ __forceinline__ Weight weight_of(const Scale& s, float l, double min_p) {
  Weight w{0, kBins, false};
  const double d = l == s.top ? 0.0 : ((double)s.top - (double)l) * s.inv_t;
  if (d < s.past) {
    const double e = exp(-d);
    w.mass = (u64)__builtin_rint(e * s.unit);
    w.bin = min((int)(d * s.per), kBins - 1);
    w.over = e >= min_p;
  }
  return w;
}

__device__ __forceinline__ u64 shfl_up64(u64 v, int o) {
  return ((u64)__shfl_up((uint32_t)(v >> 32), o, 64) << 32) | __shfl_up((uint32_t)v, o, 64);
}
// Inclusive scan over the workgroup; `sums`: kWaves entries.  Two barriers.
__device__ __forceinline__ u64 scan64(u64 v, u64* sums, u64& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const u64 u = shfl_up64(v, o);
    if (lane >= o) v += u;
  }
  if (lane == 63) sums[wave] = v;
  __syncthreads();
  u64 before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w == wave) before = total;
    total += sums[w];
  }
  __syncthreads();
  return v + before;
}

// The row's largest logit and its first index, from the parts.  Every thread of a wave gets it.
__device__ __forceinline__ float top_of(const Row& r, int parts, uint32_t* at = nullptr) {
  const int lane = threadIdx.x & 63;
  float m = -INFINITY;
  uint32_t i = 0xffffffffu;
  for (int c = lane; c < parts; c += 64) {
    const float v = r.top[c];
    const uint32_t a = r.top_at[c];
    if (v > m || (v == m && a < i)) m = v, i = a;
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const float v = __shfl_xor(m, o, 64);
    const uint32_t a = __shfl_xor(i, o, 64);
    if (v > m || (v == m && a < i)) m = v, i = a;
  }
  if (at) *at = i;
  return m;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) top_kernel(const Params p) {
  __shared__ float ms[kWaves];
  __shared__ uint32_t is[kWaves];
  const int row = blockIdx.x / p.splits, split = blockIdx.x - row * p.splits, tid = threadIdx.x;
  const Row r = row_at(p.ws, row, p.parts);
  // (the bins and the list start empty; this is the first launch of the call)
  for (int b = split * kThreads + tid; b < kBins; b += p.splits * kThreads) r.mass[b] = 0, r.count[b] = 0;
  if (split == 0 && tid == 0) *r.listed = 0;
  const T* const logits = reinterpret_cast<const T*>(p.s.logits) + row * p.s.row_stride;
  for (int c = split; c < p.parts; c += p.splits) {
    const int i0 = c * kPart + tid * kPer;
    float x[kPer], m = -INFINITY;
    uint32_t at = min(i0, p.s.V - 1);
    load(logits, i0, p.s.V, x);
#pragma unroll
    for (int e = 0; e < kPer; ++e)
      if (x[e] > m) m = x[e], at = i0 + e;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const float v = __shfl_xor(m, o, 64);
      const uint32_t a = __shfl_xor(at, o, 64);
      if (v > m || (v == m && a < at)) m = v, at = a;
    }
    if ((tid & 63) == 0) ms[tid >> 6] = m, is[tid >> 6] = at;
    __syncthreads();
    if (tid == 0) {
#pragma unroll
      for (int w = 1; w < kWaves; ++w)
        if (ms[w] > m || (ms[w] == m && is[w] < at)) m = ms[w], at = is[w];
      r.top[c] = m;
      r.top_at[c] = at;
    }
    __syncthreads();
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) histogram_kernel(const Params p) {
  __shared__ u64 mass[kBins];
  __shared__ uint32_t count[kBins];
  const int row = blockIdx.x / p.splits, split = blockIdx.x - row * p.splits, tid = threadIdx.x;
  const Ask a = ask_of(p.s, row);
  if (a.greedy || (a.k == 0 && a.top_p >= 1.0)) return;
  const Row r = row_at(p.ws, row, p.parts);
  const Scale s = scale_of(top_of(r, p.parts), a.inv_t, p.s.V);
  if (s.top == -INFINITY) return;
  for (int b = tid; b < kBins; b += kThreads) mass[b] = 0, count[b] = 0;
  __syncthreads();
  const T* const logits = reinterpret_cast<const T*>(p.s.logits) + row * p.s.row_stride;
  for (int c = split; c < p.parts; c += p.splits) {
    float x[kPer];
    load(logits, c * kPart + tid * kPer, p.s.V, x);
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const Weight w = weight_of(s, x[e], 0.0);
      if (w.mass) {
        atomicAdd(&mass[w.bin], w.mass);
        atomicAdd(&count[w.bin], 1u);
      }
    }
  }
  __syncthreads();
  for (int b = tid; b < kBins; b += kThreads)
    if (count[b]) {
      atomicAdd(&r.mass[b], mass[b]);
      atomicAdd(&r.count[b], count[b]);
    }
}

// The cuts' bins.  `sums`: kWaves entries; `out`: shared.  Every thread returns the same.
__device__ __forceinline__ Cut find_cut(const Row& r, const Ask& a, u64* sums, Cut* out) {
  constexpr int kEach = kBins / kThreads;
  const int tid = threadIdx.x;
  u64 m[kEach];
  uint32_t n[kEach];
  u64 mine = 0, count = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    m[i] = r.mass[tid * kEach + i];
    n[i] = r.count[tid * kEach + i];
    mine += m[i];
    count += n[i];
  }
  u64 total, counted;
  u64 before = scan64(mine, sums, total) - mine;
  u64 nbefore = scan64(count, sums, counted) - count;
  if (tid == 0) *out = Cut{kBins, kBins, kBins, 0, total, 0, total};
  __syncthreads();
  // the bin of the k-th element (none where fewer than k can be drawn)
  if (a.k && nbefore < (u64)a.k && nbefore + count >= (u64)a.k) {
    u64 mm = before, nn = nbefore;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if (nn < (u64)a.k && nn + n[i] >= (u64)a.k) {
        out->kbin = tid * kEach + i;
        out->kcount = (uint32_t)nn;
        out->kmass = mm;
        out->lowmass = mm + m[i];       // (for the next step: the mass up to its end)
      }
      nn += n[i];
      mm += m[i];
    }
  }
  __syncthreads();
  if (a.top_p < 1.0) {
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
        out->low = tid * kEach + i;
        out->lowmass = mm;
      }
      if ((double)end >= most && (first || (double)mm < most)) out->high = tid * kEach + i;
      mm = end;
    }
  }
  __syncthreads();
  return *out;
}

// Whether an element of this bin may or may not be kept, as the cuts fall within the bin.
__device__ __forceinline__ bool in_doubt(const Cut& c, int bin) { return (bin >= c.low && bin <= c.high) || bin == c.kbin; }

template <typename T>
__global__ void __launch_bounds__(kThreads) masses_kernel(const Params p) {
  __shared__ u64 sums[kWaves];
  __shared__ Cut shared_cut;
  const int row = blockIdx.x / p.splits, split = blockIdx.x - row * p.splits, tid = threadIdx.x;
  const Ask a = ask_of(p.s, row);
  if (a.greedy) return;
  const Row r = row_at(p.ws, row, p.parts);
  const Scale s = scale_of(top_of(r, p.parts), a.inv_t, p.s.V);
  if (s.top == -INFINITY) return;
  Cut cut{kBins, kBins, kBins, 0, 0, 0, 0};
  if (a.k || a.top_p < 1.0) {
    cut = find_cut(r, a, sums, &shared_cut);
    if (split == 0 && tid == 0) *r.cut = cut;
  }
  const int sure = min(cut.low, cut.kbin);
  const T* const logits = reinterpret_cast<const T*>(p.s.logits) + row * p.s.row_stride;
  for (int c = split; c < p.parts; c += p.splits) {
    const int i0 = c * kPart + tid * kPer;
    float x[kPer];
    load(logits, i0, p.s.V, x);
    u64 mass = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const Weight w = weight_of(s, x[e], a.min_p);
      if (w.mass && w.bin < sure && w.over) mass += w.mass;
      const bool doubt = w.mass && in_doubt(cut, w.bin);
      if (doubt) {
        const uint32_t at = atomicAdd(r.listed, 1u);
        if (at < (uint32_t)kList) r.list[at] = ((u64)order_key(x[e]) << 32) | (uint32_t)(i0 + e);
      }
    }
    u64 total;
    scan64(mass, sums, total);
    if (tid == 0) r.part_mass[c] = total;
  }
}

// The last kept element in the order: key and index; none where `some` is false.
struct Last {
  u64 at;
  bool some;
};

struct Shared {
  u64 list[kList];
  u64 part[kMaxParts];
  u64 digit_mass[256];
  uint32_t digit_count[256];
  u64 sums[kWaves];
  u64 found[4];
};

// Sorts the first n entries (a power of two).
__device__ __forceinline__ void sort(u64* v, int n) {
  for (int k = 2; k <= n; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      for (int i = threadIdx.x; i < n / 2; i += kThreads) {
        const int lo = 2 * i - (i & (j - 1)), hi = lo + j;
        const u64 x = v[lo], y = v[hi];
        if ((x > y) == ((lo & k) == 0)) v[lo] = y, v[hi] = x;
      }
      __syncthreads();
    }
}

// The last kept element, from a list of all that are in doubt.
__device__ __forceinline__ Last last_of_list(Shared& sh, const Row& r, int n, const Cut& cut, const Ask& a, const Scale& s) {
  const int tid = threadIdx.x;
  int size = 2;
  while (size < n) size <<= 1;
  for (int i = tid; i < size; i += kThreads) sh.list[i] = i < n ? r.list[i] : ~0ull;
  if (tid < 4) sh.found[tid] = 0;
  __syncthreads();
  sort(sh.list, size);
  // four entries a thread: their bins and masses
  constexpr int kEach = kList / kThreads;
  u64 m[kEach];
  int bin[kEach];
  u64 mine = 0, kmine = 0;
  uint32_t earlier = 0;                      // entries of bins before kbin
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int j = tid * kEach + i;
    Weight w{0, kBins, false};
    if (j < n) w = weight_of(s, logit_of((uint32_t)(sh.list[j] >> 32)), 0.0);
    m[i] = w.mass;
    bin[i] = w.bin;
    mine += w.mass;
    earlier += j < n && w.bin < cut.kbin;
  }
  u64 total, first_k = 0;
  if (cut.kbin < kBins) {
    scan64(earlier, sh.sums, first_k);       // where kbin's entries start
    const u64 end = first_k + (u64)(a.k - cut.kcount);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const u64 j = tid * kEach + i;
      if (j >= first_k && j < end) kmine += m[i];
    }
  }
  u64 chosen;
  scan64(kmine, sh.sums, chosen);
  const u64 kmass = cut.kbin < kBins ? cut.kmass + chosen : cut.total;
  const double limit = a.top_p * (double)kmass;
  u64 before = scan64(mine, sh.sums, total) - mine + cut.lowmass;
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
  scan64(kept, sh.sums, all);
  Last last{0, all > 0};
  if (all) last.at = sh.list[all - 1];
  return last;
}

// The same from the row itself, digit by digit of the order key.  Finds the key at which the running count
// (by_count) or mass of the elements in bins first .. last reaches `want`, and what lies before that key.
struct Digits {
  uint32_t key;
  uint32_t ties;           // elements of that key
  u64 count, mass;         // before it, from the given start on
};
template <typename T>
__device__ __forceinline__ Digits descend(Shared& sh, const T* logits, int V, const Scale& s, int first, int last, bool by_count,
                                          u64 count0, u64 mass0, u64 want_count, double want_mass) {
  const int tid = threadIdx.x;
  Digits d{0, 0, count0, mass0};
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int b = tid; b < 256; b += kThreads) sh.digit_mass[b] = 0, sh.digit_count[b] = 0;
    __syncthreads();
    for (int i0 = tid * kPer; i0 < V; i0 += kPart) {
      float x[kPer];
      load(logits, i0, V, x);
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const uint32_t key = order_key(x[e]);
        if (shift < 24 && (key >> (shift + 8)) != (d.key >> (shift + 8))) continue;
        const Weight w = weight_of(s, x[e], 0.0);
        if (w.mass == 0 || w.bin < first || w.bin > last) continue;
        atomicAdd(&sh.digit_count[(key >> shift) & 255], 1u);
        atomicAdd(&sh.digit_mass[(key >> shift) & 255], w.mass);
      }
    }
    __syncthreads();
    u64 all;
    const u64 m = tid < 256 ? sh.digit_mass[tid] : 0, c = tid < 256 ? sh.digit_count[tid] : 0;
    const u64 mend = scan64(m, sh.sums, all) + d.mass, cend = scan64(c, sh.sums, all) + d.count;
    // the first digit that reaches it; where rounding leaves none, the last that has elements
    const bool reaches = c && (by_count ? cend >= want_count : (double)mend >= want_mass);
    const bool before = by_count ? cend - c >= want_count : (double)(mend - m) >= want_mass;
    if (tid == 0) sh.found[0] = 0xffffffffull, sh.found[1] = 0;
    __syncthreads();
    if (reaches && (!before || cend - c == d.count)) atomicMin(&sh.found[0], (u64)tid);
    if (c) atomicMax(&sh.found[1], (u64)tid);
    __syncthreads();
    const uint32_t digit = (uint32_t)(sh.found[0] == 0xffffffffull ? sh.found[1] : sh.found[0]);
    __syncthreads();
    if ((uint32_t)tid == digit) sh.found[0] = cend - c, sh.found[1] = mend - m, sh.found[2] = c;
    __syncthreads();
    d.key |= digit << shift;
    d.count = sh.found[0];
    d.mass = sh.found[1];
    d.ties = (uint32_t)sh.found[2];
    __syncthreads();
  }
  return d;
}

template <typename T>
__device__ __noinline__ Last last_of_row(Shared& sh, const T* logits, int V, const Cut& cut, const Ask& a, const Scale& s) {
  const int tid = threadIdx.x;
  uint32_t key = 0xffffffffu, ties = 0;
  bool some = false;
  u64 kmass = cut.total;
  if (cut.kbin < kBins) {
    const Digits d = descend(sh, logits, V, s, cut.kbin, cut.kbin, true, cut.kcount, cut.kmass, (u64)a.k, 0.0);
    key = d.key;
    ties = (uint32_t)((u64)a.k - d.count);
    some = true;
    kmass = d.mass + ties * weight_of(s, logit_of(key), 0.0).mass;
  }
  if (cut.low < kBins) {
    const double limit = a.top_p * (double)kmass;
    const Digits d = descend(sh, logits, V, s, cut.low, cut.high, false, 0, cut.lowmass, 0, limit);
    // of its ties, those before which lies less than the limit (the row's first element in any case)
    const u64 each = weight_of(s, logit_of(d.key), 0.0).mass;
    uint32_t lo = cut.low == 0 && d.count == 0 ? 1 : 0, hi = d.ties;
    while (lo < hi) {
      const uint32_t mid = (lo + hi + 1) / 2;
      if ((double)(d.mass + (mid - 1) * each) < limit) lo = mid;
      else hi = mid - 1;
    }
    if (!some || d.key < key || (d.key == key && lo < ties)) key = d.key, ties = lo;
    some = true;
  }
  // the index of the last of its ties
  Last last{(u64)key << 32, some};
  if (ties == 0) {
    // (no tie of this key: the element before it is the last, and every index of a smaller key passes)
    last.at = ((u64)key << 32) - 1;
    return last;
  }
  u64 seen = 0;
  for (int c = 0; c < V; c += kPart) {
    float x[kPer];
    load(logits, c + tid * kPer, V, x);
    u64 mine = 0, all;
#pragma unroll
    for (int e = 0; e < kPer; ++e) mine += order_key(x[e]) == key && c + tid * kPer + e < V;
    u64 at = seen + scan64(mine, sh.sums, all) - mine;
    if (seen < ties && seen + all >= ties) {
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        if (order_key(x[e]) == key && c + tid * kPer + e < V && ++at == ties) sh.found[3] = c + tid * kPer + e;
    }
    seen += all;
    __syncthreads();
    if (seen >= ties) break;
  }
  last.at |= sh.found[3];
  return last;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) draw_kernel(const Params p) {
  __shared__ Shared sh;
  const int row = blockIdx.x, tid = threadIdx.x, V = p.s.V;
  const Ask a = ask_of(p.s, row);
  const Row r = row_at(p.ws, row, p.parts);
  uint32_t top_at;
  const float top = top_of(r, p.parts, &top_at);
  if (a.greedy || top == -INFINITY) {
    // (the parts' first indices: 0 for a row that leaves nothing)
    if (tid == 0) {
      p.s.tokens[row] = top_at;
      if (p.s.probs) p.s.probs[row] = top == -INFINITY ? 0.0f : 1.0f;
    }
    return;
  }
  const Scale s = scale_of(top, a.inv_t, V);
  const T* const logits = reinterpret_cast<const T*>(p.s.logits) + row * p.s.row_stride;
  for (int c = tid; c < p.parts; c += kThreads) sh.part[c] = r.part_mass[c];
  const bool cuts = a.k || a.top_p < 1.0;
  Cut cut{kBins, kBins, kBins, 0, 0, 0, 0};
  Last last{0, false};
  __syncthreads();
  if (cuts) {
    cut = *r.cut;
    const uint32_t n = *r.listed;
    if (n > (uint32_t)kList) {
      last = last_of_row(sh, logits, V, cut, a, s);
      __syncthreads();
      for (int c = 0; c < p.parts; ++c) {    // the kept ones among those in doubt, part by part
        float x[kPer];
        const int i0 = c * kPart + tid * kPer;
        load(logits, i0, V, x);
        u64 mass = 0, all;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          const Weight w = weight_of(s, x[e], a.min_p);
          if (w.mass && w.over && w.bin >= min(cut.low, cut.kbin) &&
              (((u64)order_key(x[e]) << 32) | (uint32_t)(i0 + e)) <= last.at)
            mass += w.mass;
        }
        scan64(mass, sh.sums, all);
        if (tid == 0) sh.part[c] += all;
      }
    } else if (n) {
      last = last_of_list(sh, r, (int)n, cut, a, s);
      for (uint32_t i = tid; i < n; i += kThreads) {
        const u64 at = sh.list[i];
        const Weight w = weight_of(s, logit_of((uint32_t)(at >> 32)), a.min_p);
        if (last.some && at <= last.at && w.over) atomicAdd(&sh.part[(uint32_t)at / kPart], w.mass);
      }
    }
    __syncthreads();
  }
  // the part that holds the drawn mass
  constexpr int kEach = kMaxParts / kThreads;
  u64 mine = 0, total;
#pragma unroll
  for (int i = 0; i < kEach; ++i) mine += tid * kEach + i < p.parts ? sh.part[tid * kEach + i] : 0;
  u64 before = scan64(mine, sh.sums, total) - mine;
  const double at = (double)p.s.uniforms[row] * (double)total;
  const u64 target = at > 0.0 ? min((u64)fmin(at, 0x1p62), total - 1) : 0;
  if (target >= before && target < before + mine) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const u64 m = tid * kEach + i < p.parts ? sh.part[tid * kEach + i] : 0;
      if (target >= before && target < before + m) sh.found[0] = tid * kEach + i, sh.found[1] = before;
      before += m;
    }
  }
  __syncthreads();
  const int i0 = (int)sh.found[0] * kPart + tid * kPer;
  before = sh.found[1];
  float x[kPer];
  u64 m[kPer];
  load(logits, i0, V, x);
  mine = 0;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    const Weight w = weight_of(s, x[e], a.min_p);
    bool keep = w.mass && w.over;
    if (cuts)
      keep = keep && (w.bin < min(cut.low, cut.kbin) ||
                      (last.some && in_doubt(cut, w.bin) && (((u64)order_key(x[e]) << 32) | (uint32_t)(i0 + e)) <= last.at));
    m[e] = keep ? w.mass : 0;
    mine += m[e];
  }
  u64 all;
  before += scan64(mine, sh.sums, all) - mine;
  if (target >= before && target < before + mine) {
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      if (target >= before && target < before + m[e]) {
        p.s.tokens[row] = i0 + e;
        if (p.s.probs) p.s.probs[row] = (float)((double)m[e] / (double)total);
      }
      before += m[e];
    }
  }
}

template <typename T>
int launch(Params p, hipStream_t stream) {
  const SampleParams& s = p.s;
  const bool greedy = !s.temperatures && !(s.temperature > 0.0f);
  const bool cuts = s.top_ks || s.top_ps || (s.top_k > 0 && s.top_k < s.V) || s.top_p < 1.0f;
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
  return rows * ((row_bytes(parts_of(V)) + 15) & ~15ll);
}

int launch_sample(int dtype, const SampleParams& s, void* workspace, hipStream_t stream) {
  Params p{s, parts_of(s.V), 1, reinterpret_cast<uint8_t*>(workspace)};
  if (dtype == SLMT_F16) return launch<Fp16>(p, stream);
  if (dtype == SLMT_BF16) return launch<Bf16>(p, stream);
  return launch<float>(p, stream);
}

}  // namespace slmt
