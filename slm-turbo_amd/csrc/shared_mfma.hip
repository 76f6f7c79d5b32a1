// Decode attention of sequences that share a prompt, over the packed per-token 4-bit paged
// cache on the matrix cores, head_dim 64, 80 and 128, any number of query heads per KV head.
// (The reference has no counterpart: its paged decode reads every sequence's whole row,
// kernels/kv_dequant_kernels.cuh:671-801.)
//
// For a sequence of L tokens whose group shares the first P of them,
//   out = sum_t e^{s_t} v_t / sum_t e^{s_t},   s_t = q . k_t / sqrt(D),
// is joined from two sums, over t < P and over P <= t < L.  The first is computed for all
// sequences of the group at once, so the prompt's keys and values are read and unpacked once
// for up to 32 columns, column = (sequence, query head of the KV head); the second for a
// sequence's own query heads.  Both are items of one list: columns, a row of the block tables,
// a range of keys in tiles of 64.
//
// The work is split by what the lengths on the device say, with no host sync: every workgroup
// computes the same schedule in LDS.  A shared item is cut into equal parts, a job each, whose
// tiles a workgroup's four waves take in turn and join through LDS; a sequence's own tiles into
// chunks, a wave each, four to a job.  Their size is what gives every workgroup one job, by the
// tiles' measured costs.  A job's result is a partial one (m, l, o); merge_kernel, next on the
// stream, joins a query head's.  (With runs of tiles over item borders instead, a workgroup had
// up to three results to join and write: 50.7 us where the jobs took 29.0, at 8 sequences of 32
// heads on 8, D = 128, over 32768 shared tokens.)
//
// A wave works on a tile by itself, from registers: lane (c = lane & 15, g = lane >> 4) reads a
// quarter of key c's codes, which is its part of K as the matrix cores' left operand, and of
// the values of keys 4 g + i the bytes at its place c, from which a byte permute makes pairs of
// keys.  Everything is transposed, so that a lane owns a column from the scores to the output:
//   S^T = K Q^T,  P^T = exp2(S^T - m),  O^T += V^T P^T    (v_mfma_f32_16x16x32_f16)
// Up to 8 columns go another way, attend_few below.
//
// Exactness: codes enter as n - 8 and the query as it is, both fp16 numbers, so a score is
// kstep (q . (n - 8)) + (kmin + 8 kstep) sum(q) with fp32 sums (log2(e) / sqrt(D) folded into
// the rulers).  (As fp16's smallest numbers, n 2^-24, codes would need a mask alone, which took
// 6 % less; but products with such a number are cut as if it had the smallest normal one's
// exponent, and 2.4e-5 of the answer was lost instead of 1.9e-7.)  Weights w = p * vstep enter as
// an fp16 number and the fp16 remainder, two products.  What p is measured against, one reference
// a column for all its sums, is set by the weights: the largest w of a column lies in fp16's top
// octaves whatever the values' steps are (kTop below); sum(p) and sum(p (vmin + 8 vstep)) stay in
// fp32.
//
// What bounds it: instructions.  A tile of 32 columns at D = 128 is some 740 vector instructions
// (300 of them unpack codes, 290 are the softmax's) beside 96 matrix ones, 5300 cycles with a
// wave a SIMD, 8200 with another beside it.  Measured, us a call with its merge (us by bytes at
// the rate of a large copy): 8 sequences of 32 heads on 8, D = 128, over 32768 shared and
// 100-700 own tokens 26.4 (7.5), of which the schedule is 4, the first loads 4, five tiles 12,
// join and write 3; 64 over 8192 and 200-2000 own 47.6 (16.6), vector units 37 % busy, matrix
// cores 12 %; 32 of 32 on 4, D = 64, in groups of four over 1001-4096 15.8 (1.3); 2 of 14 on 2
// over 150 tokens 11.3 (two launches).
#include "slmt_internal.h"

#include <algorithm>
#include <type_traits>

namespace slmt {
namespace shared {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

constexpr int TK = 64;             // keys per tile
constexpr int COLS = 16;           // columns of a set
constexpr int SETS = 2;            // sets of a shared item
constexpr int WAVES = 4;           // waves per workgroup
// What a tile costs, by the number of columns (up to 8, 16 and 32).  Few and two: in the ratio of measured cycles, where waves of
// both kinds share a SIMD (6500 and 8200 at 128 dims; alone 3000 and 5300).  One has a side each way, by whole calls with 4 and
// with 3 (32 heads on 8, D = 128, groups of four sequences): 16 over 2048 shared and 300 own tokens 27.8 and 26.3 us, 12 over 3000
// and 700 30.1 and 31.4, 8 over 4096 and 16 23.9 and 23.7; D = 80, 16 over 1000 and 200 18.5 and 18.7; 32 on 4, D = 64, 16 groups of
// two over 4096 and 300 20.2 and 20.1.
constexpr int kCostFew = 3, kCostOne = 4, kCostTwo = 4;
// With few items and up to this cost of a wave, half the workgroups do the work: one a CU, which starts and joins as soon as
// two that share it, and of parts there are half as many.  8 sequences, 32 heads of 128 values on 8, a prompt of 8192 /
// 32768 / 98304 / 131072 tokens (a wave's cost 4 / 16 / 48 / 64): 18.6 / 26.9 / 50.2 / 64.5 us a call against 19.1 / 28.8 /
// 51.3 / 61.8 with all.  Other layers, with half / with all: 32 heads of 64 on 4, as many sequences over 8192 / 32768 14.9 / 20.9
// against 15.2 / 21.1, over 98304 / 131072 (costs past the limit here too) 36.9 / 45.0 against 33.2 / 37.7; 16 of 128 on 2, four
// sequences over 32768 / 131072 18.3 / 28.6 against 20.3 / 31.5; 8 of 80 on 8, eight over 8192 / 65536 15.3 / 28.6 against 16.1 /
// 29.3.  With more items each would have too few parts to even out (eight sequences on 9 prompts: 23.3 against 22.3), and for a
// few it may be the wrong side (four prompts of eight sequences, 32 heads of 64 on 4, 4096 tokens: 17.5 against 16.3).
constexpr int kHalfCost = 48;
constexpr int kMaxTokens = 1 << 28;   // of a row of the block tables
constexpr int kMaxSeqs = 4096;     // sequences and groups of a call (their places are in LDS)
// Weights w = p vstep stay up to 2^kTop, below fp16's largest number: one past it moves the reference, so that the largest is
// 2^(kTop - kSlack).  With a remainder in units of 2^-24, a column's weights keep 21 bits down to 2^-12 of its largest one, and
// are off by no more than 2^-32 of that below.  (A reference by the scores alone leaves w to the values' steps: with steps of
// 0.02 and scores of a deviation of 2.5 the answer was off by 1.5e-6 of its norm, with 2e-4 by 1.4e-4.)  Steps of 0 count as
// fp16's smallest number: p stays up to 2^39.  A smaller slack moves the reference more often: 8 sequences over 32768 tokens
// 28.1 us with 3, 26.5 with 7 and with more.
constexpr float kTop = 15.9f, kSlack = 7.0f;
constexpr int kLeastStep = -23;    // exponent e of fp16's smallest number, in 2^(e - 1) <= x < 2^e
constexpr int kWeightRow = 144;    // bytes of a column's weights in LDS (64 fp16, and 16 that spread the rows over the banks)

template <int D>
struct Geo {
  static constexpr int KW = D == 128 ? 4 : 2;        // dwords of K codes per key and lane (32 or 16 dims)
  static constexpr bool X = D == 80;                 // 16 dims more: 2 bytes of K, a nibble of V
  static constexpr int KB = KW + (X ? 1 : 0);        // 32-dim blocks of QK
  static constexpr int VB = D == 128 ? 4 : 2;        // bytes of V per key and lane
  static constexpr int RB = D / 16;                  // 16-dim blocks of PV
  static constexpr int OROW = D + 4;                 // floats of a column in the join
  static constexpr int JOIN = WAVES * SETS * COLS * OROW * 4;
  static constexpr int WAVE = TK * 16 + 16 * kWeightRow;   // a wave's rulers and weights, where the join's sums are later
  static_assert(WAVES * WAVE <= JOIN, "the waves' parts lie in the join's");
  static constexpr int FIXED = JOIN + WAVES * SETS * COLS * 8;
  static constexpr int WGS = 2;                      // workgroups a CU holds
};

// Codes n of halves' low or second nibbles as the fp16 numbers n - 8: the nibble under an
// exponent that makes it 1024 + n or 64 + n, and one exact packed sum.
struct Exponents {                 // (in vector registers: mask and exponent are one instruction then, which takes one scalar)
  uint32_t low = 0x64006400u, high = 0x54005400u;
  __device__ __forceinline__ Exponents() {
    asm("" : "+v"(low));
    asm("" : "+v"(high));
  }
};
__device__ __forceinline__ uint32_t low_codes(uint32_t w, const Exponents& ex) {
  const uint32_t x = (w & 0x000F000Fu) | ex.low;
  return __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2v, x) + half2v{(_Float16)-1032.0f, (_Float16)-1032.0f});
}
__device__ __forceinline__ uint32_t high_codes(uint32_t w, const Exponents& ex) {
  const uint32_t x = (w & 0x00F000F0u) | ex.high;
  return __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2v, x) + half2v{(_Float16)-72.0f, (_Float16)-72.0f});
}
// The eight codes of a dword, dims 0, 4, 1, 5, 2, 6, 3, 7 of its eight.
__device__ __forceinline__ half8 codes8(uint32_t w, const Exponents& ex) {
  const uint32_t s = w >> 8;
  const uint4 r = make_uint4(low_codes(w, ex), high_codes(w, ex), low_codes(s, ex), high_codes(s, ex));
  return __builtin_bit_cast(half8, r);
}
__device__ __forceinline__ int dim_of(int e) { return (e >> 1) + 4 * (e & 1); }

// Two numbers as fp16, cut: a weight's remainder is exact either way.  (Rounded, v_cvt_pk_f16_f32: 64 sequences over 8192 tokens 48.9
// us instead of 47.5.)
__device__ __forceinline__ half2v halves(float a, float b) {
  return __builtin_bit_cast(half2v, __builtin_amdgcn_cvt_pkrtz(a, b));
}

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ float uniform_f(float x) { return __builtin_bit_cast(float, uniform(__builtin_bit_cast(int, x))); }
__device__ __forceinline__ int tiles_of(int from, int to) { return to > from ? (to - (from & ~15) + TK - 1) / TK : 0; }

// Largest i of [0, n) with a[i] <= x; a[0] <= x.
__device__ __forceinline__ int last_at_most(const int* a, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Inclusive sum over the wave's lanes.
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);   // from the lane 1, 2, 4, 8 below in a row of 16
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);   // the row's last lane to the next row
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);   // lane 31 to the upper half
  return x;
}
// The largest of the lanes up to this one; x >= 0.
__device__ __forceinline__ int wave_most(int x) {
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));
  return max(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));
}
__device__ __forceinline__ int wave_total(int x) { return __builtin_amdgcn_readlane(wave_scan(x), 63); }

// Exclusive sums of a[0 .. n) in place, their total in a[n]; one wave.
__device__ __forceinline__ void scan(int* a, int n) {
  const int lane = threadIdx.x & 63;
  int base = 0;
  for (int i = 0; i < n; i += 64) {
    const int v = i + lane < n ? a[i + lane] : 0;
    const int incl = wave_scan(v);
    if (i + lane < n) a[i + lane] = base + incl - v;
    base += __builtin_amdgcn_readlane(incl, 63);
  }
  if (lane == 0) a[n] = base;
}

// x / d of 0 <= x < 2^23, d > 0, with r about 1 / d.
__device__ __forceinline__ int divide(int x, int d, float r) {
  int q = (int)((float)x * r);
  const int rest = x - q * d;
  q += rest >= d;
  q -= rest < 0;
  return q;
}
__device__ __forceinline__ int divide(int x, int d) { return divide(x, d, __builtin_amdgcn_rcpf((float)d)); }
// flat / G, by its reciprocal in 2^-32 rounded up (at most one too many).
__device__ __forceinline__ int over_heads(const SharedParams& p, int flat) {
  const int q = p.G == 1 ? flat : (int)__umulhi((uint32_t)flat, p.G_inverse);
  return q - (q * p.G > flat);
}

// Jobs of one size, for a cost of a wave's work: tiles of a wave in each, and the reciprocals that make them.
struct Fit {
  int few, one, two, own;              // tiles of a wave, of items of up to 8, 16 and 32 columns, and of own chunks
  float rfew, rone, rtwo, rown;        // about 1 over a workgroup's; 1 over own
  __device__ __forceinline__ Fit(int cost, int G) {
    few = (cost + kCostFew - 1) / kCostFew;
    one = (cost + kCostOne - 1) / kCostOne;
    two = (cost + kCostTwo - 1) / kCostTwo;
    own = G <= 8 ? few : one;
    rfew = __builtin_amdgcn_rcpf((float)(few * WAVES));
    rone = __builtin_amdgcn_rcpf((float)(one * WAVES));
    rtwo = __builtin_amdgcn_rcpf((float)(two * WAVES));
    rown = __builtin_amdgcn_rcpf((float)own);
  }
  __device__ __forceinline__ int tiles(int columns) const {   // (copies: not an address to choose)
    const int a = few, b = one, c = two;
    return columns > COLS ? c : columns > 8 ? b : a;
  }
  __device__ __forceinline__ int parts(int all, int columns) const {
    const int n = tiles(columns) * WAVES;
    const float a = rfew, b = rone, c = rtwo;
    return divide(all + n - 1, n, columns > COLS ? c : columns > 8 ? b : a);
  }
  __device__ __forceinline__ int chunks(int all) const { return divide(all + own - 1, own, rown); }
};

// The call's jobs, in LDS, the same in all workgroups.  A job is a workgroup's part of a shared item's tiles (its waves take
// them in turn and join), or four chunks of sequences' own tiles, a wave each.
struct Schedule {
  int *start;     // [R + 1] the groups' first sequences
  int *prefix;    // [R] their shared tokens
  int *part;      // [R + 1] jobs of the groups before
  int *len;       // [B] tokens of a sequence
  int *chunk;     // [B + 1] chunks of the sequences before
  int width;      // workgroups a KV head that take jobs
  int shared, chunks;
  Fit fit;
  // the first of a sequence's tokens that its group does not read
  __device__ __forceinline__ int own_from(const SharedParams& p, int b) const {
    return p.R > 0 && b >= start[0] && b < start[p.R] ? min(prefix[last_at_most(start, p.R, b)], len[b]) : 0;
  }
  __device__ __forceinline__ int columns(const SharedParams& p, int r) const { return (start[r + 1] - start[r]) * p.G; }
  __device__ __forceinline__ int parts(const SharedParams& p, int r) const { return fit.parts(tiles_of(0, prefix[r]), columns(p, r)); }
};
__device__ __forceinline__ int sets_of(int columns) { return (columns + SETS * COLS - 1) / (SETS * COLS); }

__device__ __forceinline__ Schedule make_schedule(const SharedParams& p, int* lds) {
  const int tid = threadIdx.x, lane = tid & 63, R = p.R, B = p.B, wave = uniform(tid >> 6);
  Schedule s{lds, nullptr, nullptr, nullptr, nullptr, p.W, 0, 0, Fit(1, p.G)};
  s.prefix = s.start + R + 1;
  s.part = s.prefix + R;
  s.len = s.part + R + 1;
  s.chunk = s.len + B;
  if (wave == 0) {      // starts that never fall, whatever the caller's are: all that follows holds for them
    int most = 0;
    for (int i = 0; i <= R; i += 64) {
      int v = max(most, i + lane <= R ? min(max(p.group_start[i + lane], 0), B) : 0);
      v = wave_most(v);
      if (i + lane <= R) s.start[i + lane] = v;
      most = __builtin_amdgcn_readlane(v, 63);
    }
  } else {
    for (int i = tid - 64; i < R; i += (WAVES - 1) * 64) s.prefix[i] = min(max(p.prefix_lens[i], 0), p.max_tokens);
    for (int b = tid - 64; b < B; b += (WAVES - 1) * 64) s.len[b] = min(max(p.seq_lens[b], 0), p.max_tokens);
  }
  __syncthreads();
  for (int b = tid; b < B; b += WAVES * 64) s.chunk[b] = tiles_of(s.own_from(p, b), s.len[b]);
  __syncthreads();
  // As much a wave as makes a job for every workgroup and no more: by the work alone, then with half a job, then with a whole
  // one lost at every item's end (which always fits, where there are fewer items than workgroups).
  // (The lane's first group and sequence stay in registers.)
  const bool group = lane < R;
  const int columns0 = group ? s.columns(p, lane) : 0, sets0 = sets_of(columns0), tiles0 = group ? tiles_of(0, s.prefix[lane]) : 0;
  const int chunk0 = lane < B ? s.chunk[lane] : 0;
  auto price = [&](int columns) { return columns > COLS ? kCostTwo : columns > 8 ? kCostOne : kCostFew; };
  const int own_price = p.own_sets * (p.G <= 8 ? kCostFew : kCostOne);
  int cost = sets0 * tiles0 * price(columns0) + chunk0 * own_price, items = tiles0 > 0 ? sets0 : 0, own_items = chunk0 > 0 ? p.own_sets : 0;
  for (int r = lane + 64; r < R; r += 64) {
    const int columns = s.columns(p, r), sets = sets_of(columns), tiles = tiles_of(0, s.prefix[r]);
    cost += sets * tiles * price(columns);
    items += tiles > 0 ? sets : 0;
  }
  for (int b = lane + 64; b < B; b += 64) {
    cost += s.chunk[b] * own_price;
    own_items += s.chunk[b] > 0 ? p.own_sets : 0;
  }
  cost = wave_total(cost);
  items = wave_total(items) + wave_total(own_items) / WAVES + 1;
  const int half = p.W % 16 ? 0 : p.W / 2;         // (a multiple of the XCDs)
  if (2 * items <= half && cost <= kHalfCost * WAVES * half) s.width = half;
  for (int i = 0;; ++i) {
    const int jobs = max(s.width / 4, s.width - (i * items) / 2) * WAVES;
    s.fit = Fit(max(1, (int)((float)cost * __builtin_amdgcn_rcpf((float)jobs) + 0.999f)), p.G);
    if (i == 2) break;
    int shared = sets0 * s.fit.parts(tiles0, columns0), own = p.own_sets * s.fit.chunks(chunk0);
    for (int r = lane + 64; r < R; r += 64) shared += sets_of(s.columns(p, r)) * s.parts(p, r);
    for (int b = lane + 64; b < B; b += 64) own += p.own_sets * s.fit.chunks(s.chunk[b]);
    if (wave_total(shared) + (wave_total(own) + WAVES - 1) / WAVES <= s.width) break;
  }
  __syncthreads();
  if (wave == 0) {
    for (int r = lane; r < R; r += 64) s.part[r] = sets_of(s.columns(p, r)) * s.parts(p, r);
    scan(s.part, R);
  } else if (wave == 1) {
    for (int b = lane; b < B; b += 64) s.chunk[b] = p.own_sets * s.fit.chunks(s.chunk[b]);
    scan(s.chunk, B);
  }
  __syncthreads();
  s.shared = uniform(s.part[R]);
  s.chunks = uniform(s.chunk[B]);
  return s;
}

// Part i of n units in equal parts, the first ones larger by one where that is not even.
struct Run {
  int from, to;
};
__device__ __forceinline__ Run share_of(int n, int parts, int i) {
  const int each = uniform(divide(n, parts)), more = n - each * parts, from = i * each + min(i, more);
  return {from, from + each + (i < more)};
}

// What a wave does: tiles lo, lo + step, ... below hi of the keys klo .. khi - 1 of row seq0 of the tables, for ncols
// columns from flat0 on.
struct Work {
  int seq0, flat0, ncols, klo, khi, lo, hi, step;
  const int* len;                      // the sequences' lengths
  bool own;
};

template <int D, int S>
struct Sums {
  floatx4 o[S][D / 16];            // sums of the weights' products
  float m[S], l[S], vt[S];         // the weights' reference, their sum, the sum of their products with vmin + 8 vstep
};

// A wave's tiles: their places in the cache and the codes of the present one, in registers.  The keys whose values a lane has
// in slots e of half h are 16 i + 4 g + (e & 3), i = 2 h + (e >> 2), or with NARROW 16 (e & 3) + 8 h + 2 g + (e >> 2).
template <int D, bool NARROW>
struct Tiles {
  using GG = Geo<D>;
  static constexpr int KW = GG::KW, VB = GG::VB, SLOT = D + 8;
  uint32_t kx[4][KW], kxx[4], vx[16], vxx[16];
  uint2 rl;                            // the rulers of key `lane` of the tile
  const uint8_t *cache, *table;
  int64_t block_bytes;
  uint32_t row_bytes, last_block, head, kfrom, vfrom;
  int base, end16, esh, block_size, block_shift, grp, col;

  __device__ __forceinline__ Tiles(const SharedParams& p, const Work& wk, int kv) {
    const int lane = threadIdx.x & 63;
    col = lane & 15;
    grp = lane >> 4;
    cache = p.cache;
    last_block = p.last_block;
    row_bytes = (uint32_t)p.KV * SLOT;
    block_bytes = (int64_t)p.block_size * row_bytes;
    block_size = p.block_size;
    block_shift = p.block_shift;
    esh = p.bt64 ? 3 : 2;
    head = kv * SLOT;
    base = wk.klo & ~15;
    end16 = (wk.khi - 1) & ~15;
    table = reinterpret_cast<const uint8_t*>(p.block_tables) + (((int64_t)wk.seq0 * p.bt_stride) << esh);
    kfrom = col * row_bytes + 4 * KW * grp;
    vfrom = (NARROW ? 2 : 4) * grp * row_bytes + D / 2 + VB * col;
  }
  // offset of the 16 keys that the lane's group has in tile t (past the end: the last ones)
  __device__ __forceinline__ int64_t place(int t) const {
    const int key = min(base + t * TK + 16 * grp, end16);
    const int block = block_shift >= 0 ? key >> block_shift : key / block_size;
    const int in_block = key - block * block_size;
    const uint32_t entry = *reinterpret_cast<const uint32_t*>(table + ((int64_t)block << esh));
    return (int64_t)min(entry, last_block) * block_bytes + (uint32_t)(in_block * (int)row_bytes + head);
  }
  // 16 keys of a block, from the lane's head on: what lies past them reads as 0
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t keys16(int64_t off, int i) const {
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)off, 16 * i), hi = __builtin_amdgcn_readlane((int)(off >> 32), 16 * i);
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(cache + (((uint64_t)hi << 32) | lo)), 0, (int)(16 * row_bytes - head), 0x00027000);
  }
  __device__ __forceinline__ void load_k(int64_t off) {
    typedef uint32_t Words __attribute__((ext_vector_type(KW)));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __amdgpu_buffer_rsrc_t b = keys16(off, i);
      Words x;
      if constexpr (KW == 4) x = __builtin_bit_cast(Words, __builtin_amdgcn_raw_buffer_load_b128(b, kfrom, 0, 0));
      else x = __builtin_bit_cast(Words, __builtin_amdgcn_raw_buffer_load_b64(b, kfrom, 0, 0));
#pragma unroll
      for (int j = 0; j < KW; ++j) kx[i][j] = x[j];
      if constexpr (GG::X) kxx[i] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(b, kfrom - 4 * KW * grp + 32 + 2 * grp, 0, 0);
    }
    rl = *reinterpret_cast<const uint2*>(cache + off + (uint32_t)(col * row_bytes + D));
  }
  __device__ __forceinline__ void load_v(int64_t off) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __amdgpu_buffer_rsrc_t b = keys16(off, i);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // NARROW: keys 8 h + 2 g + u of the block, h = e >> 1, u = e & 1, in slot i + 4 u of half h
        const int slot = NARROW ? 8 * (e >> 1) + i + 4 * (e & 1) : 4 * i + e;
        const uint32_t row = (NARROW ? 8 * (e >> 1) + (e & 1) : e) * row_bytes;
        if constexpr (VB == 4) vx[slot] = __builtin_amdgcn_raw_buffer_load_b32(b, vfrom, row, 0);
        else vx[slot] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(b, vfrom, row, 0);
        if constexpr (GG::X) vxx[slot] = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(b, vfrom - VB * col + 32 + (col >> 1), row, 0);
      }
    }
  }
  // The values' products of half h's keys: each(block of 16 dims, their codes as the left operand).
  template <typename F>
  __device__ __forceinline__ void values(int h, const Exponents& ex, F each) const {
    auto give = [&](int c, const uint32_t (&w)[4]) { each(c, __builtin_bit_cast(half8, make_uint4(w[0], w[1], w[2], w[3]))); };
#pragma unroll
    for (int b = 0; b < VB; ++b) {
      uint32_t lo[4], hi[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t pair = __builtin_amdgcn_perm(vx[8 * h + 2 * e + 1], vx[8 * h + 2 * e], 0x0C000C00u | ((4u + b) << 16) | (uint32_t)b);
        lo[e] = low_codes(pair, ex);
        hi[e] = high_codes(pair, ex);
      }
      give(2 * b, lo);
      give(2 * b + 1, hi);
    }
    if constexpr (GG::X) {
      uint32_t lo[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t pair = __builtin_amdgcn_perm(vxx[8 * h + 2 * e + 1], vxx[8 * h + 2 * e], 0x0C040C00u);
        lo[e] = low_codes(pair >> (4 * (col & 1)), ex);
      }
      give(GG::RB - 1, lo);
    }
  }
};

// log2(e) / sqrt(D)
template <int D>
constexpr float kC = 1.4426950408889634f / (D == 64 ? 8.0f : D == 80 ? 8.94427190999916f : 11.313708498984761f);

// Sums over the waves' lane groups (lanes of one column).
__device__ __forceinline__ float sum_groups(float x) {
  float a, b;
  swap16(x, a, b);
  x = a + b;
  swap32(x, a, b);
  return a + b;
}
__device__ __forceinline__ float most_of_groups(float x) {
  float a, b;
  swap16(x, a, b);
  x = fmaxf(a, b);
  swap32(x, a, b);
  return fmaxf(a, b);
}

// Keys of a tile whose values' rulers are infinite or NaN (a key a lane, from kt0 on): their values are no numbers, which the
// columns that see them add by seen(key, value); the others' weights of 0 may not meet them, so they count as 0 from here.
template <typename F>
__device__ __forceinline__ void take_odd_keys(float& vmin, float& vstep, int kt0, F seen) {
  const bool odd = !(__builtin_fabsf(vmin) + __builtin_fabsf(vstep) < INFINITY);
  uint64_t left = __builtin_amdgcn_ballot_w64(odd);
  const float value = vmin + vstep;
  vmin = odd ? 0.f : vmin;
  vstep = odd ? 0.f : vstep;
#pragma unroll 1
  for (; left; left &= left - 1) {
    const int i = __builtin_ctzll(left);
    seen(kt0 + i, __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, value), i)));
  }
}

// The exponent of a value step, of 0 that of the smallest.
__device__ __forceinline__ int exponent_of(float vstep) {
  return __builtin_amdgcn_frexp_expf(fmaxf(__builtin_fabsf(vstep), 0x1p-24f));
}

// A wave's bound of the steps that it has seen, a power of two, and how far above the reference scores may lie with them.  A
// larger step moves the bound and with it the room; what does not fit there is looked at key by key.
struct Room {
  float steps = 0.f, room = kTop - kLeastStep;     // (uniform, in scalar registers)
  __device__ __forceinline__ bool odd(float vmin, float vstep) const {    // (infinite and NaN rulers too)
    return __builtin_amdgcn_ballot_w64(!(__builtin_fabsf(__builtin_fmaf(0.f, vmin, vstep)) <= steps));
  }
  __device__ __forceinline__ void take(float vstep) {
    const int e = exponent_of(wave_max(__builtin_fabsf(vstep)));
    steps = uniform_f(fmaxf(steps, __builtin_ldexpf(1.0f, e)));
    room = uniform_f(fminf(room, kTop - (float)e));
  }
};

// A column's reference at a wave's end: -infinity says that it saw no key.  Where it saw NaN scores alone no largest one was
// found either, but their sum is NaN: so is the reference then, and the joins keep it.  (As a comparison and a choice, 64
// sequences over 8192 tokens took 48.7 us instead of 47.9.)
__device__ __forceinline__ float reference_of(float m, float l) { return __builtin_fmaf(0.f, l, m); }

// S sets of 16 columns.
template <int D, int S>
__device__ __forceinline__ void attend(const SharedParams& p, const Work& wk, int kv, uint8_t* rulers, Sums<D, S>& sum) {
  using GG = Geo<D>;
  constexpr int KW = GG::KW, KB = GG::KB, RB = GG::RB;
  const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
  const Exponents ex;
  Tiles<D, false> x(p, wk, kv);
  int64_t off_next = 0;
  const bool any = wk.lo < wk.hi;
  if (any) {
    const int64_t off = x.place(wk.lo);
    off_next = x.place(wk.lo + wk.step < wk.hi ? wk.lo + wk.step : wk.lo);
    x.load_k(off);
    x.load_v(off);
  }

  // ---- the lane's columns (those past the item's repeat the last)
  half8 qh[S][KB];
  float qsum[S];
  int lim[S], lim_lo = 0x7fffffff;     // keys below lim are seen
#pragma unroll
  for (int st = 0; st < S; ++st) {
    const int flat = wk.flat0 + min(COLS * st + col, wk.ncols - 1);
    const int seq = wk.own ? wk.seq0 : wk.seq0 + over_heads(p, flat), head = kv * p.G + (wk.own ? flat : flat - (seq - wk.seq0) * p.G);
    lim[st] = wk.own ? wk.khi : min(wk.khi, wk.len[seq]);
    const uint16_t* q = p.q + (int64_t)seq * p.q_seq_stride + (int64_t)head * p.q_head_stride;
    float t = 0.f;
#pragma unroll
    for (int j = 0; j < KW; ++j) {
      const half8 y = *reinterpret_cast<const half8*>(q + 8 * (KW * grp + j));
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        qh[st][j][e] = y[dim_of(e)];
        t += (float)y[e];
      }
    }
    if constexpr (GG::X) {
      const half4 y = *reinterpret_cast<const half4*>(q + 64 + 4 * grp);
      qh[st][KW] = half8{y[0], (_Float16)0.f, y[1], (_Float16)0.f, y[2], (_Float16)0.f, y[3], (_Float16)0.f};
#pragma unroll
      for (int e = 0; e < 4; ++e) t += (float)y[e];
    }
    qsum[st] = sum_groups(t);
    lim_lo = min(lim_lo, lim[st]);
#pragma unroll
    for (int c = 0; c < RB; ++c) sum.o[st][c] = floatx4{0.f, 0.f, 0.f, 0.f};
    sum.m[st] = -INFINITY;
    sum.l[st] = sum.vt[st] = 0.f;
  }
  if (!any) return;
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) lim_lo = min(lim_lo, __shfl_xor(lim_lo, o, 64));
  lim_lo = uniform(lim_lo);
  float msub[S];                       // what is subtracted: m, 0 while that is -inf
#pragma unroll
  for (int st = 0; st < S; ++st) msub[st] = 0.f;
  Room room;

  for (int t = wk.lo; t < wk.hi; t += wk.step) {
    const int kt0 = x.base + t * TK;
    {   // the tile's rulers, a key a lane
      const float kmin = h2f((uint16_t)(x.rl.x & 0xffffu)), kstep = h2f((uint16_t)(x.rl.x >> 16));
      float vmin = h2f((uint16_t)(x.rl.y & 0xffffu)), vstep = h2f((uint16_t)(x.rl.y >> 16));
      const int key = kt0 + lane;
      const bool in = key >= wk.klo && key < wk.khi;
      vmin = in ? __builtin_fmaf(8.0f, vstep, vmin) : 0.f;     // (nor may the rulers of keys that are not seen reach the sums)
      vstep = in ? vstep : 0.f;
      if (room.odd(vmin, vstep)) {
        take_odd_keys(vmin, vstep, kt0, [&](int key, float v) {
#pragma unroll
          for (int st = 0; st < S; ++st)
            if (key < lim[st]) sum.vt[st] += v;
        });
        room.take(vstep);
      }
      __builtin_amdgcn_wave_barrier();
      *reinterpret_cast<float2*>(rulers + 8 * lane) = make_float2(__builtin_fmaf(8.0f, kstep, kmin) * kC<D>, kstep * kC<D>);
      *reinterpret_cast<float2*>(rulers + 8 * (TK + lane)) = make_float2(vmin, vstep);
      __builtin_amdgcn_wave_barrier();
    }
    floatx4 sc[S][4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      half8 a[KB];
#pragma unroll
      for (int j = 0; j < KW; ++j) a[j] = codes8(x.kx[n][j], ex);
      if constexpr (GG::X) a[KW] = codes8(x.kxx[n], ex);
#pragma unroll
      for (int st = 0; st < S; ++st) {
        sc[st][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[0], qh[st][0], floatx4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
        for (int j = 1; j < KB; ++j) sc[st][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[j], qh[st][j], sc[st][n], 0, 0, 0);
      }
    }
    if (t + wk.step < wk.hi) x.load_k(off_next);
    const bool whole = kt0 >= wk.klo && kt0 + TK <= lim_lo;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const float4* kr = reinterpret_cast<const float4*>(rulers + 8 * (16 * n + 4 * grp));
      const float4 k01 = kr[0], k23 = kr[1];
#pragma unroll
      for (int st = 0; st < S; ++st) {
        sc[st][n][0] = __builtin_fmaf(sc[st][n][0], k01.y, __builtin_fmaf(qsum[st], k01.x, -msub[st]));
        sc[st][n][1] = __builtin_fmaf(sc[st][n][1], k01.w, __builtin_fmaf(qsum[st], k01.z, -msub[st]));
        sc[st][n][2] = __builtin_fmaf(sc[st][n][2], k23.y, __builtin_fmaf(qsum[st], k23.x, -msub[st]));
        sc[st][n][3] = __builtin_fmaf(sc[st][n][3], k23.w, __builtin_fmaf(qsum[st], k23.z, -msub[st]));
      }
    }
    if (!whole) {                      // keys that a column does not see: weight 0
#pragma unroll
      for (int st = 0; st < S; ++st)
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = kt0 + 16 * n + 4 * grp + i;
            sc[st][n][i] = key >= wk.klo && key < lim[st] ? sc[st][n][i] : -INFINITY;
          }
    }
    // (scores are relative to msub)
    bool over = false;
#pragma unroll
    for (int st = 0; st < S; ++st) {
      float tmax = -INFINITY;
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) tmax = fmaxf(tmax, sc[st][n][i]);
      over |= tmax > (sum.m[st] == -INFINITY ? -INFINITY : room.room);
    }
    if (__builtin_amdgcn_ballot_w64(over)) {
      float* const exponents = reinterpret_cast<float*>(rulers + 16 * TK);
      exponents[lane] = (float)exponent_of(*reinterpret_cast<const float*>(rulers + 8 * (TK + lane) + 4));
      __builtin_amdgcn_wave_barrier();
      float most[S];                   // the largest weight's exponent
#pragma unroll
      for (int st = 0; st < S; ++st) most[st] = -INFINITY;
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const floatx4 e = *reinterpret_cast<const floatx4*>(exponents + 16 * n + 4 * grp);
#pragma unroll
        for (int st = 0; st < S; ++st)
#pragma unroll
          for (int i = 0; i < 4; ++i) most[st] = fmaxf(most[st], sc[st][n][i] + e[i]);
      }
#pragma unroll
      for (int st = 0; st < S; ++st) {
        most[st] = most_of_groups(most[st]);
        const bool grow = most[st] > (sum.m[st] == -INFINITY ? -INFINITY : kTop);
        if (!__builtin_amdgcn_ballot_w64(grow)) continue;
        const float up = grow ? most[st] - (kTop - kSlack) : 0.f;
        const float alpha = !grow ? 1.f : sum.m[st] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(-up);
        msub[st] += up;
        sum.m[st] = grow ? msub[st] : sum.m[st];
        sum.l[st] *= alpha;
        sum.vt[st] *= alpha;
#pragma unroll
        for (int c = 0; c < RB; ++c) sum.o[st][c] *= alpha;
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[st][n][i] -= up;
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {      // 32 keys
      half8 bh[S], bl[S];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const float4* vr = reinterpret_cast<const float4*>(rulers + 8 * (TK + 16 * (2 * h + n) + 4 * grp));
        const float4 v01 = vr[0], v23 = vr[1];
        const float vmin[4] = {v01.x, v01.z, v23.x, v23.z}, vstep[4] = {v01.y, v01.w, v23.y, v23.w};
#pragma unroll
        for (int st = 0; st < S; ++st) {
#pragma unroll
          for (int i = 0; i < 4; i += 2) {
            float pr[2], w[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              pr[e] = __builtin_amdgcn_exp2f(sc[st][2 * h + n][i + e]);
              sum.l[st] += pr[e];
              sum.vt[st] = __builtin_fmaf(pr[e], vmin[i + e], sum.vt[st]);
              w[e] = pr[e] * vstep[i + e];
            }
            const half2v h2 = halves(w[0], w[1]), l2 = halves(w[0] - (float)h2[0], w[1] - (float)h2[1]);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              bh[st][4 * n + i + e] = h2[e];
              bl[st][4 * n + i + e] = l2[e];
            }
          }
        }
      }
      x.values(h, ex, [&](int c, half8 a) {
#pragma unroll
        for (int st = 0; st < S; ++st) sum.o[st][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, bh[st], sum.o[st][c], 0, 0, 0);
#pragma unroll
        for (int st = 0; st < S; ++st) sum.o[st][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, bl[st], sum.o[st][c], 0, 0, 0);
      });
    }
    if (t + wk.step < wk.hi) {
      x.load_v(off_next);
      off_next = x.place(t + 2 * wk.step < wk.hi ? t + 2 * wk.step : t);
    }
  }
#pragma unroll
  for (int st = 0; st < S; ++st) {
    sum.l[st] = sum_groups(sum.l[st]);
    sum.vt[st] = sum_groups(sum.vt[st]);
    sum.m[st] = reference_of(sum.m[st], sum.l[st]);
  }
}

// Up to 8 columns, four a set.  The 16 rows of the scores' products are four columns' query limbs, and keys are their columns:
//   QK, exact: v_mfma_i32_16x16x64_i8.  A column's query is scaled by a power of two to 31-bit integers (fp16 numbers down to
//   2^-21 of its largest are exact) and cut into four signed 8-bit limbs; codes are unpacked from nibbles to bytes.  A lane then
//   has the four limbs' sums of one column (its group) for one key, which join without other lanes.
//   PV: columns 0 .. 7 of the right operand are the weights, 8 .. 15 their remainders, so one product does both; they pass
//   through LDS, a lane's four keys (one of each 16) side by side.
// Against 16 columns of which few are used: half the unpacking of K, a quarter of the softmax, half the products.  64 sequences
// with 200-2000 tokens of their own, 4 columns each, beside 8192 shared ones: 47.4 us, by 8 columns (Q = 2) 50.2, by 16 51.5.
template <int D, int Q>
__device__ __forceinline__ void attend_few(const SharedParams& p, const Work& wk, int kv, uint8_t* rulers, uint8_t* weights, Sums<D, 1>& sum) {
  using GG = Geo<D>;
  constexpr int KW = GG::KW, RB = GG::RB, KB = D == 64 ? 1 : 2;      // blocks of 64 dims (head_dim 80: 16 in the second)
  typedef int v4i __attribute__((ext_vector_type(4)));
  const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
  const Exponents ex;
  Tiles<D, true> x(p, wk, kv);
  int64_t off_next = 0;
  const bool any = wk.lo < wk.hi;
  if (any) {
    const int64_t off = x.place(wk.lo);
    off_next = x.place(wk.lo + wk.step < wk.hi ? wk.lo + wk.step : wk.lo);
    x.load_k(off);
    x.load_v(off);
  }
#pragma unroll
  for (int c = 0; c < RB; ++c) sum.o[0][c] = floatx4{0.f, 0.f, 0.f, 0.f};
  sum.m[0] = -INFINITY;
  sum.l[0] = sum.vt[0] = 0.f;
  if (!any) return;

  auto row_of = [&](int c) {           // the query row of column c
    const int flat = wk.flat0 + min(c, wk.ncols - 1);
    const int seq = wk.own ? wk.seq0 : wk.seq0 + over_heads(p, flat), head = kv * p.G + (wk.own ? flat : flat - (seq - wk.seq0) * p.G);
    return p.q + (int64_t)seq * p.q_seq_stride + (int64_t)head * p.q_head_stride;
  };
  // limb col & 3 of column 4 st + (col >> 2), its dims in the order of the unpacked codes
  v4i limbs[Q][KB];
  float scale[Q], qsum[Q];             // of column 4 st + grp
  int lim[Q], lim_lo = 0x7fffffff;
#pragma unroll
  for (int st = 0; st < Q; ++st) {
    const uint16_t* const q = row_of(4 * st + (col >> 2));
    float f[KB][16];
#pragma unroll
    for (int j = 0; j < KW; ++j) {
      const half8 y = *reinterpret_cast<const half8*>(q + 8 * (KW * grp + j));
#pragma unroll
      for (int e = 0; e < 8; ++e) f[j / 2][8 * (j & 1) + e] = (float)y[e];
    }
    if constexpr (GG::X) {
      const half4 y = *reinterpret_cast<const half4*>(q + 64 + 4 * grp);
#pragma unroll
      for (int e = 0; e < 16; ++e) f[1][e] = e < 4 ? (float)y[e] : 0.f;
    }
    float most = 0.f, t = 0.f;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        most = fmaxf(most, __builtin_fabsf(f[kb][e]));
        t += f[kb][e];
      }
    most = most_of_groups(most);
    t = sum_groups(t);
    const int sc = most > 0.f ? 30 - __builtin_amdgcn_frexp_expf(most) : 0;      // the largest below 2^30: the top limb fits
    const int shift = 8 * (col & 3);
    const uint32_t flip = (col & 3) < 3 ? 0x80u : 0u;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      uint32_t byte[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int n = (int)__builtin_rintf(__builtin_amdgcn_ldexpf(f[kb][e], sc));
        // balanced digits: n + 0x808080 = sum d 2^(8 x), limb d - 128 (the top one: the rest)
        byte[e] = ((uint32_t)((n + 0x808080) >> shift) & 0xffu) ^ flip;
      }
      uint32_t dw[4];                  // a word of codes becomes its even and its odd dims
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const int e = 8 * (d >> 1) + (d & 1);
        dw[d] = byte[e] | (byte[e + 2] << 8) | (byte[e + 4] << 16) | (byte[e + 6] << 24);
      }
      if (GG::X && kb == 1) {          // four dims, in one dword
        dw[0] = byte[0] | (byte[2] << 8) | (byte[1] << 16) | (byte[3] << 24);
        dw[1] = dw[2] = dw[3] = 0;
      }
      limbs[st][kb] = v4i{(int)dw[0], (int)dw[1], (int)dw[2], (int)dw[3]};
    }
    scale[st] = __shfl(__builtin_amdgcn_ldexpf(1.0f, -sc), 4 * grp, 64);
    qsum[st] = __shfl(t, 4 * grp, 64);
    const int flat = wk.flat0 + min(4 * st + grp, wk.ncols - 1);
    lim[st] = wk.own ? wk.khi : min(wk.khi, wk.len[wk.seq0 + over_heads(p, flat)]);
    lim_lo = min(lim_lo, lim[st]);
  }
  lim_lo = min(min(__builtin_amdgcn_readlane(lim_lo, 0), __builtin_amdgcn_readlane(lim_lo, 16)),
               min(__builtin_amdgcn_readlane(lim_lo, 32), __builtin_amdgcn_readlane(lim_lo, 48)));
  float m[Q], msub[Q], l[Q], vt[Q];    // of column 4 st + grp; l and vt: the lane's keys
#pragma unroll
  for (int st = 0; st < Q; ++st) {
    m[st] = -INFINITY;
    msub[st] = l[st] = vt[st] = 0.f;
  }
  Room room;
  // a column's value from its lane group, for the lanes that hold its sums
  auto of_column = [&](const float (&v)[Q]) {
    float a = __shfl(v[0], 16 * (col & 3), 64);
    if constexpr (Q == 2) {
      const float b = __shfl(v[1], 16 * (col & 3), 64);
      a = col & 4 ? b : a;
    }
    return a;
  };

  for (int t = wk.lo; t < wk.hi; t += wk.step) {
    const int kt0 = x.base + t * TK;
    {   // the tile's rulers, a key a lane
      const float kmin = h2f((uint16_t)(x.rl.x & 0xffffu)), kstep = h2f((uint16_t)(x.rl.x >> 16));
      float vmin = h2f((uint16_t)(x.rl.y & 0xffffu)), vstep = h2f((uint16_t)(x.rl.y >> 16));
      const int key = kt0 + lane;
      const bool in = key >= wk.klo && key < wk.khi;
      vmin = in ? __builtin_fmaf(8.0f, vstep, vmin) : 0.f;     // (nor may the rulers of keys that are not seen reach the sums)
      vstep = in ? vstep : 0.f;
      if (room.odd(vmin, vstep)) {
        take_odd_keys(vmin, vstep, kt0, [&](int key, float v) {
#pragma unroll
          for (int st = 0; st < Q; ++st)
            if (key < lim[st]) vt[st] += v;
        });
        room.take(vstep);
      }
      __builtin_amdgcn_wave_barrier();
      *reinterpret_cast<float4*>(rulers + 16 * lane) = make_float4(kmin * kC<D>, kstep * kC<D>, vmin, vstep);
      __builtin_amdgcn_wave_barrier();
    }
    float s[Q][4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      v4i b[KB];
#pragma unroll
      for (int kb = 0; kb < (GG::X ? 1 : KB); ++kb)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          b[kb][2 * w] = (int)(x.kx[n][2 * kb + w] & 0x0F0F0F0Fu);
          b[kb][2 * w + 1] = (int)((x.kx[n][2 * kb + w] >> 4) & 0x0F0F0F0Fu);
        }
      if constexpr (GG::X) b[1] = v4i{(int)((x.kxx[n] & 0x0F0Fu) | ((x.kxx[n] & 0xF0F0u) << 12)), 0, 0, 0};
#pragma unroll
      for (int st = 0; st < Q; ++st) {
        v4i c = __builtin_amdgcn_mfma_i32_16x16x64_i8(limbs[st][0], b[0], v4i{0, 0, 0, 0}, 0, 0, 0);
        if constexpr (KB == 2) c = __builtin_amdgcn_mfma_i32_16x16x64_i8(limbs[st][1], b[1], c, 0, 0, 0);
        s[st][n] = __builtin_fmaf((float)(c[2] + (c[3] << 8)), 65536.0f, (float)(c[0] + (c[1] << 8)));
      }
    }
    if (t + wk.step < wk.hi) x.load_k(off_next);
    const bool whole = kt0 >= wk.klo && kt0 + TK <= lim_lo;
    float vmin[4], vstep[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {      // key 16 n + col of the tile
      const float4 r = *reinterpret_cast<const float4*>(rulers + 16 * (16 * n + col));
      vmin[n] = r.z;
      vstep[n] = r.w;
#pragma unroll
      for (int st = 0; st < Q; ++st) {
        s[st][n] = __builtin_fmaf(s[st][n], r.y * scale[st], __builtin_fmaf(qsum[st], r.x, -msub[st]));
        if (!whole) {
          const int key = kt0 + 16 * n + col;
          s[st][n] = key >= wk.klo && key < lim[st] ? s[st][n] : -INFINITY;
        }
      }
    }
#pragma unroll
    for (int st = 0; st < Q; ++st) {
      const float tmax = fmaxf(fmaxf(s[st][0], s[st][1]), fmaxf(s[st][2], s[st][3]));
      // (scores are relative to msub)
      if (__builtin_amdgcn_ballot_w64(tmax > (m[st] == -INFINITY ? -INFINITY : room.room))) {
        float most = -INFINITY;        // the largest weight's exponent
#pragma unroll
        for (int n = 0; n < 4; ++n) most = fmaxf(most, s[st][n] + (float)exponent_of(vstep[n]));
        most = fmaxf(most, dpp_f<0x121>(most));      // over the group's 16 lanes
        most = fmaxf(most, dpp_f<0x122>(most));
        most = fmaxf(most, dpp_f<DPP_ROW_ROR4>(most));
        most = fmaxf(most, dpp_f<DPP_ROW_ROR8>(most));
        const bool grow = most > (m[st] == -INFINITY ? -INFINITY : kTop);
        const float up = grow ? most - (kTop - kSlack) : 0.f;
        const float alpha = !grow ? 1.f : m[st] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(-up);
        msub[st] += up;
        m[st] = grow ? msub[st] : m[st];
        l[st] *= alpha;
        vt[st] *= alpha;
        float both[Q];
#pragma unroll
        for (int i = 0; i < Q; ++i) both[i] = i == st ? alpha : 1.f;
        const float a = of_column(both);
#pragma unroll
        for (int c = 0; c < RB; ++c) sum.o[0][c] *= a;
#pragma unroll
        for (int n = 0; n < 4; ++n) s[st][n] -= up;
      }
      float w[4];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const float pr = __builtin_amdgcn_exp2f(s[st][n]);
        l[st] += pr;
        vt[st] = __builtin_fmaf(pr, vmin[n], vt[st]);
        w[n] = pr * vstep[n];
      }
      // (remainders have columns of their own: in units of 2^-35, at most 2^14)
      const half2v h0 = halves(w[0], w[1]), h1 = halves(w[2], w[3]);
      const half2v l0 = halves((w[0] - (float)h0[0]) * 2048.0f, (w[1] - (float)h0[1]) * 2048.0f);
      const half2v l1 = halves((w[2] - (float)h1[0]) * 2048.0f, (w[3] - (float)h1[1]) * 2048.0f);
      uint8_t* const to = weights + (4 * st + grp) * kWeightRow + 8 * col;
      *reinterpret_cast<uint2*>(to) = make_uint2(__builtin_bit_cast(uint32_t, h0), __builtin_bit_cast(uint32_t, h1));
      *reinterpret_cast<uint2*>(to + 8 * kWeightRow) = make_uint2(__builtin_bit_cast(uint32_t, l0), __builtin_bit_cast(uint32_t, l1));
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const half8 b = *reinterpret_cast<const half8*>(weights + col * kWeightRow + 64 * h + 16 * grp);
      x.values(h, ex, [&](int c, half8 a) { sum.o[0][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, sum.o[0][c], 0, 0, 0); });
    }
    __builtin_amdgcn_wave_barrier();
    if (t + wk.step < wk.hi) {
      x.load_v(off_next);
      off_next = x.place(t + 2 * wk.step < wk.hi ? t + 2 * wk.step : t);
    }
  }
#pragma unroll
  for (int st = 0; st < Q; ++st)
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) {
      l[st] += __shfl_xor(l[st], o, 64);
      vt[st] += __shfl_xor(vt[st], o, 64);
    }
  sum.m[0] = of_column(m);
  sum.l[0] = of_column(l);
  sum.vt[0] = of_column(vt);
  sum.m[0] = reference_of(sum.m[0], sum.l[0]);
#pragma unroll
  for (int c = 0; c < RB; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i) sum.o[0][c][i] = __builtin_fmaf(dpp_f<DPP_ROW_ROR8>(sum.o[0][c][i]), 0x1p-11f, sum.o[0][c][i]);
}

// The sums of the lane's column, times f, four dims at a time: put(dim, values).  With f = 0 the sums are 0 or finite.
template <int D, int S, typename F>
__device__ __forceinline__ void each_four(const Sums<D, S>& sum, int st, float f, F put) {
  using GG = Geo<D>;
  constexpr int N = 2 * GG::VB;        // dims side by side: N (4 grp + i) ...
  const int grp = (threadIdx.x & 63) >> 4;
  const float vt = f * sum.vt[st];
  auto of = [&](int c, int i) { return __builtin_fmaf(sum.o[st][c][i], f, vt); };
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int c = 0; c < N; c += 4) put(N * (4 * grp + i) + c, make_float4(of(c, i), of(c + 1, i), of(c + 2, i), of(c + 3, i)));
  if constexpr (GG::X) put(64 + 4 * grp, make_float4(of(GG::RB - 1, 0), of(GG::RB - 1, 1), of(GG::RB - 1, 2), of(GG::RB - 1, 3)));
}

// The sums of a workgroup's waves over a shared item's part, joined and written.
template <int D, int S>
__device__ __forceinline__ void join_waves(const SharedParams& p, const Work& wk, int kv, uint8_t* smem, int slot, Sums<D, S>& sum) {
  using GG = Geo<D>;
  constexpr int RB = GG::RB;
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, grp = lane >> 4, wave = uniform(tid >> 6);
  float* const join = reinterpret_cast<float*>(smem);
  float2* const jml = reinterpret_cast<float2*>(smem + GG::JOIN);
  constexpr int C = S * COLS;
  if (grp == 0)
#pragma unroll
    for (int st = 0; st < S; ++st)
      if (COLS * st + col < wk.ncols) jml[wave * C + COLS * st + col] = make_float2(sum.m[st], sum.l[st]);
  __syncthreads();
#pragma unroll
  for (int st = 0; st < S; ++st) {
    if (__builtin_amdgcn_ballot_w64(sum.m[st] == -INFINITY)) {      // (nor may what a column does not see reach the sums)
      const bool none = sum.m[st] == -INFINITY;
      sum.vt[st] = none ? 0.f : sum.vt[st];
#pragma unroll
      for (int c = 0; c < RB; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) sum.o[st][c][i] = none ? 0.f : sum.o[st][c][i];
    }
    if (COLS * st + col >= wk.ncols) continue;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) top = fmaxf(top, jml[w * C + COLS * st + col].x);
    const float f = sum.m[st] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sum.m[st] - top);
    float* const jo = join + (wave * C + COLS * st + col) * GG::OROW;
    each_four<D, S>(sum, st, f, [&](int d, float4 v) { *reinterpret_cast<float4*>(jo + d) = v; });
  }
  __syncthreads();
  const bool has = slot < p.part_slots;
  const int64_t row = ((int64_t)slot * p.KV + kv) * (SETS * COLS);
  for (int e = tid; has && e < wk.ncols * (D / 4); e += WAVES * 64) {
    const int c = e / (D / 4), d = 4 * (e % (D / 4));
    float4 v = *reinterpret_cast<const float4*>(join + c * GG::OROW + d);
#pragma unroll
    for (int w = 1; w < WAVES; ++w) {
      const float4 x = *reinterpret_cast<const float4*>(join + (w * C + c) * GG::OROW + d);
      v = make_float4(v.x + x.x, v.y + x.y, v.z + x.z, v.w + x.w);
    }
    *reinterpret_cast<float4*>(p.part_o + (row + c) * D + d) = v;
  }
  if (has && tid < wk.ncols) {
    float mm = -INFINITY, ll = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) mm = fmaxf(mm, jml[w * C + tid].x);
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float2 x = jml[w * C + tid];
      ll += x.x == -INFINITY ? 0.f : x.y * __builtin_amdgcn_exp2f(x.x - mm);
    }
    reinterpret_cast<float2*>(p.part_ml)[row + tid] = make_float2(mm, ll);
  }
  __syncthreads();                     // (before the next job's rulers and sums)
}

template <int D>
__global__ void __launch_bounds__(WAVES * 64) __attribute__((amdgpu_waves_per_eu(Geo<D>::WGS))) shared_kernel(const SharedParams p) {
  using GG = Geo<D>;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int id = blockIdx.x, run = uniform(divide(id >> 3, p.KV)), kv = (id >> 3) - run * p.KV;
  const Schedule s = make_schedule(p, reinterpret_cast<int*>(smem + GG::FIXED));
  if (id == 0) {      // for merge_kernel: where a sequence's parts are
    for (int b = tid; b < p.B; b += WAVES * 64) {
      int4 a = make_int4(0, 0, 0, 0);
      if (p.R > 0 && b >= s.start[0] && b < s.start[p.R]) {
        const int r = last_at_most(s.start, p.R, b);
        a = make_int4(s.part[r], s.parts(p, r), sets_of(s.columns(p, r)), (b - s.start[r]) * p.G);
      }
      p.records[2 * b] = a;
      p.records[2 * b + 1] = make_int4(s.chunk[b], s.fit.chunks(tiles_of(s.own_from(p, b), s.len[b])), s.len[b] > 0, 0);
    }
  }
  // Workgroup id runs on XCD id % 8.  Jobs that read the same keys stand behind one another, and an XCD has an unbroken
  // run of the shared ones and one of the others, for all KV heads at a time, since a token's heads lie side by side and
  // share cache lines.  All XCDs have as many jobs, give or take one, and of the shared ones their part.
  const int xcd = id & 7, jobs = s.shared + (s.chunks + WAVES - 1) / WAVES;
  const int from = jobs * xcd >> 3, to = jobs * (xcd + 1) >> 3;
  const float share = (float)s.shared * __builtin_amdgcn_rcpf((float)max(jobs, 1));
  auto shared_of = [&](int n) {        // exactly the whole part of n * shared / jobs: never more of one than of all
    int q = uniform((int)((float)n * share));
    const int64_t all = (int64_t)n * s.shared;
    while ((int64_t)q * jobs > all) --q;
    while ((int64_t)(q + 1) * jobs <= all && q < n) ++q;
    return q;
  };
  const int sfrom = shared_of(from), scount = shared_of(to) - sfrom, ofrom = from - sfrom, ocount = to - from - scount;
  for (int k = run; run < s.width / 8 && k < scount + ocount; k += s.width / 8) {
    Work wk;
    wk.len = s.len;
    int slot;
    if (k < scount) {
      slot = sfrom + k;
      const int r = uniform(last_at_most(s.part, p.R, slot)), rel = slot - uniform(s.part[r]);
      const int columns = uniform(s.columns(p, r)), sets = sets_of(columns), part = uniform(divide(rel, sets)), set = rel - part * sets;
      wk.seq0 = uniform(s.start[r]);
      wk.flat0 = set * SETS * COLS;
      wk.ncols = min(SETS * COLS, columns - wk.flat0);
      wk.klo = 0;
      wk.khi = uniform(s.prefix[r]);
      const int tiles = tiles_of(0, wk.khi);
      const Run run = share_of((tiles + WAVES - 1) / WAVES, uniform(s.fit.parts(tiles, columns)), part);
      wk.lo = WAVES * run.from + wave;
      wk.hi = min(WAVES * run.to, tiles);
      wk.step = WAVES;
      wk.own = false;
    } else {
      slot = (ofrom + k - scount) * WAVES + wave;
      if (slot >= s.chunks) continue;
      const int b = uniform(last_at_most(s.chunk, p.B, slot));
      wk.seq0 = b;
      wk.klo = uniform(s.own_from(p, b));
      wk.khi = uniform(s.len[b]);
      const int tiles = tiles_of(wk.klo, wk.khi);
      const int chunks = uniform(s.fit.chunks(tiles));
      int c = slot - uniform(s.chunk[b]), set = 0;
      if (p.own_sets > 1) {
        set = uniform(divide(c, chunks));
        c -= set * chunks;
      }
      wk.flat0 = set * COLS;
      wk.ncols = min(COLS, p.G - wk.flat0);
      const Run run = share_of(tiles, chunks, c);
      wk.lo = run.from;
      wk.hi = run.to;
      wk.step = 1;
      wk.own = true;
    }
    uint8_t* const wave_lds = smem + wave * GG::WAVE;
    if (wk.ncols > COLS) {
      Sums<D, SETS> sum;
      attend<D, SETS>(p, wk, kv, wave_lds, sum);
      join_waves<D, SETS>(p, wk, kv, smem, slot, sum);
      continue;
    }
    Sums<D, 1> sum;                    // (by the number of columns, the same in all of a workgroup's waves)
    if (wk.ncols <= 4) attend_few<D, 1>(p, wk, kv, wave_lds, wave_lds + 16 * TK, sum);
    else if (wk.ncols <= 8) attend_few<D, 2>(p, wk, kv, wave_lds, wave_lds + 16 * TK, sum);
    else attend<D, 1>(p, wk, kv, wave_lds, sum);
    if (!wk.own) {
      join_waves<D, 1>(p, wk, kv, smem, slot, sum);
      continue;
    }
    const int col = lane & 15;
    if (col < wk.ncols && slot < p.own_slots) {
      const int64_t row = ((int64_t)slot * p.KV + kv) * p.own_cols + col;
      each_four<D, 1>(sum, 0, 1.f, [&](int d, float4 v) { *reinterpret_cast<float4*>(p.own_o + row * D + d) = v; });
      if (lane < COLS) reinterpret_cast<float2*>(p.own_ml)[row] = make_float2(sum.m[0], sum.l[0]);
    }
  }
}

// Joins the parts of a sequence's query head: four dims a thread, the parts shared out over teams of threads.
template <int D>
__global__ void __launch_bounds__(256) merge_kernel(const SharedParams p) {
  constexpr int WIDE = D / 4, TEAMS = 256 / WIDE;
  __shared__ float4 team_o[256];
  __shared__ float2 team_ml[256];
  const int b = blockIdx.y, head = blockIdx.x, kv = head / p.G, g = head - kv * p.G, tid = threadIdx.x;
  const int4 pre = p.records[2 * b], own = p.records[2 * b + 1];
  const int team = tid / WIDE, mine = tid - team * WIDE, d = 4 * mine;
  // parts: those of the shared tokens, then those of the sequence's own
  constexpr int C = SETS * COLS;
  const int flat = pre.w + g, np = pre.y, n = np + own.y;
  const int64_t prow = ((int64_t)(pre.x + flat / C) * p.KV + kv) * C + flat % C, pstep = (int64_t)pre.z * p.KV * C;
  const int64_t orow = ((int64_t)(own.x + (g / COLS) * own.y) * p.KV + kv) * p.own_cols + g % COLS, ostep = (int64_t)p.KV * p.own_cols;
  auto ml = [&](int i) {
    return i < np ? reinterpret_cast<const float2*>(p.part_ml)[prow + i * pstep] : reinterpret_cast<const float2*>(p.own_ml)[orow + (i - np) * ostep];
  };
  auto sums = [&](int i) {
    return *reinterpret_cast<const float4*>(i < np ? p.part_o + (prow + i * pstep) * D + d : p.own_o + (orow + (i - np) * ostep) * D + d);
  };
  float top = -INFINITY, L = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
  auto add = [&](float2 x, float4 o, float to) {
    const float f = x.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(x.x - to);   // no key of the part: 0
    L = __builtin_fmaf(f, x.y, L);
    v[0] = __builtin_fmaf(f, o.x, v[0]);
    v[1] = __builtin_fmaf(f, o.y, v[1]);
    v[2] = __builtin_fmaf(f, o.z, v[2]);
    v[3] = __builtin_fmaf(f, o.w, v[3]);
  };
  constexpr int U = 4;                 // parts read at a time
  if (team < TEAMS) {
    for (int i0 = team; i0 < n; i0 += U * TEAMS) {
      float2 x[U];
      float4 o[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = min(i0 + u * TEAMS, n - 1);
        x[u] = ml(i);
        o[u] = sums(i);
        if (i0 + u * TEAMS >= n) x[u].x = -INFINITY;
      }
      float t = top;
#pragma unroll
      for (int u = 0; u < U; ++u) t = fmaxf(t, x[u].x);
      const float f = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - t);
      L *= f;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] *= f;
      top = t;
#pragma unroll
      for (int u = 0; u < U; ++u) add(x[u], o[u], top);
    }
    team_ml[tid] = make_float2(top, L);
    team_o[tid] = make_float4(v[0], v[1], v[2], v[3]);
  }
  __syncthreads();
  if (team > 0) return;
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < TEAMS; ++i) m = fmaxf(m, team_ml[i * WIDE + mine].x);
  L = v[0] = v[1] = v[2] = v[3] = 0.f;
#pragma unroll
  for (int i = 0; i < TEAMS; ++i) add(team_ml[i * WIDE + mine], team_o[i * WIDE + mine], m);
  const float rL = 1.0f / L;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = own.z ? v[i] * rL : 0.f;
  const int64_t to = (int64_t)b * p.out_seq_stride + (int64_t)head * p.out_head_stride + d;
  if (p.out_f16)
    *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p.out) + to) =
        make_uint2((uint32_t)f2h(v[0]) | ((uint32_t)f2h(v[1]) << 16), (uint32_t)f2h(v[2]) | ((uint32_t)f2h(v[3]) << 16));
  else
    *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.out) + to) = make_float4(v[0], v[1], v[2], v[3]);
}

struct Sizes {
  int W, own_sets, own_cols;
  int64_t part_slots, own_slots, records, part_o, part_ml, own_o, own_ml, bytes;
};

// Workgroups per KV head, a multiple of the XCDs: in all as many as the chip holds at a time.
Sizes sizes_of(int B, int R, int H, int KV, int D) {
  Sizes z;
  const int G = H / KV, cus = device_cu_count();
  const int slots = (D == 64 ? Geo<64>::WGS : D == 80 ? Geo<80>::WGS : Geo<128>::WGS) * (cus > 0 ? cus : 256);   // (without a device: the MI355X)
  z.W = std::max(1, slots / (8 * KV)) * 8;
  z.own_sets = (G + COLS - 1) / COLS;
  z.own_cols = std::min(G, COLS);
  z.part_slots = R ? z.W + (int64_t)B * G / (SETS * COLS) + std::min(R, B) : 0;
  z.own_slots = (int64_t)z.W * WAVES + (int64_t)B * z.own_sets;
  const int64_t prows = z.part_slots * KV * SETS * COLS, orows = z.own_slots * KV * z.own_cols;
  z.records = 0;
  z.part_o = 32 * (int64_t)B;
  z.own_o = z.part_o + prows * D * 4;
  z.part_ml = z.own_o + orows * D * 4;
  z.own_ml = z.part_ml + prows * 8;
  z.bytes = z.own_ml + orows * 8;
  return z;
}

template <int D>
int launch(const SharedParams& p, hipStream_t stream) {
  const int lds = Geo<D>::FIXED + 4 * (3 * p.R + 2 + 2 * p.B + 1);
  static const bool lds_ok = [] {   // (more than 64 KB)
    return hipFuncSetAttribute(reinterpret_cast<const void*>(shared_kernel<D>), hipFuncAttributeMaxDynamicSharedMemorySize,
                               Geo<D>::FIXED + 4 * (5 * kMaxSeqs + 3)) == hipSuccess;
  }();
  if (!lds_ok) return fail(SLMT_ERR_HIP, "shared decode: could not grant the kernel its LDS");
  hipLaunchKernelGGL((shared_kernel<D>), dim3((unsigned)(p.W * p.KV)), dim3(WAVES * 64), lds, stream, p);
  if (int rc = check_launch("shared decode")) return rc;
  hipLaunchKernelGGL((merge_kernel<D>), dim3(p.KV * p.G, (unsigned)p.B), dim3(256), 0, stream, p);
  return check_launch("shared decode merge");
}

}  // namespace shared

static int check_shared_sizes(int B, int R, int H, int KV) {
  if (B > shared::kMaxSeqs || R > shared::kMaxSeqs)
    return fail(SLMT_ERR_UNSUPPORTED, "shared decode: at most " + std::to_string(shared::kMaxSeqs) + " sequences and groups a call, got " +
                                          std::to_string(B) + " and " + std::to_string(R));
  if (H > 65535 || (int64_t)H * B > (1 << 30)) return fail(SLMT_ERR_UNSUPPORTED, "shared decode: too many heads for one launch");
  return SLMT_OK;
}

int64_t shared_workspace_bytes(int B, int R, int H, int KV, int D) {
  if (check_shared_sizes(B, R, H, KV) != SLMT_OK) return -1;
  return shared::sizes_of(B, R, H, KV, D).bytes;
}

int launch_shared(int D, SharedParams& p, int H, void* workspace, int64_t ws_bytes, hipStream_t stream) {
  if (int rc = check_shared_sizes(p.B, p.R, H, p.KV)) return rc;
  const shared::Sizes z = shared::sizes_of(p.B, p.R, H, p.KV, D);
  if ((int64_t)p.block_size * p.KV * (D + 8) >= (int64_t(1) << 31))
    return fail(SLMT_ERR_UNSUPPORTED, "shared decode: a cache block of 2 GiB or more");
  // (tiles' costs are summed up in 32 bits, tiles of a row divided in fp32)
  const int64_t items = (int64_t)p.B * z.own_sets + (p.R ? (int64_t)p.B * p.G / (shared::SETS * shared::COLS) + std::min(p.R, p.B) : 0);
  if (p.max_tokens > shared::kMaxTokens || shared::kCostTwo * ((int64_t)p.max_tokens / shared::TK + 2) * items >= (int64_t(1) << 31))
    return fail(SLMT_ERR_UNSUPPORTED, "shared decode: block tables too wide for so many sequences");
  p.G_inverse = p.G > 1 ? (uint32_t)(((uint64_t(1) << 32) + p.G - 1) / p.G) : 0;
  if (workspace == nullptr || ws_bytes < z.bytes)
    return fail(SLMT_ERR_INVALID, "shared decode: workspace of " + std::to_string(z.bytes) + " bytes required, got " + std::to_string(ws_bytes));
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return fail(SLMT_ERR_INVALID, "shared decode: the workspace must be 16-byte aligned");
  uint8_t* const ws = reinterpret_cast<uint8_t*>(workspace);
  p.W = z.W;
  p.own_sets = z.own_sets;
  p.own_cols = z.own_cols;
  p.part_slots = (int)z.part_slots;
  p.own_slots = (int)z.own_slots;
  p.records = reinterpret_cast<int4*>(ws + z.records);
  p.part_o = reinterpret_cast<float*>(ws + z.part_o);
  p.own_o = reinterpret_cast<float*>(ws + z.own_o);
  p.part_ml = reinterpret_cast<float*>(ws + z.part_ml);
  p.own_ml = reinterpret_cast<float*>(ws + z.own_ml);
  if (D == 64) return shared::launch<64>(p, stream);
  if (D == 80) return shared::launch<80>(p, stream);
  return shared::launch<128>(p, stream);
}

}  // namespace slmt
