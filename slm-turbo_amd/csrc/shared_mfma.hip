// Decode attention of sequences that share a prompt, over the packed per-token 4-bit paged
// cache on the matrix cores, head_dim 64, 80 and 128, any number of query heads per KV head.
// (The reference has no counterpart: its paged decode reads every sequence's whole row,
// kernels/kv_dequant_kernels.cuh:671-801.)
//
// For a sequence of L tokens whose group shares the first P of them,
//   out = sum_t e^{s_t} v_t / sum_t e^{s_t},   s_t = q . k_t / sqrt(D),
// is joined from two sums, over t < P and over P <= t < L.  The first is computed for all
// sequences of the group at once, so the prompt's keys and values are read and unpacked once
// for 16 columns, column = (sequence, query head of the KV head); the second for a sequence's
// own query heads.  Both are items of one list: 16 columns, a row of the block tables, a range
// of keys.  The tiles (64 keys) of all items stand behind one another, and every workgroup
// takes an equal run of them for one KV head, so the split of the work needs no lengths on the
// host.  A run's part of an item is a partial result (m, l, o); merge_kernel, next on the
// stream, joins a query head's.
//
// A wave works on a tile by itself, from registers: lane (c = lane & 15, g = lane >> 4) reads a
// quarter of key c's codes, which is its part of K as the matrix cores' left operand, and of
// the values of keys 4 g + i the bytes at its place c, from which a byte permute makes pairs of
// keys.  Everything is transposed, so that a lane owns a column from the scores to the output:
//   S^T = K Q^T,  P^T = exp2(S^T - m),  O^T += V^T P^T    (v_mfma_f32_16x16x32_f16)
//
// Exactness: codes enter as n - 8 and the query as it is, both fp16 numbers, so a score is
// kstep (q . (n - 8)) + (kmin + 8 kstep) sum(q) with fp32 sums (log2(e) / sqrt(D) folded into
// the rulers).  Weights p * vstep enter as an fp16 number and the fp16 remainder in units of
// 2^-11, two products into two accumulators, ~22 bits; sum(p) and sum(p (vmin + 8 vstep)) stay
// in fp32.
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
constexpr int COLS = 16;           // columns per item
constexpr int WAVES = 4;           // waves per workgroup
constexpr float kMargin = 4.0f;    // the weights' reference lies this far (base 2) above the largest score
constexpr int kMaxSeqs = 4096;     // sequences and groups of a call (their places are in LDS)

template <int D>
struct Geo {
  static constexpr int KW = D == 128 ? 4 : 2;        // dwords of K codes per key and lane (32 or 16 dims)
  static constexpr bool X = D == 80;                 // 16 dims more: 2 bytes of K, a nibble of V
  static constexpr int KB = KW + (X ? 1 : 0);        // 32-dim blocks of QK
  static constexpr int VB = D == 128 ? 4 : 2;        // bytes of V per key and lane
  static constexpr int RB = D / 16;                  // 16-dim blocks of PV
  static constexpr int OROW = D + 4;                 // floats of a column in the join
  static constexpr int JOIN = WAVES * COLS * OROW * 4;
  static constexpr int RULERS = WAVES * TK * 16;
  static constexpr int FIXED = JOIN + RULERS + WAVES * COLS * 8;
};

// Codes n of halves' low or second nibbles as the fp16 numbers n - 8: the nibble under an
// exponent that makes it 1024 + n or 64 + n, and one exact packed sum.
__device__ __forceinline__ uint32_t low_codes(uint32_t w) {
  const uint32_t x = (w & 0x000F000Fu) | 0x64006400u;
  return __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2v, x) + half2v{(_Float16)-1032.0f, (_Float16)-1032.0f});
}
__device__ __forceinline__ uint32_t high_codes(uint32_t w) {
  const uint32_t x = (w & 0x00F000F0u) | 0x54005400u;
  return __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2v, x) + half2v{(_Float16)-72.0f, (_Float16)-72.0f});
}
// The eight codes of a dword, dims 0, 4, 1, 5, 2, 6, 3, 7 of its eight.
__device__ __forceinline__ half8 codes8(uint32_t w) {
  const uint32_t s = w >> 8;
  const uint4 r = make_uint4(low_codes(w), high_codes(w), low_codes(s), high_codes(s));
  return __builtin_bit_cast(half8, r);
}
__device__ __forceinline__ int dim_of(int e) { return (e >> 1) + 4 * (e & 1); }

__device__ __forceinline__ int seq_len(const SharedParams& p, int b) { return min(max(p.seq_lens[b], 0), p.max_tokens); }

// Where everything is: in LDS, for all workgroups alike.
struct Schedule {
  int *start;     // [R + 1] the groups' first sequences
  int *prefix;    // [R] their shared tokens
  int *ptile;     // [R + 1] tiles of the groups before, over all their sets of columns
  int *pitem;     // [R + 1] sets of columns of the groups before
  int *own;       // [B] tokens of a sequence that its group reads
  int *otile;     // [B + 1] tiles of the sequences before
  int total, per; // tiles in all, and of a workgroup
};
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

// Exclusive sums of a[0 .. n) in place, their total in a[n]; one wave.
__device__ __forceinline__ void scan(int* a, int n) {
  const int lane = threadIdx.x & 63;
  int base = 0;
  for (int i = 0; i < n; i += 64) {
    const int v = i + lane < n ? a[i + lane] : 0;
    int incl = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int u = __shfl_up(incl, o, 64);
      if (lane >= o) incl += u;
    }
    if (i + lane < n) a[i + lane] = base + incl - v;
    base += __builtin_amdgcn_readlane(incl, 63);
  }
  if (lane == 0) a[n] = base;
}

__device__ __forceinline__ Schedule make_schedule(const SharedParams& p, int* lds) {
  const int tid = threadIdx.x, R = p.R, B = p.B, wave = tid >> 6;
  Schedule s;
  s.start = lds;
  s.prefix = s.start + R + 1;
  s.ptile = s.prefix + R;
  s.pitem = s.ptile + R + 1;
  s.own = s.pitem + R + 1;
  s.otile = s.own + B;
  if (wave == 0) {      // starts that never fall, whatever the caller's are: all that follows holds for them
    const int lane = tid & 63;
    int most = 0;
    for (int i = 0; i <= R; i += 64) {
      int v = max(most, i + lane <= R ? min(max(p.group_start[i + lane], 0), B) : 0);
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(v, o, 64);
        if (lane >= o) v = max(v, u);
      }
      if (i + lane <= R) s.start[i + lane] = v;
      most = __builtin_amdgcn_readlane(v, 63);
    }
  } else {
    for (int i = tid - 64; i < R; i += (WAVES - 1) * 64) s.prefix[i] = min(max(p.prefix_lens[i], 0), p.max_tokens);
    for (int b = tid - 64; b < B; b += (WAVES - 1) * 64) s.otile[b] = seq_len(p, b);
  }
  __syncthreads();
  for (int i = tid; i < R; i += WAVES * 64) {
    const int sets = ((s.start[i + 1] - s.start[i]) * p.G + COLS - 1) / COLS;
    s.pitem[i] = sets;
    s.ptile[i] = sets * tiles_of(0, s.prefix[i]);
  }
  for (int b = tid; b < B; b += WAVES * 64) {
    const int len = s.otile[b];
    int pre = 0;
    if (R > 0 && b >= s.start[0] && b < s.start[R]) pre = min(s.prefix[last_at_most(s.start, R, b)], len);
    s.own[b] = pre;
    s.otile[b] = tiles_of(pre, len) * p.own_sets;
  }
  __syncthreads();
  if (wave == 0) scan(s.ptile, R);
  if (wave == 1) scan(s.pitem, R);
  if (wave == 2) scan(s.otile, B);
  __syncthreads();
  s.total = __builtin_amdgcn_readfirstlane(s.ptile[R] + s.otile[B]);
  // (a multiple of the waves, which take the tiles in turn)
  s.per = max(1, (s.total + p.W * WAVES - 1) / (p.W * WAVES)) * WAVES;
  return s;
}

template <int D>
__global__ void __launch_bounds__(WAVES * 64) __attribute__((amdgpu_waves_per_eu(2))) shared_kernel(const SharedParams p) {
  using GG = Geo<D>;
  constexpr int KW = GG::KW, KB = GG::KB, VB = GG::VB, RB = GG::RB, SLOT = D + 8;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, grp = lane >> 4;
  // Workgroups of one run, for all KV heads, are 8 apart and so on one XCD: a token's heads lie
  // side by side, and share cache lines.
  const int id = blockIdx.x, run = (id / (8 * p.KV)) * 8 + (id & 7), kv = (id >> 3) % p.KV;
  float* const join = reinterpret_cast<float*>(smem);
  uint8_t* const rulers = smem + GG::JOIN + wave * TK * 16;
  float2* const jml = reinterpret_cast<float2*>(smem + GG::JOIN + GG::RULERS);
  const Schedule s = make_schedule(p, reinterpret_cast<int*>(smem + GG::FIXED));
  if (id == 0) {      // for merge_kernel: where a sequence's parts are
    for (int b = tid; b < p.B; b += WAVES * 64) {
      int4 a = make_int4(0, 0, 0, 0);
      if (p.R > 0 && b >= s.start[0] && b < s.start[p.R]) {
        const int r = last_at_most(s.start, p.R, b);
        a = make_int4(s.ptile[r], tiles_of(0, s.prefix[r]), s.pitem[r], (b - s.start[r]) * p.G);
      }
      const int mine = (s.otile[b + 1] - s.otile[b]) / p.own_sets;
      p.records[2 * b] = a;
      p.records[2 * b + 1] = make_int4(s.ptile[p.R] + s.otile[b], mine, s.per, 0);
    }
  }
  const int first = run * s.per, last = min(s.total, first + s.per);
  const uint32_t row_bytes = (uint32_t)p.KV * SLOT;
  const int64_t block_bytes = (int64_t)p.block_size * row_bytes;
  const int esh = p.bt64 ? 3 : 2;
  constexpr float kC = 1.4426950408889634f / (D == 64 ? 8.0f : D == 80 ? 8.94427190999916f : 11.313708498984761f);

  for (int at = first; at < last;) {
    // ---- the item that tile `at` belongs to
    int seq0, flat0, ncols, klo, khi, tile, tiles, item;
    const bool mine = at >= s.ptile[p.R];
    if (!mine) {
      const int r = last_at_most(s.ptile, p.R, at), n = s.start[r + 1] - s.start[r];
      seq0 = s.start[r];
      khi = s.prefix[r];
      klo = 0;
      tiles = tiles_of(0, khi);
      const int set = (at - s.ptile[r]) / tiles;
      tile = at - s.ptile[r] - set * tiles;
      flat0 = set * COLS;
      ncols = min(COLS, n * p.G - flat0);
      item = s.pitem[r] + set;
    } else {
      const int t = at - s.ptile[p.R], b = last_at_most(s.otile, p.B, t);
      seq0 = b;
      klo = s.own[b];
      khi = seq_len(p, b);
      tiles = tiles_of(klo, khi);
      const int set = (t - s.otile[b]) / tiles;
      tile = t - s.otile[b] - set * tiles;
      flat0 = set * COLS;
      ncols = min(COLS, p.G - flat0);
      item = b * p.own_sets + set;
    }
    seq0 = __builtin_amdgcn_readfirstlane(seq0);
    klo = __builtin_amdgcn_readfirstlane(klo);
    khi = __builtin_amdgcn_readfirstlane(khi);
    tile = __builtin_amdgcn_readfirstlane(tile);
    tiles = __builtin_amdgcn_readfirstlane(tiles);
    flat0 = __builtin_amdgcn_readfirstlane(flat0);
    ncols = __builtin_amdgcn_readfirstlane(ncols);
    item = __builtin_amdgcn_readfirstlane(item);
    const int count = min(tiles - tile, last - at);      // tiles of the item in this run
    at += count;

    // ---- the lane's column (those past the item's repeat the last)
    const int flat = flat0 + min(col, ncols - 1);
    const int seq = mine ? seq0 : seq0 + flat / p.G, head = kv * p.G + (mine ? flat : flat % p.G);
    const int lim = mine ? khi : min(khi, seq_len(p, seq));      // keys below it are seen
    half8 qh[KB];
    float qsum = 0.f;
    {
      const uint16_t* q = p.q + (int64_t)seq * p.q_seq_stride + (int64_t)head * p.q_head_stride;
#pragma unroll
      for (int j = 0; j < KW; ++j) {
        const half8 x = *reinterpret_cast<const half8*>(q + 8 * (KW * grp + j));
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          qh[j][e] = x[dim_of(e)];
          qsum += (float)x[e];
        }
      }
      if constexpr (GG::X) {
        const half4 x = *reinterpret_cast<const half4*>(q + 64 + 4 * grp);
        qh[KW] = half8{x[0], (_Float16)0.f, x[1], (_Float16)0.f, x[2], (_Float16)0.f, x[3], (_Float16)0.f};
#pragma unroll
        for (int e = 0; e < 4; ++e) qsum += (float)x[e];
      }
      float a, b;
      swap16(qsum, a, b);
      qsum = a + b;
      swap32(qsum, a, b);
      qsum = a + b;
    }
    int lim_lo = lim;
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) lim_lo = min(lim_lo, __shfl_xor(lim_lo, o, 64));
    lim_lo = __builtin_amdgcn_readfirstlane(lim_lo);

    // ---- keys and values of the wave's tiles
    const int base = klo & ~15, end16 = (khi - 1) & ~15;
    const uint8_t* const table = reinterpret_cast<const uint8_t*>(p.block_tables) + (((int64_t)seq0 * p.bt_stride) << esh);
    // offset of the 16 keys that the lane's group has in tile t (past the end: the last ones)
    auto place = [&](int t) -> int64_t {
      const int key = min(base + t * TK + 16 * grp, end16);
      const int block = p.block_shift >= 0 ? key >> p.block_shift : key / p.block_size;
      const int in_block = key - block * p.block_size;
      const uint32_t entry = *reinterpret_cast<const uint32_t*>(table + ((int64_t)block << esh));
      return (int64_t)min(entry, p.last_block) * block_bytes + (uint32_t)(in_block * (int)row_bytes + kv * SLOT);
    };
    uint32_t kx[4][KW], kxx[4], vx[16], vxx[16];
    uint2 rl;
    auto base_of = [&](int64_t off, int i) -> const uint8_t* {
      const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)off, 16 * i), hi = __builtin_amdgcn_readlane((int)(off >> 32), 16 * i);
      return p.cache + (((uint64_t)hi << 32) | lo);
    };
    const uint32_t kfrom = col * row_bytes + 4 * KW * grp, kxfrom = col * row_bytes + 32 + 2 * grp;
    const uint32_t vfrom = 4 * grp * row_bytes + D / 2 + VB * col, vxfrom = 4 * grp * row_bytes + D / 2 + 32 + (col >> 1);
    auto load_k = [&](int64_t off) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint8_t* const b = base_of(off, i);
#pragma unroll
        for (int j = 0; j < KW; j += 2) {
          const uint2 x = *reinterpret_cast<const uint2*>(b + kfrom + 4 * j);
          kx[i][j] = x.x;
          kx[i][j + 1] = x.y;
        }
        if constexpr (GG::X) kxx[i] = *reinterpret_cast<const uint16_t*>(b + kxfrom);
      }
      rl = *reinterpret_cast<const uint2*>(p.cache + off + (uint32_t)(col * row_bytes + D));
    };
    auto load_v = [&](int64_t off) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint8_t* const b = base_of(off, i);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (VB == 4) vx[4 * i + e] = *reinterpret_cast<const uint32_t*>(b + e * row_bytes + vfrom);
          else vx[4 * i + e] = *reinterpret_cast<const uint16_t*>(b + e * row_bytes + vfrom);
          if constexpr (GG::X) vxx[4 * i + e] = b[e * row_bytes + vxfrom];
        }
      }
    };

    floatx4 o[RB], ol[RB];             // sums of the weights' products and of their remainders'
#pragma unroll
    for (int c = 0; c < RB; ++c) o[c] = ol[c] = floatx4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, msub = 0.f;   // the weights' reference; what is subtracted (0 while it is -inf)
    float l = 0.f, vt = 0.f;

    int64_t off = 0, off_next = 0;
    if (wave < count) {
      off = place(tile + wave);
      load_k(off);
      load_v(off);
      off_next = place(tile + min(wave + WAVES, count - 1));
    }
    for (int t = wave; t < count; t += WAVES) {
      const int kt0 = base + (tile + t) * TK;
      {   // the tile's rulers, a key a lane
        const float kmin = h2f((uint16_t)(rl.x & 0xffffu)), kstep = h2f((uint16_t)(rl.x >> 16));
        const float vmin = h2f((uint16_t)(rl.y & 0xffffu)), vstep = h2f((uint16_t)(rl.y >> 16));
        __builtin_amdgcn_wave_barrier();
        *reinterpret_cast<float2*>(rulers + 8 * lane) = make_float2(__builtin_fmaf(8.0f, kstep, kmin) * kC, kstep * kC);
        *reinterpret_cast<float2*>(rulers + 8 * (TK + lane)) = make_float2(__builtin_fmaf(8.0f, vstep, vmin), vstep);
        __builtin_amdgcn_wave_barrier();
      }
      floatx4 sc[4];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        sc[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8(kx[n][0]), qh[0], floatx4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
        for (int j = 1; j < KW; ++j) sc[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8(kx[n][j]), qh[j], sc[n], 0, 0, 0);
        if constexpr (GG::X) sc[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8(kxx[n]), qh[KW], sc[n], 0, 0, 0);
      }
      load_k(off_next);
      float tmax = -INFINITY;
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const float4* kr = reinterpret_cast<const float4*>(rulers + 8 * (16 * n + 4 * grp));
        const float4 k01 = kr[0], k23 = kr[1];
        sc[n][0] = __builtin_fmaf(sc[n][0], k01.y, __builtin_fmaf(qsum, k01.x, -msub));
        sc[n][1] = __builtin_fmaf(sc[n][1], k01.w, __builtin_fmaf(qsum, k01.z, -msub));
        sc[n][2] = __builtin_fmaf(sc[n][2], k23.y, __builtin_fmaf(qsum, k23.x, -msub));
        sc[n][3] = __builtin_fmaf(sc[n][3], k23.w, __builtin_fmaf(qsum, k23.z, -msub));
      }
      const bool whole = kt0 >= klo && kt0 + TK <= lim_lo;
      if (!whole) {                    // keys that a column does not see: weight 0
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = kt0 + 16 * n + 4 * grp + i;
            sc[n][i] = key >= klo && key < lim ? sc[n][i] : -INFINITY;
          }
      }
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) tmax = fmaxf(tmax, sc[n][i]);
      // (scores are relative to msub)
      if (__builtin_amdgcn_ballot_w64(tmax > (m == -INFINITY ? -INFINITY : 0.f))) {
        float a, b;                    // over the four lane groups that hold the column
        swap16(tmax, a, b);
        tmax = fmaxf(a, b);
        swap32(tmax, a, b);
        tmax = fmaxf(a, b);
        const bool grow = tmax > (m == -INFINITY ? -INFINITY : 0.f);
        const float up = grow ? tmax + kMargin : 0.f;
        const float alpha = !grow ? 1.f : m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(-up);
        msub += up;
        m = grow ? msub : m;
        l *= alpha;
        vt *= alpha;
#pragma unroll
        for (int c = 0; c < RB; ++c) {
          o[c] *= alpha;
          ol[c] *= alpha;
        }
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[n][i] -= up;
      }
      half4 ph[4], pl[4];
      auto weights = [&](auto all) __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const float4* vr = reinterpret_cast<const float4*>(rulers + 8 * (TK + 16 * n + 4 * grp));
          const float4 v01 = vr[0], v23 = vr[1];
          float vmin[4] = {v01.x, v01.z, v23.x, v23.z}, vstep[4] = {v01.y, v01.w, v23.y, v23.w};
          if constexpr (!decltype(all)::value) {   // (nor may the rulers of keys that are not seen reach the sums)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int key = kt0 + 16 * n + 4 * grp + i;
              const bool ok = key >= klo && key < lim;
              vmin[i] = ok ? vmin[i] : 0.f;
              vstep[i] = ok ? vstep[i] : 0.f;
            }
          }
#pragma unroll
          for (int i = 0; i < 4; i += 2) {
            float pr[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              pr[e] = __builtin_amdgcn_exp2f(sc[n][i + e]);
              l += pr[e];
              vt = __builtin_fmaf(pr[e], vmin[i + e], vt);
            }
            // One rounding of the weight for both uses: through the empty asm, since the
            // compiler rounds product and conversion at once for one and apart for the
            // other, and where those differ the remainder is off by an fp16 ulp.
            uint32_t hw = __builtin_bit_cast(uint32_t, half2v{(_Float16)(pr[0] * vstep[i]), (_Float16)(pr[1] * vstep[i + 1])});
            asm("" : "+v"(hw));
            const half2v h2 = __builtin_bit_cast(half2v, hw);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              ph[n][i + e] = h2[e];
              pl[n][i + e] = (_Float16)(__builtin_fmaf(pr[e], vstep[i + e], -(float)h2[e]) * 2048.0f);
            }
          }
        }
      };
      if (whole) weights(std::true_type{});
      else weights(std::false_type{});
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const half8 bh = __builtin_shufflevector(ph[2 * h], ph[2 * h + 1], 0, 1, 2, 3, 4, 5, 6, 7);
        const half8 bl = __builtin_shufflevector(pl[2 * h], pl[2 * h + 1], 0, 1, 2, 3, 4, 5, 6, 7);
        auto products = [&](int c, const uint32_t (&w)[4]) {
          const half8 a = __builtin_bit_cast(half8, make_uint4(w[0], w[1], w[2], w[3]));
          o[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, bh, o[c], 0, 0, 0);
          ol[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, bl, ol[c], 0, 0, 0);
        };
#pragma unroll
        for (int b = 0; b < VB; ++b) {
          uint32_t lo[4], hi[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t pair = __builtin_amdgcn_perm(vx[8 * h + 2 * e + 1], vx[8 * h + 2 * e], 0x0C000C00u | ((4u + b) << 16) | (uint32_t)b);
            lo[e] = low_codes(pair);
            hi[e] = high_codes(pair);
          }
          products(2 * b, lo);
          products(2 * b + 1, hi);
        }
        if constexpr (GG::X) {
          uint32_t lo[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t pair = __builtin_amdgcn_perm(vxx[8 * h + 2 * e + 1], vxx[8 * h + 2 * e], 0x0C040C00u);
            lo[e] = low_codes(pair >> (4 * (col & 1)));
          }
          products(RB - 1, lo);
        }
      }
      load_v(off_next);
      off_next = place(tile + min(t + 2 * WAVES, count - 1));
    }

    // ---- the waves' sums, joined
    float a, b;
    swap16(l, a, b);
    l = a + b;
    swap32(l, a, b);
    l = a + b;
    swap16(vt, a, b);
    vt = a + b;
    swap32(vt, a, b);
    vt = a + b;
    __syncthreads();                   // (the last item's sums have been read)
    if (grp == 0) jml[wave * COLS + col] = make_float2(m, l);
    __syncthreads();
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) top = fmaxf(top, jml[w * COLS + col].x);
    const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
    float* const jo = join + (wave * COLS + col) * GG::OROW;
    auto sum_of = [&](int c, int i) { return f == 0.f ? 0.f : f * (__builtin_fmaf(ol[c][i], 0x1p-11f, o[c][i]) + vt); };
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      constexpr int N = 2 * VB;        // dims side by side: 2 VB (4 grp + i) ...
#pragma unroll
      for (int c = 0; c < N; c += 4)
        *reinterpret_cast<float4*>(jo + N * (4 * grp + i) + c) = make_float4(sum_of(c, i), sum_of(c + 1, i), sum_of(c + 2, i), sum_of(c + 3, i));
    }
    if constexpr (GG::X)
      *reinterpret_cast<float4*>(jo + 64 + 4 * grp) = make_float4(sum_of(RB - 1, 0), sum_of(RB - 1, 1), sum_of(RB - 1, 2), sum_of(RB - 1, 3));
    __syncthreads();
    const int64_t row = ((int64_t)(run + item) * p.KV + kv) * (mine ? p.own_cols : COLS);
    float* const part_o = mine ? p.own_o : p.part_o;
    float2* const part_ml = reinterpret_cast<float2*>(mine ? p.own_ml : p.part_ml);
    if (run + item < (mine ? p.own_slots : p.part_slots)) {
      for (int e = tid; e < ncols * (D / 4); e += WAVES * 64) {
        const int c = e / (D / 4), d = 4 * (e % (D / 4));
        float4 v = *reinterpret_cast<const float4*>(join + c * GG::OROW + d);
#pragma unroll
        for (int w = 1; w < WAVES; ++w) {
          const float4 x = *reinterpret_cast<const float4*>(join + (w * COLS + c) * GG::OROW + d);
          v = make_float4(v.x + x.x, v.y + x.y, v.z + x.z, v.w + x.w);
        }
        *reinterpret_cast<float4*>(part_o + (row + c) * D + d) = v;
      }
      if (tid < ncols) {
        float mm = -INFINITY, ll = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) mm = fmaxf(mm, jml[w * COLS + tid].x);
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
          const float2 x = jml[w * COLS + tid];
          ll += x.x == -INFINITY ? 0.f : x.y * __builtin_amdgcn_exp2f(x.x - mm);
        }
        part_ml[row + tid] = make_float2(mm, ll);
      }
    }
  }
}

// Joins the parts of a sequence's query heads of one KV head: four dims per thread, the parts
// of few heads shared out over teams of threads.
template <int D>
__global__ void __launch_bounds__(256) merge_kernel(const SharedParams p) {
  __shared__ float4 team_o[256];
  __shared__ float2 team_ml[256];
  const int b = blockIdx.x, kv = blockIdx.y, tid = threadIdx.x;
  const int4 pre = p.records[2 * b], own = p.records[2 * b + 1];
  const int per = own.z, all = p.G * (D / 4), wide = min(all, 256), teams = 256 / wide;
  const int team = tid / wide;
  for (int e0 = 0; e0 < all; e0 += wide) {
    const int e = e0 + tid - team * wide, g = min(e / (D / 4), p.G - 1), d = 4 * (e % (D / 4));
    // parts: those of the shared tokens, then those of the sequence's own
    const int flat = pre.w + g, pt = pre.x + (flat / COLS) * pre.y, ot = own.x + (g / COLS) * own.y;
    const int pw = pt / per, np = pre.y > 0 ? (pt + pre.y - 1) / per - pw + 1 : 0;
    const int ow = ot / per, no = own.y > 0 ? (ot + own.y - 1) / per - ow + 1 : 0;
    const int64_t prow = ((int64_t)(pw + pre.z + flat / COLS) * p.KV + kv) * COLS + flat % COLS;
    const int64_t orow = ((int64_t)(ow + b * p.own_sets + g / COLS) * p.KV + kv) * p.own_cols + g % COLS;
    auto ml = [&](int i) {
      return i < np ? reinterpret_cast<const float2*>(p.part_ml)[prow + (int64_t)i * p.KV * COLS]
                    : reinterpret_cast<const float2*>(p.own_ml)[orow + (int64_t)(i - np) * p.KV * p.own_cols];
    };
    float top = -INFINITY, L = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
    for (int i = team; i < np + no; i += teams) top = fmaxf(top, ml(i).x);
    for (int i = team; i < np + no; i += teams) {
      const float2 x = ml(i);
      const float4 o = *reinterpret_cast<const float4*>(i < np ? p.part_o + (prow + (int64_t)i * p.KV * COLS) * D + d
                                                               : p.own_o + (orow + (int64_t)(i - np) * p.KV * p.own_cols) * D + d);
      const float f = x.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(x.x - top);   // no key of the part: 0
      L = __builtin_fmaf(f, x.y, L);
      v[0] = __builtin_fmaf(f, o.x, v[0]);
      v[1] = __builtin_fmaf(f, o.y, v[1]);
      v[2] = __builtin_fmaf(f, o.z, v[2]);
      v[3] = __builtin_fmaf(f, o.w, v[3]);
    }
    if (teams > 1) {
      team_ml[tid] = make_float2(top, L);
      team_o[tid] = make_float4(v[0], v[1], v[2], v[3]);
      __syncthreads();
      const int mine = tid - team * wide;
      float m = -INFINITY;
      for (int i = 0; i < teams; ++i) m = fmaxf(m, team_ml[i * wide + mine].x);
      L = v[0] = v[1] = v[2] = v[3] = 0.f;
      for (int i = 0; i < teams; ++i) {
        const float2 x = team_ml[i * wide + mine];
        const float4 o = team_o[i * wide + mine];
        const float f = x.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(x.x - m);
        L = __builtin_fmaf(f, x.y, L);
        v[0] = __builtin_fmaf(f, o.x, v[0]);
        v[1] = __builtin_fmaf(f, o.y, v[1]);
        v[2] = __builtin_fmaf(f, o.z, v[2]);
        v[3] = __builtin_fmaf(f, o.w, v[3]);
      }
    }
    if (team == 0 && e < all) {
      const bool sees = seq_len(p, b) > 0;
      const float rL = 1.0f / L;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = sees ? v[i] * rL : 0.f;
      const int64_t to = (int64_t)b * p.out_seq_stride + (int64_t)(kv * p.G + g) * p.out_head_stride + d;
      if (p.out_f16)
        *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p.out) + to) =
            make_uint2((uint32_t)f2h(v[0]) | ((uint32_t)f2h(v[1]) << 16), (uint32_t)f2h(v[2]) | ((uint32_t)f2h(v[3]) << 16));
      else
        *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.out) + to) = make_float4(v[0], v[1], v[2], v[3]);
    }
  }
}

struct Sizes {
  int W, own_sets, own_cols;
  int64_t part_slots, own_slots, records, part_o, part_ml, own_o, own_ml, bytes;
};

// Runs of tiles per KV head, a multiple of the XCDs: two workgroups a CU in all, as many as its
// registers hold.
Sizes sizes_of(int B, int R, int H, int KV, int D) {
  Sizes z;
  const int G = H / KV, cus = device_cu_count();
  const int slots = 2 * (cus > 0 ? cus : 256);             // (sizes asked for without a device: the MI355X)
  z.W = std::max(1, slots / (8 * KV)) * 8;
  z.own_sets = (G + COLS - 1) / COLS;
  z.own_cols = std::min(G, COLS);
  z.part_slots = R ? z.W + (int64_t)B * G / COLS + std::min(R, B) : 0;
  z.own_slots = z.W + (int64_t)B * z.own_sets;
  const int64_t prows = z.part_slots * KV * COLS, orows = z.own_slots * KV * z.own_cols;
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
  const int lds = Geo<D>::FIXED + 4 * (4 * p.R + 3 + 2 * p.B + 1);
  static const bool lds_ok = [] {   // (more than 64 KB for many sequences)
    return hipFuncSetAttribute(reinterpret_cast<const void*>(shared_kernel<D>), hipFuncAttributeMaxDynamicSharedMemorySize,
                               Geo<D>::FIXED + 4 * (6 * kMaxSeqs + 4)) == hipSuccess;
  }();
  if (!lds_ok) return fail(SLMT_ERR_HIP, "shared decode: could not grant the kernel its LDS");
  hipLaunchKernelGGL((shared_kernel<D>), dim3((unsigned)(p.W * p.KV)), dim3(WAVES * 64), lds, stream, p);
  if (int rc = check_launch("shared decode")) return rc;
  hipLaunchKernelGGL((merge_kernel<D>), dim3((unsigned)p.B, p.KV), dim3(256), 0, stream, p);
  return check_launch("shared decode merge");
}

}  // namespace shared

static int check_shared_sizes(int B, int R, int H, int KV) {
  if (B > shared::kMaxSeqs || R > shared::kMaxSeqs)
    return fail(SLMT_ERR_UNSUPPORTED, "shared decode: at most " + std::to_string(shared::kMaxSeqs) + " sequences and groups a call, got " +
                                          std::to_string(B) + " and " + std::to_string(R));
  if (KV > 65535 || (int64_t)H * B > (1 << 30)) return fail(SLMT_ERR_UNSUPPORTED, "shared decode: too many heads for one launch");
  return SLMT_OK;
}

int64_t shared_workspace_bytes(int B, int R, int H, int KV, int D) {
  if (check_shared_sizes(B, R, H, KV) != SLMT_OK) return -1;
  return shared::sizes_of(B, R, H, KV, D).bytes;
}

int launch_shared(int D, SharedParams& p, int H, void* workspace, int64_t ws_bytes, hipStream_t stream) {
  if (int rc = check_shared_sizes(p.B, p.R, H, p.KV)) return rc;
  const shared::Sizes z = shared::sizes_of(p.B, p.R, H, p.KV, D);
  const int64_t per_row = (int64_t)p.max_tokens / shared::TK + 2;
  if (per_row * (z.own_slots + z.part_slots) >= (int64_t(1) << 31) - (int64_t(1) << 20))
    return fail(SLMT_ERR_UNSUPPORTED, "shared decode: block tables too wide for so many sequences");
  if ((int64_t)p.block_size * p.KV * (D + 8) >= (int64_t(1) << 31))
    return fail(SLMT_ERR_UNSUPPORTED, "shared decode: a cache block of 2 GiB or more");
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
