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
constexpr int COLS = 16;           // columns of a set
constexpr int SETS = 2;            // sets of a shared item
constexpr int WAVES = 4;           // waves per workgroup
constexpr int kMaxSeqs = 4096;     // sequences and groups of a call (their places are in LDS)
// A score may lie this far (base 2) above the weights' reference; one past it moves the reference, to kSlack less.  Weights
// are up to 2^8 vstep then, keep 22 bits down to 2^-17 of that, and count down to 2^-33.  Where values have steps past
// kStepLimit (fp16 holds them up to 2^16), less far, so that weights stay below fp16's largest number.
constexpr float kRoom = 8.0f, kRoomLargeSteps = -1.0f, kSlack = 4.0f;
constexpr float kStepLimit = 128.0f;

template <int D>
struct Geo {
  static constexpr int KW = D == 128 ? 4 : 2;        // dwords of K codes per key and lane (32 or 16 dims)
  static constexpr bool X = D == 80;                 // 16 dims more: 2 bytes of K, a nibble of V
  static constexpr int KB = KW + (X ? 1 : 0);        // 32-dim blocks of QK
  static constexpr int VB = D == 128 ? 4 : 2;        // bytes of V per key and lane
  static constexpr int RB = D / 16;                  // 16-dim blocks of PV
  static constexpr int OROW = D + 4;                 // floats of a column in the join
  static constexpr int JOIN = WAVES * SETS * COLS * OROW * 4;
  static constexpr int RULERS = WAVES * TK * 16;
  static constexpr int FIXED = JOIN + RULERS + WAVES * SETS * COLS * 8;
  static constexpr int WGS = 2;                      // workgroups a CU holds
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
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }
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

// The call's jobs, in LDS, the same in all workgroups.  A job is a workgroup's part of a shared item's tiles (its waves take
// them in turn and join), or four chunks of sequences' own tiles, a wave each.
struct Schedule {
  int *start;     // [R + 1] the groups' first sequences
  int *prefix;    // [R] their shared tokens
  int *part;      // [R + 1] jobs of the groups before
  int *own;       // [B] tokens of a sequence that its group reads
  int *chunk;     // [B + 1] chunks of the sequences before
  int tiles;      // at most, of a wave in a job
  int shared, jobs;
};
__device__ __forceinline__ int sets_of(const SharedParams& p, const Schedule& s, int r) {
  return ceil_div((s.start[r + 1] - s.start[r]) * p.G, SETS * COLS);
}
__device__ __forceinline__ int parts_of(const Schedule& s, int r) { return ceil_div(tiles_of(0, s.prefix[r]), s.tiles * WAVES); }

__device__ __forceinline__ Schedule make_schedule(const SharedParams& p, int* lds) {
  const int tid = threadIdx.x, lane = tid & 63, R = p.R, B = p.B, wave = uniform(tid >> 6);
  Schedule s;
  s.start = lds;
  s.prefix = s.start + R + 1;
  s.part = s.prefix + R;
  s.own = s.part + R + 1;
  s.chunk = s.own + B;
  if (wave == 0) {      // starts that never fall, whatever the caller's are: all that follows holds for them
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
    for (int b = tid - 64; b < B; b += (WAVES - 1) * 64) s.chunk[b] = seq_len(p, b);
  }
  __syncthreads();
  for (int b = tid; b < B; b += WAVES * 64) {
    const int len = s.chunk[b];
    int pre = 0;
    if (R > 0 && b >= s.start[0] && b < s.start[R]) pre = min(s.prefix[last_at_most(s.start, R, b)], len);
    s.own[b] = pre;
    s.chunk[b] = tiles_of(pre, len);
  }
  __syncthreads();
  // As many tiles a wave as make a job for every workgroup and no more.
  int all = 0;
  for (int i = lane; i < R; i += 64) all += sets_of(p, s, i) * tiles_of(0, s.prefix[i]);
  for (int b = lane; b < B; b += 64) all += p.own_sets * s.chunk[b];
  s.tiles = max(1, ceil_div(wave_total(all), p.W * WAVES));
  for (int i = 0; i < 4; ++i) {
    int shared = 0, own = 0;
    for (int r = lane; r < R; r += 64) shared += sets_of(p, s, r) * parts_of(s, r);
    for (int b = lane; b < B; b += 64) own += p.own_sets * ceil_div(s.chunk[b], s.tiles);
    if (wave_total(shared) + ceil_div(wave_total(own), WAVES) <= p.W) break;
    s.tiles += max(1, s.tiles / 4);
  }
  __syncthreads();
  if (wave == 0) {
    for (int r = lane; r < R; r += 64) s.part[r] = sets_of(p, s, r) * parts_of(s, r);
    scan(s.part, R);
  } else if (wave == 1) {
    for (int b = lane; b < B; b += 64) s.chunk[b] = p.own_sets * ceil_div(s.chunk[b], s.tiles);
    scan(s.chunk, B);
  }
  __syncthreads();
  s.shared = uniform(s.part[R]);
  s.jobs = s.shared + ceil_div(uniform(s.chunk[B]), WAVES);
  return s;
}

// What a wave does: tiles lo, lo + step, ... below hi of the keys klo .. khi - 1 of row seq0 of the tables, for ncols
// columns from flat0 on.
struct Work {
  int seq0, flat0, ncols, klo, khi, lo, hi, step;
  bool own;
};

template <int D, int S>
struct Sums {
  floatx4 o[S][D / 16];            // sums of the weights' products
  float m[S], l[S], vt[S];         // the weights' reference, their sum, the sum of their products with vmin + 8 vstep
};

template <int D, int S>
__device__ __forceinline__ void attend(const SharedParams& p, const Work& wk, int kv, uint8_t* rulers, Sums<D, S>& sum) {
  using GG = Geo<D>;
  constexpr int KW = GG::KW, KB = GG::KB, VB = GG::VB, RB = GG::RB, SLOT = D + 8;
  constexpr float kC = 1.4426950408889634f / (D == 64 ? 8.0f : D == 80 ? 8.94427190999916f : 11.313708498984761f);
  const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
  const uint32_t row_bytes = (uint32_t)p.KV * SLOT;
  const int64_t block_bytes = (int64_t)p.block_size * row_bytes;
  const int esh = p.bt64 ? 3 : 2;

  // ---- keys and values of the wave's tiles
  const int base = wk.klo & ~15, end16 = (wk.khi - 1) & ~15;
  const uint8_t* const table = reinterpret_cast<const uint8_t*>(p.block_tables) + (((int64_t)wk.seq0 * p.bt_stride) << esh);
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
      typedef uint32_t Words __attribute__((ext_vector_type(KW), aligned(8)));
      const Words x = *reinterpret_cast<const Words*>(b + kfrom);
#pragma unroll
      for (int j = 0; j < KW; ++j) kx[i][j] = x[j];
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
  int64_t off_next = 0;
  const bool any = wk.lo < wk.hi;
  if (any) {
    const int64_t off = place(wk.lo);
    const int next = wk.lo + wk.step < wk.hi ? wk.lo + wk.step : wk.lo;
    off_next = place(next);
    load_k(off);
    load_v(off);
  }

  // ---- the lane's columns (those past the item's repeat the last)
  half8 qh[S][KB];
  float qsum[S];
  int lim[S], lim_lo = 0x7fffffff;     // keys below lim are seen
#pragma unroll
  for (int st = 0; st < S; ++st) {
    const int flat = wk.flat0 + min(COLS * st + col, wk.ncols - 1);
    const int seq = wk.own ? wk.seq0 : wk.seq0 + flat / p.G, head = kv * p.G + (wk.own ? flat : flat % p.G);
    lim[st] = wk.own ? wk.khi : min(wk.khi, seq_len(p, seq));
    const uint16_t* q = p.q + (int64_t)seq * p.q_seq_stride + (int64_t)head * p.q_head_stride;
    float t = 0.f;
#pragma unroll
    for (int j = 0; j < KW; ++j) {
      const half8 x = *reinterpret_cast<const half8*>(q + 8 * (KW * grp + j));
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        qh[st][j][e] = x[dim_of(e)];
        t += (float)x[e];
      }
    }
    if constexpr (GG::X) {
      const half4 x = *reinterpret_cast<const half4*>(q + 64 + 4 * grp);
      qh[st][KW] = half8{x[0], (_Float16)0.f, x[1], (_Float16)0.f, x[2], (_Float16)0.f, x[3], (_Float16)0.f};
#pragma unroll
      for (int e = 0; e < 4; ++e) t += (float)x[e];
    }
    float a, b;
    swap16(t, a, b);
    t = a + b;
    swap32(t, a, b);
    qsum[st] = a + b;
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
  float room = kRoom;

  for (int t = wk.lo; t < wk.hi; t += wk.step) {
    const int kt0 = base + t * TK;
    {   // the tile's rulers, a key a lane
      const float kmin = h2f((uint16_t)(rl.x & 0xffffu)), kstep = h2f((uint16_t)(rl.x >> 16));
      float vmin = h2f((uint16_t)(rl.y & 0xffffu)), vstep = h2f((uint16_t)(rl.y >> 16));
      const int key = kt0 + lane;
      const bool in = key >= wk.klo && key < wk.khi;
      vmin = in ? __builtin_fmaf(8.0f, vstep, vmin) : 0.f;     // (nor may the rulers of keys that are not seen reach the sums)
      vstep = in ? vstep : 0.f;
      __builtin_amdgcn_wave_barrier();
      *reinterpret_cast<float2*>(rulers + 8 * lane) = make_float2(__builtin_fmaf(8.0f, kstep, kmin) * kC, kstep * kC);
      *reinterpret_cast<float2*>(rulers + 8 * (TK + lane)) = make_float2(vmin, vstep);
      __builtin_amdgcn_wave_barrier();
      if (room == kRoom && __builtin_amdgcn_ballot_w64(__builtin_fabsf(vstep) > kStepLimit)) {   // (rare)
        constexpr float up = kRoom - kRoomLargeSteps;
        const float alpha = __builtin_amdgcn_exp2f(-up);
        room = kRoomLargeSteps;
#pragma unroll
        for (int st = 0; st < S; ++st) {
          if (sum.m[st] == -INFINITY) continue;
          sum.m[st] = msub[st] = sum.m[st] + up;
          sum.l[st] *= alpha;
          sum.vt[st] *= alpha;
#pragma unroll
          for (int c = 0; c < RB; ++c) sum.o[st][c] *= alpha;
        }
      }
    }
    floatx4 sc[S][4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      half8 a[KB];
#pragma unroll
      for (int j = 0; j < KW; ++j) a[j] = codes8(kx[n][j]);
      if constexpr (GG::X) a[KW] = codes8(kxx[n]);
#pragma unroll
      for (int st = 0; st < S; ++st) {
        sc[st][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[0], qh[st][0], floatx4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
        for (int j = 1; j < KB; ++j) sc[st][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[j], qh[st][j], sc[st][n], 0, 0, 0);
      }
    }
    if (t + wk.step < wk.hi) load_k(off_next);
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
#pragma unroll
    for (int st = 0; st < S; ++st) {
      float tmax = -INFINITY;
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) tmax = fmaxf(tmax, sc[st][n][i]);
      // (scores are relative to msub)
      if (__builtin_amdgcn_ballot_w64(tmax > (sum.m[st] == -INFINITY ? -INFINITY : room))) {
        float a, b;                    // over the four lane groups that hold the column
        swap16(tmax, a, b);
        tmax = fmaxf(a, b);
        swap32(tmax, a, b);
        tmax = fmaxf(a, b);
        const bool grow = tmax > (sum.m[st] == -INFINITY ? -INFINITY : room);
        const float up = grow ? tmax - (room - kSlack) : 0.f;
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
            // (cut, not rounded: the remainder is exact either way)
            const auto h2 = __builtin_amdgcn_cvt_pkrtz(w[0], w[1]);
            const auto l2 = __builtin_amdgcn_cvt_pkrtz(w[0] - (float)h2[0], w[1] - (float)h2[1]);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              bh[st][4 * n + i + e] = (_Float16)h2[e];
              bl[st][4 * n + i + e] = (_Float16)l2[e];
            }
          }
        }
      }
      auto products = [&](int c, const uint32_t (&w)[4]) {
        const half8 a = __builtin_bit_cast(half8, make_uint4(w[0], w[1], w[2], w[3]));
#pragma unroll
        for (int st = 0; st < S; ++st) sum.o[st][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, bh[st], sum.o[st][c], 0, 0, 0);
#pragma unroll
        for (int st = 0; st < S; ++st) sum.o[st][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, bl[st], sum.o[st][c], 0, 0, 0);
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
    if (t + wk.step < wk.hi) {
      load_v(off_next);
      off_next = place(t + 2 * wk.step < wk.hi ? t + 2 * wk.step : t);
    }
  }
#pragma unroll
  for (int st = 0; st < S; ++st) {
    float a, b;
    swap16(sum.l[st], a, b);
    sum.l[st] = a + b;
    swap32(sum.l[st], a, b);
    sum.l[st] = a + b;
    swap16(sum.vt[st], a, b);
    sum.vt[st] = a + b;
    swap32(sum.vt[st], a, b);
    sum.vt[st] = a + b;
  }
}

// The sums of the lane's column, times f, four dims at a time: put(dim, values).
template <int D, int S, typename F>
__device__ __forceinline__ void each_four(const Sums<D, S>& sum, int st, float f, F put) {
  using GG = Geo<D>;
  constexpr int N = 2 * GG::VB;        // dims side by side: N (4 grp + i) ...
  const int grp = (threadIdx.x & 63) >> 4;
  auto of = [&](int c, int i) { return f == 0.f ? 0.f : f * (sum.o[st][c][i] + sum.vt[st]); };
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int c = 0; c < N; c += 4) put(N * (4 * grp + i) + c, make_float4(of(c, i), of(c + 1, i), of(c + 2, i), of(c + 3, i)));
  if constexpr (GG::X) put(64 + 4 * grp, make_float4(of(GG::RB - 1, 0), of(GG::RB - 1, 1), of(GG::RB - 1, 2), of(GG::RB - 1, 3)));
}

// A shared item's part by the whole workgroup: every wave its tiles, then their sums joined.
template <int D, int S>
__device__ __forceinline__ void shared_job(const SharedParams& p, const Work& wk, int kv, uint8_t* smem, int slot) {
  using GG = Geo<D>;
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, grp = lane >> 4, wave = uniform(tid >> 6);
  float* const join = reinterpret_cast<float*>(smem);
  float2* const jml = reinterpret_cast<float2*>(smem + GG::JOIN + GG::RULERS);
  Sums<D, S> sum;
  attend<D, S>(p, wk, kv, smem + GG::JOIN + wave * TK * 16, sum);
  constexpr int C = S * COLS;
  __syncthreads();                     // (the last job's sums have been read)
  if (grp == 0)
#pragma unroll
    for (int st = 0; st < S; ++st) jml[wave * C + COLS * st + col] = make_float2(sum.m[st], sum.l[st]);
  __syncthreads();
#pragma unroll
  for (int st = 0; st < S; ++st) {
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) top = fmaxf(top, jml[w * C + COLS * st + col].x);
    const float f = sum.m[st] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sum.m[st] - top);
    float* const jo = join + (wave * C + COLS * st + col) * GG::OROW;
    each_four<D, S>(sum, st, f, [&](int d, float4 v) { *reinterpret_cast<float4*>(jo + d) = v; });
  }
  __syncthreads();
  if (slot >= p.part_slots) return;
  const int64_t row = ((int64_t)slot * p.KV + kv) * (SETS * COLS);
  for (int e = tid; e < wk.ncols * (D / 4); e += WAVES * 64) {
    const int c = e / (D / 4), d = 4 * (e % (D / 4));
    float4 v = *reinterpret_cast<const float4*>(join + c * GG::OROW + d);
#pragma unroll
    for (int w = 1; w < WAVES; ++w) {
      const float4 x = *reinterpret_cast<const float4*>(join + (w * C + c) * GG::OROW + d);
      v = make_float4(v.x + x.x, v.y + x.y, v.z + x.z, v.w + x.w);
    }
    *reinterpret_cast<float4*>(p.part_o + (row + c) * D + d) = v;
  }
  if (tid < wk.ncols) {
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
}

template <int D>
__global__ void __launch_bounds__(WAVES * 64) __attribute__((amdgpu_waves_per_eu(Geo<D>::WGS))) shared_kernel(const SharedParams p) {
  using GG = Geo<D>;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int id = blockIdx.x, kv = (id >> 3) % p.KV;
  const Schedule s = make_schedule(p, reinterpret_cast<int*>(smem + GG::FIXED));
  if (id == 0) {      // for merge_kernel: where a sequence's parts are
    for (int b = tid; b < p.B; b += WAVES * 64) {
      int4 a = make_int4(0, 0, 0, 0);
      if (p.R > 0 && b >= s.start[0] && b < s.start[p.R]) {
        const int r = last_at_most(s.start, p.R, b);
        a = make_int4(s.part[r], parts_of(s, r), sets_of(p, s, r), (b - s.start[r]) * p.G);
      }
      p.records[2 * b] = a;
      p.records[2 * b + 1] = make_int4(s.chunk[b], (s.chunk[b + 1] - s.chunk[b]) / p.own_sets, seq_len(p, b) > 0, 0);
    }
  }
  // Workgroup id runs on XCD id % 8.  Jobs that read the same keys stand behind one another, and an XCD has an unbroken
  // run of them, for all KV heads at a time, since a token's heads lie side by side and share cache lines.
  const int each = ceil_div(s.jobs, 8), xcd = id & 7;
  for (int k = id / (8 * p.KV); k < each; k += p.W / 8) {
    const int job = xcd * each + k;
    if (job >= s.jobs) break;
    Work wk;
    if (job < s.shared) {
      const int r = uniform(last_at_most(s.part, p.R, job)), rel = job - uniform(s.part[r]);
      const int sets = uniform(sets_of(p, s, r)), parts = uniform(parts_of(s, r));
      const int part = rel / sets, set = rel - part * sets;
      wk.seq0 = uniform(s.start[r]);
      wk.flat0 = set * SETS * COLS;
      wk.ncols = min(SETS * COLS, uniform(s.start[r + 1] - s.start[r]) * p.G - wk.flat0);
      wk.klo = 0;
      wk.khi = uniform(s.prefix[r]);
      const int tiles = tiles_of(0, wk.khi);
      wk.lo = (int)((int64_t)part * tiles / parts) + wave;
      wk.hi = (int)((int64_t)(part + 1) * tiles / parts);
      wk.step = WAVES;
      wk.own = false;
      if (wk.ncols > COLS) shared_job<D, 2>(p, wk, kv, smem, job);
      else shared_job<D, 1>(p, wk, kv, smem, job);
    } else {
      const int chunk = (job - s.shared) * WAVES + wave;
      if (chunk >= uniform(s.chunk[p.B])) continue;
      const int b = uniform(last_at_most(s.chunk, p.B, chunk)), rel = chunk - uniform(s.chunk[b]);
      const int chunks = uniform(s.chunk[b + 1] - s.chunk[b]) / p.own_sets, set = rel / chunks, c = rel - set * chunks;
      wk.seq0 = b;
      wk.flat0 = set * COLS;
      wk.ncols = min(COLS, p.G - wk.flat0);
      wk.klo = uniform(s.own[b]);
      wk.khi = uniform(seq_len(p, b));
      const int tiles = tiles_of(wk.klo, wk.khi);
      wk.lo = (int)((int64_t)c * tiles / chunks);
      wk.hi = (int)((int64_t)(c + 1) * tiles / chunks);
      wk.step = 1;
      wk.own = true;
      Sums<D, 1> sum;
      attend<D, 1>(p, wk, kv, smem + GG::JOIN + wave * TK * 16, sum);
      const int col = lane & 15;
      if (col < wk.ncols && chunk < p.own_slots) {
        const int64_t row = ((int64_t)chunk * p.KV + kv) * p.own_cols + col;
        each_four<D, 1>(sum, 0, 1.f, [&](int d, float4 v) { *reinterpret_cast<float4*>(p.own_o + row * D + d) = v; });
        if (lane < COLS) reinterpret_cast<float2*>(p.own_ml)[row] = make_float2(sum.m[0], sum.l[0]);
      }
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
