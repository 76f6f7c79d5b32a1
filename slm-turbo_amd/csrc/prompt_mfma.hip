// Attention over whole prompts' own K and V on the matrix cores, fp16 and bf16, head_dim 64, 80 and 128:
// sequences of different lengths packed behind one another, grouped heads, causal or not.
//
// A workgroup takes 128 query rows of one sequence and query head, 32 per wave, and walks the 64-key tiles
// that they can see; where there are few workgroups, eight waves do, four the even tiles and four the odd ones, and
// where there are very few for the keys, several workgroups, whose parts a second kernel joins.  Everything is
// transposed, so a lane owns one query column from the scores to the output (both halves of the wave the same 32
// columns, each half its own keys and dims):
//   S^T = K Q^T                 (v_mfma_f32_32x32x16: A = 32 K rows, B = the lane's query)
//   P^T = exp2(c S^T - m)       (online softmax per query column; c = scale log2(e))
//   O^T += V^T P^T              (B = the lane's P^T as it comes out of S^T, A in the same order of keys)
// Scores, maxima, sums and the output accumulate in fp32.  The weights P enter the second product in the
// tensors' type, half a step of which is what the output's own rounding is off by, and the row sums add the
// same rounded weights; in fp16 the largest is near 2^6, so that small ones keep their bits (kHead).
//
// What bounds it: the matrix cores and the exponentials, which share a SIMD's issue, at the clock that the power limit
// leaves (about 1.8 GHz under long prompts).  8192 tokens, 32 q / 8 KV heads, 128 dims, bf16: 496 - 515 us, 1070 - 1110
// TFLOP/s where a large matrix product reaches 1217; the matrix cores are busy 54% of the time, the vector units 38%, and
// bank conflicts are 0.8 million cycles beside 25.5 million LDS instructions.  At 64 dims an exponential serves half as many
// products: 8192 tokens, 32 q / 4 KV heads 46% and 58%; 8 prompts of 17 to 2000 tokens, whose workgroups are of unequal length,
// 66 - 76 us, 580 - 670 TFLOP/s, 28% and 47%, so that no unit is full.  80 dims pay for 96 in the products with V and for 128 in
// LDS: 1900 tokens, 32 q / 8 KV heads 37 us, 20% and 23%.
// Tried without gain: a raised priority around the products (+1%), two heads a workgroup (-1% at 8192 tokens, +13 - 20%
// below 1000), four waves a SIMD at 64 dims.
#include "slmt_internal.h"

#include <algorithm>
#include <type_traits>

namespace slmt {
namespace prompt {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef float float16v __attribute__((ext_vector_type(16)));
typedef unsigned uint4v __attribute__((ext_vector_type(4)));

constexpr int BM = 128;    // query rows per workgroup
constexpr int BN = 64;     // keys per tile

// kHead: what the largest weight is 2 to the power of when the reference has moved, and kGrow: what a weight may grow to
// before it moves again (in powers of two as well).  fp16's smallest numbers are 2^-24 apart: with weights of 1 at most, what
// lies 2^25 below the largest would vanish however many such keys there are, and 2^17 keys of that make 1/256 of the sum; from
// 2^6 on it is 2^31 below.
template <typename T>
struct Mfma;
template <>
struct Mfma<_Float16> {
  typedef half8 V8;
  static constexpr float kHead = 6.0f, kGrow = 15.0f;
  static __device__ __forceinline__ float16v mul(V8 a, V8 b, float16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mfma<__bf16> {
  typedef bf8 V8;
  static constexpr float kHead = 0.0f, kGrow = 13.0f;
  static __device__ __forceinline__ float16v mul(V8 a, V8 b, float16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};

struct Item {
  int seq, block;      // seq < 0: none
  int q0, nq, k0, nk;  // the sequence's rows of q and of k, v
};

// Block x of the sequences' blocks of BM query rows.  Uniform over the wave.  Of `blocks`, at least as many as there
// are.  Up to kSorted sequences the blocks go by their place in the sequence, the last first: these have the most keys, and
// workgroups that start late had better be short.  More sequences fill the chip several times over and go one after
// another, the last first, so that a sequence's keys stay in the caches.  us, sorted / one after another, 32 q / 4 KV
// heads, 64 dims, 1024 tokens each: 4 sequences 34.2 / 36.3, 8 57.3 / 60.8, 16 118 / 116, 32 244 / 220 (9 to 15 sequences,
// and many of other lengths, are not measured).
constexpr int kSorted = 8;
__device__ __forceinline__ Item find_item(const PromptParams& p, int x, int blocks) {
  const int lane = threadIdx.x & 63;
  auto rows = [&](int r, int& q0, int& q1, int& k0, int& k1) {
    q0 = min(max(p.q_start[r], 0), p.N), q1 = min(max(p.q_start[r + 1], q0), p.N);
    k0 = min(max(p.k_start[r], 0), p.NK), k1 = min(max(p.k_start[r + 1], k0), p.NK);
  };
  if (p.R <= kSorted) {
    int q0, q1, k0, k1;
    rows(min(lane, p.R - 1), q0, q1, k0, k1);
    const int n = lane < p.R ? (q1 - q0 + BM - 1) / BM : 0;
    int most = 0;
    for (int r = 0; r < p.R; ++r) most = max(most, __builtin_amdgcn_readlane(n, r));
    for (int b0 = (most - 1) & ~63; b0 >= 0; b0 -= 64) {
      int from = 0;                          // blocks with place b0 + lane or a later one
      for (int r = 0; r < p.R; ++r) from += max(0, __builtin_amdgcn_readlane(n, r) - b0 - lane);
      const uint64_t past = __builtin_amdgcn_ballot_w64(from > x);
      if (!past) continue;
      const int at = 63 - __builtin_clzll(past), b = b0 + at;
      int later = 0;                         // those with a later place
      for (int r = 0; r < p.R; ++r) later += max(0, __builtin_amdgcn_readlane(n, r) - b - 1);
      const uint64_t has = __builtin_amdgcn_ballot_w64(n > b);
      const bool mine = n > b && __builtin_popcountll(has & ((1ull << lane) - 1)) == x - later;
      const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(mine));
      Item it;
      it.seq = l;
      it.block = b;
      it.q0 = __builtin_amdgcn_readlane(q0, l);
      it.nq = __builtin_amdgcn_readlane(q1, l) - it.q0;
      it.k0 = __builtin_amdgcn_readlane(k0, l);
      it.nk = __builtin_amdgcn_readlane(k1, l) - it.k0;
      return it;
    }
    return Item{-1, 0, 0, 0, 0, 0};
  }
  x = blocks - 1 - x;
  int base = 0;
  for (int r0 = 0; r0 < p.R; r0 += 64) {
    int q0, q1, k0, k1;
    rows(min(r0 + lane, p.R - 1), q0, q1, k0, k1);
    const int blocks = r0 + lane < p.R ? (q1 - q0 + BM - 1) / BM : 0;
    int incl = blocks;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(incl, o, 64);
      if (lane >= o) incl += v;
    }
    const uint64_t hit = __builtin_amdgcn_ballot_w64(base + incl > x);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      Item it;
      it.seq = r0 + l;
      it.block = x - base - (__builtin_amdgcn_readlane(incl, l) - __builtin_amdgcn_readlane(blocks, l));
      it.q0 = __builtin_amdgcn_readlane(q0, l);
      it.nq = __builtin_amdgcn_readlane(q1, l) - it.q0;
      it.k0 = __builtin_amdgcn_readlane(k0, l);
      it.nk = __builtin_amdgcn_readlane(k1, l) - it.k0;
      return it;
    }
    base += __builtin_amdgcn_readlane(incl, 63);
  }
  return Item{-1, 0, 0, 0, 0, 0};
}

// Staged K and V rows (stage: K's 64 rows, then V's), 16-byte chunks of a row in an order of its own:
// chunk g of row r sits in place g ^ swizzle(r).  The loads to LDS write lane after lane, so the order is
// made by which chunk a lane fetches.
//   K: a lane reads chunk 2 j + hf of row 32 n + col; the LDS serves lanes 0-7 and 16-23 (then 8-15 and
//      24-31, ...) together, over 256 bytes, so those rows take 16 different places.
//   V: the transposing read takes 4 keys and 64 bytes of each for half a wave; the 4 keys' chunks lie apart.
template <int D>
struct Geo {
  static constexpr int QB = D / 16;                  // 16-dim blocks of QK
  static constexpr int OB = (D + 31) / 32;           // 32-dim blocks of PV
  static constexpr int CH = D == 64 ? 8 : 16;        // chunks of a staged row (head_dim 80: the last six are not used)
  static constexpr int ROWB = CH * 16;
  static constexpr int TILE = BN * ROWB, STAGE = 2 * TILE;
  static constexpr int RPI = 64 / CH;                // rows that a wave fetches with one instruction
  static constexpr int LOADS = BN / 4 / RPI;         // instructions of a wave for its quarter of K's or V's tile
  static __device__ __forceinline__ int kswz(int r) {
    return CH == 16 ? (r & 7) | ((r >> 1) & 8) : ((r >> 1) & 3) | ((r >> 2) & 4);
  }
  static __device__ __forceinline__ int vswz(int r) { return CH == 16 ? 4 * (r & 3) : 4 * ((r >> 1) & 1); }
};

// 16 bytes per lane from base + offset to LDS at `lds` + 16 lane, without a register in between.  Counted by
// vmcnt alone: the wait before the barrier is the kernel's own.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_lds(uint32_t lds, uint32_t offset, const void* base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(offset), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void load_lds(uint32_t lds, const void* at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(at) : "memory", "m0");
}
#pragma clang diagnostic pop
__device__ __forceinline__ void wait_and_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x70);          // vmcnt(0) lgkmcnt(0), known to the compiler (in asm it waited again for the query)
  asm volatile("s_barrier" ::: "memory");
}

typedef short short4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) short4v* LdsShort4;
typedef unsigned uint2v __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) uint4v* LdsUint4;
typedef __attribute__((address_space(3))) uint2v* LdsUint2;
typedef __attribute__((address_space(3))) float* LdsFloat;

__device__ __forceinline__ float dot2(uint32_t p, float l, _Float16) {
  return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, p), f16x2{(_Float16)1.0f, (_Float16)1.0f}, l, false);
}
__device__ __forceinline__ float dot2(uint32_t p, float l, __bf16) {
  typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf2, p), bf2{(__bf16)1.0f, (__bf16)1.0f}, l, false);
}

// This workgroup's query head (the heads of a KV head on the same XCD where they are a multiple of 8: workgroups go around the XCDs).
__device__ __forceinline__ int head_of(const PromptParams& p) {
  const int x = blockIdx.x % p.H, kv = x % p.KV;
  return kv * (p.H / p.KV) + x / p.KV;
}

// A wave's part of a split of the keys: its output, reference and sum, 64 floats a register.
template <int D>
__host__ __device__ constexpr int64_t part_floats() { return (16 * Geo<D>::OB + 2) * 64; }
template <int D, typename P>
__device__ __forceinline__ P* part_of(P* parts, int64_t workgroup, int splits, int split, int w) {
  return parts + ((workgroup * splits + split) * 4 + w) * part_floats<D>();
}

// The outputs of a wave's rows from its sums o and l.
template <typename T, int D>
__device__ __forceinline__ void write_rows(const PromptParams& p, const Item& it, int h, int m0, int w, int lane,
                                           const float16v (&o)[Geo<D>::OB], float l, uint32_t mine) {
  // (a row that sees keys whose scores are all -infinity is 0 / 0, as its softmax is)
  const int col = lane & 31, hf = lane >> 5, m = m0 + 32 * w + col, shift = it.nk - it.nq;
  const bool none = p.causal ? m + shift < 0 : it.nk == 0;
  const float rl = none ? 0.0f : 1.0f / l;
  // The wave's rows go through LDS at `mine` (its part of a ring that no wave reads any more), so that whole rows are written 16
  // bytes a lane (8 bytes of 32 rows at a time took eight times the cache's write requests).
#pragma unroll
  for (int c = 0; c < Geo<D>::OB; ++c)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      if (32 * c + 8 * g >= D) continue;
      T y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = (T)(none ? 0.0f : o[c][4 * g + i] * rl);
      *(LdsUint2)(uintptr_t)(mine + col * (2 * D + 16) + 2 * (32 * c + 8 * g + 4 * hf)) = __builtin_bit_cast(uint2v, y);
    }
  __builtin_amdgcn_wave_barrier();
  T* const out = reinterpret_cast<T*>(p.out) + (int64_t)(it.q0 + m0 + 32 * w) * p.out_token + (int64_t)h * p.out_head;
  const int rows = it.nq - m0 - 32 * w;
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    const int at = 64 * i + lane, row = at / (D / 8), ch = at - row * (D / 8);
    const uint4v y = *(LdsUint4)(uintptr_t)(mine + row * (2 * D + 16) + 16 * ch);
    if (row < rows) __builtin_memcpy(out + row * p.out_token + 8 * ch, &y, 16);
  }
}

template <typename T, int D, int SP>
__global__ void __launch_bounds__(256 * SP) __attribute__((amdgpu_waves_per_eu(D == 64 ? 3 : 2)))
prompt_kernel(const PromptParams p, const int blocks, const int turn, const int splits, float* const parts) {
  using V8 = typename Mfma<T>::V8;
  using G = Geo<D>;
  constexpr int QB = G::QB, OB = G::OB;
  __shared__ __attribute__((aligned(256))) uint8_t smem[SP * 2 * G::STAGE];
  const uint32_t ldsw = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)smem;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, hf = lane >> 5;
  const int w = wave & 3, half = wave >> 2;
  const uint32_t lds0 = ldsw + half * 2 * G::STAGE;    // this half's ring
  const int h = head_of(p), kv = h / (p.H / p.KV);
  int place = blockIdx.x / p.H;
  if (turn && place >= turn) place = turn + blocks - 1 - place;
  const Item it = find_item(p, place, blocks);
  if (p.clear && blockIdx.y == 0) {                             // the rows of no sequence, spread over the workgroups
    const int head = min(max(p.q_start[0], 0), p.N), end = min(max(p.q_start[p.R], head), p.N);
    const int64_t n = ((int64_t)head + (p.N - end)) * p.H * (D / 4);
    for (int64_t i = (int64_t)blockIdx.x * (256 * SP) + tid; i < n; i += (int64_t)gridDim.x * (256 * SP)) {
      const int64_t one = i / (D / 4), row = one / p.H;
      T* const at = reinterpret_cast<T*>(p.out) + (row < head ? row : row - head + end) * p.out_token + (one - row * p.H) * p.out_head;
      *reinterpret_cast<uint2*>(at + 4 * (i - one * (D / 4))) = make_uint2(0, 0);
    }
  }
  if (it.seq < 0) return;
  const int m0 = it.block * BM, m = m0 + 32 * w + col;
  const int shift = it.nk - it.nq;           // query row m sees the keys up to m + shift
  const int last = min(m0 + BM, it.nq) - 1;
  const int seen = p.causal ? min(it.nk, max(last + shift + 1, 0)) : it.nk;
  // Tiles from `tile0` to `all` are this split's.  A half's tile t is the SP t + half'th of these.
  const int per = SP > 1 ? ((seen + BN - 1) / BN + splits - 1) / splits : 0, tile0 = SP > 1 ? (int)blockIdx.y * per : 0;
  const int kend = SP > 1 ? min(seen, (tile0 + per) * BN) : seen;
  const int all = (kend + BN - 1) / BN;
  const int ntiles = max(0, all - tile0 + SP - 1) / SP;      // rounds
  auto tile = [&](int t) { return tile0 + SP * t + half; };
  const T* const q = reinterpret_cast<const T*>(p.q) + (int64_t)(it.q0 + min(m, it.nq - 1)) * p.q_token + (int64_t)h * p.q_head;
  const T* const k = reinterpret_cast<const T*>(p.k) + (int64_t)it.k0 * p.k_token + (int64_t)kv * p.k_head;
  const T* const v = reinterpret_cast<const T*>(p.v) + (int64_t)it.k0 * p.v_token + (int64_t)kv * p.v_head;
  V8 qf[QB];
#pragma unroll
  for (int j = 0; j < QB; ++j) __builtin_memcpy(&qf[j], q + 16 * j + 8 * hf, 16);

  // ---- staging: wave w fetches rows 16 w .. 16 w + 15 of K and of V, RPI at a time
  const int srow = lane / G::CH, splace = lane & (G::CH - 1);   // of an instruction's rows
  auto chunk = [&](int swz) { return 16 * (D == 80 ? min(splace ^ swz, 9) : splace ^ swz); };
  const uint32_t koff = (uint32_t)srow * (uint32_t)(2 * p.k_token), voff = (uint32_t)srow * (uint32_t)(2 * p.v_token);
  const uint32_t cv = chunk(G::vswz(srow));  // (rows RPI apart: the same, as RPI is a multiple of 4)
  auto fetch = [&](int t, auto which) {      // K's or V's tile t into the ring's place t & 1
    constexpr bool V = decltype(which)::value;
    const uint32_t lds = lds0 + (t & 1) * G::STAGE + V * G::TILE + 16 * w * G::ROWB;
    const T* const base = V ? v : k;
    const int64_t stride = V ? p.v_token : p.k_token;
    auto at = [&](int r) { return V ? cv : chunk(G::kswz(r)); };
    const int from = tile(t) * BN;
    if (SP > 1 && from >= kend) return;
    if (from + BN <= it.nk) {                // uniform
      const T* rows = base + ((int64_t)from + 16 * w) * stride;
#pragma unroll
      for (int i = 0; i < G::LOADS; ++i) {
        load_lds(lds + i * 1024, (V ? voff : koff) + at(16 * w + i * G::RPI + srow), rows);
        rows += G::RPI * stride;
      }
    } else {                                 // rows past the sequence repeat its last: their weights are 0
#pragma unroll 1
      for (int i = 0; i < G::LOADS; ++i) {
        const int r = 16 * w + i * G::RPI + srow;
        load_lds(lds + i * 1024, reinterpret_cast<const uint8_t*>(base + (int64_t)min(from + r, it.nk - 1) * stride) + at(r));
      }
    }
  };
  using K = std::false_type;
  using V = std::true_type;

  // ---- where the lane reads: K chunk 2 j + hf of row 32 n + col; V 8 bytes of key 16 u + 8 e + 4 hf + (lane & 15) / 4
  const uint32_t kat = lds0 + col * G::ROWB + ((G::kswz(col) ^ hf) * 16);
  const int vkey = 4 * hf + ((lane & 15) >> 2);
  const uint32_t vat = lds0 + G::TILE + vkey * G::ROWB + ((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ G::vswz(vkey)) * 16 + (lane & 1) * 8;

  float16v o[OB] = {};
  float mc = -3.0e38f, l = 0.0f;             // the column's reference (times scale) and its sum over this lane's keys
  if (ntiles > 0) {                          // (all that the first tile and the second's scores need, at once)
    fetch(0, K{});
    fetch(0, V{});
  }
  if (ntiles > 1) fetch(1, K{});
  auto kread = [&](uint32_t so, int n, int j) {
    const uint4v a = *(LdsUint4)(uintptr_t)((kat ^ (32 * j)) + so + 32 * n * G::ROWB);
    return __builtin_bit_cast(V8, a);
  };
  auto vread = [&](uint32_t so, int c, int u) {        // V^T: dim 32 c + col, the keys of the weights' block u
    struct { short4v x[2]; } x;
#pragma unroll
    for (int e = 0; e < 2; ++e)
      x.x[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsShort4)(uintptr_t)((vat ^ (64 * c)) + so + (16 * u + 8 * e) * G::ROWB));
    return __builtin_bit_cast(V8, x);
  };
  // The reference moves only when weights grow past it (2^kGrow in a lane's sum of a tile, inside fp16 for each), so that
  // the sums are rescaled rarely.
  auto move = [&](float tmax) {
    float a, b;
    swap32(tmax, a, b);
    const float next = fmaxf(mc, __builtin_fmaf(fmaxf(a, b), p.scale, -Mfma<T>::kHead));
    const float alpha = __builtin_amdgcn_exp2f(mc - next);
    mc = next;
    l *= alpha;
#pragma unroll
    for (int c = 0; c < OB; ++c) o[c] *= alpha;
  };
  constexpr float kMost = 1 << (int)Mfma<T>::kGrow;
  auto grown = [&](float sum) { return __builtin_amdgcn_ballot_w64(sum > kMost) != 0; };
  // weights of 16 keys, from eight scores of the lane
  auto weights = [&](const float16v& s, int first) {
    V8 pb;
#pragma unroll
    for (int i = 0; i < 8; ++i) pb[i] = (T)__builtin_amdgcn_exp2f(__builtin_fmaf(s[first + i], p.scale, -mc));
    return pb;
  };
  auto sum8 = [&](V8 pb) {
    const uint4v x = __builtin_bit_cast(uint4v, pb);
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) sum = dot2(x[e], sum, T{});
    return sum;
  };

  // Keys that the column sees, and of the wave's rows those that the last sees and those that all see.
  const int see = p.causal ? min(it.nk, m + shift + 1) : it.nk;
  const int wsee = min(kend, p.causal ? m0 + 32 * w + 32 + shift : it.nk);
  const int wall = p.causal ? min(it.nk, m0 + 32 * w + 1 + shift) : it.nk;
  // ---- tiles that all of the wave's rows see whole (the waves go from this loop to the next one each at a tile of
  // its own: their fetches and barriers are the same in both)
  const int nwhole = max(0, min(all, max(0, wall) / BN) - tile0 - half + SP - 1) / SP;
  // A tile's weights are multiplied with V one tile later, so that the next tile's softmax runs beside those products:
  // round t has K's tile t and V's tile t - 1 in LDS and fetches the ones after them.
  V8 pb[4];
  auto products = [&](uint32_t so) {
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int c = 0; c < OB; ++c) o[c] = Mfma<T>::mul(vread(so, c, u), pb[u], o[c]);
  };
  auto whole = [&](int t, auto at, auto first) {       // (the tiles' places are immediate offsets of the reads)
    constexpr uint32_t so = decltype(at)::value * G::STAGE, before = (decltype(at)::value ^ 1) * G::STAGE;
    if constexpr (!decltype(first)::value) {
      if (t + 1 < ntiles) fetch(t + 1, K{});
      fetch(t, V{});
    }
    // (all reads of the first 32 keys before their first product, those of the next 32 between them)
    float16v s[2] = {};
    V8 ka[2][QB];
#pragma unroll
    for (int j = 0; j < QB; ++j) ka[0][j] = kread(so, 0, j);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < QB; ++j) {
      ka[1][j] = kread(so, 1, j);
      s[0] = Mfma<T>::mul(ka[0][j], qf[j], s[0]);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < QB; ++j) s[1] = Mfma<T>::mul(ka[1][j], qf[j], s[1]);
    // Weights against the reference as it is; a maximum is formed, and the weights again, only where their sum shows
    // that they have grown past it.
    V8 next[4];
    float sum = 0.0f;
    auto weigh = [&] {
      float part[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        next[u] = weights(s[u >> 1], 8 * (u & 1));
        part[u] = sum8(next[u]);
      }
      sum = (part[0] + part[1]) + (part[2] + part[3]);
    };
    if constexpr (!decltype(first)::value) {
      products(before);
      weigh();
    }
    if (decltype(first)::value || __builtin_expect(grown(sum), 0)) {
      float tmax = -INFINITY;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) tmax = fmaxf(tmax, s[n][i]);
      move(tmax);
      weigh();
    }
    l += sum;
#pragma unroll
    for (int u = 0; u < 4; ++u) pb[u] = next[u];
    wait_and_barrier();
  };
  wait_and_barrier();
  int t = 0;
  if (nwhole > 0) {
    using S0 = std::integral_constant<int, 0>;
    using S1 = std::integral_constant<int, 1>;
    whole(t++, S0{}, std::true_type{});
    for (; t + 2 <= nwhole; t += 2) {
      whole(t, S1{}, std::false_type{});
      whole(t + 1, S0{}, std::false_type{});
    }
    if (t < nwhole) whole(t++, S1{}, std::false_type{});
  }
  // ---- the others, and the last one's products: of each tile the halves that one of the wave's rows sees
  for (; t <= ntiles; ++t) {
    if (t > 0 && t + 1 < ntiles) fetch(t + 1, K{});
    if (t > 0 && t < ntiles) fetch(t, V{});
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int k0 = tile(t - 1) * BN + 32 * n;
      if (t == 0 || k0 >= wsee) continue;
      const uint32_t so = ((t - 1) & 1) * G::STAGE + n * 32 * G::ROWB;
      bool odd = false;
      if (k0 + 32 > wall) {                  // a masked value that is no number times 0 would be none either
        float16v z = {};
#pragma unroll
        for (int c = 0; c < OB; ++c)         // (head_dim 80: its last 16 rows of dims repeat others)
#pragma unroll
          for (int u = 0; u < 2; ++u) z = Mfma<T>::mul(vread(so, c, u), V8{}, z);
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) sum += z[i];
        odd = __builtin_amdgcn_ballot_w64(sum != 0.0f) != 0;
      }
      if (__builtin_expect(!odd, 1)) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int c = 0; c < OB; ++c) o[c] = Mfma<T>::mul(vread(so, c, u), pb[2 * n + u], o[c]);
      } else {
        // one key at a time, added to the columns that see it
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll 1
          for (int x = 0; x < 16; ++x) {
            const int xh = x >> 3, xe = x & 7;
            const bool sees = k0 + 16 * u + 8 * (xe >> 2) + 4 * xh + (xe & 3) < see;
            V8 pk{};
#pragma unroll
            for (int e = 0; e < 8; ++e) pk[e] = hf == xh && e == xe ? pb[2 * n + u][e] : (T)0.0f;
#pragma unroll
            for (int c = 0; c < OB; ++c) {
              V8 va = vread(so, c, u);
#pragma unroll
              for (int e = 0; e < 8; ++e) va[e] = hf == xh && e == xe ? va[e] : (T)0.0f;
              const float16v one = Mfma<T>::mul(va, pk, float16v{});
#pragma unroll
              for (int i = 0; i < 16; ++i) o[c][i] += sees ? one[i] : 0.0f;
            }
          }
      }
    }
    if (t < ntiles && tile(t) * BN < wsee) {
      float16v s[2] = {};
      float tmax = -INFINITY;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const int k0 = tile(t) * BN + 32 * n;
        if (k0 >= wsee) continue;
        V8 ka[QB];
#pragma unroll
        for (int j = 0; j < QB; ++j) ka[j] = kread((t & 1) * G::STAGE, n, j);
#pragma unroll
        for (int j = 0; j < QB; ++j) s[n] = Mfma<T>::mul(ka[j], qf[j], s[n]);
        // s[n][i]: key 8 (i / 4) + 4 hf + i % 4 of the 32
        if (k0 + 32 > wall) {
          const int left = see - k0 - 4 * hf;
#pragma unroll
          for (int i = 0; i < 16; ++i) s[n][i] = 8 * (i >> 2) + (i & 3) < left ? s[n][i] : -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) tmax = fmaxf(tmax, s[n][i]);
      }
      if (__builtin_amdgcn_ballot_w64(__builtin_fmaf(tmax, p.scale, -mc) > Mfma<T>::kHead + 8.0f)) move(tmax);
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        if (tile(t) * BN + 32 * n >= wsee) continue;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          pb[2 * n + u] = weights(s[n], 8 * u);
          l += sum8(pb[2 * n + u]);
        }
      }
    }
    wait_and_barrier();
  }
  float a, b;
  swap32(l, a, b);
  l = a + b;
  // The halves' parts of a column join in the first one's registers, by way of the rings that no wave reads any more.
  constexpr int PART = (16 * OB + 2) * 256;  // bytes of a wave's output, reference and sum, one float a lane behind another
  constexpr int OROW = 2 * D + 16;
  static_assert((SP > 1 ? 4 * PART : 0) + 4 * 32 * OROW <= SP * 2 * G::STAGE, "the parts and the waves' rows fit the rings");
  if constexpr (SP > 1) {
    const uint32_t at = ldsw + w * PART + 4 * lane;
    if (half) {
#pragma unroll
      for (int c = 0; c < OB; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) *(LdsFloat)(uintptr_t)(at + (16 * c + i) * 256) = o[c][i];
      *(LdsFloat)(uintptr_t)(at + 16 * OB * 256) = mc;
      *(LdsFloat)(uintptr_t)(at + (16 * OB + 1) * 256) = l;
    }
    wait_and_barrier();
    if (half) return;
    const float mo = *(LdsFloat)(uintptr_t)(at + 16 * OB * 256), lo = *(LdsFloat)(uintptr_t)(at + (16 * OB + 1) * 256);
    const float next = fmaxf(mc, mo), x = __builtin_amdgcn_exp2f(mc - next), y = __builtin_amdgcn_exp2f(mo - next);
    l = l * x + lo * y;
    mc = next;
#pragma unroll
    for (int c = 0; c < OB; ++c)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[c][i] = o[c][i] * x + *(LdsFloat)(uintptr_t)(at + (16 * c + i) * 256) * y;
  }
  if constexpr (SP > 1) {
    if (splits > 1) {                        // this split's part, lane after lane as it is in the registers
      if (m0 + 32 * w >= it.nq) return;
      float* const at = part_of<D>(parts, blockIdx.x, splits, blockIdx.y, w) + lane;
#pragma unroll
      for (int c = 0; c < OB; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) at[(16 * c + i) * 64] = o[c][i];
      at[16 * OB * 64] = mc;
      at[(16 * OB + 1) * 64] = l;
      return;
    }
  }
  write_rows<T, D>(p, it, h, m0, w, lane, o, l, ldsw + (SP > 1 ? 4 * PART : 0) + w * 32 * OROW);
}

// Joins the splits' parts, with the reference moved to the largest of theirs.  A part's registers are all in flight at
// once, and the next part's behind them (one after another they took 17 us a split at 128 dims).
template <typename T, int D>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 2)))
join_kernel(const PromptParams p, const int blocks, const int splits, const float* parts) {
  constexpr int OB = Geo<D>::OB;
  __shared__ __attribute__((aligned(256))) uint8_t smem[4 * 32 * (2 * D + 16)];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Item it = find_item(p, blockIdx.x / p.H, blocks);
  const int m0 = it.block * BM;
  if (it.seq < 0 || m0 + 32 * w >= it.nq) return;
  auto part = [&](int s) { return part_of<D>(parts, blockIdx.x, splits, min(s, splits - 1), w) + lane; };
  float mc = -3.0e38f;
  for (int s = 0; s < splits; ++s) mc = fmaxf(mc, part(s)[16 * OB * 64]);
  float16v o[OB] = {};
  float l = 0.0f, now[16 * OB + 2], next[16 * OB + 2];
  auto load = [&](int s, float* x) {
    const float* const at = part(s);
#pragma unroll
    for (int i = 0; i < 16 * OB + 2; ++i) x[i] = at[i * 64];
    __builtin_amdgcn_sched_barrier(0);
  };
  load(0, now);
#pragma unroll 1
  for (int s = 0; s < splits; ++s) {
    load(s + 1, next);
    const float x = __builtin_amdgcn_exp2f(now[16 * OB] - mc);
    l += now[16 * OB + 1] * x;
#pragma unroll
    for (int c = 0; c < OB; ++c)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[c][i] += now[16 * c + i] * x;
#pragma unroll
    for (int i = 0; i < 16 * OB + 2; ++i) now[i] = next[i];
  }
  const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)smem;
  write_rows<T, D>(p, it, head_of(p), m0, w, lane, o, l, lds + w * 32 * (2 * D + 16));
}

// Query blocks of all sequences, or a few more: each takes (rows + BM - 1) / BM, rounded down.
int64_t blocks_of(int N, int R) { return (N + (BM - 1) * (int64_t)R) / BM; }

// Workgroups that share a block's keys where the blocks leave most of the chip idle: as many as make one for each CU, each with
// ten tiles at least, or at 64 dims, where the next ones' start hides behind the first ones' end, two for each CU with
// sixteen; and no more than the join is worth, which reads them all (64 rows of 14 heads at 64 dims over 16384 keys, 16
// shares: 15 us for these and 16 for the join).  us, without / with: 32 q / 8 KV heads, 128 dims, a row over 4096 keys 54 / 23, over 32768 391 / 82, 128 rows over 8192
// 105 / 42, 512 over 32768 397 / 276; prompts of 4 q heads, 2048 tokens, 128 dims 33 / 25, 4096, 64 dims 40 / 32.  Eight tiles a share: 14 q heads, 64
// dims, 1500 tokens 19.4 / 21.4, 4 q heads, 1100 tokens 15.7 / 16.5.
constexpr int kMostSplits = 16;
int splits_of(int D, int N, int NK, int R, int H) {
  const int64_t grid = blocks_of(N, R) * H, cus = device_cu_count(), tiles = NK / R / BN;
  const int64_t one = std::min(cus / grid, tiles / 10), two = D == 64 ? std::min(2 * cus / grid, tiles / 16) : 1;
  return (int)std::min<int64_t>(std::max<int64_t>(1, std::max(one, two)), kMostSplits);
}

template <typename T, int D>
int launch_dim(const PromptParams& p, float* parts, int64_t floats, hipStream_t stream) {
  const int64_t n = blocks_of(p.N, p.R), grid = n * p.H;
  if (const int rc = check_grid("prompt attention", grid, 256)) return rc;
  const int cus = device_cu_count();
  // Few workgroups and many keys: two halves of eight waves share a workgroup's keys.  us, without / with, 128 dims, 32 q
  // heads, 1000 tokens 26.0 / 24.2, 2000 (511 workgroups) 49.5 / 51.5, 300 12.6 / 13.1; 64 dims, 32 q heads, 1500 tokens (384
  // workgroups) 24.2 / 22.0, 2900 (736) 54.4 / 57.8; 4 q heads, 4096 tokens 47.1 / 38.2.
  if (grid <= (D == 64 ? 2 : 1) * (int64_t)cus && p.NK >= 512 * (int64_t)p.R) {
    const int most = splits_of(D, p.N, p.NK, p.R, p.H), splits = floats >= grid * most * 4 * part_floats<D>() ? most : 1;
    hipLaunchKernelGGL((prompt_kernel<T, D, 2>), dim3((unsigned)grid, splits), dim3(512), 0, stream, p, (int)n, 0, splits, parts);
    if (splits > 1) hipLaunchKernelGGL((join_kernel<T, D>), dim3((unsigned)grid), dim3(256), 0, stream, p, (int)n, splits, parts);
    return check_launch("prompt attention");
  }
  // Two workgroups a CU and no more: the ones behind the first round go in rising order, so that a CU that holds one of
  // the longest blocks gets one of the shortest beside it.  us, falling / so, 32 q heads, 128 dims, 1500 tokens 37.6 / 35.8,
  // 2000 50.9 / 47.7; 80 dims, 1900 38.0 / 36.4.  (64 dims hold three a CU and have no gain: 54.8 / 56.2 and 24.1 / 23.4.)
  const int turn = p.causal && D != 64 && grid > cus && grid <= 2 * (int64_t)cus ? (cus + p.H - 1) / p.H : 0;
  hipLaunchKernelGGL((prompt_kernel<T, D, 1>), dim3((unsigned)grid), dim3(256), 0, stream, p, (int)n, turn, 1, nullptr);
  return check_launch("prompt attention");
}

template <typename T>
int launch(int D, const PromptParams& p, float* parts, int64_t floats, hipStream_t stream) {
  return D == 64   ? launch_dim<T, 64>(p, parts, floats, stream)
         : D == 80 ? launch_dim<T, 80>(p, parts, floats, stream)
                   : launch_dim<T, 128>(p, parts, floats, stream);
}

}  // namespace prompt

int64_t prompt_workspace_bytes(int D, int N, int NK, int R, int H) {
  if (N == 0 || R == 0) return 0;
  const int splits = prompt::splits_of(D, N, NK, R, H);
  const int64_t part = D == 64 ? prompt::part_floats<64>() : D == 80 ? prompt::part_floats<80>() : prompt::part_floats<128>();
  return splits > 1 ? prompt::blocks_of(N, R) * H * splits * 4 * part * (int64_t)sizeof(float) : 0;
}

int launch_prompt(int D, int dtype, const PromptParams& p, void* workspace, int64_t bytes, hipStream_t stream) {
  float* const parts = reinterpret_cast<float*>(workspace);
  const int64_t floats = workspace ? bytes / (int64_t)sizeof(float) : 0;
  return dtype == SLMT_BF16 ? prompt::launch<__bf16>(D, p, parts, floats, stream) : prompt::launch<_Float16>(D, p, parts, floats, stream);
}

}  // namespace slmt
