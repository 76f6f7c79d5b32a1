// Attention over whole prompts' own K and V on the matrix cores, fp16 and bf16, head_dim 64, 80 and 128:
// sequences of different lengths packed behind one another, grouped heads, causal or not.
//
// A workgroup takes 128 query rows of one sequence and query head, 32 per wave, and walks the 64-key tiles
// that they can see.  Everything is transposed, so a lane owns one query column from the scores to the
// output (both halves of the wave the same 32 columns, each half its own keys and dims):
//   S^T = K Q^T                 (v_mfma_f32_32x32x16: A = 32 K rows, B = the lane's query)
//   P^T = exp2(c S^T - m)       (online softmax per query column; c = scale log2(e))
//   O^T += V^T P^T              (B = the lane's P^T as it comes out of S^T, A in the same order of keys)
// Scores, maxima, sums and the output accumulate in fp32.  The weights P enter the second product in the
// tensors' type, half a step of which is what the output's own rounding is off by, and the row sums add the
// same rounded weights.
#include "slmt_internal.h"

#include <type_traits>

namespace slmt {
namespace prompt {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef float float16v __attribute__((ext_vector_type(16)));
typedef unsigned uint4v __attribute__((ext_vector_type(4)));

constexpr int BM = 128;    // query rows per workgroup
constexpr int BN = 64;     // keys per tile

template <typename T>
struct Mfma;
template <>
struct Mfma<_Float16> {
  typedef half8 V8;
  static __device__ __forceinline__ float16v mul(V8 a, V8 b, float16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mfma<__bf16> {
  typedef bf8 V8;
  static __device__ __forceinline__ float16v mul(V8 a, V8 b, float16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};

struct Item {
  int seq, block;      // seq < 0: none
  int q0, nq, k0, nk;  // the sequence's rows of q and of k, v
};

// Block x of the sequences' blocks of BM query rows, one sequence after another.  Uniform over the wave.
__device__ __forceinline__ Item find_item(const PromptParams& p, int x) {
  const int lane = threadIdx.x & 63;
  int base = 0;
  for (int r0 = 0; r0 < p.R; r0 += 64) {
    const int r = min(r0 + lane, p.R - 1);
    const int q0 = min(max(p.q_start[r], 0), p.N), q1 = min(max(p.q_start[r + 1], q0), p.N);
    const int k0 = min(max(p.k_start[r], 0), p.NK), k1 = min(max(p.k_start[r + 1], k0), p.NK);
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

template <typename T, int D>
__global__ void __launch_bounds__(256) prompt_kernel(const PromptParams p) {
  using V8 = typename Mfma<T>::V8;
  constexpr int QB = D / 16;                 // 16-dim blocks of QK
  constexpr int OB = (D + 31) / 32;          // 32-dim blocks of PV
  constexpr int KROW = D + 8, VROW = BN + 8; // staged rows, elements
  __shared__ __attribute__((aligned(16))) T ks[BN * KROW];
  __shared__ __attribute__((aligned(16))) T vs[OB * 32 * VROW];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, col = lane & 31, hf = lane >> 5;
  const int h = blockIdx.x % p.H;
  const Item it = find_item(p, blockIdx.x / p.H);
  if (it.seq < 0) return;
  const int kv = h / (p.H / p.KV);
  const int m0 = it.block * BM, m = m0 + 32 * w + col;
  const int shift = it.nk - it.nq;           // query row m sees the keys up to m + shift
  const int last = min(m0 + BM, it.nq) - 1;
  const int kend = p.causal ? min(it.nk, max(last + shift + 1, 0)) : it.nk;
  const int ntiles = (kend + BN - 1) / BN;
  const T* const q = reinterpret_cast<const T*>(p.q) + (int64_t)(it.q0 + min(m, it.nq - 1)) * p.q_token + (int64_t)h * p.q_head;
  const T* const k = reinterpret_cast<const T*>(p.k) + (int64_t)it.k0 * p.k_token + (int64_t)kv * p.k_head;
  const T* const v = reinterpret_cast<const T*>(p.v) + (int64_t)it.k0 * p.v_token + (int64_t)kv * p.v_head;
  V8 qf[QB];
#pragma unroll
  for (int j = 0; j < QB; ++j) __builtin_memcpy(&qf[j], q + 16 * j + 8 * hf, 16);
  float16v o[OB] = {};
  float mx = -INFINITY, l = 0.0f;            // of this lane's keys for l, of the column for mx
  for (int i = tid; i < (OB * 32 - D) * VROW; i += 256) vs[D * VROW + i] = (T)0.0f;
  for (int t = 0; t < ntiles; ++t) {
    __syncthreads();
    // rows past the sequence are zeros, so that nothing of the next one reaches a product
    for (int i = tid; i < BN * (D / 8); i += 256) {
      const int row = i / (D / 8), c = i - row * (D / 8);
      const int key = t * BN + row;
      uint4v kx = {0, 0, 0, 0}, vx = {0, 0, 0, 0};
      if (key < it.nk) {
        __builtin_memcpy(&kx, k + (int64_t)key * p.k_token + 8 * c, 16);
        __builtin_memcpy(&vx, v + (int64_t)key * p.v_token + 8 * c, 16);
      }
      __builtin_memcpy(ks + row * KROW + 8 * c, &kx, 16);
      T e[8];
      __builtin_memcpy(e, &vx, 16);
#pragma unroll
      for (int d = 0; d < 8; ++d) vs[(8 * c + d) * VROW + row] = e[d];
    }
    __syncthreads();
    float16v s[2];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      s[n] = float16v{};
#pragma unroll
      for (int j = 0; j < QB; ++j) {
        V8 a;
        __builtin_memcpy(&a, __builtin_assume_aligned(ks + (32 * n + col) * KROW + 16 * j + 8 * hf, 16), 16);
        s[n] = Mfma<T>::mul(a, qf[j], s[n]);
      }
    }
    // s[n][i]: key 32 n + 8 (i / 4) + 4 hf + i % 4 of the tile
    const int k0 = t * BN;
    const bool whole = k0 + BN <= it.nk && (!p.causal || k0 + BN - 1 <= m0 + 32 * __builtin_amdgcn_readfirstlane(w) + shift);
    const int see = p.causal ? min(it.nk, m + shift + 1) : it.nk;     // keys that the column sees
    float tmax = -INFINITY;
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int key = k0 + 32 * n + 8 * (i >> 2) + 4 * hf + (i & 3);
        if (!whole) s[n][i] = key < see ? s[n][i] : -INFINITY;
        tmax = fmaxf(tmax, s[n][i]);
      }
    float a, b;
    swap32(tmax, a, b);
    const float next = fmaxf(mx, fmaxf(a, b));
    const float base = next == -INFINITY ? 0.0f : next * p.scale;     // (a column that has seen no key: weights 0)
    const float alpha = __builtin_amdgcn_exp2f(mx * p.scale - base);
    mx = next;
    l *= alpha;
#pragma unroll
    for (int c = 0; c < OB; ++c) o[c] *= alpha;
    V8 pb[4];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const T e = (T)__builtin_amdgcn_exp2f(__builtin_fmaf(s[n][i], p.scale, -base));
        pb[2 * n + (i >> 3)][i & 7] = e;
        l += (float)e;
      }
    auto vt = [&](int c, int u) {            // V^T: dim 32 c + col, the keys of pb[u]
      struct { uint2 x[2]; } x;
#pragma unroll
      for (int g = 0; g < 2; ++g)
        x.x[g] = *reinterpret_cast<const uint2*>(vs + (32 * c + col) * VROW + 16 * u + 8 * g + 4 * hf);
      return __builtin_bit_cast(V8, x);
    };
    bool odd = false;
    if (!whole) {                            // a masked value that is no number times 0 would be none either
      float16v z = {};
#pragma unroll
      for (int c = 0; c < OB; ++c)
#pragma unroll
        for (int u = 0; u < 4; ++u) z = Mfma<T>::mul(vt(c, u), V8{}, z);
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 16; ++i) sum += z[i];
      odd = __builtin_amdgcn_ballot_w64(sum != 0.0f) != 0;
    }
    if (!odd) {
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int c = 0; c < OB; ++c) o[c] = Mfma<T>::mul(vt(c, u), pb[u], o[c]);
    } else {
      // one key at a time, added to the columns that see it
#pragma unroll
      for (int u = 0; u < 4; ++u)
        for (int x = 0; x < 16; ++x) {
          const int xh = x >> 3, xe = x & 7;
          const bool sees = k0 + 16 * u + 8 * (xe >> 2) + 4 * xh + (xe & 3) < see;
          V8 pk{};
#pragma unroll
          for (int e = 0; e < 8; ++e) pk[e] = hf == xh && e == xe ? pb[u][e] : (T)0.0f;
#pragma unroll
          for (int c = 0; c < OB; ++c) {
            V8 va = vt(c, u);
#pragma unroll
            for (int e = 0; e < 8; ++e) va[e] = hf == xh && e == xe ? va[e] : (T)0.0f;
            const float16v add = Mfma<T>::mul(va, pk, float16v{});
#pragma unroll
            for (int i = 0; i < 16; ++i) o[c][i] += sees ? add[i] : 0.0f;
          }
        }
    }
  }
  float a, b;
  swap32(l, a, b);
  l = a + b;
  if (m >= it.nq) return;
  // (a row that sees keys whose scores are all -infinity is 0 / 0, as its softmax is)
  const bool none = p.causal ? m + shift < 0 : it.nk == 0;
  const float rl = none ? 0.0f : 1.0f / l;
  T* const out = reinterpret_cast<T*>(p.out) + (int64_t)(it.q0 + m) * p.out_token + (int64_t)h * p.out_head;
#pragma unroll
  for (int c = 0; c < OB; ++c)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * c + 8 * g + 4 * hf;
      if (d >= D) continue;
      T y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = (T)(none ? 0.0f : o[c][4 * g + i] * rl);
      __builtin_memcpy(out + d, y, 8);
    }
}

template <typename T>
int launch(int D, const PromptParams& p, hipStream_t stream) {
  const int64_t blocks = ((int64_t)p.N / BM + p.R) * p.H;
  if (blocks > 0x7fffffff) return fail(SLMT_ERR_UNSUPPORTED, "prompt attention: too many query blocks");
  const dim3 grid((unsigned)blocks), block(256);
  if (D == 64) hipLaunchKernelGGL((prompt_kernel<T, 64>), grid, block, 0, stream, p);
  else if (D == 80) hipLaunchKernelGGL((prompt_kernel<T, 80>), grid, block, 0, stream, p);
  else hipLaunchKernelGGL((prompt_kernel<T, 128>), grid, block, 0, stream, p);
  return check_launch("prompt attention");
}

}  // namespace prompt

int launch_prompt(int D, int dtype, const PromptParams& p, hipStream_t stream) {
  return dtype == SLMT_BF16 ? prompt::launch<__bf16>(D, p, stream) : prompt::launch<_Float16>(D, p, stream);
}

}  // namespace slmt
