// Rotary positions: queries and keys turned by their tokens' positions, and the same joined with the
// quantize-on-write store, so that a decode step's keys go from the projection to the packed cache
// without being written in between.
//
// Pair i of a head's first `rotary_dim` dims, (2i, 2i + 1) or (i, i + rotary_dim / 2), turns by
// a = position * inv_freq[i]:  (y1, y2) = (x1 c - x2 s, x2 c + x1 s), c = scale cos a, s = scale sin a.
// The angle is the exact product: positions of 10^5 times an fp32 frequency have no fraction left in
// fp32, so it is formed in fp64, with what that rounds off (from 2^29 on, the product has more than 53 bits) beside
// it, and reduced there (Cody and Waite, pi/2 in two parts): angles of up to 2^52.  The Taylor sums of
// sine and cosine on [-pi/4, pi/4] run in fp64 too; c and s are then rounded to fp32 once.  The rotation
// is in fp32, every product rounded by itself, and each result is rounded to the tensors' type once.
// The joined form's cache bytes are those of the rotation followed by the store, bit for bit.
//
// A workgroup takes the (token, head) rows of a few tokens: it forms their cosines and sines once, in
// LDS, for all heads, and turns the rows 8 dims per lane.  A lane of the half layout needs the 8 dims
// `rotary_dim / 2` away as well and reads them itself: they are in its row's cache lines.
//
// Memory bounds the large calls: the joined form of 7001 tokens, 32 + 2 * 8 heads of 128 dims, moves its 151 MB in 28 us
// where they come from the caches and 34 from memory (4.4 - 5.3 TB/s; a large copy 4.7).  A decode step (64 tokens of these
// heads, 1.4 MB) is latency, 3.8 us; 3001 tokens of 12 + 2 heads in bf16, half of the head turned, take 8.2 us of the 4.6
// that the bytes need: one round of workgroups, each of which reads its positions and frequencies, forms the angles in
// fp64 and only then turns its rows; its waves wait for 60% of their time.  (Rows read ahead of the angles: 9.5 us.)
#include "store_row.h"

namespace slmt {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 8;      // tokens of a workgroup

// cos(a) and sin(a) of a = position * frequency, each times scale, rounded to fp32 once.
__device__ __forceinline__ float2 turn(double position, double frequency, double scale) {
  const double a = position * frequency, rest = __builtin_fma(position, frequency, -a);
  const double k = __builtin_rint(a * 0.63661977236758134308);        // 2 / pi
  double r = __builtin_fma(-k, 1.5707963267948965580, a);             // pi / 2, its first 53 bits
  r = __builtin_fma(-k, 6.1232339957367658860e-17, r) + rest;         // and the next
  const double r2 = r * r;
  double s = -1.0 / 1307674368000.0;                                  // 1 / 15!
  s = __builtin_fma(s, r2, 1.0 / 6227020800.0);
  s = __builtin_fma(s, r2, -1.0 / 39916800.0);
  s = __builtin_fma(s, r2, 1.0 / 362880.0);
  s = __builtin_fma(s, r2, -1.0 / 5040.0);
  s = __builtin_fma(s, r2, 1.0 / 120.0);
  s = __builtin_fma(s, r2, -1.0 / 6.0);
  s = __builtin_fma(s * r2, r, r);
  double c = 1.0 / 20922789888000.0;                                  // 1 / 16!
  c = __builtin_fma(c, r2, -1.0 / 87178291200.0);
  c = __builtin_fma(c, r2, 1.0 / 479001600.0);
  c = __builtin_fma(c, r2, -1.0 / 3628800.0);
  c = __builtin_fma(c, r2, 1.0 / 40320.0);
  c = __builtin_fma(c, r2, -1.0 / 720.0);
  c = __builtin_fma(c, r2, 1.0 / 24.0);
  c = __builtin_fma(c, r2, -0.5);
  c = __builtin_fma(c, r2, 1.0);
  const int quarter = (int)(k - 4.0 * __builtin_floor(0.25 * k));     // 0 .. 3
  const double cc = quarter & 1 ? s : c, ss = quarter & 1 ? c : s;
  return make_float2((float)((quarter == 1 || quarter == 2 ? -cc : cc) * scale),
                     (float)((quarter >= 2 ? -ss : ss) * scale));
}

typedef __bf16 Bf16;
typedef _Float16 Fp16;

// Eight values from and to an address that is a multiple of their size.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float* x) {
  T raw[8];
  __builtin_memcpy(raw, p, sizeof(raw));
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = (float)raw[e];
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const T* y) {
  __builtin_memcpy(p, y, 8 * sizeof(T));
}

struct Params {
  RotaryParams r;
  uint32_t rows, per_split, tokens;     // a token's rows (query heads, then KV heads); of one split; tokens of a workgroup
};

// Eight turned dims d0 .. d0 + 7 of the row at `row`; cs: the token's cosines and sines.
// HALF8: the half layout with rotary_dim a multiple of 16, so that the eight lie on one side.
template <typename T, bool HALF8>
__device__ __forceinline__ void rotate8(const RotaryParams& r, const T* row, int d0, const float2* cs, T* y) {
#pragma clang fp contract(off)
  const int rot = r.rotary_dim, half = rot >> 1;
  float x[8];
  load8(row + d0, x);
  if (HALF8) {
    if (d0 < rot) {
      const bool low = d0 < half;
      const int i0 = low ? d0 : d0 - half;
      float o[8];
      load8(row + (low ? d0 + half : d0 - half), o);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float a = x[e] * cs[i0 + e].x, b = o[e] * cs[i0 + e].y;
        x[e] = low ? a - b : a + b;
      }
    }
  } else if (r.interleaved) {
#pragma unroll
    for (int e = 0; e < 8; e += 2)
      if (d0 + e < rot) {
        const float2 t = cs[(d0 + e) >> 1];
        const float x1 = x[e], x2 = x[e + 1];
        x[e] = x1 * t.x - x2 * t.y;
        x[e + 1] = x2 * t.x + x1 * t.y;
      }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int d = d0 + e;
      if (d < rot) {
        const bool low = d < half;
        const float2 t = cs[low ? d : d - half];
        const float o = (float)row[low ? d + half : d - half];
        const float a = x[e] * t.x, b = o * t.y;
        x[e] = low ? a - b : a + b;
      }
    }
  }
  __builtin_amdgcn_wave_barrier();           // (a row turned in place: all of its lanes read before one writes)
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = (T)x[e];
}

template <typename T, int D, bool HALF8, bool STORE>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const Params p) {
  constexpr int LANES = D == 64 ? 8 : 16, SLOT = D + 8;
  __shared__ float2 cs[kMaxTokens][D / 2];
  const RotaryParams& r = p.r;
  const int tid = threadIdx.x;
  const uint32_t t0 = blockIdx.x * p.tokens, tokens = min(p.tokens, (uint32_t)r.N - t0);
  const uint32_t half = r.rotary_dim >> 1;
  for (uint32_t i = tid; i < tokens * half; i += kThreads) {
    const uint32_t t = i / half, f = i - t * half;
    const int64_t pos = r.pos64 ? reinterpret_cast<const int64_t*>(r.positions)[t0 + t]
                                : reinterpret_cast<const int32_t*>(r.positions)[t0 + t];
    cs[t][f] = turn((double)pos, (double)r.inv_freq[f], r.scale);
  }
  __syncthreads();
  const int lane = tid & (LANES - 1);
  const int d0 = 8 * min(lane, D / 8 - 1);
  const bool writes = lane < D / 8;             // idle lanes repeat the row's last dims
  const uint32_t first = blockIdx.y * p.per_split, n = min(p.per_split, p.rows - first);
  for (uint32_t i = tid / LANES; i < tokens * n; i += kThreads / LANES) {
    const uint32_t t = i / n, row = first + (i - t * n);
    const int64_t token = t0 + t;
    T y[8];
    if (row < (uint32_t)r.H) {
      rotate8<T, HALF8>(r, reinterpret_cast<const T*>(r.q) + token * r.q_token + (int64_t)row * r.q_head, d0, cs[t], y);
      if (writes) store8(reinterpret_cast<T*>(r.q_out) + token * r.q_out_token + (int64_t)row * r.q_out_head + d0, y);
      continue;
    }
    const uint32_t h = row - r.H;
    const T* const key = reinterpret_cast<const T*>(r.k) + token * r.k_token + (int64_t)h * r.k_head;
    if constexpr (!STORE) {
      rotate8<T, HALF8>(r, key, d0, cs[t], y);
      if (writes) store8(reinterpret_cast<T*>(r.k_out) + token * r.k_out_token + (int64_t)h * r.k_out_head + d0, y);
    } else {
      const int64_t slot = r.slots[token];
      Eight v;
      __builtin_memcpy(&v, reinterpret_cast<const T*>(r.v) + token * r.v_token + (int64_t)h * r.v_head + d0, 16);
      rotate8<T, HALF8>(r, key, d0, cs[t], y);
      const Eight k = __builtin_bit_cast(Eight, y);
      if (r.k_out && writes)
        store8(reinterpret_cast<T*>(r.k_out) + token * r.k_out_token + (int64_t)h * r.k_out_head + d0, y);
      float kmin, kstep, vmin, vstep;
      row_ruler<LANES, D != 128>(k, kmin, kstep);
      row_ruler<LANES, D != 128>(v, vmin, vstep);
      const uint32_t kc = codes(k, kmin, kstep, 1.0f / kstep);
      const uint32_t vc = codes(v, vmin, vstep, 1.0f / vstep);
      if (slot < 0 || slot >= r.num_slots) continue;
      uint8_t* const dst = r.cache + (slot * r.KV + h) * (int64_t)SLOT;
      if (writes) {
        *reinterpret_cast<uint32_t*>(dst + 4 * lane) = kc;
        *reinterpret_cast<uint32_t*>(dst + D / 2 + 4 * lane) = vc;
      }
      if (lane == 0) {
        const uint32_t r0 = (uint32_t)f2h(kmin) | ((uint32_t)f2h(kstep) << 16);
        const uint32_t r1 = (uint32_t)f2h(vmin) | ((uint32_t)f2h(vstep) << 16);
        *reinterpret_cast<uint2*>(dst + D) = make_uint2(r0, r1);
      }
    }
  }
}

template <typename T, int D, bool STORE>
int launch(const RotaryParams& r, hipStream_t stream) {
  constexpr uint32_t flight = kThreads / (D == 64 ? 8 : 16);       // rows that a workgroup turns at a time
  Params p;
  p.r = r;
  p.rows = (uint32_t)(r.H + (r.k ? r.KV : 0));
  // A workgroup holds about as many rows as it turns at a time: several tokens of few heads, and a part of
  // a token of many where there are too few tokens to fill the chip.
  p.tokens = p.rows >= flight || r.N <= 512 ? 1 : (flight / p.rows < (uint32_t)kMaxTokens ? flight / p.rows : kMaxTokens);
  const uint32_t blocks = ((uint32_t)r.N + p.tokens - 1) / p.tokens;
  uint32_t splits = (p.rows + flight - 1) / flight, most = 1024 / blocks;
  if (splits > most) splits = most ? most : 1;
  p.per_split = (p.rows + splits - 1) / splits;
  splits = (p.rows + p.per_split - 1) / p.per_split;
  if (const int rc = check_grid("rotary", blocks, kThreads)) return rc;
  const dim3 grid(blocks, splits);
  if (!r.interleaved && r.rotary_dim % 16 == 0)
    hipLaunchKernelGGL((rotary_kernel<T, D, true, STORE>), grid, dim3(kThreads), 0, stream, p);
  else
    hipLaunchKernelGGL((rotary_kernel<T, D, false, STORE>), grid, dim3(kThreads), 0, stream, p);
  return check_launch("rotary");
}

template <typename T, bool STORE>
int launch_dim(int D, const RotaryParams& r, hipStream_t stream) {
  return D == 64 ? launch<T, 64, STORE>(r, stream) : D == 80 ? launch<T, 80, STORE>(r, stream) : launch<T, 128, STORE>(r, stream);
}

}  // namespace

int launch_rotary(int D, int dtype, const RotaryParams& r, hipStream_t stream) {
  if (r.N == 0 || r.H + (r.k ? r.KV : 0) == 0) return SLMT_OK;
  if (r.cache) return launch_dim<Fp16, true>(D, r, stream);
  if (dtype == SLMT_BF16) return launch_dim<Bf16, false>(D, r, stream);
  if (dtype == SLMT_F16) return launch_dim<Fp16, false>(D, r, stream);
  return launch_dim<float, false>(D, r, stream);
}

}  // namespace slmt
