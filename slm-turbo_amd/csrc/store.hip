// Quantize-on-write store into the packed per-token 4-bit paged cache.
//
// Same arithmetic as the reference's kv_quantize_store_kernel
// (kernels/kv_dequant_kernels.cuh:816-919), laid out for CDNA4: 8 dims per lane, so
// a (token, kv head) row is 8 lanes at head_dim 64 and 16 at 80 and 128 (6 of them
// idle at 80), and a wave takes 8 or 4 rows.  K and V are one 16-byte load and one
// 4-byte store each per lane; minima and maxima go over packed fp16 pairs and DPP
// within the row's lanes.  Every fp32 operation is rounded separately (contraction
// off) so codes and fp16 rulers are bit-exact with the reference.
//
// Long prompts move each byte once (7001 tokens, 8 KV heads of 128 dims: 28.5 MB read and
// 7.2 MB written by the counters, in 10.2 us), and what bounds them is the launch and each
// wave's one chain of load, reduction and store, not the memory: rotating over 430 MB of
// buffers, so that all of it comes from HBM, takes 6 % longer than passes over one set,
// which the Infinity Cache holds.  2 dims per lane, a wave per row, byte stores and the
// compiler's division took 23.1 us.
#include "store_row.h"

namespace slmt {

namespace {

constexpr int kThreads = 256;

template <int D>
__global__ void __launch_bounds__(kThreads)
quantize_store_kernel(const uint16_t* __restrict__ key, int64_t key_stride,
                      const uint16_t* __restrict__ value, int64_t value_stride,
                      uint8_t* __restrict__ cache, int64_t num_slots,
                      const int64_t* __restrict__ slot_mapping, uint32_t rows, uint32_t KV) {
  constexpr int SLOT = D + 8, HALF = D / 2;
  constexpr int LANES = D == 64 ? 8 : 16;
  const int lane = threadIdx.x & (LANES - 1);
  const uint32_t row = blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
  const uint32_t rw = min(row, rows - 1);             // lanes past the end repeat the last row and store nothing
  const uint32_t t = rw / KV, h = rw - t * KV;
  // The row is quantized whether or not its slot is valid and only the stores
  // test it: with an early exit on the slot the row's K/V loads were issued
  // after the slot's had returned, two dependent round trips per call.
  const int64_t slot = slot_mapping[t];
  const int d0 = 8 * min(lane, D / 8 - 1);            // idle lanes re-read the row's last dims
  const Eight k = load_eight(key + t * key_stride + (int64_t)h * D + d0);
  const Eight v = load_eight(value + t * value_stride + (int64_t)h * D + d0);
  float kmin, kstep, vmin, vstep;
  row_ruler<LANES, D != 128>(k, kmin, kstep);
  row_ruler<LANES, D != 128>(v, vmin, vstep);
  const uint32_t kc = codes(k, kmin, kstep, 1.0f / kstep);
  const uint32_t vc = codes(v, vmin, vstep, 1.0f / vstep);

  // padding token / out of range: no store
  if (row >= rows || slot < 0 || slot >= num_slots) return;
  uint8_t* dst = cache + (slot * KV + h) * (int64_t)SLOT;
  if (lane < D / 8) {
    *reinterpret_cast<uint32_t*>(dst + 4 * lane) = kc;
    *reinterpret_cast<uint32_t*>(dst + HALF + 4 * lane) = vc;
  }
  if (lane == 0) {
    const uint32_t r0 = (uint32_t)f2h(kmin) | ((uint32_t)f2h(kstep) << 16);
    const uint32_t r1 = (uint32_t)f2h(vmin) | ((uint32_t)f2h(vstep) << 16);
    *reinterpret_cast<uint2*>(dst + D) = make_uint2(r0, r1);   // slot base is 8-byte aligned
  }
}

}  // namespace

int launch_quantize_store(const void* key, int64_t key_stride, const void* value,
                          int64_t value_stride, void* cache, int64_t num_slots,
                          const int64_t* slot_mapping, int64_t N, int KV, int D,
                          hipStream_t stream) {
  if (N == 0) return SLMT_OK;
  // (row numbers are 32-bit: 2^32 rows of K alone would not fit the device)
  const int64_t rows = N * KV, per_block = kThreads / (D == 64 ? 8 : 16);
  const int64_t blocks = (rows + per_block - 1) / per_block;
  if (rows >= (int64_t(1) << 32) - kThreads || blocks > 0x7fffffffLL)
    return fail(SLMT_ERR_UNSUPPORTED, "store: too many tokens for one launch");
  const dim3 grid((unsigned)blocks), block(kThreads);
  auto k = reinterpret_cast<const uint16_t*>(key);
  auto v = reinterpret_cast<const uint16_t*>(value);
  auto c = reinterpret_cast<uint8_t*>(cache);
  switch (D) {
    case 64:
      hipLaunchKernelGGL(quantize_store_kernel<64>, grid, block, 0, stream, k, key_stride, v,
                         value_stride, c, num_slots, slot_mapping, (uint32_t)rows, (uint32_t)KV);
      break;
    case 80:
      hipLaunchKernelGGL(quantize_store_kernel<80>, grid, block, 0, stream, k, key_stride, v,
                         value_stride, c, num_slots, slot_mapping, (uint32_t)rows, (uint32_t)KV);
      break;
    case 128:
      hipLaunchKernelGGL(quantize_store_kernel<128>, grid, block, 0, stream, k, key_stride, v,
                         value_stride, c, num_slots, slot_mapping, (uint32_t)rows, (uint32_t)KV);
      break;
    default:
      return fail(SLMT_ERR_INVALID, "store: head_dim must be 64/80/128, got " + std::to_string(D));
  }
  return check_launch("store");
}

}  // namespace slmt
