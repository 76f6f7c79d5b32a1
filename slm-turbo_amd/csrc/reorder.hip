// The beams' cache rows after a selection: row j of a request becomes a copy of its parent's
// row.  Blocks that are full are never written again, so their table entries are copied and
// beams share them; in the block that is still filling every beam has a block of its own,
// whose tokens are copied, in all layers.  (The reference has no beam search.)
//
// In place, for any parents: a thread reads its 16 bytes (or its table column) of all W beams'
// parents before it writes any of them, and no other thread touches these bytes.
// (More than 8 rows: with the places of those that move listed in LDS.)
//
// Bound by memory where it moves much: 16 requests of 8 beams, of which half take over
// another's row, 32 layers of 8 heads, D = 128, blocks of 16: 35.7 MB read and written in 9.5 us
// a call, 3.7 TB/s (6.9 us at the rate of a large copy).  A launch otherwise: 4 beams, 22
// layers of 4 heads, D = 64: 6.5 us a call, the host's, 3.6 in the kernel.
#include "slmt_internal.h"

#include <algorithm>

namespace slmt {
namespace reorder {

constexpr int kThreads = 256;

// blockIdx: x unit of the block or table column, y layer (one more for the tables), z request.
// WMAX: beams that a thread holds; Unit: what it moves of each.
template <int WMAX, typename Unit, typename Entry>
__global__ void __launch_bounds__(kThreads) reorder_kernel(const ReorderParams p) {
  const int r = blockIdx.z, layer = blockIdx.y;
  const int32_t* const parents = p.parents + (int64_t)r * p.W;
  Entry* const tables = reinterpret_cast<Entry*>(p.block_tables) + (int64_t)r * p.W * p.bt_stride;
  const int len = max(p.seq_lens[r], 0);
  const int col = len / p.block_size, filled = len - col * p.block_size;
  const int at = blockIdx.x * kThreads + threadIdx.x;
  if (layer == p.layers) {             // table entries of the full blocks
    if (at >= min(col, p.columns)) return;
    Entry e[WMAX];
#pragma unroll
    for (int j = 0; j < WMAX; ++j) {
      const int from = j < p.W ? parents[j] : -1;
      e[j] = tables[(int64_t)(from >= 0 && from < p.W ? from : j < p.W ? j : 0) * p.bt_stride + at];
    }
#pragma unroll
    for (int j = 0; j < WMAX; ++j) {
      const int from = j < p.W ? parents[j] : -1;
      if (from >= 0 && from < p.W && from != j) tables[(int64_t)j * p.bt_stride + at] = e[j];
    }
    return;
  }
  if (col >= p.columns) return;        // (a row without room for another token)
  const int64_t bytes = (int64_t)filled * p.row_bytes;    // a multiple of 8
  const int64_t from_byte = (int64_t)at * sizeof(Unit);
  const bool half = sizeof(Unit) == 16 && from_byte + 8 == bytes;
  const int64_t block_bytes = (int64_t)p.block_size * p.row_bytes;
  uint8_t* const cache = p.caches[layer] + from_byte;
  Unit v[WMAX];
  if constexpr (WMAX <= 8) {           // every thread finds the rows' places by itself
    if (from_byte >= bytes) return;
    uint8_t* to[WMAX];
#pragma unroll
    for (int j = 0; j < WMAX; ++j) {
      to[j] = nullptr;
      if (j >= p.W) continue;
      const int from = parents[j];
      if (from < 0 || from >= p.W || from == j) continue;
      const int64_t src = tables[(int64_t)from * p.bt_stride + col], dst = tables[(int64_t)j * p.bt_stride + col];
      if (src < 0 || src >= p.num_blocks || dst < 0 || dst >= p.num_blocks) continue;
      to[j] = cache + dst * block_bytes;
      const uint8_t* const s = cache + src * block_bytes;
      if (half) *reinterpret_cast<uint2*>(&v[j]) = *reinterpret_cast<const uint2*>(s);
      else v[j] = *reinterpret_cast<const Unit*>(s);
    }
#pragma unroll
    for (int j = 0; j < WMAX; ++j) {
      if (to[j] == nullptr) continue;
      if (half) *reinterpret_cast<uint2*>(to[j]) = *reinterpret_cast<const uint2*>(&v[j]);
      else *reinterpret_cast<Unit*>(to[j]) = v[j];
    }
    return;
  }
  if ((int64_t)blockIdx.x * kThreads * (int64_t)sizeof(Unit) >= bytes) return;
  // Of more rows those that move are listed first, by a thread each: their places would not stay in registers beside their bytes
  // (2 requests of 64 beams, 64 rows to move, 32 layers of 8 heads, D = 128: 45 us without the list, 18 with it; 4 of 32 50 and
  // 12.5; 1 of 4, which takes the other way, would be 6.5 instead of 6.4).
  __shared__ int64_t froms[WMAX], tos[WMAX];
  __shared__ int moved;
  if (threadIdx.x < 64) {
    const int j = threadIdx.x, from = j < p.W ? parents[j] : -1;
    int64_t src = -1, dst = -1;
    if (from >= 0 && from < p.W && from != j) {
      src = tables[(int64_t)from * p.bt_stride + col];
      dst = tables[(int64_t)j * p.bt_stride + col];
    }
    const bool moves = src >= 0 && src < p.num_blocks && dst >= 0 && dst < p.num_blocks;
    const uint64_t who = __builtin_amdgcn_ballot_w64(moves);
    if (moves) {
      const int i = __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
      froms[i] = src * block_bytes;
      tos[i] = dst * block_bytes;
    }
    if (j == 0) moved = __builtin_popcountll(who);
  }
  __syncthreads();
  if (from_byte >= bytes) return;
  const int n = __builtin_amdgcn_readfirstlane(moved);
#pragma unroll
  for (int j = 0; j < WMAX; ++j) {
    if (j >= n) continue;
    const uint8_t* const s = cache + froms[j];
    if (half) *reinterpret_cast<uint2*>(&v[j]) = *reinterpret_cast<const uint2*>(s);
    else v[j] = *reinterpret_cast<const Unit*>(s);
  }
#pragma unroll
  for (int j = 0; j < WMAX; ++j) {
    if (j >= n) continue;
    uint8_t* const t = cache + tos[j];
    if (half) *reinterpret_cast<uint2*>(t) = *reinterpret_cast<const uint2*>(&v[j]);
    else *reinterpret_cast<Unit*>(t) = v[j];
  }
}

template <int WMAX, typename Unit>
int launch(const ReorderParams& p, hipStream_t stream) {
  const int64_t units = ((int64_t)(p.block_size - 1) * p.row_bytes + sizeof(Unit) - 1) / sizeof(Unit);
  const int64_t x = std::max<int64_t>(1, (std::max<int64_t>(units, p.tables ? p.columns : 0) + kThreads - 1) / kThreads);
  const dim3 grid((unsigned)x, p.layers + (p.tables ? 1 : 0), p.R);
  if (int rc = check_grid("reorder beams", x, kThreads)) return rc;
  if (p.bt64) hipLaunchKernelGGL((reorder_kernel<WMAX, Unit, int64_t>), grid, dim3(kThreads), 0, stream, p);
  else hipLaunchKernelGGL((reorder_kernel<WMAX, Unit, int32_t>), grid, dim3(kThreads), 0, stream, p);
  return check_launch("reorder beams");
}

}  // namespace reorder

int launch_reorder(const ReorderParams& p, hipStream_t stream) {
  // 16 bytes where every block starts at a multiple of 16, and the fewest units that hold the beams, in registers.  16 requests
  // of 8 beams, 32 layers of 8 heads, D = 128, us in the kernel: 10.6; by 8 bytes 12.9; with 16 units 13.9.  4 requests of 32
  // beams, us a call: 12.5; by 8 bytes with 64 units 18.0.  (64 units of 16 bytes are all of a thread's registers.)
  bool wide = ((int64_t)p.block_size * p.row_bytes) % 16 == 0;
  for (int i = 0; i < p.layers; ++i) wide = wide && (reinterpret_cast<uintptr_t>(p.caches[i]) & 15) == 0;
  if (p.W <= 4) return wide ? reorder::launch<4, uint4>(p, stream) : reorder::launch<4, uint2>(p, stream);
  if (p.W <= 8) return wide ? reorder::launch<8, uint4>(p, stream) : reorder::launch<8, uint2>(p, stream);
  if (p.W <= 16) return wide ? reorder::launch<16, uint4>(p, stream) : reorder::launch<16, uint2>(p, stream);
  if (p.W <= 32) return wide ? reorder::launch<32, uint4>(p, stream) : reorder::launch<32, uint2>(p, stream);
  return reorder::launch<64, uint2>(p, stream);
}

}  // namespace slmt
