// A serving step's metadata from its requests' lengths: positions, slots, sequence lengths and the
// block-table entries of the blocks that the step's tokens open, in one launch.
//
// Request r brings q_r tokens behind c_r cached ones.  With start_r = sum q_s (s < r), token t of
// request r sits at position p = c_r + t - start_r, in column p / block_size of its table row; columns
// from ceil(c_r / block_size) on are new and take the next blocks of the free list, requests and
// columns in order:
//   need_r = ceil((c_r + q_r) / bs) - ceil(c_r / bs),   first free block = free_start + sum need_s (s < r).
// A workgroup takes kTokens tokens and goes through the requests kThreads at a time: two scans (tokens,
// then blocks), and a search for each of its tokens in the ends that the first scan left in LDS.
// Every workgroup repeats the scans up to its own last token, so none waits for another; the first one
// goes through all requests and writes what there is per request.  A new column is written by the
// token that opens it, and only older columns are read: no order between the workgroups is needed.
//
// Sums saturate at the step's token capacity, which keeps them in 32 bits whatever the lengths hold.
//
// It is latency all through: the bytes (16 a token, 8 a request) are 0.5 us of copying at most, and a launch of
// anything takes 3.8 us in a row of them.  us: 3.4 for 32 requests of a token each, 6.7 for 200 with 27 thousand
// tokens together (27 workgroups), 6.4 for 96 with 130 thousand; torch's forms of the same take 270 - 300.
#include "slmt_internal.h"

namespace slmt {
namespace {

constexpr int kThreads = 256, kPerThread = 4, kTokens = kThreads * kPerThread;

struct Params {
  const int32_t *query_lens, *context_lens;
  int R;
  void* tables;
  int64_t table_stride;
  int columns;
  const void* free_blocks;
  int num_free;
  const int32_t* free_start;
  int block_size, N;
  int32_t *query_start, *seq_lens;
  int64_t *positions, *slots;
  int32_t* free_end;
};

// Inclusive scan over the workgroup of a sum that saturates at `most`; returns this thread's value and
// the total.  (`sums`: one entry per wave; two barriers.)
__device__ __forceinline__ uint32_t scan(uint32_t v, uint32_t most, uint32_t* sums, uint32_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t u = __shfl_up(v, o, 64);
    if (lane >= o) v = min(v + u, most);
  }
  if (lane == 63) sums[wave] = v;
  __syncthreads();
  uint32_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    if (w == wave) before = total;
    total = min(total + sums[w], most);
  }
  __syncthreads();
  return min(v + before, most);
}

template <typename Entry>
__global__ void __launch_bounds__(kThreads) step_metadata_kernel(const Params p) {
  __shared__ uint32_t sums[kThreads / 64];
  __shared__ uint32_t ends[kThreads];        // the requests' last token + 1
  __shared__ int4 info[kThreads];            // first position - first token, held columns, first free block, tokens' end
  Entry* const tables = reinterpret_cast<Entry*>(p.tables);
  const Entry* const free_blocks = reinterpret_cast<const Entry*>(p.free_blocks);
  const int tid = threadIdx.x, bs = p.block_size;
  const uint32_t N = p.N, t0 = blockIdx.x * (uint32_t)kTokens, t1 = min(t0 + kTokens, N);
  const bool all = blockIdx.x == 0;
  const int64_t capacity = min((int64_t)p.columns * bs, (int64_t)0x7fffffff);
  const uint32_t free_start = p.free_start ? (uint32_t)max(*p.free_start, 0) : 0u;
  uint32_t base = 0, taken = 0;              // tokens and new blocks of the requests before this round's
  for (int r0 = 0; r0 < p.R && (all || base < t1); r0 += kThreads) {
    const int r = r0 + tid;
    uint32_t q = 0;
    int32_t ctx = 0;
    if (r < p.R) {
      q = (uint32_t)max(p.query_lens[r], 0);
      ctx = (int32_t)min((int64_t)max(p.context_lens[r], 0), capacity);
    }
    uint32_t round;
    const uint32_t end = min(base + scan(min(q, N), N, sums, round), N);
    // (this round's part of the request; where the sum is cut at N, so are its tokens)
    const uint32_t before = __shfl_up(end, 1, 64);
    if ((tid & 63) == 63) sums[tid >> 6] = end;
    __syncthreads();
    const uint32_t start = tid == 0 ? base : (tid & 63) ? before : sums[(tid >> 6) - 1];
    __syncthreads();
    const uint32_t tokens = end - start;
    // those that the row has columns for, and the columns that they open
    const uint32_t fit = (uint32_t)min((int64_t)tokens, capacity - ctx);
    const uint32_t held = (uint32_t)(((int64_t)ctx + bs - 1) / bs);
    const uint32_t need = (uint32_t)(((int64_t)ctx + fit + bs - 1) / bs) - held;
    uint32_t opened;
    const uint32_t first = taken + scan(need, 0x7fffffffu, sums, opened) - need;
    // blocks that are left for them, and the tokens that then have a slot
    const int64_t left = (int64_t)p.num_free - free_start - first;
    const uint32_t got = (uint32_t)max(min((int64_t)need, left), (int64_t)0);
    const uint32_t live = got == need ? fit : (uint32_t)max((int64_t)(held + got) * bs - ctx, (int64_t)0);
    ends[tid] = end;
    info[tid] = make_int4((int)((uint32_t)ctx - start), (int)held, (int)(free_start + first), (int)(start + live));
    if (all && r < p.R) {
      p.query_start[r + 1] = (int32_t)end;
      p.seq_lens[r] = ctx + (int32_t)live;
      if (r == 0) p.query_start[0] = 0;
    }
    __syncthreads();
    const uint32_t last = min(base + round, N);
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      const uint32_t t = t0 + i * kThreads + tid;
      if (t < base || t >= last || t >= t1) continue;
      int lo = 0;                            // the first request of the round that ends past t
#pragma unroll
      for (int step = kThreads / 2; step; step >>= 1)
        if (ends[lo + step - 1] <= t) lo += step;
      const int4 a = info[lo];
      const uint32_t pos = (uint32_t)a.x + t;
      const uint32_t col = pos / (uint32_t)bs, in = pos - col * bs;
      int64_t slot = -1;
      if (t < (uint32_t)a.w) {
        Entry* const at = tables + (int64_t)(r0 + lo) * p.table_stride + col;
        Entry block;
        if (col >= (uint32_t)a.y) {
          block = free_blocks[(uint32_t)a.z + (col - (uint32_t)a.y)];
          if (in == 0) *at = block;
        } else {
          block = *at;
        }
        slot = (int64_t)block * bs + in;
      }
      p.positions[t] = pos;
      p.slots[t] = slot;
    }
    base = last;
    taken += opened;
    __syncthreads();
  }
  // padding (base is the number of the step's tokens here, or reaches past this workgroup's)
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const uint32_t t = t0 + i * kThreads + tid;
    if (t < t1 && t >= base) {
      p.positions[t] = 0;
      p.slots[t] = -1;
    }
  }
  if (all && tid == 0) {
    if (p.R == 0) p.query_start[0] = 0;
    *p.free_end = (int32_t)min((uint64_t)free_start + taken, (uint64_t)0x7fffffff);
  }
}

}  // namespace

int launch_step_metadata(const int32_t* query_lens, const int32_t* context_lens, int num_reqs, void* block_tables,
                         int bt64, int64_t table_stride, int columns, const void* free_blocks, int num_free,
                         const int32_t* free_start, int block_size, int num_tokens, int32_t* query_start,
                         int32_t* seq_lens, int64_t* positions, int64_t* slots, int32_t* free_end,
                         hipStream_t stream) {
  Params p{query_lens, context_lens, num_reqs,  block_tables, table_stride, columns, free_blocks, num_free, free_start,
           block_size, num_tokens,   query_start, seq_lens,   positions,    slots,   free_end};
  const dim3 grid((unsigned)(num_tokens > kTokens ? ((int64_t)num_tokens + kTokens - 1) / kTokens : 1)), block(kThreads);
  if (bt64)
    hipLaunchKernelGGL(step_metadata_kernel<int64_t>, grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL(step_metadata_kernel<int32_t>, grid, block, 0, stream, p);
  return check_launch("step metadata");
}

}  // namespace slmt
