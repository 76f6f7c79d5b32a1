// extern "C" entry points of libslmturbo_hip.so (declared in include/slmturbo.h).
//
// This layer replaces the reference's pybind11/ATen launchers
// (kernels/kv_dequant_cuda.cu:53-456): it validates sizes, strides and
// alignment with the same phase-prefixed wording as the reference's
// TORCH_CHECKs, then enqueues the kernels on the caller's stream (the
// reference used the legacy default stream).  Nothing here allocates.
#include "slmt_internal.h"

#include <mutex>
#include <string>

namespace slmt {

namespace {
thread_local std::string g_error;
thread_local int g_status = SLMT_OK;
}

void set_error(const std::string& msg) { g_error = msg; }
void clear_error() {
  g_error.clear();
  g_status = SLMT_OK;
}
int fail(int code, const std::string& msg) {
  g_error = msg;
  g_status = code;
  return code;
}
int last_status() { return g_status == SLMT_OK ? SLMT_ERR_INVALID : g_status; }
int check_launch(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(SLMT_ERR_HIP, std::string(what) + ": launch failed: " + hipGetErrorString(e));
  return SLMT_OK;
}

int check_grid(const char* what, int64_t workgroups, int threads) {
  if (workgroups * threads <= 0xffffffffll) return SLMT_OK;
  return fail(SLMT_ERR_UNSUPPORTED, std::string(what) + ": too many rows for a launch (" + std::to_string(workgroups) + " workgroups)");
}

int device_cu_count() {
  static std::mutex mu;
  static int counts[64] = {0};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return -1;
  std::lock_guard<std::mutex> lock(mu);
  if (counts[dev] == 0) {
    int n = 0;
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess) return -1;
    counts[dev] = n;
  }
  return counts[dev];
}

namespace {

bool head_dim_ok(int D) { return D == 64 || D == 80 || D == 128; }
bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
std::string s(int64_t v) { return std::to_string(v); }

int block_shift_of(int bs) {
  if (bs <= 0 || (bs & (bs - 1)) != 0) return -1;
  int k = 0;
  while ((1 << k) < bs) ++k;
  return k;
}

AttnParams blank_params() {
  AttnParams p{};
  p.block_shift = -1;
  p.min_tiles = 4;
  return p;
}

// Shared checks of the contiguous-source entry points.
int check_contig(const char* phase, const void* q, const void* kp, const void* vp, const void* r[4],
                 int H, int KVt, int KV, int S, int D, const float* out) {
  if (!head_dim_ok(D)) return fail(SLMT_ERR_INVALID, std::string(phase) + ": head_dim must be 64/80/128, got " + s(D));
  if (KV <= 0 || H <= 0 || H % KV != 0)
    return fail(SLMT_ERR_INVALID, std::string(phase) + ": num_kv_heads " + s(KV) + " must divide query heads " + s(H));
  if (KV > KVt)
    return fail(SLMT_ERR_INVALID, std::string(phase) + ": num_kv_heads " + s(KV) +
                                      " exceeds the packed KV heads " + s(KVt));
  if (S < 0) return fail(SLMT_ERR_INVALID, std::string(phase) + ": sequence length must be >= 0");
  if (!q || !kp || !vp || !out || !r[0] || !r[1] || !r[2] || !r[3])
    return fail(SLMT_ERR_INVALID, std::string(phase) + ": null pointer argument");
  if (!aligned(q, 16) || !aligned(kp, 8) || !aligned(vp, 8) || !aligned(out, 8))
    return fail(SLMT_ERR_INVALID, std::string(phase) + ": q must be 16-byte, packed KV and out 8-byte aligned");
  return SLMT_OK;
}

// Rows of `dim` elements of 2 bytes: element (t, h, d) at base + t * token + h * head + d.
struct Rows {
  const void* base;
  int64_t token, head;
  int tokens, heads, dim;
  Rows merged() const { return head == dim ? Rows{base, token, 0, tokens, 1, heads * dim} : *this; }   // (heads side by side)
  // one element past the last, in elements from the base
  int64_t end() const { return (tokens - 1) * token + (heads - 1) * head + dim; }
  bool dense() const { return end() == (int64_t)tokens * heads * dim; }
  // whether a row of a head lies among elements lo .. hi - 1 from the base
  bool within(int64_t lo, int64_t hi) const {
    for (int h = 0; h < heads; ++h) {
      const int64_t at = lo - h * head;
      const int64_t t = at >= dim && token > 0 ? (at - dim) / token + 1 : 0;   // the first one that ends past lo
      if (t < tokens && t * token + dim > at && t * token + h * head < hi) return true;
    }
    return false;
  }
};
// Whether two tensors share elements.  (Exact where one of them has no gaps or both have the same token stride, as parts of one
// buffer have; other layouts are taken not to.)
bool share(const Rows& a, const Rows& b) {
  const Rows x = a.merged(), y = b.merged();
  if (!x.tokens || !y.tokens) return false;
  const int64_t apart = (int64_t)((uintptr_t)y.base - (uintptr_t)x.base) >> 1;
  if (apart >= x.end() || -apart >= y.end()) return false;
  if (x.dense()) return y.within(-apart, x.end() - apart);
  if (y.dense()) return x.within(apart, y.end() + apart);
  const int64_t token = x.tokens > 1 ? x.token : y.token;
  if (token <= 0 || (x.tokens > 1 && y.tokens > 1 && x.token != y.token)) return false;
  for (int h = 0; h < x.heads; ++h)
    for (int g = 0; g < y.heads; ++g) {
      // row u of y starts at - (t - u) token behind row t of x: before that one's end, and its own is past that one's start
      const int64_t at = apart + g * y.head - h * x.head;
      int64_t d = at >= 0 ? at / token : -((token - 1 - at) / token);        // t - u: floor(at / token), and one more
      for (int i = 0; i < 2; ++i, ++d)
        if (d < x.tokens && -d < y.tokens && at - d * token < x.dim && d * token - at < y.dim) return true;
    }
  return false;
}

int check_workspace(const char* phase, int B, int H, int KV, int D, const void* ws, int64_t ws_bytes) {
  const int64_t need = attention_workspace_bytes(B, H, KV, D);
  if (need < 0) return last_status();
  if (!ws || ws_bytes < need)
    return fail(SLMT_ERR_INVALID, std::string(phase) + ": workspace of " + s(need) + " bytes required, got " + s(ws_bytes));
  return SLMT_OK;
}

}  // namespace

int decode_paged_batched(const void* q, int64_t q_seq_stride, int64_t q_head_stride, const void* kv_cache,
                         int64_t num_blocks, int block_size, const void* block_tables, int block_table_bits,
                         int64_t block_table_stride, const int32_t* seq_lens, int fixed_seq_len, int num_seqs,
                         int num_heads, int num_kv_heads, int head_dim, void* out, int out_dtype,
                         int64_t out_seq_stride, int64_t out_head_stride, void* workspace, int64_t workspace_bytes,
                         hipStream_t stream, bool clear_counters) {
  const char* ph = "paged decode";
  if (!head_dim_ok(head_dim)) return fail(SLMT_ERR_INVALID, "paged decode: head_dim must be 64/80/128, got " + s(head_dim));
  if (num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0)
    return fail(SLMT_ERR_INVALID, "H not divisible by num_kv_heads");
  if (block_size <= 0) return fail(SLMT_ERR_INVALID, "paged decode: block_size must be positive, got " + s(block_size));
  if (block_table_bits != 32 && block_table_bits != 64)
    return fail(SLMT_ERR_INVALID, "paged decode: block table must be int32 or int64");
  if (out_dtype != SLMT_OUT_F32 && out_dtype != SLMT_OUT_F16)
    return fail(SLMT_ERR_INVALID, "paged decode: out dtype must be fp32 or fp16");
  if (num_seqs < 0) return fail(SLMT_ERR_INVALID, "paged decode: num_seqs must be >= 0");
  if (!seq_lens && fixed_seq_len < 0) return fail(SLMT_ERR_INVALID, "paged decode: seq_len must be >= 0");
  if (num_seqs == 0) return SLMT_OK;
  if (!q || !kv_cache || !block_tables || !out) return fail(SLMT_ERR_INVALID, "paged decode: null pointer argument");
  if (!aligned(q, 16) || (q_seq_stride % 8) || (q_head_stride % 8))
    return fail(SLMT_ERR_INVALID, "paged decode: q must be 16-byte aligned with strides that are multiples of 8");
  if (!aligned(out, out_dtype == SLMT_OUT_F32 ? 8 : 4) || (out_seq_stride & 1) || (out_head_stride & 1))
    return fail(SLMT_ERR_INVALID, "paged decode: out must be aligned with even strides");
  if (!aligned(kv_cache, 8)) return fail(SLMT_ERR_INVALID, "paged decode: kv_cache must be 8-byte aligned");
  int rc = check_workspace(ph, num_seqs, num_heads, num_kv_heads, head_dim, workspace, workspace_bytes);
  if (rc != SLMT_OK) return rc;
  AttnParams p = blank_params();
  p.q = reinterpret_cast<const uint16_t*>(q);
  p.q_seq_stride = q_seq_stride;
  p.q_head_stride = q_head_stride;
  p.cache = reinterpret_cast<const uint8_t*>(kv_cache);
  p.block_tables = block_tables;
  p.bt_stride = block_table_stride;
  p.bt64 = block_table_bits == 64;
  p.block_size = block_size;
  p.block_shift = block_shift_of(block_size);
  p.cache_kv = num_kv_heads;
  p.num_blocks = num_blocks;
  p.seq_lens = seq_lens;
  p.fixed_len = fixed_seq_len;
  p.B = num_seqs;
  p.H = num_heads;
  p.G = num_heads / num_kv_heads;
  p.out = out;
  p.out_f16 = out_dtype == SLMT_OUT_F16;
  p.out_seq_stride = out_seq_stride;
  p.out_head_stride = out_head_stride;
  return launch_attention(SRC_PAGED, head_dim, p, workspace, workspace_bytes, stream, clear_counters);
}

}  // namespace slmt

using namespace slmt;

extern "C" {

const char* slmt_last_error(void) { return g_error.c_str(); }

int slmt_abi_version(void) { return SLMT_ABI_VERSION; }

int64_t slmt_attention_workspace_bytes(int num_seqs, int num_heads, int num_kv_heads, int head_dim) {
  clear_error();
  if (!head_dim_ok(head_dim)) return fail(SLMT_ERR_INVALID, "workspace: head_dim must be 64/80/128, got " + s(head_dim)), -1;
  return attention_workspace_bytes(num_seqs, num_heads, num_kv_heads, head_dim);
}

int slmt_quantize_store(const void* key, int64_t key_token_stride, const void* value,
                        int64_t value_token_stride, void* kv_cache, int64_t num_blocks,
                        int block_size, const int64_t* slot_mapping, int64_t num_tokens,
                        int num_kv_heads, int head_dim, slmt_stream_t stream) {
  clear_error();
  if (!head_dim_ok(head_dim)) return fail(SLMT_ERR_INVALID, "store: head_dim must be 64/80/128, got " + s(head_dim));
  if (num_tokens < 0 || num_kv_heads <= 0 || block_size <= 0 || num_blocks < 0)
    return fail(SLMT_ERR_INVALID, "store: invalid sizes (N=" + s(num_tokens) + ", KV=" + s(num_kv_heads) +
                                      ", block_size=" + s(block_size) + ")");
  if (num_tokens == 0) return SLMT_OK;
  if (!key || !value || !kv_cache || !slot_mapping) return fail(SLMT_ERR_INVALID, "store: null pointer argument");
  if (key_token_stride < (int64_t)num_kv_heads * head_dim || value_token_stride < (int64_t)num_kv_heads * head_dim)
    return fail(SLMT_ERR_INVALID, "store: token stride smaller than KV*D");
  if ((key_token_stride & 1) || (value_token_stride & 1) || !aligned(key, 4) || !aligned(value, 4) ||
      !aligned(kv_cache, 8))
    return fail(SLMT_ERR_INVALID, "store: key/value rows must be 4-byte aligned and the cache 8-byte aligned");
  return launch_quantize_store(key, key_token_stride, value, value_token_stride, kv_cache,
                               num_blocks * (int64_t)block_size, slot_mapping, num_tokens,
                               num_kv_heads, head_dim, reinterpret_cast<hipStream_t>(stream));
}

static int quantize_per_channel(int nt, const void* const* x, int num_kv_heads, int seq_len, int head_dim,
                                void* const* packed, void* const* scale, void* const* zero, slmt_stream_t stream) {
  clear_error();
  if (!head_dim_ok(head_dim))
    return fail(SLMT_ERR_INVALID, "quantize: head_dim must be 64/80/128, got " + s(head_dim));
  if (num_kv_heads < 0 || seq_len <= 0)
    return fail(SLMT_ERR_INVALID, "quantize: need KV >= 0 and S >= 1 (got KV=" + s(num_kv_heads) + ", S=" + s(seq_len) + ")");
  if (num_kv_heads == 0) return SLMT_OK;
  for (int i = 0; i < nt; ++i) {
    if (!x[i] || !packed[i] || !scale[i] || !zero[i]) return fail(SLMT_ERR_INVALID, "quantize: null pointer argument");
    if (!aligned(x[i], 4) || !aligned(scale[i], 2) || !aligned(zero[i], 2))
      return fail(SLMT_ERR_INVALID, "quantize: x must be 4-byte aligned");
  }
  return launch_quantize_per_channel(nt, x, num_kv_heads, seq_len, head_dim, packed, scale, zero,
                                     reinterpret_cast<hipStream_t>(stream));
}

int slmt_quantize_per_channel(const void* x, int num_kv_heads, int seq_len, int head_dim, void* packed,
                              void* scale, void* zero, slmt_stream_t stream) {
  return quantize_per_channel(1, &x, num_kv_heads, seq_len, head_dim, &packed, &scale, &zero, stream);
}

int slmt_quantize_kv_per_channel(const void* k, const void* v, int num_kv_heads, int seq_len, int head_dim,
                                 void* k_packed, void* k_scale, void* k_zero, void* v_packed, void* v_scale,
                                 void* v_zero, slmt_stream_t stream) {
  const void* x[2] = {k, v};
  void *packed[2] = {k_packed, v_packed}, *scale[2] = {k_scale, v_scale}, *zero[2] = {k_zero, v_zero};
  return quantize_per_channel(2, x, num_kv_heads, seq_len, head_dim, packed, scale, zero, stream);
}

int slmt_quantize_with_rulers(const void* x, int64_t x_head_stride, int64_t x_seq_stride, int num_kv_heads,
                              int seq_len, int head_dim, const void* scale, const void* zero, void* packed,
                              int64_t out_head_stride, int64_t out_seq_stride, slmt_stream_t stream) {
  clear_error();
  if (!head_dim_ok(head_dim))
    return fail(SLMT_ERR_INVALID, "quantize_tensor: head_dim must be 64/80/128, got " + s(head_dim));
  if (num_kv_heads < 0 || seq_len < 0)
    return fail(SLMT_ERR_INVALID, "quantize_tensor: need KV >= 0 and S >= 0");
  if (num_kv_heads == 0 || seq_len == 0) return SLMT_OK;
  if (!x || !scale || !zero || !packed) return fail(SLMT_ERR_INVALID, "quantize_tensor: null pointer argument");
  if ((x_head_stride & 1) || (x_seq_stride & 1) || !aligned(x, 4) || !aligned(scale, 4) || !aligned(zero, 4))
    return fail(SLMT_ERR_INVALID, "quantize_tensor: x rows and the rulers must be 4-byte aligned (even strides)");
  if ((seq_len > 1 && (x_seq_stride < head_dim || out_seq_stride < head_dim / 2)) ||
      (num_kv_heads > 1 && (x_head_stride < head_dim || out_head_stride < head_dim / 2)))
    return fail(SLMT_ERR_INVALID, "quantize_tensor: strides smaller than a row");
  return launch_quantize_rulers(x, x_head_stride, x_seq_stride, num_kv_heads, seq_len, head_dim, scale, zero,
                                packed, out_head_stride, out_seq_stride, reinterpret_cast<hipStream_t>(stream));
}

int slmt_decode_paged_batched(const void* q, int64_t q_seq_stride, int64_t q_head_stride,
                              const void* kv_cache, int64_t num_blocks, int block_size,
                              const void* block_tables, int block_table_bits, int64_t block_table_stride,
                              const int32_t* seq_lens, int fixed_seq_len, int num_seqs, int num_heads,
                              int num_kv_heads, int head_dim, void* out, int out_dtype,
                              int64_t out_seq_stride, int64_t out_head_stride, void* workspace,
                              int64_t workspace_bytes, slmt_stream_t stream) {
  clear_error();
  return decode_paged_batched(q, q_seq_stride, q_head_stride, kv_cache, num_blocks, block_size, block_tables,
                              block_table_bits, block_table_stride, seq_lens, fixed_seq_len, num_seqs, num_heads,
                              num_kv_heads, head_dim, out, out_dtype, out_seq_stride, out_head_stride, workspace,
                              workspace_bytes, reinterpret_cast<hipStream_t>(stream), false);
}

int64_t slmt_chunk_workspace_bytes(int64_t num_tokens, int num_reqs, int num_heads, int num_kv_heads, int head_dim,
                                   int max_seq_len) {
  clear_error();
  if (!head_dim_ok(head_dim)) return fail(SLMT_ERR_INVALID, "workspace: head_dim must be 64/80/128, got " + s(head_dim)), -1;
  if (num_tokens < 0 || num_reqs < 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0)
    return fail(SLMT_ERR_INVALID, "workspace: invalid sizes"), -1;
  return chunk_workspace_bytes(num_tokens, num_reqs, num_heads, num_kv_heads, head_dim, max_seq_len);
}

int slmt_chunk_paged(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* kv_cache,
                     int64_t num_blocks, int block_size, const void* block_tables, int block_table_bits,
                     int64_t block_table_stride, const int32_t* query_start_loc, const int32_t* seq_lens,
                     int max_seq_len, int num_tokens, int num_reqs, int num_heads, int num_kv_heads, int head_dim,
                     void* out, int out_dtype, int64_t out_token_stride, int64_t out_head_stride, void* workspace,
                     int64_t workspace_bytes, slmt_stream_t stream) {
  clear_error();
  if (!head_dim_ok(head_dim)) return fail(SLMT_ERR_INVALID, "chunk: head_dim must be 64/80/128, got " + s(head_dim));
  if (num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0)
    return fail(SLMT_ERR_INVALID, "H not divisible by num_kv_heads");
  const int shift = block_shift_of(block_size);
  if (shift < 4) return fail(SLMT_ERR_INVALID, "chunk: block_size must be a power of two of at least 16, got " + s(block_size));
  if (block_table_bits != 32 && block_table_bits != 64)
    return fail(SLMT_ERR_INVALID, "chunk: block table must be int32 or int64");
  if (out_dtype != SLMT_OUT_F32 && out_dtype != SLMT_OUT_F16)
    return fail(SLMT_ERR_INVALID, "chunk: out dtype must be fp32 or fp16");
  if (num_tokens < 0 || num_reqs < 0 || num_blocks < 0 || num_blocks >= (int64_t(1) << 31))
    return fail(SLMT_ERR_INVALID, "chunk: invalid sizes");
  if ((int64_t)num_tokens * (num_heads / num_kv_heads) >= (int64_t(1) << 31) - 64)
    return fail(SLMT_ERR_UNSUPPORTED, "chunk: too many query rows for one launch");
  if (num_tokens == 0 || num_reqs == 0) return SLMT_OK;
  if (!q || !kv_cache || !block_tables || !query_start_loc || !seq_lens || !out)
    return fail(SLMT_ERR_INVALID, "chunk: null pointer argument");
  if (!aligned(q, 16) || (q_token_stride % 8) || (q_head_stride % 8))
    return fail(SLMT_ERR_INVALID, "chunk: q must be 16-byte aligned with strides that are multiples of 8");
  if (!aligned(out, out_dtype == SLMT_OUT_F32 ? 8 : 4) || (out_token_stride & 1) || (out_head_stride & 1))
    return fail(SLMT_ERR_INVALID, "chunk: out must be aligned with even strides");
  if (!aligned(kv_cache, 8)) return fail(SLMT_ERR_INVALID, "chunk: kv_cache must be 8-byte aligned");
  ChunkParams p{};
  p.q = reinterpret_cast<const uint16_t*>(q);
  p.q_seq_stride = q_token_stride;
  p.q_head_stride = q_head_stride;
  p.cache = reinterpret_cast<const uint8_t*>(kv_cache);
  p.block_tables = block_tables;
  p.bt_stride = block_table_stride;
  p.bt64 = block_table_bits == 64;
  p.block_shift = shift;
  p.query_start = query_start_loc;
  p.seq_lens = seq_lens;
  p.N = num_tokens;
  p.R = num_reqs;
  p.G = num_heads / num_kv_heads;
  p.KV = num_kv_heads;
  p.out = out;
  p.out_f16 = out_dtype == SLMT_OUT_F16;
  p.out_seq_stride = out_token_stride;
  p.out_head_stride = out_head_stride;
  return launch_chunk(head_dim, p, max_seq_len, workspace, workspace_bytes, reinterpret_cast<hipStream_t>(stream));
}

int slmt_decode_paged(const void* q, const void* kv_cache, int64_t num_blocks, int block_size,
                      const int64_t* block_table, int seq_len, int num_heads, int num_kv_heads,
                      int head_dim, float* out, void* workspace, int64_t workspace_bytes,
                      slmt_stream_t stream) {
  // One request = a batch of one with a fixed length and an int64 block row.
  if (seq_len < 0) {
    clear_error();
    return fail(SLMT_ERR_INVALID, "paged decode: seq_len must be >= 0");
  }
  return slmt_decode_paged_batched(q, (int64_t)num_heads * head_dim, head_dim, kv_cache, num_blocks,
                                   block_size, block_table, 64, 0, nullptr, seq_len, 1, num_heads,
                                   num_kv_heads, head_dim, out, SLMT_OUT_F32,
                                   (int64_t)num_heads * head_dim, head_dim, workspace, workspace_bytes,
                                   stream);
}

int slmt_decode_per_token(const void* q, const void* k_packed, const void* k_min, const void* k_step,
                          const void* v_packed, const void* v_min, const void* v_step, int num_heads,
                          int kv_tensor_heads, int num_kv_heads, int seq_len, int head_dim, int block_n,
                          float* out, void* workspace, int64_t workspace_bytes, slmt_stream_t stream) {
  clear_error();
  const char* ph = "per-token decode";
  if (block_n != 32 && block_n != 64)
    return fail(SLMT_ERR_INVALID, "per-token decode: BLOCK_N must be 32 or 64, got " + s(block_n));
  const void* r[4] = {k_min, k_step, v_min, v_step};
  int rc = check_contig(ph, q, k_packed, v_packed, r, num_heads, kv_tensor_heads, num_kv_heads, seq_len, head_dim, out);
  if (rc != SLMT_OK) return rc;
  rc = check_workspace(ph, 1, num_heads, num_kv_heads, head_dim, workspace, workspace_bytes);
  if (rc != SLMT_OK) return rc;
  // one short sequence: split over (KV head, key chunk) when the shape allows it
  rc = launch_decode_split(true, q, k_packed, v_packed, r, num_heads, num_heads / num_kv_heads, seq_len, head_dim, 1,
                           out, workspace, workspace_bytes, reinterpret_cast<hipStream_t>(stream));
  if (rc != SLMT_ERR_UNSUPPORTED) return rc;
  AttnParams p = blank_params();
  p.q = reinterpret_cast<const uint16_t*>(q);
  p.q_seq_stride = (int64_t)num_heads * head_dim;
  p.q_head_stride = head_dim;
  p.kp = reinterpret_cast<const uint8_t*>(k_packed);
  p.vp = reinterpret_cast<const uint8_t*>(v_packed);
  p.kr0 = reinterpret_cast<const uint16_t*>(k_min);
  p.kr1 = reinterpret_cast<const uint16_t*>(k_step);
  p.vr0 = reinterpret_cast<const uint16_t*>(v_min);
  p.vr1 = reinterpret_cast<const uint16_t*>(v_step);
  p.s_rows = seq_len;
  p.fixed_len = seq_len;
  p.B = 1;
  p.H = num_heads;
  p.G = num_heads / num_kv_heads;
  p.out = out;
  p.out_seq_stride = (int64_t)num_heads * head_dim;
  p.out_head_stride = head_dim;
  return launch_attention(SRC_TOKEN, head_dim, p, workspace, workspace_bytes, reinterpret_cast<hipStream_t>(stream));
}

int slmt_decode_per_channel(const void* q, const void* k_packed, const void* k_scale, const void* k_zero,
                            const void* v_packed, const void* v_scale, const void* v_zero, int num_heads,
                            int kv_tensor_heads, int num_kv_heads, int seq_len, int head_dim, int block_n,
                            int use_quant, float* out, void* workspace, int64_t workspace_bytes,
                            slmt_stream_t stream) {
  clear_error();
  const char* ph = "kv_dequant_decode";
  if (block_n != 32 && block_n != 64)
    return fail(SLMT_ERR_INVALID, "kv_dequant_decode: BLOCK_N must be 32 or 64, got " + s(block_n));
  const void* r[4] = {k_scale, k_zero, v_scale, v_zero};
  int rc = check_contig(ph, q, k_packed, v_packed, r, num_heads, kv_tensor_heads, num_kv_heads, seq_len, head_dim, out);
  if (rc != SLMT_OK) return rc;
  rc = check_workspace(ph, 1, num_heads, num_kv_heads, head_dim, workspace, workspace_bytes);
  if (rc != SLMT_OK) return rc;
  // one short sequence: split over (KV head, key chunk) when the shape allows it
  rc = launch_decode_split(false, q, k_packed, v_packed, r, num_heads, num_heads / num_kv_heads, seq_len, head_dim,
                           use_quant, out, workspace, workspace_bytes, reinterpret_cast<hipStream_t>(stream));
  if (rc != SLMT_ERR_UNSUPPORTED) return rc;
  AttnParams p = blank_params();
  p.q = reinterpret_cast<const uint16_t*>(q);
  p.q_seq_stride = (int64_t)num_heads * head_dim;
  p.q_head_stride = head_dim;
  p.kp = reinterpret_cast<const uint8_t*>(k_packed);
  p.vp = reinterpret_cast<const uint8_t*>(v_packed);
  p.kr0 = reinterpret_cast<const uint16_t*>(k_scale);
  p.kr1 = reinterpret_cast<const uint16_t*>(k_zero);
  p.vr0 = reinterpret_cast<const uint16_t*>(v_scale);
  p.vr1 = reinterpret_cast<const uint16_t*>(v_zero);
  p.use_quant = use_quant ? 1 : 0;
  p.s_rows = seq_len;
  p.fixed_len = seq_len;
  p.B = 1;
  p.H = num_heads;
  p.G = num_heads / num_kv_heads;
  p.out = out;
  p.out_seq_stride = (int64_t)num_heads * head_dim;
  p.out_head_stride = head_dim;
  return launch_attention(SRC_CHANNEL, head_dim, p, workspace, workspace_bytes, reinterpret_cast<hipStream_t>(stream));
}

int slmt_prefill_per_channel(const void* q, const void* k_packed, const void* k_scale, const void* k_zero,
                             const void* v_packed, const void* v_scale, const void* v_zero, int num_heads,
                             int kv_tensor_heads, int num_kv_heads, int num_queries, int seq_len, int head_dim,
                             int block_m, int block_n, int causal, int use_quant, float* out, void* workspace,
                             int64_t workspace_bytes, slmt_stream_t stream) {
  clear_error();
  const char* ph = "kv_dequant_prefill";
  if (block_m != 16 && block_m != 32)
    return fail(SLMT_ERR_INVALID, "kv_dequant_prefill: BLOCK_M must be 16 or 32, got " + s(block_m));
  if (block_n != 32 && block_n != 64)
    return fail(SLMT_ERR_INVALID, "kv_dequant_prefill: BLOCK_N must be 32 or 64, got " + s(block_n));
  const bool combo_ok = (block_m == 16 && block_n == 32) || head_dim == 64;
  if (!combo_ok)
    return fail(SLMT_ERR_INVALID, "kv_dequant_prefill: (BLOCK_M=" + s(block_m) + ", BLOCK_N=" + s(block_n) +
                                      ") does not fit the 48 KB shared budget for head_dim=" + s(head_dim) +
                                      ". Use BLOCK_M=16, BLOCK_N=32 for D>=80.");
  const void* r[4] = {k_scale, k_zero, v_scale, v_zero};
  int rc = check_contig(ph, q, k_packed, v_packed, r, num_heads, kv_tensor_heads, num_kv_heads, seq_len, head_dim, out);
  if (rc != SLMT_OK) return rc;
  if (num_queries < 0) return fail(SLMT_ERR_INVALID, "kv_dequant_prefill: M must be >= 0");
  if (num_queries == 0) return SLMT_OK;
  if (head_dim == 80) {   // its documented argument, though the kernel uses none of it
    rc = check_workspace(ph, num_queries, num_heads, num_kv_heads, head_dim, workspace, workspace_bytes);
    if (rc != SLMT_OK) return rc;
  }
  return launch_prefill_mfma(q, k_packed, k_scale, k_zero, v_packed, v_scale, v_zero, num_heads,
                             num_heads / num_kv_heads, num_queries, seq_len, head_dim, causal, use_quant, out,
                             reinterpret_cast<hipStream_t>(stream));
}

int slmt_step_metadata(const int32_t* query_lens, const int32_t* context_lens, int num_reqs, void* block_tables,
                       int block_table_bits, int64_t block_table_stride, int max_blocks, const void* free_blocks,
                       int num_free, const int32_t* free_start, int block_size, int num_tokens,
                       int32_t* query_start_loc, int32_t* seq_lens, int64_t* positions, int64_t* slot_mapping,
                       int32_t* free_end, slmt_stream_t stream) {
  clear_error();
  if (num_reqs < 0 || max_blocks < 0 || num_free < 0 || num_tokens < 0 || num_tokens > 0x7fffffff - 1024)
    return fail(SLMT_ERR_INVALID, "step metadata: invalid sizes (requests=" + s(num_reqs) + ", max_blocks=" +
                                      s(max_blocks) + ", free blocks=" + s(num_free) + ", tokens=" + s(num_tokens) + ")");
  if (block_size <= 0) return fail(SLMT_ERR_INVALID, "step metadata: block_size must be positive, got " + s(block_size));
  if (block_table_bits != 32 && block_table_bits != 64)
    return fail(SLMT_ERR_INVALID, "step metadata: block table must be int32 or int64");
  if (num_reqs > 1 && block_table_stride < max_blocks)
    return fail(SLMT_ERR_INVALID, "step metadata: block table rows overlap");
  if (!query_start_loc || !free_end || (num_tokens && (!positions || !slot_mapping)) ||
      (num_reqs && (!query_lens || !context_lens || !seq_lens)) || (num_reqs && max_blocks && !block_tables) ||
      (num_free && !free_blocks))
    return fail(SLMT_ERR_INVALID, "step metadata: null pointer argument");
  // Workgroups read the inputs and the tables' old columns for themselves while others write: nothing written may lie among what
  // is read, or among what else is written.
  struct Range { const void* p; int64_t bytes; };
  const int64_t R = num_reqs, N = num_tokens, entry = block_table_bits / 8;
  const Range reads[] = {{query_lens, 4 * R}, {context_lens, 4 * R}, {free_blocks, num_free * entry}, {free_start, 4}};
  const Range writes[] = {{query_start_loc, 4 * (R + 1)}, {seq_lens, 4 * R}, {positions, 8 * N}, {slot_mapping, 8 * N},
                          {free_end, 4}};
  auto meet = [](const Range& x, const Range& y) {
    const uintptr_t a = (uintptr_t)x.p, b = (uintptr_t)y.p;
    return a && b && x.bytes && y.bytes && a < b + (uintptr_t)y.bytes && b < a + (uintptr_t)x.bytes;
  };
  auto in_tables = [&](const Range& x) {     // (between a row's columns and the next row there may be anything)
    const int64_t at = (int64_t)((uintptr_t)x.p - (uintptr_t)block_tables), row = max_blocks * entry, step = block_table_stride * entry;
    if (!x.p || !x.bytes || !block_tables || !R || !row) return false;
    const int64_t r = at >= row && R > 1 ? (at - row) / step + 1 : 0;    // the first row that ends past x's start
    return r < R && r * step + row > at && r * step < at + x.bytes;
  };
  for (const Range& w : writes)
    for (const Range& r : reads)
      if (meet(w, r)) return fail(SLMT_ERR_INVALID, "step metadata: an output overlaps an input");
  for (const Range& r : reads)
    if (in_tables(r)) return fail(SLMT_ERR_INVALID, "step metadata: an input overlaps the block tables");
  for (const Range& w : writes)
    if (in_tables(w)) return fail(SLMT_ERR_INVALID, "step metadata: an output overlaps the block tables");
  for (const Range& w : writes)
    for (const Range& x : writes)
      if (&w < &x && meet(w, x)) return fail(SLMT_ERR_INVALID, "step metadata: outputs overlap");
  return launch_step_metadata(query_lens, context_lens, num_reqs, block_tables, block_table_bits == 64,
                              block_table_stride, max_blocks, free_blocks, num_free, free_start, block_size, num_tokens,
                              query_start_loc, seq_lens, positions, slot_mapping, free_end,
                              reinterpret_cast<hipStream_t>(stream));
}

static int check_rotary(const char* ph, const RotaryParams& r, int D, int position_bits) {
  const std::string phase(ph);
  if (!head_dim_ok(D)) return fail(SLMT_ERR_INVALID, phase + ": head_dim must be 64/80/128, got " + s(D));
  if (r.N < 0 || r.H < 0 || r.KV < 0 || (int64_t)r.H + r.KV > 65536)
    return fail(SLMT_ERR_INVALID, phase + ": invalid sizes (N=" + s(r.N) + ", H=" + s(r.H) + ", KV=" + s(r.KV) + ")");
  if (r.rotary_dim < 2 || r.rotary_dim > D || (r.rotary_dim & 1))
    return fail(SLMT_ERR_INVALID, phase + ": rotary_dim must be even and at most head_dim, got " + s(r.rotary_dim));
  if (position_bits != 32 && position_bits != 64)
    return fail(SLMT_ERR_INVALID, phase + ": positions must be int32 or int64");
  if (r.N == 0) return SLMT_OK;
  if ((r.H && (!r.q || !r.q_out)) || !r.positions || !r.inv_freq)
    return fail(SLMT_ERR_INVALID, phase + ": null pointer argument");
  return SLMT_OK;
}

int slmt_rotary(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k, int64_t k_token_stride,
                int64_t k_head_stride, void* q_out, int64_t q_out_token_stride, int64_t q_out_head_stride, void* k_out,
                int64_t k_out_token_stride, int64_t k_out_head_stride, int num_tokens, int num_heads, int num_kv_heads,
                int head_dim, int dtype, const void* positions, int position_bits, const float* inv_freq,
                int rotary_dim, int interleaved, double scale, slmt_stream_t stream) {
  clear_error();
  RotaryParams r{q, k, nullptr, q_out, k_out, q_token_stride, q_head_stride, k_token_stride, k_head_stride, 0, 0,
                 q_out_token_stride, q_out_head_stride, k_out_token_stride, k_out_head_stride, num_tokens, num_heads,
                 num_kv_heads, positions, position_bits == 64, inv_freq, rotary_dim, interleaved ? 1 : 0, scale,
                 nullptr, 0, nullptr};
  const int rc = check_rotary("rotary", r, head_dim, position_bits);
  if (rc != SLMT_OK) return rc;
  if (dtype != SLMT_F32 && dtype != SLMT_F16 && dtype != SLMT_BF16)
    return fail(SLMT_ERR_INVALID, "rotary: dtype must be fp32, fp16 or bf16");
  if (num_tokens == 0) return SLMT_OK;
  if (num_kv_heads && (!k || !k_out)) return fail(SLMT_ERR_INVALID, "rotary: null pointer argument");
  if (num_kv_heads == 0) r.k = nullptr;
  return launch_rotary(head_dim, dtype, r, reinterpret_cast<hipStream_t>(stream));
}

int slmt_rotary_quantize_store(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* key,
                               int64_t key_token_stride, int64_t key_head_stride, const void* value,
                               int64_t value_token_stride, int64_t value_head_stride, void* q_out,
                               int64_t q_out_token_stride, int64_t q_out_head_stride, void* key_out,
                               int64_t key_out_token_stride, int64_t key_out_head_stride, void* kv_cache,
                               int64_t num_blocks, int block_size, const int64_t* slot_mapping, int num_tokens,
                               int num_heads, int num_kv_heads, int head_dim, const void* positions,
                               int position_bits, const float* inv_freq, int rotary_dim, int interleaved,
                               double scale, slmt_stream_t stream) {
  clear_error();
  RotaryParams r{q, key, value, q_out, key_out, q_token_stride, q_head_stride, key_token_stride, key_head_stride,
                 value_token_stride, value_head_stride, q_out_token_stride, q_out_head_stride, key_out_token_stride,
                 key_out_head_stride, num_tokens, num_heads, num_kv_heads, positions, position_bits == 64, inv_freq,
                 rotary_dim, interleaved ? 1 : 0, scale, reinterpret_cast<uint8_t*>(kv_cache),
                 num_blocks * (int64_t)block_size, slot_mapping};
  const int rc = check_rotary("rotary store", r, head_dim, position_bits);
  if (rc != SLMT_OK) return rc;
  if (num_kv_heads <= 0 || block_size <= 0 || num_blocks < 0)
    return fail(SLMT_ERR_INVALID, "rotary store: invalid sizes (KV=" + s(num_kv_heads) + ", block_size=" + s(block_size) + ")");
  if (num_tokens == 0) return SLMT_OK;
  if (!key || !value || !kv_cache || !slot_mapping) return fail(SLMT_ERR_INVALID, "rotary store: null pointer argument");
  if (!aligned(kv_cache, 8)) return fail(SLMT_ERR_INVALID, "rotary store: the cache must be 8-byte aligned");
  return launch_rotary(head_dim, SLMT_F16, r, reinterpret_cast<hipStream_t>(stream));
}

int slmt_prompt_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k,
                          int64_t k_token_stride, int64_t k_head_stride, const void* v, int64_t v_token_stride,
                          int64_t v_head_stride, const int32_t* query_start_loc, const int32_t* key_start_loc,
                          int num_seqs, int num_tokens, int num_keys, int num_heads, int num_kv_heads, int head_dim,
                          int dtype, int causal, double scale, void* out, int64_t out_token_stride,
                          int64_t out_head_stride, int clear_rest, void* workspace, int64_t workspace_bytes,
                          slmt_stream_t stream) {
  clear_error();
  if (!head_dim_ok(head_dim)) return fail(SLMT_ERR_INVALID, "prompt attention: head_dim must be 64/80/128, got " + s(head_dim));
  if (num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0)
    return fail(SLMT_ERR_INVALID, "H not divisible by num_kv_heads");
  if (dtype != SLMT_F16 && dtype != SLMT_BF16)
    return fail(SLMT_ERR_INVALID, "prompt attention: dtype must be fp16 or bf16");
  if (num_seqs < 0 || num_tokens < 0 || num_keys < 0) return fail(SLMT_ERR_INVALID, "prompt attention: invalid sizes");
  // (times log2(e) it is fp32's: of a scale that is 0 there, a masked score's -infinity would make no number)
  if (!(scale >= 1.0e-38 && scale <= 3.0e38 / 1.4427))
    return fail(SLMT_ERR_INVALID, "prompt attention: scale must be positive and finite, from 1e-38 to 2e38");
  if (num_seqs == 0 || num_tokens == 0) return SLMT_OK;
  if (!q || !out || !query_start_loc || (num_keys && (!k || !v)))
    return fail(SLMT_ERR_INVALID, "prompt attention: null pointer argument");
  if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || ((q_token_stride | q_head_stride | k_token_stride |
      k_head_stride | v_token_stride | v_head_stride) & 7))
    return fail(SLMT_ERR_INVALID, "prompt attention: q, k and v must be 16-byte aligned with strides that are multiples of 8");
  if (!aligned(out, 8) || ((out_token_stride | out_head_stride) & 3))
    return fail(SLMT_ERR_INVALID, "prompt attention: out must be 8-byte aligned with strides that are multiples of 4");
  if (!aligned(workspace, 4)) return fail(SLMT_ERR_INVALID, "prompt attention: the workspace must be 4-byte aligned");
  if (out == k || out == v) return fail(SLMT_ERR_INVALID, "prompt attention: out must not be k or v");
  const Rows o{out, out_token_stride, out_head_stride, num_tokens, num_heads, head_dim};
  if (share(o, Rows{k, k_token_stride, k_head_stride, num_keys, num_kv_heads, head_dim}) ||
      share(o, Rows{v, v_token_stride, v_head_stride, num_keys, num_kv_heads, head_dim}))
    return fail(SLMT_ERR_INVALID, "prompt attention: out overlaps k or v");
  const bool itself = out == q && (num_tokens == 1 || out_token_stride == q_token_stride) &&
                      (num_heads == 1 || out_head_stride == q_head_stride);
  if (!itself && share(o, Rows{q, q_token_stride, q_head_stride, num_tokens, num_heads, head_dim}))
    return fail(SLMT_ERR_INVALID, "prompt attention: out must be q itself or not overlap it");
  if (k_token_stride < 0 || v_token_stride < 0 || k_token_stride >= (1 << 28) || v_token_stride >= (1 << 28))
    return fail(SLMT_ERR_UNSUPPORTED, "prompt attention: token strides of k and v must be below 2^28 elements");
  PromptParams p{q, k, v, out, q_token_stride, q_head_stride, k_token_stride, k_head_stride, v_token_stride,
                 v_head_stride, out_token_stride, out_head_stride, query_start_loc,
                 key_start_loc ? key_start_loc : query_start_loc, num_seqs, num_tokens, num_keys, num_heads,
                 num_kv_heads, causal ? 1 : 0, clear_rest ? 1 : 0, (float)(scale * 1.4426950408889634)};
  return launch_prompt(head_dim, dtype, p, workspace, workspace_bytes, reinterpret_cast<hipStream_t>(stream));
}

int64_t slmt_prompt_workspace_bytes(int num_tokens, int num_keys, int num_seqs, int num_heads, int head_dim) {
  clear_error();
  if (!head_dim_ok(head_dim)) return fail(SLMT_ERR_INVALID, "prompt attention: head_dim must be 64/80/128, got " + s(head_dim)), -1;
  if (num_heads <= 0 || num_seqs < 0 || num_tokens < 0 || num_keys < 0)
    return fail(SLMT_ERR_INVALID, "prompt attention: invalid sizes"), -1;
  return prompt_workspace_bytes(head_dim, num_tokens, num_keys, num_seqs, num_heads);
}

static int check_sample(int num_rows, int vocab) {
  if (num_rows < 0 || vocab <= 0)
    return fail(SLMT_ERR_INVALID, "sample: invalid sizes (rows=" + s(num_rows) + ", vocab=" + s(vocab) + ")");
  return SLMT_OK;
}

int64_t slmt_sample_workspace_bytes(int num_rows, int vocab) {
  clear_error();
  if (check_sample(num_rows, vocab) != SLMT_OK) return -1;
  return sample_workspace_bytes(num_rows, vocab);
}

int slmt_sample_tokens(const void* logits, int dtype, int64_t row_stride, int num_rows, int vocab, const float* uniforms,
                       const float* temperatures, double temperature, const int32_t* top_ks, int top_k,
                       const float* top_ps, double top_p, const float* min_ps, double min_p, int64_t* tokens,
                       float* probs, void* workspace, int64_t workspace_bytes, slmt_stream_t stream) {
  clear_error();
  const int rc = check_sample(num_rows, vocab);
  if (rc != SLMT_OK) return rc;
  if (dtype != SLMT_F32 && dtype != SLMT_F16 && dtype != SLMT_BF16)
    return fail(SLMT_ERR_INVALID, "sample: dtype must be fp32, fp16 or bf16");
  if (!temperatures && !(temperature >= 0.0)) return fail(SLMT_ERR_INVALID, "sample: temperature must be >= 0");
  if (!top_ks && top_k < 0) return fail(SLMT_ERR_INVALID, "sample: top_k must be >= 0, got " + s(top_k));
  if (!top_ps && !(top_p >= 0.0 && top_p <= 1.0)) return fail(SLMT_ERR_INVALID, "sample: top_p must lie in [0, 1]");
  if (!min_ps && !(min_p >= 0.0 && min_p <= 1.0)) return fail(SLMT_ERR_INVALID, "sample: min_p must lie in [0, 1]");
  if (num_rows == 0) return SLMT_OK;
  if (!logits || !uniforms || !tokens) return fail(SLMT_ERR_INVALID, "sample: null pointer argument");
  const int64_t need = sample_workspace_bytes(num_rows, vocab);
  if (need < 0) return last_status();
  if (need && (!workspace || !aligned(workspace, 16) || workspace_bytes < need))
    return fail(SLMT_ERR_INVALID, "sample: workspace of " + s(need) + " bytes required, got " + s(workspace_bytes));
  SampleParams sp{logits, row_stride, num_rows, vocab, uniforms, temperatures, top_ps, min_ps, top_ks,
                  (float)temperature, (float)top_p, (float)min_p, top_k, tokens, probs};
  return launch_sample(dtype, sp, workspace, reinterpret_cast<hipStream_t>(stream));
}

static int check_shared(int num_seqs, int num_groups, int num_heads, int num_kv_heads, int head_dim) {
  if (!head_dim_ok(head_dim)) return fail(SLMT_ERR_INVALID, "shared decode: head_dim must be 64/80/128, got " + s(head_dim));
  if (num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0)
    return fail(SLMT_ERR_INVALID, "H not divisible by num_kv_heads");
  if (num_seqs < 0 || num_groups < 0)
    return fail(SLMT_ERR_INVALID, "shared decode: invalid sizes (sequences=" + s(num_seqs) + ", groups=" + s(num_groups) + ")");
  return SLMT_OK;
}

int64_t slmt_shared_workspace_bytes(int num_seqs, int num_groups, int num_heads, int num_kv_heads, int head_dim) {
  clear_error();
  if (check_shared(num_seqs, num_groups, num_heads, num_kv_heads, head_dim) != SLMT_OK) return -1;
  return shared_workspace_bytes(num_seqs, num_groups, num_heads, num_kv_heads, head_dim);
}

int slmt_decode_paged_shared(const void* q, int64_t q_seq_stride, int64_t q_head_stride, const void* kv_cache,
                             int64_t num_blocks, int block_size, const void* block_tables, int block_table_bits,
                             int64_t block_table_stride, int max_blocks, const int32_t* seq_lens,
                             const int32_t* group_start_loc, const int32_t* prefix_lens, int num_groups, int num_seqs,
                             int num_heads, int num_kv_heads, int head_dim, void* out, int out_dtype,
                             int64_t out_seq_stride, int64_t out_head_stride, void* workspace, int64_t workspace_bytes,
                             slmt_stream_t stream) {
  clear_error();
  const int rc = check_shared(num_seqs, num_groups, num_heads, num_kv_heads, head_dim);
  if (rc != SLMT_OK) return rc;
  if (block_size <= 0 || block_size % 16 != 0)
    return fail(SLMT_ERR_INVALID, "shared decode: block_size must be a multiple of 16, got " + s(block_size));
  if (block_table_bits != 32 && block_table_bits != 64)
    return fail(SLMT_ERR_INVALID, "shared decode: block table must be int32 or int64");
  if (out_dtype != SLMT_OUT_F32 && out_dtype != SLMT_OUT_F16) return fail(SLMT_ERR_INVALID, "shared decode: out must be fp32 or fp16");
  if (num_blocks < 0 || num_blocks > 0x7fffffff || max_blocks < 0)
    return fail(SLMT_ERR_INVALID, "shared decode: invalid sizes (blocks=" + s(num_blocks) + ", max_blocks=" + s(max_blocks) + ")");
  if (num_seqs == 0) return SLMT_OK;
  if (!q || !out || !seq_lens || !group_start_loc || (num_groups && !prefix_lens))
    return fail(SLMT_ERR_INVALID, "shared decode: null pointer argument");
  if (num_blocks == 0 || !kv_cache || !block_tables) max_blocks = 0;      // (nothing can be seen)
  if (max_blocks && !aligned(kv_cache, 8)) return fail(SLMT_ERR_INVALID, "shared decode: the cache must be 8-byte aligned");
  if (!aligned(q, 16) || ((q_seq_stride | q_head_stride) & 7))
    return fail(SLMT_ERR_INVALID, "shared decode: q must be 16-byte aligned with strides that are multiples of 8");
  if (!aligned(out, out_dtype == SLMT_OUT_F16 ? 8 : 16) || ((out_seq_stride | out_head_stride) & 3))
    return fail(SLMT_ERR_INVALID, "shared decode: out's rows must be aligned to four elements");
  SharedParams p{};
  p.q = reinterpret_cast<const uint16_t*>(q);
  p.q_seq_stride = q_seq_stride;
  p.q_head_stride = q_head_stride;
  p.cache = reinterpret_cast<const uint8_t*>(kv_cache);
  p.last_block = num_blocks ? (uint32_t)(num_blocks - 1) : 0;
  p.block_tables = block_tables;
  p.bt_stride = block_table_stride;
  p.bt64 = block_table_bits == 64;
  p.block_size = block_size;
  p.block_shift = block_shift_of(block_size);
  const int64_t tokens = (int64_t)max_blocks * block_size;
  p.max_tokens = (int)(tokens < 0x7fffff00 ? tokens : 0x7fffff00);
  p.seq_lens = seq_lens;
  p.group_start = group_start_loc;
  p.prefix_lens = prefix_lens;
  p.B = num_seqs;
  p.R = num_groups;
  p.G = num_heads / num_kv_heads;
  p.KV = num_kv_heads;
  p.out = out;
  p.out_f16 = out_dtype == SLMT_OUT_F16;
  p.out_seq_stride = out_seq_stride;
  p.out_head_stride = out_head_stride;
  return launch_shared(head_dim, p, num_heads, workspace, workspace_bytes, reinterpret_cast<hipStream_t>(stream));
}

static int check_beam(int num_requests, int num_beams, int vocab, int num_candidates) {
  if (num_requests < 0 || vocab <= 0)
    return fail(SLMT_ERR_INVALID, "beam select: invalid sizes (requests=" + s(num_requests) + ", vocab=" + s(vocab) + ")");
  if (num_beams < 1 || num_beams > 64 || num_candidates < 1 || num_candidates > 64)
    return fail(SLMT_ERR_UNSUPPORTED, "beam select: beams and candidates must lie in 1 .. 64, got " + s(num_beams) + " and " + s(num_candidates));
  if (vocab > 4194304) return fail(SLMT_ERR_UNSUPPORTED, "beam select: vocabularies go up to 4194304 entries, got " + s(vocab));
  if ((int64_t)num_requests * num_beams > 0x7fffffff) return fail(SLMT_ERR_UNSUPPORTED, "beam select: too many rows for a launch");
  return SLMT_OK;
}

int64_t slmt_beam_workspace_bytes(int num_requests, int num_beams, int vocab, int num_candidates) {
  clear_error();
  if (check_beam(num_requests, num_beams, vocab, num_candidates) != SLMT_OK) return -1;
  return beam_workspace_bytes(num_requests, num_beams, vocab, num_candidates);
}

int slmt_beam_select(const void* logits, int dtype, int64_t row_stride, int num_requests, int num_beams, int vocab,
                     const float* scores, const uint8_t* finished, const int32_t* lengths, double length_penalty,
                     int64_t eos_token, int64_t pad_token, int num_candidates, int keep_rows, int64_t* tokens,
                     int32_t* parents, float* out_scores, uint8_t* out_finished, int32_t* out_lengths, void* workspace,
                     int64_t workspace_bytes, slmt_stream_t stream) {
  clear_error();
  const int rc = check_beam(num_requests, num_beams, vocab, num_candidates);
  if (rc != SLMT_OK) return rc;
  if (dtype != SLMT_F32 && dtype != SLMT_F16 && dtype != SLMT_BF16)
    return fail(SLMT_ERR_INVALID, "beam select: dtype must be fp32, fp16 or bf16");
  if (!(length_penalty > -1e6 && length_penalty < 1e6)) return fail(SLMT_ERR_INVALID, "beam select: length_penalty must be finite");
  if (length_penalty != 0.0 && !lengths) return fail(SLMT_ERR_INVALID, "beam select: length_penalty needs lengths");
  if (pad_token < 0 || pad_token >= vocab) return fail(SLMT_ERR_INVALID, "beam select: pad_token must be a token, got " + s(pad_token));
  if (keep_rows && num_candidates != num_beams)
    return fail(SLMT_ERR_INVALID, "beam select: keep_rows needs as many candidates as beams, got " + s(num_candidates) + " and " + s(num_beams));
  if (out_lengths && !lengths) return fail(SLMT_ERR_INVALID, "beam select: lengths out need lengths");
  if (num_requests == 0) return SLMT_OK;
  if (!logits || !scores || !tokens || !parents || !out_scores) return fail(SLMT_ERR_INVALID, "beam select: null pointer argument");
  const int64_t rows = (int64_t)num_requests * num_beams, size = dtype == SLMT_F32 ? 4 : 2;
  if (row_stride < 0 || (reinterpret_cast<uintptr_t>(logits) & (size - 1)))
    return fail(SLMT_ERR_INVALID, "beam select: logits must be aligned to their type");
  // Workgroups of other requests read while one writes.
  struct Range { const void* p; int64_t bytes; };
  const int64_t n = (int64_t)num_requests * num_candidates;
  const Range reads[] = {{logits, ((rows - 1) * row_stride + vocab) * size}, {scores, 4 * rows}, {finished, rows}, {lengths, 4 * rows}};
  const Range writes[] = {{tokens, 8 * n}, {parents, 4 * n}, {out_scores, 4 * n}, {out_finished, n}, {out_lengths, 4 * n}};
  auto meet = [](const Range& x, const Range& y) {
    const uintptr_t a = (uintptr_t)x.p, b = (uintptr_t)y.p;
    return a && b && a < b + (uintptr_t)y.bytes && b < a + (uintptr_t)x.bytes;
  };
  for (const Range& w : writes) {
    for (const Range& r : reads)
      if (meet(w, r)) return fail(SLMT_ERR_INVALID, "beam select: an output overlaps an input");
    for (const Range& x : writes)
      if (&w < &x && meet(w, x)) return fail(SLMT_ERR_INVALID, "beam select: outputs overlap");
  }
  const int64_t need = beam_workspace_bytes(num_requests, num_beams, vocab, num_candidates);
  if (!workspace || !aligned(workspace, 16) || workspace_bytes < need)
    return fail(SLMT_ERR_INVALID, "beam select: workspace of " + s(need) + " bytes required, got " + s(workspace_bytes));
  const BeamParams b{logits, row_stride, num_requests, num_beams, vocab, num_candidates, scores, finished, lengths,
                     length_penalty, eos_token, pad_token, keep_rows ? 1 : 0, tokens, parents, out_scores, out_finished, out_lengths};
  return launch_beam(dtype, b, workspace, reinterpret_cast<hipStream_t>(stream));
}

int slmt_reorder_beams(void* const* kv_caches, int num_layers, int64_t layer_stride, int64_t num_blocks, int block_size,
                       int num_kv_heads, int head_dim, void* block_tables, int block_table_bits, int64_t block_table_stride, int max_blocks,
                       const int32_t* seq_lens, const int32_t* parents, int num_requests, int num_beams, slmt_stream_t stream) {
  clear_error();
  if (!head_dim_ok(head_dim)) return fail(SLMT_ERR_INVALID, "reorder beams: head_dim must be 64/80/128, got " + s(head_dim));
  if (num_layers < 0 || num_blocks < 0 || num_kv_heads <= 0 || block_size <= 0 || max_blocks < 0 || num_requests < 0)
    return fail(SLMT_ERR_INVALID, "reorder beams: invalid sizes (layers=" + s(num_layers) + ", blocks=" + s(num_blocks) + ", KV=" +
                                      s(num_kv_heads) + ", block_size=" + s(block_size) + ", requests=" + s(num_requests) + ")");
  if (num_beams < 1 || num_beams > 64) return fail(SLMT_ERR_UNSUPPORTED, "reorder beams: beams must lie in 1 .. 64, got " + s(num_beams));
  if (num_requests > 65535) return fail(SLMT_ERR_UNSUPPORTED, "reorder beams: too many requests for a launch");
  if (block_table_bits != 32 && block_table_bits != 64)
    return fail(SLMT_ERR_INVALID, "reorder beams: block table must be int32 or int64");
  if (block_table_stride < max_blocks) return fail(SLMT_ERR_INVALID, "reorder beams: block table rows overlap");
  const int64_t block_bytes = (int64_t)block_size * num_kv_heads * (head_dim + 8);
  if (block_bytes >= (int64_t(1) << 31)) return fail(SLMT_ERR_UNSUPPORTED, "reorder beams: a cache block of 2 GiB or more");
  if (num_requests == 0 || max_blocks == 0) return SLMT_OK;
  if (!block_tables || !seq_lens || !parents || (num_layers && !kv_caches))
    return fail(SLMT_ERR_INVALID, "reorder beams: null pointer argument");
  // Every layer's blocks are moved by workgroups of their own, in place: no bytes of two layers may be the same.
  bool rising = true;
  const uintptr_t bytes = (uintptr_t)(num_blocks * block_bytes);
  auto at = [&](int i) { return reinterpret_cast<uintptr_t>(layer_stride ? kv_caches[0] : kv_caches[i]) + (uintptr_t)(layer_stride * i); };
  for (int i = 0; i < num_layers; ++i) {
    if (!at(i)) return fail(SLMT_ERR_INVALID, "reorder beams: null pointer argument");
    if (at(i) & 7) return fail(SLMT_ERR_INVALID, "reorder beams: the caches must be 8-byte aligned");
    rising = rising && (i == 0 || at(i) >= at(i - 1) + bytes);
  }
  for (int i = 0; i < num_layers && !rising; ++i)
    for (int j = 0; j < i; ++j)
      if (at(i) < at(j) + bytes && at(j) < at(i) + bytes) return fail(SLMT_ERR_INVALID, "reorder beams: two caches overlap");
  ReorderParams p{};
  p.num_blocks = num_blocks;
  p.block_size = block_size;
  p.row_bytes = num_kv_heads * (head_dim + 8);
  p.block_tables = block_tables;
  p.bt64 = block_table_bits == 64;
  p.bt_stride = block_table_stride;
  p.columns = max_blocks;
  p.seq_lens = seq_lens;
  p.parents = parents;
  p.R = num_requests;
  p.W = num_beams;
  int done = 0;
  do {      // (the entries that the copies read are not among those that the first launch moves)
    p.tables = done == 0;
    p.layers = 0;
    while (p.layers < kReorderLayers && done < num_layers) p.caches[p.layers++] = reinterpret_cast<uint8_t*>(at(done++));
    const int rc = launch_reorder(p, reinterpret_cast<hipStream_t>(stream));
    if (rc != SLMT_OK) return rc;
  } while (done < num_layers);
  return SLMT_OK;
}

int slmt_kernel_timing(int enable) {
  clear_error();
  return set_kernel_timing(enable != 0);
}

const char* slmt_kernel_timing_kernel(void) { return kernel_timing_kernel(); }

int slmt_kernel_timing_read(float* us, int max_n) {
  clear_error();
  if (us == nullptr && max_n > 0) return fail(SLMT_ERR_INVALID, "timing: output array is null"), -1;
  return read_kernel_timing(us, max_n);
}

}  // extern "C"
