// The paged-attention entry points as operators of torch's dispatcher (torch.ops.tokquay_amd.*).
//
// Each operator is a thin call into the C ABI (include/tokquay_amd.h) on the current HIP stream of
// the pool's device: shapes and strides are read off the tensors, the status is turned into a
// torch error. Registering them makes the kernels visible to whatever records torch programs
// (FX / make_fx graphs, torch.library tooling); their fake (shape-only) implementations are
// registered from Python (tokquay_amd/torch_ops.py). The tensor-level checks with the reference's
// messages live in tokquay_amd/ops.py, which calls these operators.
//
// Schemas follow tokquay_amd/ops.py: out-variants that write their outputs (and, for the write
// variants, the pool) in place, annotated as mutations.

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include <algorithm>
#include <cmath>
#include <string>
#include <tuple>
#include <utility>
#include <vector>

#include "tokquay_amd.h"

namespace {

void check(tq_status s, const char* what) {
  if (s == TQ_OK) return;
  std::string msg = std::string(what) + " failed: " + tq_status_string(s);
  if (s == TQ_ERR_HIP) msg += std::string(" (") + tq_last_hip_error() + ")";
  TORCH_CHECK(false, msg);
}

// The current stream of t's device, which is the current device until the end of the expression that names it:
// the handle of a device's default stream is null, and a launch on null goes to whichever device is current.
class stream_of {
 public:
  explicit stream_of(const at::Tensor& t)
      : guard_(t.device()), stream_(c10::hip::getCurrentHIPStream(t.device().index()).stream()) {}
  operator void*() const { return stream_; }

 private:
  c10::DeviceGuard guard_;
  void* stream_;
};

// ---- argument checks: everything a kernel would read or write past is refused before any launch.
// Values inside the tensors (block ids, slots, lengths, orders) are checked by the kernels
// themselves and reported through d_error.

struct Pool {
  int64_t blocks;
  int32_t layers, heads, block_size, head_dim;
  at::Device device;
};

Pool pool_of(const char* op, const at::Tensor& pool, int64_t layer) {
  TORCH_CHECK(pool.dim() == 6 && pool.size(2) == 2 && pool.scalar_type() == at::kFloat && pool.is_contiguous() &&
                  pool.is_cuda(),
              op, ": pool must be a contiguous float32 [num_blocks, n_layer, 2, n_head, block_size, d_head] tensor "
              "on a HIP device");
  TORCH_CHECK(pool.size(5) == 64, op, ": only d_head 64 is supported, got ", pool.size(5));
  TORCH_CHECK(layer >= 0 && layer < pool.size(1), op, ": layer ", layer, " out of range [0, ", pool.size(1), ")");
  return {pool.size(0), (int32_t)pool.size(1), (int32_t)pool.size(3), (int32_t)pool.size(4), (int32_t)pool.size(5),
          pool.device()};
}

void on_device(const char* op, const char* name, const at::Tensor& t, const Pool& p) {
  TORCH_CHECK(t.device() == p.device, op, ": ", name, " is on ", t.device(), ", the pool on ", p.device);
}

// A float32 row tensor [N, H, D] or [N, H*D] with at least `rows` rows, each row's H*D elements
// contiguous (any row stride). Returns the row stride in elements.
int64_t rows_of(const char* op, const char* name, const at::Tensor& t, int64_t rows, const Pool& p) {
  on_device(op, name, t, p);
  const int64_t width = (int64_t)p.heads * p.head_dim;
  bool ok = t.scalar_type() == at::kFloat;
  if (t.dim() == 3)
    ok = ok && t.size(1) == p.heads && t.size(2) == p.head_dim && t.stride(2) == 1 && t.stride(1) == p.head_dim;
  else if (t.dim() == 2)
    ok = ok && t.size(1) == width && t.stride(1) == 1;
  else
    ok = false;
  TORCH_CHECK(ok, op, ": ", name, " must be float32 [N, ", p.heads, ", ", p.head_dim, "] or [N, ", width,
              "] with contiguous rows");
  TORCH_CHECK(t.size(0) >= rows, op, ": ", name, " has ", t.size(0), " rows, needs ", rows);
  TORCH_CHECK(rows <= 1 || t.stride(0) >= width, op, ": ", name, "'s rows overlap (row stride ", t.stride(0), ")");
  return t.size(0) > 1 ? t.stride(0) : width;
}

// A contiguous integer vector with at least `n` entries.
void vector_of(const char* op, const char* name, const at::Tensor& t, at::ScalarType dtype, int64_t n,
               const Pool& p) {
  on_device(op, name, t, p);
  TORCH_CHECK(t.scalar_type() == dtype && t.is_contiguous(), op, ": ", name, " must be a contiguous ", dtype,
              " tensor");
  TORCH_CHECK(t.numel() >= n, op, ": ", name, " has ", t.numel(), " entries, needs ", n);
}

// An int32 [B, max_blocks] block-table tensor with at least `rows` rows and contiguous rows.
// Returns its row stride in elements.
int64_t tables_of(const char* op, const char* name, const at::Tensor& t, int64_t rows, const Pool& p) {
  on_device(op, name, t, p);
  TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == 2 && (t.size(1) <= 1 || t.stride(1) == 1),
              op, ": ", name, " must be an int32 [B, max_blocks] tensor with contiguous rows");
  TORCH_CHECK(t.size(0) >= rows, op, ": ", name, " has ", t.size(0), " rows, needs ", rows);
  TORCH_CHECK(rows <= 1 || t.stride(0) >= t.size(1), op, ": ", name, "'s rows overlap");
  return t.size(0) > 1 ? t.stride(0) : t.size(1);
}

template <typename T>
T* ptr(const c10::optional<at::Tensor>& t) {
  return t.has_value() ? static_cast<T*>(t->data_ptr()) : nullptr;
}

void error_word_of(const char* op, const c10::optional<at::Tensor>& t, const Pool& p) {
  if (t.has_value()) vector_of(op, "d_error", *t, at::kInt, 1, p);
}

size_t workspace_of(const char* op, const c10::optional<at::Tensor>& t, const Pool& p) {
  if (!t.has_value()) return 0;
  on_device(op, "workspace", *t, p);
  TORCH_CHECK(t->is_contiguous(), op, ": workspace must be contiguous");
  return t->numel() * t->element_size();
}

void cache_write(at::Tensor pool, int64_t layer, const at::Tensor& k, const at::Tensor& v,
                 const at::Tensor& slot_mapping, const c10::optional<at::Tensor>& d_error) {
  const char* op = "tokquay_amd::cache_write";
  const Pool p = pool_of(op, pool, layer);
  vector_of(op, "slot_mapping", slot_mapping, at::kLong, 0, p);
  const int64_t n = slot_mapping.numel();
  const int64_t ks = rows_of(op, "k", k, n, p), vs = rows_of(op, "v", v, n, p);
  error_word_of(op, d_error, p);
  check(tq_cache_write(pool.data_ptr<float>(), p.blocks, p.layers, p.heads, p.block_size, p.head_dim, (int32_t)layer,
                       k.data_ptr<float>(), ks, v.data_ptr<float>(), vs, slot_mapping.data_ptr<int64_t>(), n,
                       ptr<int32_t>(d_error), stream_of(pool)),
        "tq_cache_write");
}

// The checks shared by the decode variants; returns the number of sequences.
int64_t decode_args(const char* op, const Pool& p, const at::Tensor& out, const at::Tensor& q,
                    const at::Tensor& block_tables, const at::Tensor& context_lens,
                    const c10::optional<at::Tensor>& d_error, const c10::optional<at::Tensor>& seq_order) {
  vector_of(op, "context_lens", context_lens, at::kInt, 0, p);
  const int64_t n = context_lens.numel();
  TORCH_CHECK(n <= INT32_MAX, op, ": too many sequences");
  rows_of(op, "out", out, n, p);
  rows_of(op, "q", q, n, p);
  tables_of(op, "block_tables", block_tables, n, p);
  if (seq_order.has_value()) vector_of(op, "seq_order", *seq_order, at::kInt, n, p);
  error_word_of(op, d_error, p);
  return n;
}

void paged_decode(at::Tensor out, const at::Tensor& q, const at::Tensor& pool, int64_t layer,
                  const at::Tensor& block_tables, const at::Tensor& context_lens, int64_t max_context_len,
                  double scale, int64_t partition_tokens, const c10::optional<at::Tensor>& workspace,
                  const c10::optional<at::Tensor>& d_error, const c10::optional<at::Tensor>& seq_order) {
  const char* op = "tokquay_amd::paged_decode";
  const Pool p = pool_of(op, pool, layer);
  const int64_t n = decode_args(op, p, out, q, block_tables, context_lens, d_error, seq_order);
  const size_t ws = workspace_of(op, workspace, p);
  check(tq_paged_decode(out.data_ptr<float>(), rows_of(op, "out", out, n, p), q.data_ptr<float>(),
                        rows_of(op, "q", q, n, p), pool.data_ptr<float>(), p.blocks, p.layers, p.heads, p.block_size,
                        p.head_dim, (int32_t)layer, block_tables.data_ptr<int32_t>(),
                        tables_of(op, "block_tables", block_tables, n, p), (int32_t)block_tables.size(1),
                        context_lens.data_ptr<int32_t>(), ptr<int32_t>(seq_order), (int32_t)n,
                        (int32_t)max_context_len, (float)scale, (int32_t)partition_tokens, ptr<void>(workspace), ws,
                        ptr<int32_t>(d_error), stream_of(pool)),
        "tq_paged_decode");
}

void paged_decode_write(at::Tensor out, const at::Tensor& q, const at::Tensor& k_new, const at::Tensor& v_new,
                        at::Tensor pool, int64_t layer, const at::Tensor& block_tables,
                        const at::Tensor& context_lens, int64_t max_context_len, double scale,
                        int64_t partition_tokens, const c10::optional<at::Tensor>& workspace,
                        const c10::optional<at::Tensor>& d_error, const c10::optional<at::Tensor>& seq_order) {
  const char* op = "tokquay_amd::paged_decode_write";
  const Pool p = pool_of(op, pool, layer);
  const int64_t n = decode_args(op, p, out, q, block_tables, context_lens, d_error, seq_order);
  const int64_t ks = rows_of(op, "k_new", k_new, n, p), vs = rows_of(op, "v_new", v_new, n, p);
  const size_t ws = workspace_of(op, workspace, p);
  check(tq_paged_decode_write(out.data_ptr<float>(), rows_of(op, "out", out, n, p), q.data_ptr<float>(),
                              rows_of(op, "q", q, n, p), k_new.data_ptr<float>(), ks, v_new.data_ptr<float>(), vs,
                              pool.data_ptr<float>(), p.blocks, p.layers, p.heads, p.block_size, p.head_dim,
                              (int32_t)layer, block_tables.data_ptr<int32_t>(),
                              tables_of(op, "block_tables", block_tables, n, p), (int32_t)block_tables.size(1),
                              context_lens.data_ptr<int32_t>(), ptr<int32_t>(seq_order), (int32_t)n,
                              (int32_t)max_context_len, (float)scale, (int32_t)partition_tokens, ptr<void>(workspace),
                              ws, ptr<int32_t>(d_error), stream_of(pool)),
        "tq_paged_decode_write");
}

// The checks shared by the prefill variants: q rows, out rows, tables, cu_seqlens_q and q_start.
// Returns the number of sequences.
int64_t prefill_args(const char* op, const Pool& p, const at::Tensor& out, const at::Tensor& q, const char* out_name,
                     const char* q_name, const char* tables_name, const at::Tensor& block_tables,
                     const at::Tensor& cu_seqlens_q, const at::Tensor& q_start) {
  vector_of(op, "q_start", q_start, at::kInt, 0, p);
  const int64_t n = q_start.numel();
  vector_of(op, "cu_seqlens_q", cu_seqlens_q, at::kInt, n + 1, p);
  TORCH_CHECK(cu_seqlens_q.numel() == n + 1, op, ": cu_seqlens_q must have num_seqs + 1 entries");
  TORCH_CHECK(q.dim() >= 1 && q.size(0) <= INT32_MAX, op, ": ", q_name, " has too many rows");
  rows_of(op, q_name, q, q.size(0), p);
  rows_of(op, out_name, out, q.size(0), p);
  tables_of(op, tables_name, block_tables, n, p);
  return n;
}

void paged_prefill(at::Tensor out, const at::Tensor& q, const at::Tensor& pool, int64_t layer,
                   const at::Tensor& block_tables, const at::Tensor& cu_seqlens_q, const at::Tensor& q_start,
                   int64_t max_query_len, double scale, const c10::optional<at::Tensor>& d_error,
                   const c10::optional<at::Tensor>& seq_order) {
  const char* op = "tokquay_amd::paged_prefill";
  const Pool p = pool_of(op, pool, layer);
  const int64_t n = prefill_args(op, p, out, q, "out", "q", "block_tables", block_tables, cu_seqlens_q, q_start);
  if (seq_order.has_value()) vector_of(op, "seq_order", *seq_order, at::kInt, n, p);
  error_word_of(op, d_error, p);
  const int64_t nq = q.size(0);
  check(tq_paged_prefill(out.data_ptr<float>(), rows_of(op, "out", out, nq, p), q.data_ptr<float>(),
                         rows_of(op, "q", q, nq, p), pool.data_ptr<float>(), p.blocks, p.layers, p.heads,
                         p.block_size, p.head_dim, (int32_t)layer, block_tables.data_ptr<int32_t>(),
                         tables_of(op, "block_tables", block_tables, n, p), (int32_t)block_tables.size(1),
                         cu_seqlens_q.data_ptr<int32_t>(), q_start.data_ptr<int32_t>(), ptr<int32_t>(seq_order),
                         (int32_t)n, (int32_t)nq,
                         (int32_t)max_query_len, (float)scale, ptr<int32_t>(d_error), stream_of(pool)),
        "tq_paged_prefill");
}

void paged_mixed(at::Tensor dec_out, const at::Tensor& dec_q, const at::Tensor& k_new, const at::Tensor& v_new,
                 const at::Tensor& dec_block_tables, const at::Tensor& context_lens, int64_t max_context_len,
                 at::Tensor pre_out, const at::Tensor& pre_q, const at::Tensor& pre_block_tables,
                 const at::Tensor& cu_seqlens_q, const at::Tensor& q_start, int64_t max_query_len, at::Tensor pool,
                 int64_t layer, double scale, int64_t partition_tokens, const c10::optional<at::Tensor>& workspace,
                 const c10::optional<at::Tensor>& d_error, const c10::optional<at::Tensor>& seq_order) {
  const char* op = "tokquay_amd::paged_mixed";
  const Pool p = pool_of(op, pool, layer);
  const int64_t nd = decode_args(op, p, dec_out, dec_q, dec_block_tables, context_lens, d_error, seq_order);
  const int64_t ks = rows_of(op, "k_new", k_new, nd, p), vs = rows_of(op, "v_new", v_new, nd, p);
  const int64_t np = prefill_args(op, p, pre_out, pre_q, "pre_out", "pre_q", "pre_block_tables", pre_block_tables,
                                  cu_seqlens_q, q_start);
  const int64_t nq = pre_q.size(0);
  const size_t ws = workspace_of(op, workspace, p);
  check(tq_paged_mixed(dec_out.data_ptr<float>(), rows_of(op, "dec_out", dec_out, nd, p), dec_q.data_ptr<float>(),
                       rows_of(op, "dec_q", dec_q, nd, p), k_new.data_ptr<float>(), ks, v_new.data_ptr<float>(), vs,
                       dec_block_tables.data_ptr<int32_t>(),
                       tables_of(op, "dec_block_tables", dec_block_tables, nd, p), (int32_t)dec_block_tables.size(1),
                       context_lens.data_ptr<int32_t>(), ptr<int32_t>(seq_order), (int32_t)nd,
                       (int32_t)max_context_len, (int32_t)partition_tokens, pre_out.data_ptr<float>(),
                       rows_of(op, "pre_out", pre_out, nq, p), pre_q.data_ptr<float>(),
                       rows_of(op, "pre_q", pre_q, nq, p), pre_block_tables.data_ptr<int32_t>(),
                       tables_of(op, "pre_block_tables", pre_block_tables, np, p), (int32_t)pre_block_tables.size(1),
                       cu_seqlens_q.data_ptr<int32_t>(), q_start.data_ptr<int32_t>(), (int32_t)np, (int32_t)nq,
                       (int32_t)max_query_len, pool.data_ptr<float>(), p.blocks, p.layers, p.heads, p.block_size,
                       p.head_dim, (int32_t)layer, (float)scale, ptr<void>(workspace), ws, ptr<int32_t>(d_error),
                       stream_of(pool)),
        "tq_paged_mixed");
}

void paged_gather(at::Tensor k_out, at::Tensor v_out, const at::Tensor& pool, int64_t layer,
                  const at::Tensor& block_tables, const c10::optional<at::Tensor>& d_error) {
  const char* op = "tokquay_amd::paged_gather";
  const Pool p = pool_of(op, pool, layer);
  TORCH_CHECK(block_tables.dim() == 2, op, ": block_tables must be an int32 [B, max_blocks] tensor");
  const int64_t n = block_tables.size(0);
  const int64_t ts = tables_of(op, "block_tables", block_tables, n, p);
  // The gathered copies: [B, H, max_blocks * block_size, D], contiguous.
  const std::vector<int64_t> shape{n, p.heads, block_tables.size(1) * p.block_size, p.head_dim};
  for (const auto& [name, t] : {std::pair<const char*, const at::Tensor&>{"k_out", k_out}, {"v_out", v_out}}) {
    on_device(op, name, t, p);
    TORCH_CHECK(t.scalar_type() == at::kFloat && t.is_contiguous() && t.sizes() == at::IntArrayRef(shape), op, ": ",
                name, " must be a contiguous float32 tensor of shape ", at::IntArrayRef(shape));
  }
  error_word_of(op, d_error, p);
  check(tq_paged_gather(k_out.data_ptr<float>(), v_out.data_ptr<float>(), pool.data_ptr<float>(), p.blocks, p.layers,
                        p.heads, p.block_size, p.head_dim, (int32_t)layer, block_tables.data_ptr<int32_t>(), ts,
                        (int32_t)block_tables.size(1), (int32_t)n, ptr<int32_t>(d_error), stream_of(pool)),
        "tq_paged_gather");
}

void argmax_rows(const at::Tensor& logits, at::Tensor out) {
  const char* op = "tokquay_amd::argmax_rows";
  TORCH_CHECK(logits.is_cuda() && logits.scalar_type() == at::kFloat && logits.dim() == 2 &&
                  (logits.size(1) <= 1 || logits.stride(1) == 1),
              op, ": logits must be a float32 [rows, vocab] tensor on a HIP device with contiguous rows");
  TORCH_CHECK(logits.size(0) <= 1 || logits.stride(0) >= logits.size(1), op, ": logits' rows overlap");
  TORCH_CHECK(out.device() == logits.device() && out.scalar_type() == at::kLong && out.is_contiguous() &&
                  out.numel() >= logits.size(0),
              op, ": out must be a contiguous int64 tensor with one entry per row, on the logits' device");
  const int64_t stride = logits.size(0) > 1 ? logits.stride(0) : logits.size(1);
  check(tq_argmax_rows(out.data_ptr<int64_t>(), logits.data_ptr<float>(), logits.size(0), logits.size(1), stride,
                       stream_of(logits)),
        "tq_argmax_rows");
}

void linear(at::Tensor out, const at::Tensor& x, const at::Tensor& weight, const c10::optional<at::Tensor>& bias,
            bool gelu) {
  const char* op = "tokquay_amd::linear";
  TORCH_CHECK(x.is_cuda() && x.scalar_type() == at::kFloat && x.dim() == 2 && (x.size(1) <= 1 || x.stride(1) == 1), op,
              ": x must be a float32 [rows, K] tensor on a HIP device with contiguous rows");
  const int64_t M = x.size(0), K = x.size(1);
  TORCH_CHECK(M <= 1 || x.stride(0) >= K, op, ": x's rows overlap");
  TORCH_CHECK(weight.device() == x.device() && weight.scalar_type() == at::kFloat && weight.dim() == 2 &&
                  weight.size(1) == K && weight.is_contiguous(),
              op, ": weight must be a contiguous float32 [N, K] tensor on x's device");
  const int64_t N = weight.size(0);
  TORCH_CHECK(!bias.has_value() || (bias->device() == x.device() && bias->scalar_type() == at::kFloat &&
                                    bias->dim() == 1 && bias->size(0) == N && bias->is_contiguous()),
              op, ": bias must be a contiguous float32 [N] tensor on x's device");
  TORCH_CHECK(out.device() == x.device() && out.scalar_type() == at::kFloat && out.dim() == 2 && out.size(0) == M &&
                  out.size(1) == N && (N <= 1 || out.stride(1) == 1),
              op, ": out must be a float32 [rows, N] tensor on x's device with contiguous rows");
  TORCH_CHECK(M <= 1 || out.stride(0) >= N, op, ": out's rows overlap");
  TORCH_CHECK(M <= INT32_MAX && N <= INT32_MAX && K <= INT32_MAX, op, ": sizes past int32");
  // Per call, from torch's allocator: safe on any stream and under graph capture.
  const size_t bytes = tq_linear_workspace_size((int32_t)M, (int32_t)N, (int32_t)K);
  at::Tensor workspace;
  if (bytes > 0) workspace = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
  check(tq_linear(out.data_ptr<float>(), M > 1 ? out.stride(0) : N, x.data_ptr<float>(), M > 1 ? x.stride(0) : K,
                  (int32_t)M, weight.data_ptr<float>(), ptr<float>(bias), (int32_t)N, (int32_t)K, gelu ? 1 : 0,
                  bytes > 0 ? workspace.data_ptr() : nullptr, bytes, stream_of(x)),
        "tq_linear");
}

// ---- rotated cache append, chunk attention and draft verification: pools of three types, grouped heads

int32_t dtype_of(at::ScalarType t) {
  return t == at::kFloat ? TQ_F32 : t == at::kHalf ? TQ_F16 : t == at::kBFloat16 ? TQ_BF16 : -1;
}

// A contiguous pool of one of the types, with heads of 64 or 128 dims.
Pool typed_pool_of(const char* op, const at::Tensor& pool, int64_t layer, bool float32) {
  const bool type = pool.scalar_type() == at::kHalf || pool.scalar_type() == at::kBFloat16 ||
                    (float32 && pool.scalar_type() == at::kFloat);
  TORCH_CHECK(pool.dim() == 6 && pool.size(2) == 2 && type && pool.is_contiguous() && pool.is_cuda(), op,
              ": pool must be a contiguous ", float32 ? "float32, float16 or bfloat16" : "float16 or bfloat16",
              " [num_blocks, n_layer, 2, n_kv_head, block_size, d_head] tensor on a HIP device");
  TORCH_CHECK(pool.size(5) == 64 || pool.size(5) == 128, op, ": only d_head 64 and 128 are supported, got ",
              pool.size(5));
  TORCH_CHECK(layer >= 0 && layer < pool.size(1), op, ": layer ", layer, " out of range [0, ", pool.size(1), ")");
  TORCH_CHECK(pool.size(0) >= 1 && pool.size(3) >= 1 && pool.size(4) >= 1 && pool.size(4) <= 1024 &&
                  pool.size(0) <= INT32_MAX && pool.size(1) <= INT32_MAX && pool.size(3) <= 65535,
              op, ": pool must hold blocks and heads, in blocks of at most 1024 slots");
  return {pool.size(0), (int32_t)pool.size(1), (int32_t)pool.size(3), (int32_t)pool.size(4), (int32_t)pool.size(5),
          pool.device()};
}

// Rows [N, heads, d_head] or [N, heads * d_head] of the pool's type, each row's elements contiguous, rows `align`
// bytes aligned. `heads` 0: any number (3-dimensional tensors tell it, others by their width); it is returned.
int64_t typed_rows_of(const char* op, const char* name, const at::Tensor& t, int64_t rows, int64_t& heads,
                      const at::Tensor& pool, const Pool& p, int64_t align) {
  on_device(op, name, t, p);
  TORCH_CHECK(t.scalar_type() == pool.scalar_type(), op, ": ", name, " must be of the pool's type ",
              pool.scalar_type(), ", got ", t.scalar_type());
  bool ok = t.dim() == 3 ? t.size(2) == p.head_dim && t.stride(2) == 1 && (t.size(1) <= 1 || t.stride(1) == p.head_dim)
                         : t.dim() == 2 && t.size(1) % p.head_dim == 0 && (t.size(1) <= 1 || t.stride(1) == 1);
  if (ok) {
    const int64_t has = t.dim() == 3 ? t.size(1) : t.size(1) / p.head_dim;
    ok = has >= 1 && has <= 65535 && (heads == 0 || has == heads);
    if (ok) heads = has;
  }
  TORCH_CHECK(ok, op, ": ", name, " must be [N, heads, ", p.head_dim, "] or [N, heads * ", p.head_dim,
              "] with contiguous rows", heads > 0 ? " of " + std::to_string(heads) + " heads" : std::string());
  const int64_t width = heads * p.head_dim;
  TORCH_CHECK(t.size(0) >= rows, op, ": ", name, " has ", t.size(0), " rows, needs ", rows);
  const int64_t stride = t.size(0) > 1 ? t.stride(0) : width;
  TORCH_CHECK(rows <= 1 || stride >= width, op, ": ", name, "'s rows overlap (row stride ", stride, ")");
  TORCH_CHECK((uintptr_t)t.data_ptr() % align == 0 && (rows <= 1 || stride * t.element_size() % align == 0), op, ": ",
              name, "'s rows must be ", align, "-byte aligned");
  return rows <= 1 ? width : stride;
}

void norm_of(const char* op, const char* name, const c10::optional<at::Tensor>& t, const at::Tensor& pool,
             const Pool& p) {
  if (!t.has_value()) return;
  on_device(op, name, *t, p);
  TORCH_CHECK(t->scalar_type() == pool.scalar_type() && t->dim() == 1 && t->size(0) == p.head_dim &&
                  t->is_contiguous() && (uintptr_t)t->data_ptr() % 16 == 0,
              op, ": ", name, " must be a contiguous, 16-byte aligned [", p.head_dim, "] tensor of the pool's type");
}

void rope_cache_write(at::Tensor q_out, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, at::Tensor pool,
                      int64_t layer, const at::Tensor& slot_mapping, const at::Tensor& positions,
                      const at::Tensor& table, bool interleaved, const c10::optional<at::Tensor>& q_norm,
                      const c10::optional<at::Tensor>& k_norm, double eps, const c10::optional<at::Tensor>& d_error) {
  const char* op = "tokquay_amd::rope_cache_write";
  const Pool p = typed_pool_of(op, pool, layer, true);
  vector_of(op, "slot_mapping", slot_mapping, at::kLong, 0, p);
  const int64_t n = slot_mapping.numel();
  vector_of(op, "positions", positions, at::kLong, n, p);
  int64_t heads = 0, kv_heads = p.heads;
  const int64_t qs = typed_rows_of(op, "q", q, n, heads, pool, p, 16);
  const int64_t os = typed_rows_of(op, "q_out", q_out, n, heads, pool, p, 16);
  const int64_t ks = typed_rows_of(op, "k", k, n, kv_heads, pool, p, 16);
  const int64_t vs = typed_rows_of(op, "v", v, n, kv_heads, pool, p, 16);
  on_device(op, "table", table, p);
  TORCH_CHECK(table.scalar_type() == at::kFloat && table.dim() == 2 && table.is_contiguous() &&
                  (uintptr_t)table.data_ptr() % 16 == 0 && table.size(1) >= 16 && table.size(1) <= p.head_dim &&
                  table.size(1) % 16 == 0,
              op, ": table must be a contiguous float32 [positions, rotary] tensor, rotary a multiple of 16 up to ",
              p.head_dim);
  norm_of(op, "q_norm", q_norm, pool, p);
  norm_of(op, "k_norm", k_norm, pool, p);
  TORCH_CHECK(eps >= 0, op, ": eps must not be negative, got ", eps);
  TORCH_CHECK(p.blocks <= UINT32_MAX / p.block_size, op, ": pool has more than 2^32 - 1 slots");
  TORCH_CHECK(n <= 0xffff0000LL / (heads + 2 * kv_heads), op, ": too many rows for their heads");
  TORCH_CHECK(n == 0 || table.size(0) >= 1, op, ": table has no positions");
  error_word_of(op, d_error, p);
  check(tq_rope_cache_write(q_out.data_ptr(), os, q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs,
                            pool.data_ptr(), p.blocks, p.layers, (int32_t)heads, p.heads, p.block_size, p.head_dim,
                            (int32_t)layer, slot_mapping.data_ptr<int64_t>(), positions.data_ptr<int64_t>(),
                            table.data_ptr<float>(), table.size(0), (int32_t)table.size(1), interleaved ? 1 : 0,
                            ptr<void>(q_norm), ptr<void>(k_norm), (float)eps, n, dtype_of(pool.scalar_type()),
                            ptr<int32_t>(d_error), stream_of(pool)),
        "tq_rope_cache_write");
}

// An int64 [rows, words] tensor of masks of max_query_len bits.
void masks_of(const char* op, const at::Tensor& t, int64_t rows, int64_t max_query_len, at::Device device) {
  TORCH_CHECK(t.device() == device && t.scalar_type() == at::kLong && t.dim() == 2 && t.size(0) == rows &&
                  t.is_contiguous() && t.size(1) <= 0x3fffffff && t.size(1) >= (max_query_len + 63) / 64,
              op, ": masks must be a contiguous int64 [", rows, ", words] tensor of at least ", max_query_len,
              " bits a row on ", device);
}

// paged_chunk, or paged_tree where there are masks.
void attend(const char* op, at::Tensor& out, const at::Tensor& q, const at::Tensor& pool, int64_t layer,
            const at::Tensor& block_tables, const at::Tensor& cu_seqlens_q, const at::Tensor& q_start,
            const at::Tensor* masks, int64_t max_query_len, int64_t max_context_len, double scale,
            const c10::optional<at::Tensor>& workspace, const c10::optional<at::Tensor>& d_error) {
  const Pool p = typed_pool_of(op, pool, layer, false);
  vector_of(op, "q_start", q_start, at::kInt, 0, p);
  const int64_t n = q_start.numel();
  TORCH_CHECK(n <= INT32_MAX, op, ": too many sequences");
  vector_of(op, "cu_seqlens_q", cu_seqlens_q, at::kInt, n + 1, p);
  TORCH_CHECK(cu_seqlens_q.numel() == n + 1, op, ": cu_seqlens_q must have num_seqs + 1 entries");
  TORCH_CHECK(q.dim() >= 1 && q.size(0) <= INT32_MAX, op, ": q has too many rows");
  const int64_t rows = q.size(0);
  int64_t heads = 0;
  const int64_t qs = typed_rows_of(op, "q", q, rows, heads, pool, p, 16);
  const int64_t os = typed_rows_of(op, "out", out, rows, heads, pool, p, 8);
  TORCH_CHECK(heads % p.heads == 0, op, ": ", heads, " query heads are no multiple of the pool's ", p.heads);
  const int64_t ts = tables_of(op, "block_tables", block_tables, n, p);
  TORCH_CHECK(block_tables.size(1) <= INT32_MAX, op, ": block_tables has too many columns");
  TORCH_CHECK(max_query_len >= 0 && max_query_len <= INT32_MAX && max_context_len >= 0 &&
                  max_context_len <= 1 << 30, op, ": max_query_len and max_context_len must be lengths, contexts up to 2^30");
  TORCH_CHECK(std::isfinite((float)scale), op, ": scale must be a finite float32, got ", scale);
  if (n > 0 && rows > 0 && max_query_len > 0) {
    TORCH_CHECK(max_query_len <= (INT32_MAX - 65536) / heads, op, ": max_query_len is too long for ", heads, " heads");
    TORCH_CHECK(max_context_len >= 1 && block_tables.size(1) >= 1, op,
                ": max_context_len and block_tables must have room for the sequences");
    TORCH_CHECK(pool.numel() / p.blocks <= INT32_MAX, op, ": a block of the pool has too many elements");
  }
  if (masks != nullptr) masks_of(op, *masks, rows, max_query_len, q.device());
  error_word_of(op, d_error, p);
  size_t ws = workspace_of(op, workspace, p);
  const size_t need = (masks != nullptr ? tq_paged_tree_workspace_size : tq_paged_chunk_workspace_size)(
      (int32_t)n, (int32_t)heads, p.heads, p.head_dim, (int32_t)rows, (int32_t)max_query_len, (int32_t)max_context_len);
  at::Tensor own;  // from torch's allocator: safe on any stream and under graph capture
  void* at_ws = ptr<void>(workspace);
  if (need > 0 && !workspace.has_value()) {
    own = at::empty({(int64_t)need}, pool.options().dtype(at::kByte));
    at_ws = own.data_ptr();
    ws = need;
  }
  if (masks != nullptr)
    check(tq_paged_tree(out.data_ptr(), os, q.data_ptr(), qs, pool.data_ptr(), p.blocks, p.layers, (int32_t)heads,
                        p.heads, p.block_size, p.head_dim, (int32_t)layer, block_tables.data_ptr<int32_t>(), ts,
                        (int32_t)block_tables.size(1), cu_seqlens_q.data_ptr<int32_t>(), q_start.data_ptr<int32_t>(),
                        masks->data_ptr<int64_t>(), masks->size(1), (int32_t)n, (int32_t)rows, (int32_t)max_query_len,
                        (int32_t)max_context_len, (float)scale, dtype_of(pool.scalar_type()), at_ws, ws,
                        ptr<int32_t>(d_error), stream_of(pool)),
          "tq_paged_tree");
  else
    check(tq_paged_chunk(out.data_ptr(), os, q.data_ptr(), qs, pool.data_ptr(), p.blocks, p.layers, (int32_t)heads,
                         p.heads, p.block_size, p.head_dim, (int32_t)layer, block_tables.data_ptr<int32_t>(), ts,
                         (int32_t)block_tables.size(1), cu_seqlens_q.data_ptr<int32_t>(), q_start.data_ptr<int32_t>(),
                         (int32_t)n, (int32_t)rows, (int32_t)max_query_len, (int32_t)max_context_len, (float)scale,
                         dtype_of(pool.scalar_type()), at_ws, ws, ptr<int32_t>(d_error), stream_of(pool)),
          "tq_paged_chunk");
}

void paged_chunk(at::Tensor out, const at::Tensor& q, const at::Tensor& pool, int64_t layer,
                 const at::Tensor& block_tables, const at::Tensor& cu_seqlens_q, const at::Tensor& q_start,
                 int64_t max_query_len, int64_t max_context_len, double scale,
                 const c10::optional<at::Tensor>& workspace, const c10::optional<at::Tensor>& d_error) {
  attend("tokquay_amd::paged_chunk", out, q, pool, layer, block_tables, cu_seqlens_q, q_start, nullptr, max_query_len,
         max_context_len, scale, workspace, d_error);
}

void paged_tree(at::Tensor out, const at::Tensor& q, const at::Tensor& pool, int64_t layer,
                const at::Tensor& block_tables, const at::Tensor& cu_seqlens_q, const at::Tensor& q_start,
                const at::Tensor& masks, int64_t max_query_len, int64_t max_context_len, double scale,
                const c10::optional<at::Tensor>& workspace, const c10::optional<at::Tensor>& d_error) {
  attend("tokquay_amd::paged_tree", out, q, pool, layer, block_tables, cu_seqlens_q, q_start, &masks, max_query_len,
         max_context_len, scale, workspace, d_error);
}

// A [rows, vocab] tensor with contiguous rows on p's device; its row stride.
int64_t vocab_rows_of(const char* op, const char* name, const at::Tensor& t, int64_t rows, int64_t vocab) {
  TORCH_CHECK(t.dim() == 2 && t.size(0) == rows && t.size(1) == vocab && (vocab <= 1 || t.stride(1) == 1), op, ": ",
              name, " must be [", rows, ", ", vocab, "] with contiguous rows");
  TORCH_CHECK(rows <= 1 || t.stride(0) >= vocab, op, ": ", name, "'s rows overlap");
  return rows > 1 ? t.stride(0) : vocab;
}

void verify_drafts(at::Tensor tokens, at::Tensor accepted, const at::Tensor& logits,
                   const c10::optional<at::Tensor>& draft_probs, const at::Tensor& draft_tokens,
                   const at::Tensor& uniforms, const at::Tensor& temperature, const at::Tensor& cu_seqlens_q,
                   const c10::optional<at::Tensor>& d_error) {
  const char* op = "tokquay_amd::verify_drafts";
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && dtype_of(logits.scalar_type()) >= 0, op,
              ": logits must be a float32, float16 or bfloat16 [rows, vocab] tensor on a HIP device");
  const int64_t rows = logits.size(0), vocab = logits.size(1), n = temperature.numel();
  TORCH_CHECK(rows <= INT32_MAX && vocab >= 1 && vocab <= 1 << 21 && n <= INT32_MAX, op,
              ": logits must have 1 to 2097152 columns");
  const int64_t ls = vocab_rows_of(op, "logits", logits, rows, vocab);
  const auto vector = [&](const char* name, const at::Tensor& t, at::ScalarType type, int64_t entries) {
    TORCH_CHECK(t.device() == logits.device() && t.scalar_type() == type && t.dim() == 1 && t.is_contiguous() &&
                    t.numel() == entries,
                op, ": ", name, " must be a contiguous ", type, " [", entries, "] tensor on the logits' device");
  };
  vector("draft_tokens", draft_tokens, at::kLong, rows);
  vector("uniforms", uniforms, at::kFloat, rows);
  vector("temperature", temperature, at::kFloat, n);
  vector("cu_seqlens_q", cu_seqlens_q, at::kInt, n + 1);
  vector("accepted", accepted, at::kInt, n);
  if (d_error.has_value()) vector("d_error", *d_error, at::kInt, 1);
  TORCH_CHECK(tokens.device() == logits.device() && tokens.scalar_type() == at::kLong && tokens.dim() == 2 &&
                  tokens.size(0) == n && tokens.size(1) >= 1 && tokens.size(1) <= INT32_MAX && tokens.is_contiguous(),
              op, ": tokens must be a contiguous int64 [", n, ", max_query_len] tensor on the logits' device");
  int64_t ps = vocab;
  if (draft_probs.has_value()) {
    TORCH_CHECK(draft_probs->device() == logits.device() && draft_probs->scalar_type() == at::kFloat, op,
                ": draft_probs must be a float32 tensor on the logits' device");
    ps = vocab_rows_of(op, "draft_probs", *draft_probs, rows, vocab);
  }
  const size_t need = tq_verify_drafts_workspace_size((int32_t)n, (int32_t)rows, (int32_t)vocab);
  at::Tensor workspace;
  if (need > 0) workspace = at::empty({(int64_t)need}, logits.options().dtype(at::kByte));
  check(tq_verify_drafts(tokens.data_ptr<int64_t>(), accepted.data_ptr<int32_t>(), logits.data_ptr(), ls,
                         ptr<float>(draft_probs), ps, draft_tokens.data_ptr<int64_t>(), uniforms.data_ptr<float>(),
                         temperature.data_ptr<float>(), cu_seqlens_q.data_ptr<int32_t>(), (int32_t)n, (int32_t)rows,
                         (int32_t)tokens.size(1), (int32_t)vocab, dtype_of(logits.scalar_type()),
                         need > 0 ? workspace.data_ptr() : nullptr, need, ptr<int32_t>(d_error), stream_of(logits)),
        "tq_verify_drafts");
}

// ---- trees of drafted tokens, sampling, copies of blocks

// A pool whose slots are copied: a block's places of one slot number fit 31 bits, its address 16 bytes.
void slots_of(const char* op, const at::Tensor& pool) {
  TORCH_CHECK((uintptr_t)pool.data_ptr() % 16 == 0, op, ": pool must be 16-byte aligned");
  TORCH_CHECK(pool.numel() / (pool.size(0) * pool.size(4)) <= 1 << 30, op, ": a slot of the pool has too many elements");
}

// A contiguous vector with `entries` entries (any number: -1) on `device`.
void exactly(const char* op, const char* name, const at::Tensor& t, at::ScalarType type, int64_t entries, at::Device device) {
  TORCH_CHECK(t.device() == device && t.scalar_type() == type && t.dim() == 1 && t.is_contiguous() &&
                  (entries < 0 || t.numel() == entries) && t.numel() <= INT32_MAX,
              op, ": ", name, " must be a contiguous ", type, " [", entries < 0 ? std::string("N") : std::to_string(entries),
              "] tensor on ", device);
}

// One launch takes 2^32 - 1 threads.
void launchable(const char* op, const char* what, int64_t groups, int64_t threads) {
  TORCH_CHECK(groups <= 0xffffffffLL / threads, op, ": ", what);
}

void tree_layout(at::Tensor positions, at::Tensor masks, const at::Tensor& parents, const at::Tensor& cu_seqlens_q,
                 const at::Tensor& q_start, int64_t max_query_len, const c10::optional<at::Tensor>& d_error) {
  const char* op = "tokquay_amd::tree_layout";
  const at::Device device = parents.device();
  TORCH_CHECK(parents.is_cuda(), op, ": parents must be on a HIP device");
  exactly(op, "parents", parents, at::kInt, -1, device);
  exactly(op, "q_start", q_start, at::kInt, -1, device);
  const int64_t rows = parents.numel(), n = q_start.numel();
  exactly(op, "cu_seqlens_q", cu_seqlens_q, at::kInt, n + 1, device);
  exactly(op, "positions", positions, at::kLong, rows, device);
  TORCH_CHECK(max_query_len >= 0 && max_query_len <= INT32_MAX, op, ": max_query_len must be a length");
  launchable(op, "q_start has too many sequences", n + 1, 64 * std::min<int64_t>(8, std::max<int64_t>(1, (max_query_len + 63) / 64)));
  masks_of(op, masks, rows, max_query_len, device);
  if (d_error.has_value()) exactly(op, "d_error", *d_error, at::kInt, 1, device);
  check(tq_tree_layout(positions.data_ptr<int64_t>(), masks.data_ptr<int64_t>(), masks.size(1),
                       parents.data_ptr<int32_t>(), cu_seqlens_q.data_ptr<int32_t>(), q_start.data_ptr<int32_t>(),
                       (int32_t)n, (int32_t)rows, (int32_t)max_query_len, ptr<int32_t>(d_error), stream_of(parents)),
        "tq_tree_layout");
}

void sample_tokens(at::Tensor tokens, const at::Tensor& logits, const at::Tensor& uniforms, const at::Tensor& temperature,
                   const c10::optional<at::Tensor>& top_k, const c10::optional<at::Tensor>& top_p,
                   const c10::optional<at::Tensor>& min_p, const c10::optional<at::Tensor>& cu_seqlens_q,
                   const c10::optional<at::Tensor>& d_error) {
  const char* op = "tokquay_amd::sample_tokens";
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && dtype_of(logits.scalar_type()) >= 0, op,
              ": logits must be a float32, float16 or bfloat16 [rows, vocab] tensor on a HIP device");
  const int64_t rows = logits.size(0), vocab = logits.size(1);
  const at::Device device = logits.device();
  TORCH_CHECK(rows <= INT32_MAX && vocab >= 1 && vocab <= 1 << 21, op, ": logits must have 1 to 2097152 columns");
  launchable(op, "logits has too many rows", rows, 1024);
  launchable(op, "logits has too many rows", rows * ((vocab + 8191) / 8192), 256);
  const int64_t ls = vocab_rows_of(op, "logits", logits, rows, vocab);
  exactly(op, "temperature", temperature, at::kFloat, cu_seqlens_q.has_value() ? -1 : rows, device);
  const int64_t n = temperature.numel();
  if (cu_seqlens_q.has_value()) exactly(op, "cu_seqlens_q", *cu_seqlens_q, at::kInt, n + 1, device);
  if (top_k.has_value()) exactly(op, "top_k", *top_k, at::kInt, n, device);
  if (top_p.has_value()) exactly(op, "top_p", *top_p, at::kFloat, n, device);
  if (min_p.has_value()) exactly(op, "min_p", *min_p, at::kFloat, n, device);
  exactly(op, "uniforms", uniforms, at::kFloat, rows, device);
  exactly(op, "tokens", tokens, at::kLong, rows, device);
  if (d_error.has_value()) exactly(op, "d_error", *d_error, at::kInt, 1, device);
  const size_t need = tq_sample_tokens_workspace_size((int32_t)rows, (int32_t)vocab);
  at::Tensor workspace;
  if (need > 0) workspace = at::empty({(int64_t)need}, logits.options().dtype(at::kByte));
  check(tq_sample_tokens(tokens.data_ptr<int64_t>(), logits.data_ptr(), ls, uniforms.data_ptr<float>(),
                         temperature.data_ptr<float>(), ptr<int32_t>(top_k), ptr<float>(top_p), ptr<float>(min_p),
                         ptr<int32_t>(cu_seqlens_q), (int32_t)n, (int32_t)rows, (int32_t)vocab,
                         dtype_of(logits.scalar_type()), need > 0 ? workspace.data_ptr() : nullptr, need,
                         ptr<int32_t>(d_error), stream_of(logits)),
        "tq_sample_tokens");
}

void accept_tree(at::Tensor tokens, at::Tensor path, at::Tensor counts, const at::Tensor& sampled,
                 const at::Tensor& draft_tokens, const at::Tensor& parents, const at::Tensor& cu_seqlens_q,
                 const c10::optional<at::Tensor>& pool, const c10::optional<at::Tensor>& block_tables,
                 const c10::optional<at::Tensor>& q_start, const c10::optional<at::Tensor>& d_error) {
  const char* op = "tokquay_amd::accept_tree";
  const at::Device device = sampled.device();
  TORCH_CHECK(sampled.is_cuda(), op, ": sampled must be on a HIP device");
  exactly(op, "sampled", sampled, at::kLong, -1, device);
  exactly(op, "counts", counts, at::kInt, -1, device);
  const int64_t rows = sampled.numel(), n = counts.numel();
  exactly(op, "draft_tokens", draft_tokens, at::kLong, rows, device);
  exactly(op, "parents", parents, at::kInt, rows, device);
  exactly(op, "cu_seqlens_q", cu_seqlens_q, at::kInt, n + 1, device);
  const auto per_seq = [&](const char* name, const at::Tensor& t, at::ScalarType type, int64_t columns) {
    TORCH_CHECK(t.device() == device && t.scalar_type() == type && t.dim() == 2 && t.size(0) == n && t.size(1) >= 1 &&
                    (columns < 0 || t.size(1) == columns) && t.size(1) <= INT32_MAX && t.is_contiguous(),
                op, ": ", name, " must be a contiguous ", type, " [", n, ", max_path] tensor on ", device);
  };
  per_seq("tokens", tokens, at::kLong, -1);
  per_seq("path", path, at::kInt, tokens.size(1));
  if (d_error.has_value()) exactly(op, "d_error", *d_error, at::kInt, 1, device);
  TORCH_CHECK(pool.has_value() == block_tables.has_value() && pool.has_value() == q_start.has_value(), op,
              ": pool, block_tables and q_start go together");
  Pool p{1, 1, 1, 1, 64, device};
  int64_t ts = 0;
  if (pool.has_value()) {
    p = typed_pool_of(op, *pool, 0, true);
    TORCH_CHECK(p.device == device, op, ": pool is on ", p.device, ", sampled on ", device);
    slots_of(op, *pool);
    ts = tables_of(op, "block_tables", *block_tables, n, p);
    TORCH_CHECK(block_tables->size(1) <= INT32_MAX, op, ": block_tables has too many columns");
    exactly(op, "q_start", *q_start, at::kInt, n, device);
  }
  // A workgroup takes 256 pieces of 16 bytes.
  const int64_t pieces = pool.has_value() ? pool->numel() / (pool->size(0) * pool->size(4)) * pool->element_size() / 16 : 1;
  launchable(op, "counts has too many sequences", n * ((pieces + 255) / 256), 256);
  check(tq_accept_tree(tokens.data_ptr<int64_t>(), path.data_ptr<int32_t>(), counts.data_ptr<int32_t>(),
                       (int32_t)tokens.size(1), sampled.data_ptr<int64_t>(), draft_tokens.data_ptr<int64_t>(),
                       parents.data_ptr<int32_t>(), cu_seqlens_q.data_ptr<int32_t>(), (int32_t)n, (int32_t)rows,
                       ptr<void>(pool), p.blocks, p.layers, p.heads, p.block_size, p.head_dim,
                       pool.has_value() ? dtype_of(pool->scalar_type()) : TQ_F32, ptr<int32_t>(block_tables), ts,
                       block_tables.has_value() ? (int32_t)block_tables->size(1) : 0, ptr<int32_t>(q_start),
                       ptr<int32_t>(d_error), stream_of(sampled)),
        "tq_accept_tree");
}

// The same with outputs of their own, which take the host less here than before the call (accept_tree 9.3 -> 7.1 us).
at::Tensor fresh(const at::Tensor& like, at::ScalarType type, at::IntArrayRef sizes) {
  return at::empty(sizes, like.options().dtype(type));
}

std::tuple<at::Tensor, at::Tensor> new_tree_layout(const at::Tensor& parents, const at::Tensor& cu_seqlens_q,
                                                   const at::Tensor& q_start, int64_t max_query_len,
                                                   const c10::optional<at::Tensor>& d_error) {
  TORCH_CHECK(max_query_len >= 0 && max_query_len <= INT32_MAX, "tokquay_amd::tree_layout: max_query_len must be a length");
  at::Tensor positions = fresh(parents, at::kLong, {parents.numel()});
  at::Tensor masks = fresh(parents, at::kLong, {parents.numel(), (max_query_len + 63) / 64});
  tree_layout(positions, masks, parents, cu_seqlens_q, q_start, max_query_len, d_error);
  return {positions, masks};
}

at::Tensor new_sample_tokens(const at::Tensor& logits, const at::Tensor& uniforms, const at::Tensor& temperature,
                             const c10::optional<at::Tensor>& top_k, const c10::optional<at::Tensor>& top_p,
                             const c10::optional<at::Tensor>& min_p, const c10::optional<at::Tensor>& cu_seqlens_q,
                             const c10::optional<at::Tensor>& d_error) {
  // Rows of no sequence, which the call leaves alone, have -1.
  at::Tensor tokens = cu_seqlens_q.has_value() ? at::full({uniforms.numel()}, -1, logits.options().dtype(at::kLong))
                                               : fresh(logits, at::kLong, {uniforms.numel()});
  sample_tokens(tokens, logits, uniforms, temperature, top_k, top_p, min_p, cu_seqlens_q, d_error);
  return tokens;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> new_accept_tree(
    const at::Tensor& sampled, const at::Tensor& draft_tokens, const at::Tensor& parents, const at::Tensor& cu_seqlens_q,
    int64_t max_path, const c10::optional<at::Tensor>& pool, const c10::optional<at::Tensor>& block_tables,
    const c10::optional<at::Tensor>& q_start, const c10::optional<at::Tensor>& d_error) {
  const int64_t n = cu_seqlens_q.numel() - 1;
  TORCH_CHECK(n >= 0 && max_path >= 1 && max_path <= INT32_MAX,
              "tokquay_amd::accept_tree: cu_seqlens_q must have num_seqs + 1 entries, and max_path be a length above 0");
  at::Tensor tokens = fresh(sampled, at::kLong, {n, max_path}), path = fresh(sampled, at::kInt, {n, max_path});
  at::Tensor counts = fresh(sampled, at::kInt, {n});
  accept_tree(tokens, path, counts, sampled, draft_tokens, parents, cu_seqlens_q, pool, block_tables, q_start, d_error);
  return {tokens, path, counts};
}

void copy_blocks(at::Tensor pool, const at::Tensor& src_blocks, const at::Tensor& dst_blocks,
                 const c10::optional<at::Tensor>& num_slots, const c10::optional<at::Tensor>& d_error) {
  const char* op = "tokquay_amd::copy_blocks";
  const Pool p = typed_pool_of(op, pool, 0, true);
  slots_of(op, pool);
  exactly(op, "src_blocks", src_blocks, at::kInt, -1, p.device);
  const int64_t n = src_blocks.numel();
  TORCH_CHECK(n <= 1 << 20, op, ": src_blocks has more than 1048576 entries");
  exactly(op, "dst_blocks", dst_blocks, at::kInt, n, p.device);
  if (num_slots.has_value()) exactly(op, "num_slots", *num_slots, at::kInt, n, p.device);
  // A workgroup takes 8 KiB, for every 256 pairs.
  const int64_t share = 8192 * std::max<int64_t>(1, (n + 255) / 256), block = pool.numel() / p.blocks * pool.element_size();
  launchable(op, "src_blocks has too many blocks of this size", n * ((block + share - 1) / share), 256);
  if (d_error.has_value()) exactly(op, "d_error", *d_error, at::kInt, 1, p.device);
  check(tq_copy_blocks(pool.data_ptr(), p.blocks, p.layers, p.heads, p.block_size, p.head_dim,
                       dtype_of(pool.scalar_type()), src_blocks.data_ptr<int32_t>(), dst_blocks.data_ptr<int32_t>(),
                       ptr<int32_t>(num_slots), (int32_t)n, ptr<int32_t>(d_error), stream_of(pool)),
        "tq_copy_blocks");
}

}  // namespace

TORCH_LIBRARY(tokquay_amd, m) {
  m.def("cache_write(Tensor(a!) pool, int layer, Tensor k, Tensor v, Tensor slot_mapping, Tensor(b!)? d_error) -> ()");
  m.def("paged_decode(Tensor(a!) out, Tensor q, Tensor pool, int layer, Tensor block_tables, Tensor context_lens, "
        "int max_context_len, float scale, int partition_tokens, Tensor(b!)? workspace, Tensor(c!)? d_error, "
        "Tensor? seq_order) -> ()");
  m.def("paged_decode_write(Tensor(a!) out, Tensor q, Tensor k_new, Tensor v_new, Tensor(b!) pool, int layer, "
        "Tensor block_tables, Tensor context_lens, int max_context_len, float scale, int partition_tokens, "
        "Tensor(c!)? workspace, Tensor(d!)? d_error, Tensor? seq_order) -> ()");
  m.def("paged_prefill(Tensor(a!) out, Tensor q, Tensor pool, int layer, Tensor block_tables, Tensor cu_seqlens_q, "
        "Tensor q_start, int max_query_len, float scale, Tensor(b!)? d_error, Tensor? seq_order) -> ()");
  m.def("paged_mixed(Tensor(a!) dec_out, Tensor dec_q, Tensor k_new, Tensor v_new, Tensor dec_block_tables, "
        "Tensor context_lens, int max_context_len, Tensor(b!) pre_out, Tensor pre_q, Tensor pre_block_tables, "
        "Tensor cu_seqlens_q, Tensor q_start, int max_query_len, Tensor(c!) pool, int layer, float scale, "
        "int partition_tokens, Tensor(d!)? workspace, Tensor(e!)? d_error, Tensor? seq_order) -> ()");
  m.def("paged_gather(Tensor(a!) k_out, Tensor(b!) v_out, Tensor pool, int layer, Tensor block_tables, "
        "Tensor(c!)? d_error) -> ()");
  m.def("argmax_rows(Tensor logits, Tensor(a!) out) -> ()");
  m.def("linear(Tensor(a!) out, Tensor x, Tensor weight, Tensor? bias, bool gelu) -> ()");
  m.def("rope_cache_write(Tensor(a!) q_out, Tensor q, Tensor k, Tensor v, Tensor(b!) pool, int layer, "
        "Tensor slot_mapping, Tensor positions, Tensor table, bool interleaved, Tensor? q_norm, Tensor? k_norm, "
        "float eps, Tensor(c!)? d_error) -> ()");
  m.def("paged_chunk(Tensor(a!) out, Tensor q, Tensor pool, int layer, Tensor block_tables, Tensor cu_seqlens_q, "
        "Tensor q_start, int max_query_len, int max_context_len, float scale, Tensor(b!)? workspace, "
        "Tensor(c!)? d_error) -> ()");
  m.def("verify_drafts(Tensor(a!) tokens, Tensor(b!) accepted, Tensor logits, Tensor? draft_probs, "
        "Tensor draft_tokens, Tensor uniforms, Tensor temperature, Tensor cu_seqlens_q, Tensor(c!)? d_error) -> ()");
  m.def("tree_layout(Tensor(a!) positions, Tensor(b!) masks, Tensor parents, Tensor cu_seqlens_q, Tensor q_start, "
        "int max_query_len, Tensor(c!)? d_error) -> ()");
  m.def("paged_tree(Tensor(a!) out, Tensor q, Tensor pool, int layer, Tensor block_tables, Tensor cu_seqlens_q, "
        "Tensor q_start, Tensor masks, int max_query_len, int max_context_len, float scale, Tensor(b!)? workspace, "
        "Tensor(c!)? d_error) -> ()");
  m.def("sample_tokens(Tensor(a!) tokens, Tensor logits, Tensor uniforms, Tensor temperature, Tensor? top_k, "
        "Tensor? top_p, Tensor? min_p, Tensor? cu_seqlens_q, Tensor(b!)? d_error) -> ()");
  m.def("accept_tree(Tensor(a!) tokens, Tensor(b!) path, Tensor(c!) counts, Tensor sampled, Tensor draft_tokens, "
        "Tensor parents, Tensor cu_seqlens_q, Tensor(d!)? pool, Tensor? block_tables, Tensor? q_start, "
        "Tensor(e!)? d_error) -> ()");
  m.def("tree_layout.new(Tensor parents, Tensor cu_seqlens_q, Tensor q_start, int max_query_len, "
        "Tensor(a!)? d_error) -> (Tensor, Tensor)");
  m.def("sample_tokens.new(Tensor logits, Tensor uniforms, Tensor temperature, Tensor? top_k, Tensor? top_p, Tensor? min_p, "
        "Tensor? cu_seqlens_q, Tensor(a!)? d_error) -> Tensor");
  m.def("accept_tree.new(Tensor sampled, Tensor draft_tokens, Tensor parents, Tensor cu_seqlens_q, int max_path, "
        "Tensor(a!)? pool, Tensor? block_tables, Tensor? q_start, Tensor(b!)? d_error) -> (Tensor, Tensor, Tensor)");
  m.def("copy_blocks(Tensor(a!) pool, Tensor src_blocks, Tensor dst_blocks, Tensor? num_slots, Tensor(b!)? d_error) -> ()");
}

TORCH_LIBRARY_IMPL(tokquay_amd, CUDA, m) {
  m.impl("cache_write", &cache_write);
  m.impl("paged_decode", &paged_decode);
  m.impl("paged_decode_write", &paged_decode_write);
  m.impl("paged_prefill", &paged_prefill);
  m.impl("paged_mixed", &paged_mixed);
  m.impl("paged_gather", &paged_gather);
  m.impl("argmax_rows", &argmax_rows);
  m.impl("linear", &linear);
  m.impl("rope_cache_write", &rope_cache_write);
  m.impl("paged_chunk", &paged_chunk);
  m.impl("verify_drafts", &verify_drafts);
  m.impl("tree_layout", &tree_layout);
  m.impl("paged_tree", &paged_tree);
  m.impl("sample_tokens", &sample_tokens);
  m.impl("accept_tree", &accept_tree);
  m.impl("tree_layout.new", &new_tree_layout);
  m.impl("sample_tokens.new", &new_sample_tokens);
  m.impl("accept_tree.new", &new_accept_tree);
  m.impl("copy_blocks", &copy_blocks);
}
