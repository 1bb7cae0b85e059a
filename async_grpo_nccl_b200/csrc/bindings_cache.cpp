// Python bindings of the operators on a paged cache that is read in whole chunks (launchers_cache.h).
#include "bindings_cache.h"

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <limits>

#include "bindings_layers.h"
#include "launchers.h"

namespace {

using namespace cache_args;

// Whether the first `cols` columns of `a` and those of `b`, as many rows of bf16, have nothing in common; both may be columns of one buffer.
bool apart(const Tensor& a, const Tensor& b, int64_t cols) {
  const int64_t n = a.size(0);
  if (n == 0) return true;
  const auto* x = static_cast<const c10::BFloat16*>(a.data_ptr());
  const auto* y = static_cast<const c10::BFloat16*>(b.data_ptr());
  if (y >= x + (n - 1) * a.stride(0) + cols || x >= y + (n - 1) * b.stride(0) + cols) return true;
  const int64_t pitch = a.stride(0);
  if (n == 1 || pitch <= 0 || b.stride(0) != pitch) return false;
  const int64_t column = ((y - x) % pitch + pitch) % pitch;
  return column >= cols && column + cols <= pitch;
}

void kv_cache_read(const Tensor& k_cache, const Tensor& v_cache, const Tensor& slots, Tensor& qkv, int64_t Hq, int64_t Hkv, int64_t D,
                   const OptTensor& status, const OptTensor& k_scale, const OptTensor& v_scale) {
  const char* op = "kv_cache_read";
  TORCH_CHECK(Hq >= 0 && Hkv > 0 && (D == 64 || D == 128), op, ": head_dim must be 64 or 128");
  written_rows(qkv, (Hq + 2 * Hkv) * D, op, "qkv");
  const agrpo::PagedCache c = cache(k_cache, v_cache, k_scale, v_scale, qkv.device(), D, op);
  TORCH_CHECK(c.Hkv == Hkv, op, ": cache of ", std::to_string(Hkv), " kv heads");
  ints(slots, qkv.device(), 0, op, "slots");
  TORCH_CHECK(slots.numel() == qkv.size(0), op, ": a slot for each row");
  vectors(qkv.size(0), c.Hkv, op);
  status_word(status, qkv.device(), op);
  const c10::cuda::CUDAGuard guard(qkv.device());
  agrpo::launch_kv_cache_read(c, slots.data_ptr<int>(), qkv.data_ptr(), qkv.stride(0), (int)(Hq * D), (int)((Hq + Hkv) * D), (int)qkv.size(0),
                              int_ptr(status), at::cuda::getCurrentCUDAStream());
}

void paged_chunk_attn(const Tensor& qkv, const Tensor& k_cache, const Tensor& v_cache, const Tensor& block_tables, const Tensor& seq_lens,
                      const Tensor& q_starts, Tensor& out, int64_t Hq, int64_t Hkv, int64_t D, double softmax_scale, const OptTensor& status,
                      const OptTensor& k_scale, const OptTensor& v_scale) {
  const char* op = "paged_chunk_attn";
  TORCH_CHECK(D == 64 || D == 128, op, ": head_dim must be 64 or 128");
  TORCH_CHECK(Hkv > 0 && Hq > 0 && Hq % Hkv == 0 && Hq / Hkv <= 32, op, ": 1 to 32 query heads per kv head");
  rows(qkv, Hq * D, op, "qkv");
  const torch::Device dev = qkv.device();
  written_rows(out, Hq * D, op, "out");
  TORCH_CHECK(out.device() == dev && out.size(0) == qkv.size(0) && out.size(1) == Hq * D, op, ": out [rows, Hq * D] on the device of the rows");
  TORCH_CHECK(apart(qkv, out, Hq * D), op, ": out must not be qkv or overlap its q heads");
  const agrpo::PagedCache c = cache(k_cache, v_cache, k_scale, v_scale, dev, D, op);
  TORCH_CHECK(c.Hkv == Hkv, op, ": cache of ", std::to_string(Hkv), " kv heads");
  TORCH_CHECK(c.block_size == 16 || c.block_size == 32 || c.block_size == 64 || c.block_size == 128, op, ": block size 16, 32, 64 or 128");
  ints(q_starts, dev, 1, op, "q_starts");
  const int64_t B = q_starts.numel() - 1;
  ints(seq_lens, dev, B, op, "seq_lens");
  TORCH_CHECK(block_tables.scalar_type() == torch::kInt32 && block_tables.device() == dev && block_tables.dim() == 2 && block_tables.size(0) >= B &&
                  (block_tables.size(1) <= 1 || block_tables.stride(1) == 1), op, ": block_tables int32 [sequences, blocks], inner stride 1");
  TORCH_CHECK(B <= 8192 && block_tables.size(1) * c.block_size < (int64_t(1) << 30), op, ": at most 8192 sequences of 2^30 tokens");
  // in 32 bits, also times log2 e, and not a subnormal number: hidden scores are -inf, which times zero would be no number
  TORCH_CHECK(softmax_scale >= std::numeric_limits<float>::min() && softmax_scale <= std::numeric_limits<float>::max() / 1.5, op,
              ": softmax_scale must be a positive number of 32 bits");
  for (const OptTensor* s : {&k_scale, &v_scale}) TORCH_CHECK(!given(*s) || aligned16(**s), op, ": scales must be 16-byte aligned");
  status_word(status, dev, op);
  const c10::cuda::CUDAGuard guard(dev);
  agrpo::ChunkAttnArgs a;
  a.q = qkv.data_ptr();
  a.ldq = qkv.stride(0);
  a.out = out.data_ptr();
  a.ldo = out.stride(0);
  a.block_tables = block_tables.data_ptr<int>();
  a.table_pitch = block_tables.stride(0);
  a.max_blocks = (int)block_tables.size(1);
  a.seq_lens = seq_lens.data_ptr<int>();
  a.q_starts = q_starts.data_ptr<int>();
  a.B = (int)B;
  a.Tq = (int)qkv.size(0);
  a.Hq = (int)Hq;
  a.softmax_scale = (float)softmax_scale;
  a.status = int_ptr(status);
  if (a.Tq == 0 || a.B == 0) return;
  TORCH_CHECK(agrpo::paged_chunk_attn_tiles(a, c) < (int64_t(1) << 31), op, ": too many rows for tables of this width");
  if (a.Tq == 1) a.ldq = Hq * D;  // the pitch of a single row means nothing
  // Parts of units that several CTAs share: from the allocator, so that calls on several streams or in several graphs do not meet in it.
  const int sms = launch_num_sms();
  const Tensor scratch = at::empty({agrpo::paged_chunk_attn_scratch(a, c, sms)}, qkv.options().dtype(torch::kUInt8));
  agrpo::launch_paged_chunk_attn(a, c, sms, scratch.data_ptr(), at::cuda::getCurrentCUDAStream());
}

}  // namespace

#define NOGIL py::call_guard<py::gil_scoped_release>()

void bind_cache_ops(py::module_& m) {
  m.def("kv_cache_read", &kv_cache_read, py::arg("k_cache"), py::arg("v_cache"), py::arg("slots"), py::arg("qkv"), py::arg("Hq"), py::arg("Hkv"),
        py::arg("D"), py::arg("status") = py::none(), py::arg("k_scale") = py::none(), py::arg("v_scale") = py::none(), NOGIL,
        "Keys and values of the cache slots `slots` (int32, one a row; negative: the row stays as it is) into the k and v columns of the rows of "
        "`qkv` [rows, (Hq + 2 Hkv) D]: the inverse of kv_cache_write, for a bf16 or an 8-bit cache.");
  m.def("paged_chunk_attn", &paged_chunk_attn, py::arg("qkv"), py::arg("k_cache"), py::arg("v_cache"), py::arg("block_tables"), py::arg("seq_lens"),
        py::arg("q_starts"), py::arg("out"), py::arg("Hq"), py::arg("Hkv"), py::arg("D"), py::arg("softmax_scale"), py::arg("status") = py::none(),
        py::arg("k_scale") = py::none(), py::arg("v_scale") = py::none(), NOGIL,
        "Attention of the newest tokens of every sequence over the paged cache that already holds them. Sequence b owns the rows q_starts[b] .. "
        "q_starts[b + 1] of `qkv` (q heads in the first Hq D columns) and seq_lens[b] tokens of the cache; its row i of n sees the keys 0 .. "
        "seq_lens[b] - n + i, a row that sees none is zero. Rows behind the last sequence are left as they are. Starts that go back "
        "anywhere compute nothing, and the status word says so. Cache [blocks, Hkv, block size, D], "
        "bf16 or e4m3 with scale bytes. Nothing here reads the lengths on the host: a captured call follows them. For the same reason the kernel is "
        "chosen by the average of rows over all sequences, and for 1024 rows (tokens times query heads of a kv head) a sequence over 8 bits the "
        "cache is converted to bf16 in a workspace of up to 128 MB if full tables fit there: leave out sequences without rows, and pass tables as "
        "wide as the longest sequence needs (a view will do).");
}
