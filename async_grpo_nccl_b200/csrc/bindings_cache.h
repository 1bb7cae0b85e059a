// Argument checks that the operators on a paged cache share. Numbers go into messages as text: printing one through a stream ends the process
// where the compiler's C++ library is not the one that the interpreter has loaded.
#pragma once
#include <torch/extension.h>

#include "launchers_cache.h"

namespace cache_args {

using torch::Tensor;
using OptTensor = c10::optional<torch::Tensor>;

inline bool given(const OptTensor& t) { return t.has_value() && t->defined(); }
inline bool aligned16(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }
inline int* int_ptr(const OptTensor& t) { return given(t) ? t->data_ptr<int>() : nullptr; }

// int32 on the device of the call, contiguous, at least n entries
inline void ints(const Tensor& t, const torch::Device& dev, int64_t n, const char* op, const char* name) {
  TORCH_CHECK(t.scalar_type() == torch::kInt32 && t.device() == dev && t.is_contiguous() && t.numel() >= n, op, ": ", name, " int32, contiguous, at least ", std::to_string(n),
              " entries, on the device of the rows");
}
inline void status_word(const OptTensor& t, const torch::Device& dev, const char* op) {
  if (given(t)) ints(*t, dev, 1, op, "status");
}
// bf16 rows on a GPU, read or written in 16-byte pieces
inline void rows(const Tensor& t, int64_t cols, const char* op, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.scalar_type() == torch::kBFloat16, op, ": ", name, " bf16 CUDA tensor");
  TORCH_CHECK(t.dim() == 2 && t.size(1) >= cols && (t.size(1) <= 1 || t.stride(1) == 1), op, ": ", name, " [rows, >= ", std::to_string(cols), "], inner stride 1");
  TORCH_CHECK(t.size(0) <= 1 || t.stride(0) % 8 == 0, op, ": ", name, " row pitch must be a multiple of 8 elements");
  TORCH_CHECK(t.numel() == 0 || aligned16(t), op, ": ", name, " must be 16-byte aligned");
  TORCH_CHECK(t.size(0) < (int64_t(1) << 31), op, ": ", name, " has too many rows");
}
inline void written_rows(const Tensor& t, int64_t cols, const char* op, const char* name) {
  rows(t, cols, op, name);
  TORCH_CHECK(t.size(0) <= 1 || t.stride(0) >= cols, op, ": ", name, " rows overlap");
}
// the kernels count the K and V vectors of a call in 31 bits
inline void vectors(int64_t rows, int64_t heads, const char* op) { TORCH_CHECK(rows * 2 * heads < (int64_t(1) << 31), op, ": too many rows"); }
// k and v [blocks, heads, block size, D] of one type: bf16, or e4m3 with scale bytes [blocks, heads, block size]
inline agrpo::PagedCache cache(const Tensor& k, const Tensor& v, const OptTensor& ks, const OptTensor& vs, const torch::Device& dev, int64_t D, const char* op) {
  TORCH_CHECK(k.dim() == 4 && k.sizes() == v.sizes() && k.is_contiguous() && v.is_contiguous() && k.size(3) == D, op,
              ": cache [blocks, kv heads of this rank, block size, D]");
  TORCH_CHECK(k.scalar_type() == v.scalar_type() && k.device() == dev && v.device() == dev, op, ": both caches of one type, on the device of the rows");
  TORCH_CHECK(aligned16(k) && aligned16(v), op, ": cache must be 16-byte aligned");
  TORCH_CHECK(k.size(0) > 0 && k.size(1) > 0 && k.size(2) > 0 && k.size(0) * k.size(2) < (int64_t(1) << 31), op, ": cache without slots or with too many");
  agrpo::PagedCache c;
  c.k = k.data_ptr();
  c.v = v.data_ptr();
  c.num_blocks = (int)k.size(0);
  c.Hkv = (int)k.size(1);
  c.block_size = (int)k.size(2);
  c.D = (int)D;
  if (k.scalar_type() == torch::kBFloat16) {
    TORCH_CHECK(!given(ks) && !given(vs), op, ": a bf16 cache has no scales");
    return c;
  }
  TORCH_CHECK(k.scalar_type() == torch::kFloat8_e4m3fn, op, ": cache bf16 or float8_e4m3fn");
  TORCH_CHECK(D == 64 || D == 128, op, ": an 8-bit cache has head_dim 64 or 128");
  TORCH_CHECK(given(ks) && given(vs), op, ": an 8-bit cache needs k_scale and v_scale");
  for (const Tensor* t : {&*ks, &*vs})
    TORCH_CHECK(t->scalar_type() == torch::kUInt8 && t->device() == dev && t->is_contiguous() && t->dim() == 3 && t->size(0) == k.size(0) &&
                    t->size(1) == k.size(1) && t->size(2) == k.size(2), op, ": scales uint8 [blocks, kv heads, block size]");
  c.k_scale = ks->data_ptr<uint8_t>();
  c.v_scale = vs->data_ptr<uint8_t>();
  return c;
}

}  // namespace cache_args
