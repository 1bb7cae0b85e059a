// Attention of the newest tokens of every sequence over the paged cache that already holds them.
//
// Sequence b has n = q_starts[b + 1] - q_starts[b] rows and L = seq_lens[b] tokens in the cache; its row i sees the keys 0 .. L - n + i.
// o = sum_k softmax_k(q.k s) v; a row that sees nothing is zero.
//
// One warp a row and head: a lane holds D / 32 dims, the running maximum and sum are those of the online softmax.
#include <cuda_bf16.h>

#include "../common/ptx.cuh"
#include "../launchers.h"
#include "../launchers_cache.h"
#include "kv8.cuh"

namespace agrpo {

namespace {

template <int D, bool k8>
__global__ void __launch_bounds__(128) paged_chunk_attn_kernel(ChunkAttnArgs a, PagedCache c, float scale_log2) {
  constexpr int kPer = D / 32;
  const int lane = threadIdx.x & 31;
  if (blockIdx.x == 0) {  // sequences whose rows are not rows of q: reported, and without rows
    for (int b = threadIdx.x; b < a.B; b += 128)
      if (a.q_starts[b] < 0 || a.q_starts[b + 1] < a.q_starts[b] || a.q_starts[b + 1] > a.Tq) report_status(a.status, kStatusBadIndex);
  }
  const long long item = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  const int row = static_cast<int>(item / a.Hq), head = static_cast<int>(item % a.Hq);
  if (row >= a.Tq) return;
  int lo = 0, hi = a.B;  // the last sequence that starts at or before the row
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (a.q_starts[mid] <= row) lo = mid;
    else hi = mid;
  }
  const int b = lo;
  if (row < a.q_starts[b] || row >= a.q_starts[b + 1]) return;  // behind the last sequence
  const int n = a.q_starts[b + 1] - a.q_starts[b];
  int len = a.seq_lens[b];
  if (len > static_cast<long long>(a.max_blocks) * c.block_size) {
    report_status(a.status, kStatusBadIndex);
    len = 0;
  }
  const int see = len - n + (row - a.q_starts[b]) + 1;
  const int kvh = head / (a.Hq / c.Hkv);
  const auto* qp = static_cast<const __nv_bfloat16*>(a.q) + row * a.ldq + static_cast<long long>(head) * D + lane * kPer;
  float q[kPer], o[kPer];
  for (int i = 0; i < kPer; ++i) {
    q[i] = __bfloat162float(qp[i]) * scale_log2;
    o[i] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  const auto load = [&](const void* base, const unsigned char* scale, long long at, float (&x)[kPer]) {
    if (k8) {
      const auto* p = static_cast<const uint8_t*>(base) + at * D + lane * kPer;
      uint32_t w = 0;
      for (int i = 0; i < kPer; ++i) w |= static_cast<uint32_t>(p[i]) << (8 * i);
      const uint2 v = kv8_decode4(w, kv8_scale(scale[at]));
      const uint32_t u[2] = {v.x, v.y};
      for (int i = 0; i < kPer; ++i) x[i] = __uint_as_float(i & 1 ? u[i / 2] & 0xffff0000u : u[i / 2] << 16);
    } else {
      const auto* p = static_cast<const __nv_bfloat16*>(base) + at * D + lane * kPer;
      for (int i = 0; i < kPer; ++i) x[i] = __bfloat162float(p[i]);
    }
  };
  for (int k = 0; k < see; ++k) {
    const int blk = a.block_tables[b * a.table_pitch + k / c.block_size];
    if (blk < 0 || blk >= c.num_blocks) {
      report_status(a.status, kStatusBadIndex);
      continue;
    }
    const long long at = (static_cast<long long>(blk) * c.Hkv + kvh) * c.block_size + k % c.block_size;
    float x[kPer], s = 0.f;
    load(c.k, c.k_scale, at, x);
    for (int i = 0; i < kPer; ++i) s += q[i] * x[i];
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    const float m_new = fmaxf(m, s);
    const float alpha = m == -INFINITY ? 0.f : exp2f(m - m_new), pr = exp2f(s - m_new);
    load(c.v, c.v_scale, at, x);
    for (int i = 0; i < kPer; ++i) o[i] = o[i] * alpha + pr * x[i];
    l = l * alpha + pr;
    m = m_new;
  }
  auto* op = static_cast<__nv_bfloat16*>(a.out) + row * a.ldo + static_cast<long long>(head) * D + lane * kPer;
  for (int i = 0; i < kPer; ++i) op[i] = __float2bfloat16(see > 0 ? o[i] / l : 0.f);
}

}  // namespace

void launch_paged_chunk_attn(const ChunkAttnArgs& a, const PagedCache& c, cudaStream_t s) {
  if (a.Tq == 0 || a.B == 0) return;
  const float scale_log2 = a.softmax_scale * 1.4426950408889634f;
  const unsigned blocks = static_cast<unsigned>((static_cast<long long>(a.Tq) * a.Hq + 3) / 4);
  const auto run = [&](auto kernel) {
    kernel<<<blocks, 128, 0, s>>>(a, c, scale_log2);
    check_cuda(cudaGetLastError(), "paged_chunk_attn");
  };
  const bool k8 = c.k_scale != nullptr;
  if (c.D == 128) k8 ? run(paged_chunk_attn_kernel<128, true>) : run(paged_chunk_attn_kernel<128, false>);
  else k8 ? run(paged_chunk_attn_kernel<64, true>) : run(paged_chunk_attn_kernel<64, false>);
}

}  // namespace agrpo
