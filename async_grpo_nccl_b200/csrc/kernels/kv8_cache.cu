// KV cache in 8 bits: written from the rows of a prefill, written by a decode step with its rotation, read back into rows.
// All move bytes: a vector of D bf16 values is 2 D bytes on one side and D + 1 on the other. 16384 rows of 8 kv heads of 128 written and 16000 read back: 200 MB in
// 41 - 45 us (4.4 - 4.9 TB/s), about as long each; what is left above the 31 us of memory is the address arithmetic, a third of the instructions,
// and that a row is loaded when its slot is known (rows without a slot are not read). The bf16 cache read back: 16000 rows of 8 heads 22.8 us (5.7 TB/s).
#include <cuda_bf16.h>

#include "../common/ptx.cuh"
#include "../launchers.h"
#include "../launchers_cache.h"
#include "kv8.cuh"
#include "rope.cuh"

namespace agrpo {

namespace {

constexpr int kThreads = 256;

// Largest of the values of the `kLanes` lanes that share a vector.
template <int kLanes>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// 16 bf16 values: a whole sector at once where they lie on one.
__device__ __forceinline__ bool on_sector(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 31) == 0; }
__device__ __forceinline__ void load16(const __nv_bfloat16* p, uint4& a, uint4& b) {
  if (on_sector(p)) {
    uint32_t r[8];
    ld_global_32b(p, r);
    a = make_uint4(r[0], r[1], r[2], r[3]);
    b = make_uint4(r[4], r[5], r[6], r[7]);
  } else {
    a = reinterpret_cast<const uint4*>(p)[0];
    b = reinterpret_cast<const uint4*>(p)[1];
  }
}
__device__ __forceinline__ void store16(__nv_bfloat16* p, const uint4& a, const uint4& b) {
  if (on_sector(p)) {
    const uint32_t r[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    st_global_32b(p, r);
  } else {
    reinterpret_cast<uint4*>(p)[0] = a;
    reinterpret_cast<uint4*>(p)[1] = b;
  }
}

// Where vector `vec` of a call lies: row t, heads [0, Hkv) of K, then of V. 32-bit arithmetic: with 64-bit divisions the kernels were bound by them (16384 rows of 8 kv
// heads, written and read back: 61 us; more than one vector a group of lanes took longer).
struct Vector {
  unsigned t;
  int head;
  bool is_v;
};
__device__ __forceinline__ Vector vector_at(unsigned vec, int Hkv) {
  Vector x;
  x.t = vec / (2u * Hkv);
  const int which = static_cast<int>(vec - x.t * (2u * Hkv));
  x.is_v = which >= Hkv;
  x.head = x.is_v ? which - Hkv : which;
  return x;
}
// Its place in the cache, counted in vectors; -1: none. `first` lane reports a slot behind the cache.
__device__ __forceinline__ long long place_of(const PagedCache& c, int slot, int head, bool first, int* status) {
  if (slot < 0) return -1;
  const int block = slot / c.block_size;
  if (block >= c.num_blocks) {
    if (first) report_status(status, kStatusBadIndex);
    return -1;
  }
  return (static_cast<long long>(block) * c.Hkv + head) * c.block_size + (slot - block * c.block_size);
}

// D / 16 lanes a vector, 32 bytes of bf16 each: what is done once a lane (where the vector lies, its power) takes as many instructions as 16 values do.
template <int D>
__global__ void __launch_bounds__(kThreads)
kv8_write_kernel(const __nv_bfloat16* __restrict__ qkv, long long pitch, int k_col0, int v_col0, const int* __restrict__ slots, PagedCache c,
                 unsigned vectors, int* status) {
  constexpr int kLanes = D / 16;
  const int lane = threadIdx.x % kLanes;
  const unsigned vec = blockIdx.x * (kThreads / kLanes) + threadIdx.x / kLanes;
  uint4 x = make_uint4(0u, 0u, 0u, 0u), y = x;
  long long at = -1;
  const Vector w = vector_at(min(vec, vectors - 1), c.Hkv);
  if (vec < vectors) at = place_of(c, slots[w.t], w.head, lane == 0, status);
  if (at >= 0) {
    load16(qkv + w.t * pitch + (w.is_v ? v_col0 : k_col0) + w.head * D + lane * 16, x, y);
  }
  const int byte = kv8_scale_byte(group_max<kLanes>(max(kv8_top(x), kv8_top(y))));
  if (at < 0) return;
  const uint2 a = kv8_encode(x, byte), b = kv8_encode(y, byte);
  *reinterpret_cast<uint4*>(static_cast<uint8_t*>(w.is_v ? c.v : c.k) + at * D + lane * 16) = make_uint4(a.x, a.y, b.x, b.y);
  if (lane == 0) (w.is_v ? c.v_scale : c.k_scale)[at] = static_cast<uint8_t>(byte);
}

// D / 16 lanes a vector: 16 codes (or 32 bytes of bf16) each.
template <int D, bool k8>
__global__ void __launch_bounds__(kThreads)
kv_cache_read_kernel(PagedCache c, const int* __restrict__ slots, __nv_bfloat16* __restrict__ qkv, long long pitch, int k_col0, int v_col0,
                     unsigned vectors, int* status) {
  constexpr int kLanes = D / 16;
  const int lane = threadIdx.x % kLanes;
  const unsigned vec = blockIdx.x * (kThreads / kLanes) + threadIdx.x / kLanes;
  if (vec >= vectors) return;
  const Vector w = vector_at(vec, c.Hkv);
  const long long at = place_of(c, slots[w.t], w.head, lane == 0, status);
  if (at < 0) return;
  __nv_bfloat16* dst = qkv + w.t * pitch + (w.is_v ? v_col0 : k_col0) + w.head * D + lane * 16;
  const void* src = w.is_v ? c.v : c.k;
  if (k8) {
    const uint4 x = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(src) + at * D + lane * 16);
    const Kv8Scale s = kv8_scale((w.is_v ? c.v_scale : c.k_scale)[at]);
    const uint2 a = kv8_decode4(x.x, s), b = kv8_decode4(x.y, s), d = kv8_decode4(x.z, s), e = kv8_decode4(x.w, s);
    store16(dst, make_uint4(a.x, a.y, b.x, b.y), make_uint4(d.x, d.y, e.x, e.y));
  } else {
    uint4 a, b;
    load16(static_cast<const __nv_bfloat16*>(src) + at * D + lane * 16, a, b);
    store16(dst, a, b);
  }
}

// One CTA: 16 tokens of a sequence, all heads of K and V.
template <int D>
__global__ void __launch_bounds__(kThreads) kv8_unpack_kernel(const __grid_constant__ ChunkAttnArgs a, PagedCache c, PagedCache to, int* __restrict__ table) {
  constexpr int kLanes = D / 16;
  pdl_wait();
  pdl_launch();
  const int per_page = c.block_size / 16;
  const int at = blockIdx.x / per_page, part = blockIdx.x - at * per_page;  // block of the new cache
  const int b = at / a.max_blocks, i = at - b * a.max_blocks;
  if (i * c.block_size + part * 16 >= a.seq_lens[b] || a.q_starts[b + 1] == a.q_starts[b]) return;
  int page = a.block_tables[b * a.table_pitch + i];
  if (page < 0 || page >= c.num_blocks) {
    if (threadIdx.x == 0) report_status(a.status, kStatusBadIndex);
    page = 0;
  }
  if (threadIdx.x == 0 && part == 0) table[at] = at;
  const int lane = threadIdx.x % kLanes;
#pragma unroll 4
  for (int vec = threadIdx.x / kLanes; vec < 2 * c.Hkv * 16; vec += kThreads / kLanes) {  // 16 tokens of a head of K, .. of V
    const bool is_v = vec >= c.Hkv * 16;
    const int head = (vec >> 4) - (is_v ? c.Hkv : 0);
    const long long in_page = static_cast<long long>(head) * c.block_size + part * 16 + (vec & 15);
    const long long src = static_cast<long long>(page) * c.Hkv * c.block_size + in_page, dst = static_cast<long long>(at) * c.Hkv * c.block_size + in_page;
    const uint4 x = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(is_v ? c.v : c.k) + src * D + lane * 16);
    const Kv8Scale s = kv8_scale((is_v ? c.v_scale : c.k_scale)[src]);
    const uint2 d = kv8_decode4(x.x, s), e = kv8_decode4(x.y, s), f = kv8_decode4(x.z, s), g = kv8_decode4(x.w, s);
    const uint32_t y[8] = {d.x, d.y, e.x, e.y, f.x, f.y, g.x, g.y};
    st_global_32b(static_cast<__nv_bfloat16*>(is_v ? to.v : to.k) + dst * D + lane * 16, y);
  }
}

// One CTA a row; D / 16 lanes a head, each with 8 values of the lower half of the head and the 8 that they are rotated with. The rotated
// key is rounded to bf16, as the row keeps it, before it is quantised: a token's entry is the same from a decode step as from a prefill.
template <int D>
__global__ void __launch_bounds__(128)
rope_kv8_write_decode_kernel(__nv_bfloat16* __restrict__ qkv, long long pitch, const float* __restrict__ cos_t, const float* __restrict__ sin_t,
                             int max_pos, const int* __restrict__ block_tables, long long table_pitch, int max_blocks,
                             const int* __restrict__ seq_lens, PagedCache c, int Hq, int* status) {
  pdl_wait();
  pdl_launch();
  constexpr int kLanes = D / 16, kHalf = D / 2;
  const int b = blockIdx.x, lane = threadIdx.x % kLanes;
  const int len = seq_lens[b];
  const int pos = len > 0 ? len - 1 : 0;
  const int p = pos >= max_pos ? max_pos - 1 : pos;
  int blk = -1;
  if (len > 0) {
    blk = pos / c.block_size < max_blocks ? block_tables[b * table_pitch + pos / c.block_size] : -1;
    if (blk < 0 || blk >= c.num_blocks) {
      if (threadIdx.x == 0) report_status(status, kStatusBadIndex);
      blk = -1;
    }
  }
  const int heads = Hq + 2 * c.Hkv;
  const int per = 128 / kLanes;
  for (int h0 = 0; h0 < heads; h0 += per) {
    const int h = h0 + threadIdx.x / kLanes;
    const bool on = h < heads, is_v = h >= Hq + c.Hkv;
    uint4 lo = make_uint4(0u, 0u, 0u, 0u), hi = lo;
    uint4* x = reinterpret_cast<uint4*>(qkv + b * pitch + static_cast<long long>(h) * D + lane * 8);
    if (on) {
      lo = x[0];
      hi = x[kHalf / 8];
    }
    if (on && !is_v) {
      const float* cr = cos_t + static_cast<long long>(p) * kHalf + lane * 8;
      const float* sr = sin_t + static_cast<long long>(p) * kHalf + lane * 8;
      float cv[8], sv[8];
      *reinterpret_cast<float4*>(cv) = *reinterpret_cast<const float4*>(cr);
      *reinterpret_cast<float4*>(cv + 4) = *reinterpret_cast<const float4*>(cr + 4);
      *reinterpret_cast<float4*>(sv) = *reinterpret_cast<const float4*>(sr);
      *reinterpret_cast<float4*>(sv + 4) = *reinterpret_cast<const float4*>(sr + 4);
      uint32_t* l = reinterpret_cast<uint32_t*>(&lo);
      uint32_t* u = reinterpret_cast<uint32_t*>(&hi);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float a0 = __uint_as_float(l[i] << 16), a1 = __uint_as_float(l[i] & 0xffff0000u);
        float b0 = __uint_as_float(u[i] << 16), b1 = __uint_as_float(u[i] & 0xffff0000u);
        rope_rotate(a0, b0, cv[2 * i], sv[2 * i]);
        rope_rotate(a1, b1, cv[2 * i + 1], sv[2 * i + 1]);
        l[i] = pack_bf16x2(a0, a1);
        u[i] = pack_bf16x2(b0, b1);
      }
      x[0] = lo;
      x[kHalf / 8] = hi;
    }
    const int byte = kv8_scale_byte(group_max<kLanes>(max(kv8_top(lo), kv8_top(hi))));
    if (!on || h < Hq || blk < 0) continue;
    const int kh = is_v ? h - Hq - c.Hkv : h - Hq;
    const long long at = (static_cast<long long>(blk) * c.Hkv + kh) * c.block_size + pos % c.block_size;
    uint8_t* codes = static_cast<uint8_t*>(is_v ? c.v : c.k) + at * D + lane * 8;
    *reinterpret_cast<uint2*>(codes) = kv8_encode(lo, byte);
    *reinterpret_cast<uint2*>(codes + kHalf) = kv8_encode(hi, byte);
    if (lane == 0) (is_v ? c.v_scale : c.k_scale)[at] = static_cast<uint8_t>(byte);
  }
}

}  // namespace

static unsigned blocks_of(unsigned vectors, int lanes) { return (vectors + kThreads / lanes - 1) / (kThreads / lanes); }

void launch_kv8_write(const void* qkv, long long pitch, int k_col0, int v_col0, const int* slots, const PagedCache& c, int T, int* status,
                      cudaStream_t s) {
  const unsigned vectors = static_cast<unsigned>(T) * 2u * c.Hkv;
  if (vectors == 0) return;
  const auto run = [&](auto kernel) {
    kernel<<<blocks_of(vectors, c.D / 16), kThreads, 0, s>>>(static_cast<const __nv_bfloat16*>(qkv), pitch, k_col0, v_col0, slots, c, vectors, status);
    check_cuda(cudaGetLastError(), "kv8_write");
  };
  if (c.D == 128) run(kv8_write_kernel<128>);
  else run(kv8_write_kernel<64>);
}

void launch_kv_cache_read(const PagedCache& c, const int* slots, void* qkv, long long pitch, int k_col0, int v_col0, int T, int* status,
                          cudaStream_t s) {
  const unsigned vectors = static_cast<unsigned>(T) * 2u * c.Hkv;
  if (vectors == 0) return;
  const auto run = [&](auto kernel) {
    kernel<<<blocks_of(vectors, c.D / 16), kThreads, 0, s>>>(c, slots, static_cast<__nv_bfloat16*>(qkv), pitch, k_col0, v_col0, vectors, status);
    check_cuda(cudaGetLastError(), "kv_cache_read");
  };
  const bool k8 = c.k_scale != nullptr;
  if (c.D == 128) k8 ? run(kv_cache_read_kernel<128, true>) : run(kv_cache_read_kernel<128, false>);
  else k8 ? run(kv_cache_read_kernel<64, true>) : run(kv_cache_read_kernel<64, false>);
}

void launch_rope_kv8_write_decode(void* qkv, long long pitch, const float* cos_t, const float* sin_t, int max_pos, const int* block_tables,
                                  long long table_pitch, int max_blocks, const int* seq_lens, const PagedCache& c, int B, int Hq, int* status,
                                  cudaStream_t s) {
  if (B == 0) return;
  const auto run = [&](auto kernel) {
    launch_kernel(kernel, dim3(B), dim3(128), 0, s, "rope_kv8_write_decode", static_cast<__nv_bfloat16*>(qkv), pitch, cos_t, sin_t, max_pos,
                  block_tables, table_pitch, max_blocks, seq_lens, c, Hq, status);
  };
  if (c.D == 128) {
    AGRPO_PREFER_SMEM(rope_kv8_write_decode_kernel<128>);
    run(rope_kv8_write_decode_kernel<128>);
  } else {
    AGRPO_PREFER_SMEM(rope_kv8_write_decode_kernel<64>);
    run(rope_kv8_write_decode_kernel<64>);
  }
}

void launch_kv8_unpack(const ChunkAttnArgs& a, const PagedCache& c, const PagedCache& to, int* table, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>(to.num_blocks * (c.block_size / 16)));
  if (c.D == 128) launch_kernel(kv8_unpack_kernel<128>, grid, dim3(kThreads), 0, s, "kv8_unpack", a, c, to, table);
  else launch_kernel(kv8_unpack_kernel<64>, grid, dim3(kThreads), 0, s, "kv8_unpack", a, c, to, table);
}

}  // namespace agrpo
