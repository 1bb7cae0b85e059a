// Attention of the newest tokens of every sequence over the paged cache that already holds them.
//
// Sequence b has n = q_starts[b + 1] - q_starts[b] rows and L = seq_lens[b] tokens in the cache; its row i sees the keys 0 .. L - n + i.
// o = sum_k softmax_k(q.k s) v; a row that sees nothing is zero. Softmax in one pass: running maximum and sum, fp32. The query heads of a kv head are
// rows of one unit (row = token * G + head), so that a key is loaded once for the group. How the work is dealt out: paged_line.cuh. Up to 16 rows a
// sequence: paged_few_attn.cu. This file: more rows, bound by the tensor cores and by the exponentials (16 a cycle and SM: 128 x 128 of them take as long as
// the two products of a tile).
//
// A unit is two tiles of 128 rows, which share the keys and values. S = Q K^T and O += P V run on tcgen05 with S, P and O in tensor memory, a thread a row; one
// tile's softmax runs beside the other's products. Keys and values come page by page into a ring. 8-bit cache: eight warps bring the codes into shared memory, each
// thread what it will need, and turn them into the bf16 tiles that the products read (kv8.cuh); for sequences of many rows that is done once, ahead (kUnpackRows).
#include <cuda_bf16.h>

#include <algorithm>
#include <type_traits>

#include "../common/f32x2.cuh"
#include "../common/ptx.cuh"
#include "../common/tensormap.h"
#include "../launchers.h"
#include "../launchers_cache.h"
#include "kv8.cuh"
#include "paged_line.cuh"

namespace agrpo {

namespace {

constexpr int kBN = 128;  // keys a tile
// A bf16 tile of keys in shared memory: 8 rows of 128 bytes (64 columns, swizzled) are an atom, an 8-row group holds its D / 64 atoms side by side.
// So a whole page is one copy, whatever its length, and both products find equal strides between groups.
template <int D>
constexpr int kGroupBytes = D / 64 * 1024;

constexpr int kExtra = 1;      // a unit's beginning and end, in tiles
constexpr int kSeqRoom = 128;  // sequences that a CTA has at hand

template <int D, bool k8>
struct Shape {
  static constexpr int kRows = 256;                           // rows of a unit
  static constexpr int kSlotBytes = kBN * D * 2;              // a tile of K or V in bf16
  static constexpr int kQBytes = 2 * 128 * D * 2;
  static constexpr int kSlots = k8 ? 4 : 5;
  static constexpr int kRaw = k8 ? 2 : 0;                     // tiles of codes under way: one of K, one of V
  static constexpr int kMmaWarp = 8, kLoadWarp = 9;
  static constexpr int kConvWarp = 12;                        // 8 bits: five warpgroups, registers dealt out anew; warps 10 and 11 do nothing
  static constexpr int kCleanWarp = 10;                       // bf16
  static constexpr int kThreads = k8 ? 640 : 352;
  static constexpr int kRingOff = kQBytes;
  static constexpr int kRawOff = kRingOff + kSlots * kSlotBytes;
  static constexpr int kScaleOff = kRawOff + kRaw * kBN * D;
  static constexpr int kBarOff = kScaleOff + kRaw * kBN;
  static constexpr int kSeqOff = kBarOff + 256;
  static constexpr int kSmem = kSeqOff + kSeqRoom * 12 + 1024;  // with room to align
  static_assert(kSmem <= 232448, "shared memory");
  static_assert(kSlots * kSlotBytes >= 32768, "the line of 8192 sequences is measured in the ring's memory");
};

// 16 or 4 bytes into shared memory, zeros where `on` is false (nothing is read then).
__device__ __forceinline__ void cp_async_16(void* dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_4(void* dst, const void* src, bool on) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(on ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
// 8 bits: registers of the warpgroups, 128 x (144 + 144 + 64 + 64 + 64) = the launch's 640 x 96.
template <bool kOn, int kLeft>
__device__ __forceinline__ void give_registers() {
  if (kOn) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLeft));
}
template <bool kOn, int kMore>
__device__ __forceinline__ void take_registers() {
  if (kOn) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kMore));
}

// Pieces from, from + 32, .. of a bf16 tile of V: piece i is row i / 8, bytes (i % 8) * 16 of its atoms.
template <int D>
__device__ __forceinline__ uint4* piece(uint8_t* v, int i) {
  return reinterpret_cast<uint4*>(v + (i >> 6) * kGroupBytes<D> + (i & 63) * 16);
}
template <int D>
__device__ __forceinline__ bool some_odd(uint8_t* v, int from, int end) {
  uint32_t nan = 0u;
#pragma unroll 1
  for (int i = from; i < end; i += 32) {
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      const uint4 y = piece<D>(v, i)[c * 64];
      nan = times_zero(y.x, times_zero(y.y, times_zero(y.z, times_zero(y.w, nan))));
    }
  }
  return (nan & 0x7fff7fffu) != 0u;
}
template <int D>
__device__ __noinline__ void only_finite_rows(uint8_t* v, int from, int end) {
  for (int i = from; i < end; i += 32) {
    for (int c = 0; c < D / 64; ++c) {
      const uint4 y = piece<D>(v, i)[c * 64];
      piece<D>(v, i)[c * 64] = make_uint4(only_finite(y.x), only_finite(y.y), only_finite(y.z), only_finite(y.w));
    }
  }
}
// What was taken out of the products, at a piece's end: values that are no numbers at the keys from .. to - 1, for the rows that see them (up to `pos`). Adds them
// to O (a warp's rows, `tO` in tensor memory); 8 bits, where a vector that holds a NaN is all NaN: returns one in place of the row's sum l. Apart from the kernel's
// code, whose size counts.
template <int D, bool k8>
__device__ __noinline__ float add_taken_out(const LineParams& p, int b, int kvh, int from, int to, int pos, uint32_t tO, float l) {
  const auto row_of = [&](int key) -> long long {
    const int page = p.a.block_tables[b * p.a.table_pitch + key / p.c.block_size];
    if (page < 0 || page >= p.c.num_blocks) return -1;
    return (static_cast<long long>(page) * p.c.Hkv + kvh) * p.c.block_size + (key & (p.c.block_size - 1));
  };
  if (k8) {
    for (int key = from; key < min(to, pos + 1); ++key) {
      const long long row = row_of(key);
      if (row >= 0 && p.c.v_scale[row] == kKv8NanByte) l = __uint_as_float(0x7fffffffu);
    }
    __syncwarp();
    return l;
  }
#pragma unroll 1
  for (int c = 0; c < D / 32; ++c) {
    uint32_t o[32];
    tmem_ld_32x32(tO + c * 32, o);
    tc_wait_ld();
#pragma unroll 1
    for (int key = from; key < to; ++key) {
      const long long row = row_of(key);
      if (row < 0 || key > pos) continue;
      const auto* src = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.c.v) + row * D + c * 32);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint4 x = src[i];
        const uint32_t y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float lo = __uint_as_float(o[i * 8 + 2 * k]), hi = __uint_as_float(o[i * 8 + 2 * k + 1]);
          if (!is_finite(y[k])) lo += __uint_as_float(y[k] << 16);
          if (!is_finite(y[k] >> 16)) hi += __uint_as_float(y[k] & 0xffff0000u);
          o[i * 8 + 2 * k] = __float_as_uint(lo);
          o[i * 8 + 2 * k + 1] = __float_as_uint(hi);
        }
      }
    }
    __syncwarp();
    uint32_t lo[16], hi[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      lo[i] = o[i];
      hi[i] = o[16 + i];
    }
    tmem_st_32x16(tO + c * 32, lo);
    tmem_st_32x16(tO + c * 32 + 16, hi);
  }
  tc_wait_st();
  return l;
}

template <int D, bool k8>
__global__ void __launch_bounds__(Shape<D, k8>::kThreads, 1)
paged_chunk_attn_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                        const __grid_constant__ LineParams p) {
  using S = Shape<D, k8>;
  constexpr int kChunks = D / 64;
  constexpr uint32_t kIdescS = umma_idesc_bf16(128, kBN, 0, 0);
  constexpr uint32_t kIdescO = umma_idesc_bf16(128, D, 0, 1);
  constexpr uint32_t kColO = 256, kColP = 64;  // tensor memory: S of both tiles, O of both; P in the upper half of its S

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = smem + S::kRingOff;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBarOff);
  uint64_t* full = bars;               // [kSlots]; item 2 i is K of the CTA's tile i, 2 i + 1 its V, item i is in slot i % kSlots
  uint64_t* empty = bars + 5;          // [kSlots]
  uint64_t* q_full = bars + 10;
  uint64_t* q_empty = bars + 11;
  uint64_t* s_full = bars + 12;        // [2]: of the tiles of Q, as all that follow
  uint64_t* p_ready = bars + 14;
  uint64_t* o_done = bars + 16;        // after a piece's last product
  uint64_t* o_free = bars + 18;
  uint64_t* p_half = bars + 20;        // P of the upper 64 keys (bf16 cache)
  uint64_t* cleaned = bars + 22;       // [kSlots], bf16: V of a tile that had to be cleaned is
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 27);
  volatile int* odd = reinterpret_cast<volatile int*>(bars + 28);  // set once a value was taken out of the products
  int* status = p.a.status;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kSlots; ++i) {
      mbar_init(full + i, k8 ? 4 : 1);
      mbar_init(empty + i, k8 ? 1 : 2);
      mbar_init(cleaned + i, 1);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full + i, 1);
      mbar_init(p_ready + i, 4);
      mbar_init(p_half + i, 4);
      mbar_init(o_done + i, 1);
      mbar_init(o_free + i, 4);
    }
    fence_mbar_init();
    *odd = 0;
  }
  if (warp == S::kMmaWarp) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  pdl_wait();
  pdl_launch();
  measure_line<S::kThreads, kBN, kExtra>(p, reinterpret_cast<int*>(ring));
  const Share share = find_share<kBN, kExtra, 1>(p, reinterpret_cast<const int*>(ring), blockIdx.x, gridDim.x);
  const SeqCache near = {reinterpret_cast<int*>(smem + S::kSeqOff), share.b, kSeqRoom};
  near.fill(p);
  fence_proxy_async_smem();  // the line lies where the ring's copies go next
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  Walk<kBN, kExtra> w;  // every warp walks by itself
  w.start(p, share, near);
  const auto to_clean = [](int j, int keys, int hidden) { return keys < (j + 1) * kBN || hidden < (j + 1) * kBN; };

  if (warp == S::kLoadWarp) {
    give_registers<k8, 64>();
    // ---------------------------------------------------------------- copies
    // The first tile of a piece goes ahead of its Q, which has to wait for the last products with the one before. (8 bits: Q alone comes from here.)
    int item = 0, n_q = 0;
    bool ok = true;
    for (; w.more() && ok; w.next(p)) {
      const int* table = p.a.block_tables + w.b * p.a.table_pitch;
      const int keys = unit_keys(p, w.s, w.qb);
      const int bs = p.c.block_size;
      const auto page_id = [&](int j) {
        const int key = j * kBN + lane * bs;
        int id = lane * bs < kBN && key < keys ? table[key / bs] : 0;
        if (id < 0 || id >= p.c.num_blocks) {
          report_status(status, kStatusBadIndex);
          id = 0;
        }
        return id;
      };
      int id = k8 ? 0 : page_id(w.j0);
      for (int j = w.j0; j < (k8 ? w.j0 + 1 : w.j1) && ok; ++j) {
        if (!k8) {
          const int pages = (min(kBN, keys - j * kBN) + bs - 1) / bs;  // none in a unit without keys
          const long long row = (static_cast<long long>(id) * p.c.Hkv + w.kvh) * bs;
          if (j + 1 < w.j1) id = page_id(j + 1);
#pragma unroll 1
          for (int v = 0; v < 2 && ok; ++v, ++item) {
            const int slot = item % S::kSlots, round = item / S::kSlots;
            if (round > 0 && !mbar_wait(empty + slot, (round - 1) & 1)) {
              report_status(status, kStatusWaitEmptyTimeout);
              ok = false;
              break;
            }
            __syncwarp();
            if (lane == 0) mbar_expect_tx(full + slot, pages * bs * D * 2);
            __syncwarp();
            if (lane < pages)
              tma_load_4d(ring + slot * S::kSlotBytes + lane * (bs / 8) * kGroupBytes<D>, v ? &tmV : &tmK, full + slot, 0, 0, 0, static_cast<int>(row >> 3));
          }
        }
        if (j == w.j0 && ok) {
          if (n_q > 0 && !mbar_wait(q_empty, (n_q - 1) & 1)) {
            report_status(status, kStatusWaitEmptyTimeout);
            ok = false;
            break;
          }
          ++n_q;
          const int boxes = w.tokens(p) > p.tile_tokens ? 2 : 1;
          __syncwarp();
          if (lane == 0) mbar_expect_tx(q_full, boxes * kChunks * p.G * p.tile_tokens * 128);
          __syncwarp();
          if (lane < boxes * kChunks) {
            const int box = lane / kChunks, ch = lane % kChunks;
            tma_load_3d(smem + box * (128 * D * 2) + ch * (128 * 128), &tmQ, q_full, ch * 64, w.kvh * p.G, w.s.row0 + w.qb * p.tokens + box * p.tile_tokens);
          }
        }
      }
    }
  } else if (warp == S::kMmaWarp) {
    give_registers<k8, 64>();
    // ---------------------------------------------------------------- products
    const uint32_t aQ = smem_u32(smem), aRing = smem_u32(ring);
    int tile = 0, n_q = 0;          // tiles and pieces so far
    int n_p[2] = {0, 0};            // of each tile of Q: softmaxes waited for
    int n_o[2] = {0, 0};            // pieces finished
    uint32_t n_clean = 0;           // of each slot: parity of its cleanings (a bit)
    bool ok = true;
    const auto wait = [&](uint64_t* bar, int parity, int code) {
      if (ok && !mbar_wait(bar, parity)) {
        report_status(status, code);
        ok = false;
      }
      return ok;
    };
    const auto slot_wait = [&](int item) { return wait(full + item % S::kSlots, (item / S::kSlots) & 1, kStatusWaitFullTimeout); };
    const auto scores = [&](int t, int item) {  // S_t = Q_t K^T
      if (elect_one()) {
        const uint32_t q = aQ + t * (128 * D * 2), k = aRing + (item % S::kSlots) * S::kSlotBytes;
        // 8 bits: unrolled, the descriptors would take more registers than these warps have left
#pragma unroll(k8 ? 1 : D / 16)
        for (int i = 0; i < D / 16; ++i) {
          tc_mma_f16(tmem + t * 128, umma_smem_desc(q + (i / 4) * (128 * 128) + (i % 4) * 32, 16, 1024),
                     umma_smem_desc(k + (i / 4) * 1024 + (i % 4) * 32, 16, kGroupBytes<D>), kIdescS, i > 0 ? 1u : 0u);
        }
        tc_commit(s_full + t);
      }
      __syncwarp();
    };
    // O_t (+)= P_t V, 16 keys a step. Both caches take a tile's keys from the middle on, then from the beginning: equal values, equal sums.
    const auto values = [&](auto steps, int t, int item, int from, bool first) {
      if (elect_one()) {
        const uint32_t v = aRing + (item % S::kSlots) * S::kSlotBytes;
#pragma unroll(k8 ? 1 : decltype(steps)::value)
        for (int s = 0; s < decltype(steps)::value; ++s) {
          const int i = (from + s) % (kBN / 16);
          tc_mma_f16_ts(tmem + kColO + t * 128, tmem + t * 128 + kColP + i * 8, umma_smem_desc(v + i * 2 * kGroupBytes<D>, 1024, kGroupBytes<D>), kIdescO,
                        (!first || s > 0) ? 1u : 0u);
        }
      }
      __syncwarp();
    };
    const auto commit = [&](uint64_t* bar) {
      if (elect_one()) tc_commit(bar);
      __syncwarp();
    };
    for (; w.more() && ok; w.next(p)) {
      const int keys = unit_keys(p, w.s, w.qb), hidden = first_hidden(p, w.s, w.qb);
      if (!wait(q_full, n_q++ & 1, kStatusWaitFullTimeout)) break;
      const int end[2] = {w.end_of(p, 0), w.end_of(p, 1)};
      if (!slot_wait(2 * tile)) break;
      tc_fence_after();
      for (int t = 0; t < 2; ++t)
        if (w.j0 < end[t]) scores(t, 2 * tile);
      commit(empty + (2 * tile) % S::kSlots);
      for (int j = w.j0; j < w.j1 && ok; ++j, ++tile) {
        const bool more = j + 1 < w.j1;
        if (!more) commit(q_empty);
        if (!slot_wait(2 * tile + 1)) break;
        bool cleaning = !k8 && to_clean(j, keys, hidden);
        const auto is_clean = [&] {
          const int slot = (2 * tile + 1) % S::kSlots;
          if (cleaning) wait(cleaned + slot, (n_clean >> slot) & 1, kStatusWaitFullTimeout);
          if (cleaning) n_clean ^= 1u << slot;
          cleaning = false;
          return ok;
        };
        for (int t = 0; t < 2 && ok; ++t) {
          if (j >= end[t]) continue;
          if (j == w.j0 && n_o[t] > 0 && !wait(o_free + t, (n_o[t] - 1) & 1, kStatusWaitTmemEmptyTimeout)) break;
          // The upper half's products run beside the lower half's exponentials (4096 tokens behind 12288: 694 -> 669 us in a
          // short loop; in one of seconds the power limit makes it 795). 8 bits: no gain, the warps that
          // convert are behind.
          using Half = std::integral_constant<int, kBN / 32>;
          if (!k8) {
            if (!wait(p_half + t, n_p[t] & 1, kStatusWaitTmemFullTimeout) || !is_clean()) break;
            tc_fence_after();
            values(Half{}, t, 2 * tile + 1, kBN / 32, j == w.j0);
          }
          if (!wait(p_ready + t, n_p[t]++ & 1, kStatusWaitTmemFullTimeout)) break;
          tc_fence_after();
          if (k8) values(std::integral_constant<int, kBN / 16>{}, t, 2 * tile + 1, kBN / 32, j == w.j0);
          else values(Half{}, t, 2 * tile + 1, 0, false);
          if (j + 1 >= end[t]) {
            commit(o_done + t);
            ++n_o[t];
          } else {  // over the P that the products before have read
            if (!slot_wait(2 * tile + 2)) break;
            tc_fence_after();
            scores(t, 2 * tile + 2);
          }
        }
        if (!is_clean()) break;
        commit(empty + (2 * tile + 1) % S::kSlots);
        if (more) {
          slot_wait(2 * tile + 2);  // where no tile of Q takes part any more, it still counts as read
          commit(empty + (2 * tile + 2) % S::kSlots);
        }
      }
    }
  } else if (!k8 && warp >= S::kCleanWarp) {
    // ---------------------------------------------------------------- values that must not meet a probability of zero
    // Rows of V behind the last key (whatever the page held before) become zero, and so do values that are no numbers at keys that some rows do not see. A
    // warp for that, as soon as V is there: the warp that issues the products took 8 us of 85 for it (24 sequences of up to 900 new tokens), this one 3. It takes part
    // in the release of every slot, so that it is never a round of the ring ahead or behind.
    int item = 0;
    bool ok = true;
    for (; w.more() && ok; w.next(p)) {
      const int keys = unit_keys(p, w.s, w.qb), hidden = first_hidden(p, w.s, w.qb);
      for (int i = 2 * w.j0; i < 2 * w.j1; ++i, ++item) {
        const int slot = item % S::kSlots, j = i >> 1;
        if (!mbar_wait(full + slot, (item / S::kSlots) & 1)) {
          report_status(status, kStatusWaitFullTimeout);
          ok = false;
          break;
        }
        __syncwarp();
        if (!(i & 1) || !to_clean(j, keys, hidden)) {
          if (lane == 0) mbar_arrive(empty + slot);
          continue;
        }
        uint8_t* v = ring + slot * S::kSlotBytes;
        const int from = max(hidden - j * kBN, 0), end = max(min(keys - j * kBN, kBN), 0);
        if (some_odd<D>(v, from * 8 + lane, end * 8)) {
          only_finite_rows<D>(v, from * 8 + lane, end * 8);
          *odd = 1;
        }
#pragma unroll 1
        for (int i = end * 8 + lane; i < kBN * 8; i += 32) {
#pragma unroll
          for (int c = 0; c < kChunks; ++c) piece<D>(v, i)[c * 64] = make_uint4(0u, 0u, 0u, 0u);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(cleaned + slot);
          mbar_arrive(empty + slot);
        }
      }
    }
  } else if (k8 && warp >= S::kConvWarp) {
    give_registers<k8, 64>();
    // ---------------------------------------------------------------- 8 bits to bf16
    // 16 codes a thread and step. A warp has 8 rows of every 32 (two steps for them if D = 128): eight lanes take four pieces of a row and the other
    // four of the next one, so that their 16-byte writes fall into eight different bank groups. A thread copies the pieces that it will turn into bf16
    // itself, so nobody waits for anybody else's copies. (Bulk copies of pages of 16 tokens, 2 KB, took 54 cycles each to issue.)
    const int v = (warp - S::kConvWarp) >> 2, cw = (warp - S::kConvWarp) & 3;  // four warps for K, four for V, with slots of their own
    constexpr int kPerRows = D / 64;             // steps for the same rows
    uint8_t* raw = smem + S::kRawOff + v * (kBN * D) + (cw * 32 + lane) * 16;
    uint8_t* raw_scale = smem + S::kScaleOff + v * kBN + cw * 32;
    const auto* codes = static_cast<const uint8_t*>(v ? p.c.v : p.c.k);
    const auto* scales = v ? p.c.v_scale : p.c.k_scale;
    const int sub = lane >> 2;                   // row of the eight
    Walk<kBN, kExtra> a = w;                             // the copies' walk
    int a_j = a.j0, page = 0;
    // Blocks of the table that hold this warp's rows of the tile: lane i < 4 those from row 32 i + 8 cw on.
    const auto pages = [&] {
      if (!a.more()) return;
      const int key = a_j * kBN + (lane & 3) * 32 + cw * 8;
      page = key < unit_keys(p, a.s, a.qb) ? p.a.block_tables[a.b * p.a.table_pitch + key / p.c.block_size] : 0;
    };
    const auto copy = [&] {
      if (a.more()) {
        if (page < 0 || page >= p.c.num_blocks) {
          report_status(status, kStatusBadIndex);
          page = 0;
        }
        const int bs = p.c.block_size;
        const int valid = unit_keys(p, a.s, a.qb) - a_j * kBN;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int r = q * 32 + cw * 8 + sub;
          const long long row = (static_cast<long long>(__shfl_sync(0xffffffffu, page, q)) * p.c.Hkv + a.kvh) * bs + ((a_j * kBN + r) & (bs - 1));
#pragma unroll
          for (int h = 0; h < kPerRows; ++h) {
            const int piece = D == 128 ? (lane & 3) + 4 * ((sub & 1) ^ h) : lane & 3;
            cp_async_16(raw + (q * kPerRows + h) * 2048, codes + row * D + piece * 16, r < valid);
          }
        }
        // the factors' bytes: four rows a lane
        const int pq = __shfl_sync(0xffffffffu, page, lane >> 1 & 3), r = (lane >> 1 & 3) * 32 + cw * 8 + (lane & 1) * 4;
        if (lane < 8) {
          const long long row = (static_cast<long long>(pq) * p.c.Hkv + a.kvh) * bs + ((a_j * kBN + r) & (bs - 1));
          cp_async_4(raw_scale + lane * 4, scales + row, r < valid);
        }
        if (++a_j == a.j1) {
          a.next(p);
          a_j = a.j0;
        }
        pages();
      }
    };
    pages();
    copy();
    int item = v;
    bool ok = true;
    for (; w.more() && ok; w.next(p)) {
      for (int j = w.j0; j < w.j1; ++j, item += 2) {
        const int slot = item % S::kSlots, round = item / S::kSlots;
        cp_async_wait_all();
        __syncwarp();
        // of row 32 (lane / 8) + 8 cw + lane % 8. Behind the last key the codes are zero, and the factor has to be a number
        const int left = unit_keys(p, w.s, w.qb) - j * kBN - cw * 8;
        const int r = (lane >> 3) * 32 + (lane & 7);
        int byte = r < left ? raw_scale[lane] : 0;
        if (v && byte == kKv8NanByte && j * kBN + cw * 8 + r >= first_hidden(p, w.s, w.qb)) {
          byte = 0;
          *odd = 1;
        }
        const Kv8Scale s = kv8_scale(byte);
        const bool twice = __any_sync(0xffffffffu, s.twice);         // some value above 448 * 2^7
        if (round > 0 && !mbar_wait(empty + slot, (round - 1) & 1)) {
          report_status(status, kStatusWaitEmptyTimeout);
          ok = false;
          break;
        }
        uint8_t* dst = ring + slot * S::kSlotBytes + cw * kGroupBytes<D> + sub * 128;
        const auto convert = [&](auto both) {
#pragma unroll 2
          for (int q = 0; q < 4; ++q) {
            Kv8Scale f;
            f.first = __shfl_sync(0xffffffffu, s.first, q * 8 + sub);
            f.second = decltype(both)::value ? __shfl_sync(0xffffffffu, s.second, q * 8 + sub) : 0u;
            f.twice = decltype(both)::value ? __shfl_sync(0xffffffffu, static_cast<int>(s.twice), q * 8 + sub) != 0 : false;
#pragma unroll
            for (int h = 0; h < kPerRows; ++h) {
              const uint4 x = *reinterpret_cast<const uint4*>(raw + (q * kPerRows + h) * 2048);
              const uint2 e = kv8_decode4(x.x, f), g = kv8_decode4(x.y, f), y = kv8_decode4(x.z, f), z = kv8_decode4(x.w, f);
              uint8_t* row = dst + q * 4 * kGroupBytes<D> + (D == 128 ? ((sub & 1) ^ h) * 1024 : 0);
              const int ch = (lane & 3) * 2;
              *reinterpret_cast<uint4*>(row + ((ch ^ sub) << 4)) = make_uint4(e.x, e.y, g.x, g.y);
              *reinterpret_cast<uint4*>(row + (((ch + 1) ^ sub) << 4)) = make_uint4(y.x, y.y, z.x, z.y);
            }
          }
        };
        if (twice) convert(std::true_type{});
        else convert(std::false_type{});
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(full + slot);
        copy();
      }
    }
    cp_async_wait_all();
  } else if (warp < S::kMmaWarp) {
    take_registers<k8, 144>();
    // ---------------------------------------------------------------- softmax, results
    const int t = warp >> 2, quarter = warp & 3;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t tO = tmem + lanes + kColO + t * 128, tS = tmem + lanes + t * 128;
    const int r = quarter * 32 + lane;  // row of the tile
    const int r_tok = r / p.G, r_head = r - r_tok * p.G;
    int tile = 0, n_o = 0;
    bool ok = true;
    if (threadIdx.x == 0) p.desc[blockIdx.x] = make_int4(0, 0, 0, 0);
    int flat = share.before;
    for (; w.more() && ok; flat += w.length(), w.next(p)) {
      const int rows = max(min(p.tile_tokens, w.tokens(p) - t * p.tile_tokens), 0) * p.G;  // of this tile
      const bool busy = quarter * 32 < rows;                                               // the warp has rows
      const int end = w.end_of(p, t);
      const int tile_pos = w.s.len - w.s.n + w.qb * p.tokens + t * p.tile_tokens;  // position of the tile's first row
      const int first_pos = tile_pos + quarter * 32 / p.G;                         // of the warp's first row
      const int pos = tile_pos + r_tok;                                            // the row sees the keys up to its position
      float m = -INFINITY;
      float2 l2 = make_float2(0.f, 0.f);
      for (int j = w.j0; j < end; ++j, ++tile) {
        if (!mbar_wait(s_full + t, tile & 1)) {
          report_status(status, kStatusWaitTmemFullTimeout);
          ok = false;
          break;
        }
        tc_fence_after();
        if (busy) {
          const int key0 = j * kBN;
          const int see = pos - key0;                                         // columns up to this one
          // Rescales O and l where the maximum grew by more than 2^8. The products of the tile before are complete: the scores were issued after them.
          const auto raise = [&](float mx) {
            mx *= p.scale_log2;
            float alpha = 1.f;
            if (mx > m + 8.f) {
              alpha = m == -INFINITY ? 0.f : exp2f(m - mx);
              m = mx;
            }
            if (__any_sync(0xffffffffu, alpha != 1.f) && j > w.j0) {
#pragma unroll 1
              for (int c = 0; c < D / 32; ++c) {
                uint32_t o[32];
                tmem_ld_32x32(tO + c * 32, o);
                tc_wait_ld();
                uint32_t a[16], b[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                  a[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                  b[i] = __float_as_uint(__uint_as_float(o[16 + i]) * alpha);
                }
                tmem_st_32x16(tO + c * 32, a);
                tmem_st_32x16(tO + c * 32 + 16, b);
              }
            }
            l2.x *= alpha;
            l2.y *= alpha;
          };
          const auto top = [&](const uint32_t (&s)[32], float (&mx)[4]) {
#pragma unroll
            for (int i = 0; i < 32; i += 2) mx[i / 2 & 3] = max3(mx[i / 2 & 3], __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
          };
          const auto exponentials = [&](const uint32_t (&s)[32], uint32_t dst) {  // 32 columns of P
            const float base = m == -INFINITY ? 0.f : m;
            const float2 sc = make_float2(p.scale_log2, p.scale_log2), neg = make_float2(-base, -base);
            uint32_t pk[16];
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              const float2 z = fma2(make_float2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), sc, neg);
              const float2 e = make_float2(exp2f(z.x), exp2f(z.y));
              l2 = add2(l2, e);
              pk[i / 2] = pack_bf16x2(e.x, e.y);
            }
            tmem_st_32x16(dst, pk);
          };
          const auto half_done = [&] {
            if (k8) return;
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_half + t);
          };
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
          if (first_pos < key0 + kBN - 1) {
            // Some row of the warp does not see the whole tile: 32 columns at a time, in a loop. A unit has one or two such tiles; unrolled, their code
            // came from L2 every time (3.5 us a tile, 1.2 for the others).
            const auto hide = [&](int c, uint32_t (&s)[32]) {
              const int n = see - c * 32;
              const uint32_t seen = n < 0 ? 0u : (n >= 31 ? 0xffffffffu : (2u << n) - 1u);
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (!((seen >> i) & 1u)) s[i] = 0xff800000u;
            };
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
              uint32_t s[32];
              tmem_ld_32x32(tS + c * 32, s);
              tc_wait_ld();
              hide(c, s);
              top(s, mx);
            }
            raise(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])));
#pragma unroll 1
            for (int c = 3; c >= 0; --c) {  // backwards: P of 32 columns lies over columns that have been read
              uint32_t s[32];
              tmem_ld_32x32(tS + c * 32, s);
              tc_wait_ld();
              hide(c, s);
              exponentials(s, tS + kColP + c * 16);
              if (c == 2) half_done();
            }
          } else {
            uint32_t s0[32], s1[32];
            tmem_ld_32x32(tS, s0);
            tmem_ld_32x32(tS + 32, s1);
            tc_wait_ld();
            top(s0, mx);
            top(s1, mx);
            tmem_ld_32x32(tS + 64, s0);
            tmem_ld_32x32(tS + 96, s1);
            tc_wait_ld();
            top(s0, mx);
            top(s1, mx);
            raise(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])));
            // the upper half first: P lies over it
            exponentials(s0, tS + kColP + 32);
            exponentials(s1, tS + kColP + 48);
            half_done();
            tmem_ld_32x32(tS, s0);
            tmem_ld_32x32(tS + 32, s1);
            tc_wait_ld();
            exponentials(s0, tS + kColP);
            exponentials(s1, tS + kColP + 16);
          }
          tc_wait_st();
        } else if (!k8 && lane == 0) {
          mbar_arrive(p_half + t);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_ready + t);
      }
      if (!ok) break;
      float l = l2.x + l2.y;
      const bool any = end > w.j0;  // else O holds nothing of this piece
      if (any && !mbar_wait(o_done + t, n_o++ & 1)) {
        report_status(status, kStatusWaitTmemFullTimeout);
        ok = false;
        break;
      }
      tc_fence_after();
      if (any && busy && __any_sync(0xffffffffu, *odd != 0))  // one answer for the warp
        l = add_taken_out<D, k8>(p, w.b, w.kvh, max(first_hidden(p, w.s, w.qb), w.j0 * kBN), min(unit_keys(p, w.s, w.qb), w.j1 * kBN), pos, tO, l);
      if (busy) {
        const bool whole = w.whole(), valid = r < rows;
        // a lane's stores are a row of their own: whole 32-byte sectors where the output's rows allow it
        const bool wide = ((reinterpret_cast<uintptr_t>(p.a.out) | static_cast<uintptr_t>(p.a.ldo * 2)) & 31) == 0;
        const float inv = l != 0.f ? 1.f / l : 0.f;
        const long long part = static_cast<long long>(w.part(blockIdx.x)) * S::kRows + t * 128 + r;
        auto* dst = static_cast<__nv_bfloat16*>(p.a.out) + (w.s.row0 + w.qb * p.tokens + t * p.tile_tokens + r_tok) * p.a.ldo +
                    static_cast<long long>(w.kvh * p.G + r_head) * D;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          tmem_ld_32x32(tO + c * 32, o);
          tc_wait_ld();
          if (!any) {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0u;
          }
          if (valid && whole) {
#pragma unroll
            for (int i = 0; i < 32; i += 16) {
              uint32_t y[8];
#pragma unroll
              for (int k = 0; k < 8; ++k) y[k] = pack_bf16x2(__uint_as_float(o[i + 2 * k]) * inv, __uint_as_float(o[i + 2 * k + 1]) * inv);
              if (wide) {
                st_global_32b(dst + c * 32 + i, y);
              } else {
                *reinterpret_cast<uint4*>(dst + c * 32 + i) = make_uint4(y[0], y[1], y[2], y[3]);
                *reinterpret_cast<uint4*>(dst + c * 32 + i + 8) = make_uint4(y[4], y[5], y[6], y[7]);
              }
            }
          } else if (valid) {
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
              uint32_t y[8];
#pragma unroll
              for (int k = 0; k < 8; ++k) y[k] = o[i + k];
              st_global_32b(p.part_o + part * D + c * 32 + i, y);
            }
          }
        }
        if (valid && !whole) *reinterpret_cast<float2*>(p.part_ml + part * 2) = make_float2(m, l);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0 && any) mbar_arrive(o_free + t);
      if (threadIdx.x == 0 && w.j0 == 0 && w.j1 < w.nk)
        p.desc[blockIdx.x] = make_int4(w.s.row0 + w.qb * p.tokens, w.tokens(p), w.kvh, w.last_worker(share, flat));
    }
  } else {
    give_registers<k8, 64>();
  }

  tc_fence_before();
  __syncthreads();
  if (warp == S::kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int D, bool k8>
void launch(LineParams p, int num_sms, void* scratch, cudaStream_t s) {
  using S = Shape<D, k8>;
  p.tile_tokens = 128 / p.G;
  p.tokens = 2 * p.tile_tokens;
  place_scratch(p, scratch, num_sms, S::kRows);
  const uint64_t dims[3] = {static_cast<uint64_t>(D), static_cast<uint64_t>(p.a.Hq), static_cast<uint64_t>(p.a.Tq)};
  const uint64_t pitch[2] = {static_cast<uint64_t>(D), static_cast<uint64_t>(p.a.ldq)};
  const uint32_t box[3] = {64, static_cast<uint32_t>(p.G), static_cast<uint32_t>(p.tile_tokens)};
  const CUtensorMap tq = make_tmap_nd<3>(p.a.q, dims, pitch, box);
  CUtensorMap tk = tq, tv = tq;  // 8 bits: not used
  if (!k8) {
    // 64 columns, the 8 rows of a group, the columns' chunks, groups
    const uint64_t kdims[4] = {64, 8, D / 64, static_cast<uint64_t>(p.c.num_blocks) * p.c.Hkv * p.c.block_size / 8};
    const uint64_t kpitch[3] = {D, 64, 8 * D};
    const uint32_t kbox[4] = {64, 8, D / 64, static_cast<uint32_t>(p.c.block_size / 8)};
    tk = make_tmap_nd<4>(p.c.k, kdims, kpitch, kbox);
    tv = make_tmap_nd<4>(p.c.v, kdims, kpitch, kbox);
  }
  auto kernel = paged_chunk_attn_kernel<D, k8>;
  AGRPO_SET_MAX_DYN_SMEM(kernel, S::kSmem, "paged_chunk_attn smem attr");
  launch_kernel(kernel, dim3(num_sms), dim3(S::kThreads), S::kSmem, s, "paged_chunk_attn", tq, tk, tv, p);
  launch_combine<D>(p, num_sms, s);
}

// Rows of a unit: 8 or 16 (the kernel of few rows) where the sequences have so many on average, else 256. (32 sequences of 2 to 6 rows of a group of 7 over 500
// - 4000 tokens, bf16: 46 us here, 62 us in units of 16.) The lengths are the device's, so the average counts sequences without rows: a few long prompts among hundreds of
// idle ones take units of 8, single tokens beside one long prompt units of 256. The results are right, the time is not the best.
int unit_rows(const ChunkAttnArgs& a, const PagedCache& c) {
  const int G = a.Hq / c.Hkv;
  const long long rows = static_cast<long long>(a.Tq) * G;
  if (G <= 8 && rows <= 8ll * a.B) return 8;
  return G <= 16 && rows <= 16ll * a.B ? 16 : 256;
}

// An 8-bit cache is converted to bf16 once, ahead of the attention, where every key would otherwise be converted for four units or more (on average): a tile of keys
// takes a unit 1.4 times as long from 8 bits as from bf16, and writing it out as long as a third of such a tile. 4096 rows of 28 heads behind 12288 tokens
// 955 -> 676 us (short loops); four units over 16000 tokens 51.4 -> 49.8, three 51.5 -> 54. Up to about the size of L2, where the copy stays; it is the allocator's again
// after the call. The copy has room for full tables, whatever the lengths: tables wider than the longest sequence needs may be too wide for it.
constexpr long long kUnpackMost = 128ll << 20;
constexpr long long kUnpackRows = 1024;  // of a sequence
struct Unpacked {
  long long table = 0, cache = 0;  // bytes; 0: the keys are converted by the attention
};
Unpacked unpacked(const ChunkAttnArgs& a, const PagedCache& c) {
  Unpacked u;
  const long long blocks = static_cast<long long>(a.B) * a.max_blocks;
  const long long bytes = blocks * c.Hkv * c.block_size * c.D * 2;
  if (c.k_scale == nullptr || static_cast<long long>(a.Tq) * (a.Hq / c.Hkv) < kUnpackRows * a.B || 2 * bytes > kUnpackMost) return u;
  u.table = (blocks * 4 + 255) / 256 * 256;
  u.cache = bytes;
  return u;
}

}  // namespace

long long paged_chunk_attn_tiles(const ChunkAttnArgs& a, const PagedCache& c) {
  const int rows = unit_rows(a, c), G = a.Hq / c.Hkv;
  const long long units = a.Tq / (rows == 256 ? 2 * (128 / G) : rows / G) + std::min(a.B, a.Tq);
  const long long keys = static_cast<long long>(a.max_blocks) * c.block_size;
  return units * c.Hkv * (rows == 256 ? keys / kBN + 2 : keys / 16 + 6);  // with each one's beginning, and a tile that is not full
}

long long paged_chunk_attn_scratch(const ChunkAttnArgs& a, const PagedCache& c, int num_sms) {
  const long long line = line_scratch(num_sms, unit_rows(a, c), c.D);
  const Unpacked u = unpacked(a, c);
  return u.cache ? (line + 255) / 256 * 256 + u.table + 2 * u.cache : line;
}

void launch_paged_chunk_attn(const ChunkAttnArgs& a, const PagedCache& c, int num_sms, void* scratch, cudaStream_t s) {
  if (a.Tq == 0 || a.B == 0) return;
  const int rows = unit_rows(a, c);
  if (rows <= 16) return launch_paged_few_attn(a, c, rows, num_sms, scratch, s);
  LineParams p = {};
  p.a = a;
  p.c = c;
  p.G = a.Hq / c.Hkv;
  p.scale_log2 = a.softmax_scale * 1.4426950408889634f;
  const Unpacked u = unpacked(a, c);
  if (u.cache) {
    auto* table = static_cast<uint8_t*>(scratch) + (line_scratch(num_sms, rows, c.D) + 255) / 256 * 256;
    p.c.k = table + u.table;
    p.c.v = table + u.table + u.cache;
    p.c.k_scale = p.c.v_scale = nullptr;
    p.c.num_blocks = a.B * a.max_blocks;
    p.a.block_tables = reinterpret_cast<int*>(table);
    p.a.table_pitch = a.max_blocks;
    launch_kv8_unpack(a, c, p.c, reinterpret_cast<int*>(table), s);
    return c.D == 128 ? launch<128, false>(p, num_sms, scratch, s) : launch<64, false>(p, num_sms, scratch, s);
  }
  const bool k8 = c.k_scale != nullptr;
  if (c.D == 128) k8 ? launch<128, true>(p, num_sms, scratch, s) : launch<128, false>(p, num_sms, scratch, s);
  else k8 ? launch<64, true>(p, num_sms, scratch, s) : launch<64, false>(p, num_sms, scratch, s);
}

}  // namespace agrpo
