// Attention of the newest tokens of every sequence over the paged cache that already holds them.
//
// Sequence b has n = q_starts[b + 1] - q_starts[b] rows and L = seq_lens[b] tokens in the cache; its row i sees the keys 0 .. L - n + i.
// o = sum_k softmax_k(q.k s) v; a row that sees nothing is zero. Softmax in one pass: running maximum and sum, fp32.
//
// The query heads of a kv head are rows of one tile (row = token * G + head), so that a tile of keys is loaded once for the group.
// S = Q K^T and O += P V run on tcgen05 with S, P and O in tensor memory, a thread a row. Two forms:
//  * kFew: up to 32 rows a unit (decode steps, drafts), bound by the cache's bytes. The 32 rows are loaded into all four quarters of the
//    128-row tile and each of the four softmax warps works on its own 32 of a tile's 128 keys, with a maximum and a sum of its own;
//    the quarters of O are added at the end of a unit. A step of the chain is a quarter of what one warp would take for it.
//  * otherwise two tiles of 128 rows share the keys and values, bound by the tensor cores and by the exponentials (16 a cycle and SM: 128 x 128
//    of them take as long as the products of a tile). One tile's softmax runs beside the other's products.
//
// Work is cut by key tiles, not by rows: all (sequence, kv head, rows) units in a line, their tiles counted through, every CTA takes an equal
// share of the line. A CTA that gets a part of a unit leaves (O, m, l) in the workspace, and a second kernel adds the parts. So a single
// long sequence fills the machine as a batch of ragged ones does, and nothing depends on lengths that the host would have to know.
//
// 8-bit cache: four warps, or four for K and four for V, bring the codes into shared memory, each thread what it will need, and turn them into the
// bf16 tiles that the products read (kv8.cuh).
#include <cuda_bf16.h>

#include <type_traits>

#include "../common/f32x2.cuh"
#include "../common/ptx.cuh"
#include "../common/tensormap.h"
#include "../launchers.h"
#include "../launchers_cache.h"
#include "kv8.cuh"

namespace agrpo {

namespace {

constexpr int kBN = 128;  // keys a tile
// A bf16 tile of keys in shared memory: 8 rows of 128 bytes (64 columns, swizzled) are an atom, an 8-row group holds its D / 64 atoms side by side.
// So a whole page is one copy, whatever its length, and both products find equal strides between groups.
template <int D>
constexpr int kGroupBytes = D / 64 * 1024;
constexpr int kSmemLimit = 232448;

template <int D, bool k8, bool kFew>
struct Shape {
  static constexpr int kTiles = kFew ? 1 : 2;                 // 128-row tiles of Q
  static constexpr int kRows = kFew ? 32 : 256;               // rows of a unit
  static constexpr int kSlotBytes = kBN * D * 2;              // a tile of K or V in bf16
  static constexpr int kQBytes = kTiles * 128 * D * 2;
  static constexpr int kSlots = k8 ? (kFew ? 3 : 4) : (kFew ? 6 : 5);
  static constexpr int kConvGroups = k8 ? (kFew ? 2 : 1) : 0;  // of four warps
  // Item 2 i is K of the CTA's tile i, 2 i + 1 its V. Two groups fill slots of their own, one for K and two for V: in a ring for both, a group
  // could not tell by a barrier's parity whether the other's tile before last has been read.
  __device__ static __forceinline__ int slot(int item) { return kConvGroups == 2 ? ((item & 1) ? 1 + ((item >> 1) & 1) : 0) : item % kSlots; }
  __device__ static __forceinline__ int round(int item) { return kConvGroups == 2 ? ((item & 1) ? item >> 2 : item >> 1) : item / kSlots; }
  static constexpr int kDepth = kFew ? 3 : 2;                  // tiles of codes that a group has under way
  static constexpr int kRaw = kConvGroups * kDepth;
  static constexpr int kSoftWarps = 4 * kTiles;
  static constexpr int kMmaWarp = kSoftWarps, kLoadWarp = kSoftWarps + 1;
  // Four warpgroups where registers are dealt out anew (kShares): two warps of the third do nothing.
  static constexpr bool kShares = k8 && !kFew;
  static constexpr int kConvWarp = kSoftWarps + (kShares ? 4 : 2);
  static constexpr int kThreads = (kConvWarp + 4 * kConvGroups) * 32;
  static constexpr int kRingOff = kQBytes;
  static constexpr int kRawOff = kRingOff + kSlots * kSlotBytes;
  static constexpr int kScaleOff = kRawOff + kRaw * kBN * D;
  static constexpr int kBarOff = kScaleOff + kRaw * kBN;
  static constexpr int kBytes = kBarOff + 512;
  static constexpr int kSmem = kBytes + 1024;                 // room to align
  static_assert(kSmem <= kSmemLimit, "shared memory");
};

struct Params {
  ChunkAttnArgs a;
  PagedCache c;
  int G, tokens;      // query heads a kv head; tokens a unit
  int tile_tokens;    // tokens a 128-row tile (kFew: a unit)
  float scale_log2;
  float* part_o;      // [CTAs, 2, kRows, D]
  float* part_ml;     // [CTAs, 2, kRows, 2]
  int4* desc;         // [CTAs, 2]: the unit that starts in the CTA and ends in a later one
};

struct Seq {
  int row0, n, len;
  bool bad;
};
__device__ __forceinline__ Seq load_seq(const Params& p, int b) {
  Seq s;
  s.row0 = p.a.q_starts[b];
  const int end = p.a.q_starts[b + 1];
  s.len = max(p.a.seq_lens[b], 0);
  s.bad = s.row0 < 0 || end < s.row0 || end > p.a.Tq;
  s.n = s.bad ? 0 : end - s.row0;
  if (s.len > p.a.max_blocks * p.c.block_size) {
    s.bad = true;
    s.len = 0;
  }
  return s;
}
// Keys that the last row of unit qb sees, and tiles of them. A unit without keys still has a tile: its rows are zeros to be written.
__device__ __forceinline__ int unit_keys(const Params& p, const Seq& s, int qb) {
  return max(s.len - s.n + min(s.n, (qb + 1) * p.tokens), 0);
}
__device__ __forceinline__ int unit_tiles(const Params& p, const Seq& s, int qb) { return max(1, (unit_keys(p, s, qb) + kBN - 1) / kBN); }
__device__ __forceinline__ int num_units(const Params& p, const Seq& s) { return (s.n + p.tokens - 1) / p.tokens; }

// A CTA's walk along the line of tiles: one piece (tiles [j0, j1) of a unit) after the other. Every warp walks by itself.
struct Walk {
  Seq s;
  int b, kvh, qb, j0, j1, nk, left;

  __device__ __forceinline__ void start(const Params& p, const int* at) {
    b = at[0];
    kvh = at[1];
    qb = at[2];
    j0 = at[3];
    left = at[4];
    if (left > 0) {
      s = load_seq(p, b);
      clip(p);
    }
  }
  __device__ __forceinline__ bool more() const { return left > 0; }
  __device__ __forceinline__ void clip(const Params& p) {
    nk = unit_tiles(p, s, qb);
    j1 = min(nk, j0 + left);
  }
  __device__ __forceinline__ void next(const Params& p) {
    left -= j1 - j0;
    if (left <= 0) return;
    j0 = 0;
    if (++qb == num_units(p, s)) {
      qb = 0;
      if (++kvh == p.c.Hkv) {
        kvh = 0;
        do s = load_seq(p, ++b);
        while (s.n == 0);
      }
    }
    clip(p);
  }
  __device__ __forceinline__ int tokens(const Params& p) const { return min(p.tokens, s.n - qb * p.tokens); }
  // Tiles of this piece that tile t of Q takes part in: [j0, end).
  __device__ __forceinline__ int end_of(const Params& p, int t) const {
    const int tok = min(p.tile_tokens * (t + 1), tokens(p));
    if (tok <= p.tile_tokens * t) return j0;
    const int keys = s.len - s.n + qb * p.tokens + tok;
    return max(j0, min(j1, (keys + kBN - 1) / kBN));
  }
};

// Where this CTA starts on the line: sums the tiles of all sequences (`pref`, B ints of shared memory), takes its share. at = {sequence, kv
// head, unit, tile, tiles, tiles before its first, tiles in all}.
template <int kThreads>
__device__ __forceinline__ void find_share(const Params& p, int* pref, int* at) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int base = 0; base < p.a.B; base += kThreads) {
    const int b = base + threadIdx.x;
    Seq s = {0, 0, 0, false};
    if (b < p.a.B) s = load_seq(p, b);
    if (s.bad && blockIdx.x == 0) report_status(p.a.status, kStatusBadIndex);
    const int units = num_units(p, s);
    int mine = 0;
    if (units <= 8)
      for (int q = 0; q < units; ++q) mine += unit_tiles(p, s, q);
    for (unsigned big = __ballot_sync(0xffffffffu, units > 8); big != 0; big &= big - 1) {
      const int src = __ffs(big) - 1;
      Seq o = s;
      o.n = __shfl_sync(0xffffffffu, s.n, src);
      o.len = __shfl_sync(0xffffffffu, s.len, src);
      const int total = num_units(p, o);
      int sum = 0;
      for (int q = lane; q < total; q += 32) sum += unit_tiles(p, o, q);
      sum = __reduce_add_sync(0xffffffffu, sum);
      if (lane == src) mine = sum;
    }
    if (b < p.a.B) pref[b] = mine * p.c.Hkv;
  }
  __syncthreads();
  if (warp == 0) {
    int run = 0;
    for (int base = 0; base < p.a.B; base += 32) {
      int v = base + lane < p.a.B ? pref[base + lane] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      v += run;
      run = __shfl_sync(0xffffffffu, v, 31);
      if (base + lane < p.a.B) pref[base + lane] = v;
    }
    __syncwarp();
    const int x0 = static_cast<int>(static_cast<long long>(run) * blockIdx.x / gridDim.x);
    const int x1 = static_cast<int>(static_cast<long long>(run) * (blockIdx.x + 1) / gridDim.x);
    int b = 0, kvh = 0, qb = 0, j = 0;
    if (x1 > x0) {
      int hi = p.a.B - 1;
      while (b < hi) {
        const int mid = (b + hi) / 2;
        if (pref[mid] > x0) hi = mid;
        else b = mid + 1;
      }
      const int before = b > 0 ? pref[b - 1] : 0;
      const int per = (pref[b] - before) / p.c.Hkv;
      int r = x0 - before;
      kvh = r / per;
      r -= kvh * per;
      const Seq s = load_seq(p, b);
      for (int q0 = 0;; q0 += 32) {
        const int q = q0 + lane;
        const int nk = q < num_units(p, s) ? unit_tiles(p, s, q) : 0;
        int inc = nk;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int u = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += u;
        }
        const unsigned past = __ballot_sync(0xffffffffu, inc > r);
        if (past != 0) {
          const int src = __ffs(past) - 1;
          qb = q0 + src;
          j = r - __shfl_sync(0xffffffffu, inc - nk, src);
          break;
        }
        const int all = __shfl_sync(0xffffffffu, inc, 31);
        if (all == 0) break;  // cannot be: the line would end here
        r -= all;
      }
    }
    if (lane == 0) {
      at[0] = b;
      at[1] = kvh;
      at[2] = qb;
      at[3] = j;
      at[4] = x1 - x0;
      at[5] = x0;
      at[6] = run;
    }
  }
  fence_proxy_async_smem();  // the sums lie where the ring's copies go next
  __syncthreads();
}

// 16 or 4 bytes into shared memory, zeros where `on` is false (nothing is read then).
__device__ __forceinline__ void cp_async_16(void* dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_4(void* dst, const void* src, bool on) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(on ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <bool kOn, int kLeft>
__device__ __forceinline__ void give_registers() {
  if (kOn) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLeft));
}

template <int D, bool k8, bool kFew>
__global__ void __launch_bounds__(Shape<D, k8, kFew>::kThreads, 1)
paged_chunk_attn_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                        const __grid_constant__ Params p) {
  using S = Shape<D, k8, kFew>;
  constexpr int kChunks = D / 64;
  constexpr uint32_t kIdescS = umma_idesc_bf16(128, kBN, 0, 0);
  constexpr uint32_t kIdescO = umma_idesc_bf16(128, D, 0, 1);
  // tensor memory: two buffers of S; kFew: O, then two buffers of P of their own (what a warp's keys leave out of a row stays zero there);
  // else: two O, and P in the upper half of its S
  constexpr uint32_t kColO = 256, kColP = kFew ? 384 : 64;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = smem + S::kRingOff;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBarOff);
  uint64_t* full = bars;               // [kSlots]
  uint64_t* empty = bars + 6;          // [kSlots]
  uint64_t* q_full = bars + 12;
  uint64_t* q_empty = bars + 13;
  uint64_t* s_full = bars + 14;        // [2]
  uint64_t* p_ready = bars + 16;       // [2]
  uint64_t* o_done = bars + 18;        // [2]: after a piece's last product (of tile t); kFew: [0] after every one, [1] after the last. Softmax may be two
                                       // products ahead at a piece's end, which one barrier for all of them could not tell from being done
  uint64_t* o_free = bars + 20;        // [2]
  uint64_t* soft = bars + 22;          // kFew: the softmax warps among themselves
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 23);
  int* at = reinterpret_cast<int*>(bars + 24);
  int* status = p.a.status;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kSlots; ++i) {
      mbar_init(full + i, k8 ? 4 : 1);
      mbar_init(empty + i, 1);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, kFew ? 5 : 1);
    mbar_init(soft, 4);
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full + i, 1);
      mbar_init(p_ready + i, 4);
      mbar_init(o_done + i, 1);
      mbar_init(o_free + i, 4);
    }
    fence_mbar_init();
  }
  if (warp == S::kMmaWarp) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  pdl_wait();
  pdl_launch();
  find_share<S::kThreads>(p, reinterpret_cast<int*>(ring), at);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  Walk w;
  w.start(p, at);

  // kShares: 128 x (168 + 168 + 72 + 104) registers = 512 x 128
  if (warp == S::kLoadWarp) {
    give_registers<S::kShares, 72>();
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
            const int slot = S::slot(item), round = S::round(item);
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
          constexpr int kBoxes = kFew ? 4 : S::kTiles;   // kFew: the same rows in all four quarters
          const int row0 = w.s.row0 + w.qb * p.tokens;
          __syncwarp();
          const int tok = w.tokens(p);
          const int boxes = kFew || tok > p.tile_tokens ? kBoxes : 1;
          if (lane == 0) mbar_expect_tx(q_full, boxes * kChunks * p.G * p.tile_tokens * 128);
          __syncwarp();
          if (lane < boxes * kChunks) {
            const int box = lane / kChunks, ch = lane % kChunks;
            uint8_t* dst = kFew ? smem + ch * (128 * 128) + box * (32 * 128) : smem + box * (128 * D * 2) + ch * (128 * 128);
            tma_load_3d(dst, &tmQ, q_full, ch * 64, w.kvh * p.G, row0 + (kFew ? 0 : box * p.tile_tokens));
          }
        }
      }
    }
  } else if (warp == S::kMmaWarp) {
    give_registers<S::kShares, 72>();
    // ---------------------------------------------------------------- products
    const uint32_t aQ = smem_u32(smem), aRing = smem_u32(ring);
    int tile = 0, n_q = 0;          // tiles and pieces so far
    int n_p[2] = {0, 0};            // softmaxed tiles of each buffer waited for
    int n_o[2] = {0, 0};            // pieces whose O has been started
    bool ok = true;
    const auto wait = [&](uint64_t* bar, int parity, int code) {
      if (ok && !mbar_wait(bar, parity)) {
        report_status(status, code);
        ok = false;
      }
      return ok;
    };
    const auto slot_wait = [&](int item) { return wait(full + S::slot(item), S::round(item) & 1, kStatusWaitFullTimeout); };
    const auto scores = [&](int t, int item, uint32_t col) {  // S = Q_t K^T
      if (elect_one()) {
        const uint32_t q = aQ + t * (128 * D * 2), k = aRing + S::slot(item) * S::kSlotBytes;
#pragma unroll 1  // unrolled, the descriptors would stay in registers from one tile to the next
        for (int i = 0; i < D / 16; ++i) {
          tc_mma_f16(tmem + col, umma_smem_desc(q + (i / 4) * (128 * 128) + (i % 4) * 32, 16, 1024),
                     umma_smem_desc(k + (i / 4) * 1024 + (i % 4) * 32, 16, kGroupBytes<D>), kIdescS, i > 0 ? 1u : 0u);
        }
        tc_commit(s_full + (col >> 7));
      }
      __syncwarp();
    };
    const auto values = [&](int item, uint32_t col_p, uint32_t col_o, bool first) {  // O (+)= P V
      if (elect_one()) {
        const uint32_t v = aRing + S::slot(item) * S::kSlotBytes;
#pragma unroll 1
        for (int i = 0; i < kBN / 16; ++i)
          tc_mma_f16_ts(tmem + col_o, tmem + col_p + i * 8, umma_smem_desc(v + i * 2 * kGroupBytes<D>, 1024, kGroupBytes<D>), kIdescO, (!first || i > 0) ? 1u : 0u);
      }
      __syncwarp();
    };
    const auto commit = [&](uint64_t* bar) {
      if (elect_one()) tc_commit(bar);
      __syncwarp();
    };
    // Rows of V behind the last visible key: whatever the page held before, 0 * NaN would reach every row. (The converting warps do it for 8 bits.)
    const auto clear_tail = [&](int item, int valid) {
      if (k8 || valid >= kBN) return;
      uint8_t* v = ring + S::slot(item) * S::kSlotBytes;
      for (int i = max(valid, 0) * 8 + lane; i < kBN * 8; i += 32) {  // row i / 8, bytes (i % 8) * 16 of its atoms
#pragma unroll
        for (int c = 0; c < kChunks; ++c) *reinterpret_cast<uint4*>(v + (i >> 6) * kGroupBytes<D> + c * 1024 + (i & 63) * 16) = make_uint4(0u, 0u, 0u, 0u);
      }
      fence_proxy_async_smem();
      __syncwarp();
    };
    for (; w.more() && ok; w.next(p)) {
      const int keys = unit_keys(p, w.s, w.qb);
      if (!wait(q_full, n_q++ & 1, kStatusWaitFullTimeout)) break;
      if (kFew) {
        if (!slot_wait(2 * tile)) break;
        tc_fence_after();
        scores(0, 2 * tile, (tile & 1) * 128);
        commit(empty + S::slot(2 * tile));
        for (int j = w.j0; j < w.j1; ++j, ++tile) {
          if (j + 1 < w.j1) {
            const int item = 2 * tile + 2;
            if (!slot_wait(item)) break;
            tc_fence_after();
            scores(0, item, ((tile + 1) & 1) * 128);
            commit(empty + S::slot(item));
          }
          if (j + 1 >= w.j1) commit(q_empty);
          if (j == w.j0 && n_o[0] > 0 && !wait(o_free, (n_o[0] - 1) & 1, kStatusWaitTmemEmptyTimeout)) break;
          if (!slot_wait(2 * tile + 1)) break;
          clear_tail(2 * tile + 1, keys - j * kBN);
          if (!wait(p_ready + (tile & 1), (tile >> 1) & 1, kStatusWaitTmemFullTimeout)) break;
          tc_fence_after();
          values(2 * tile + 1, kColP + (tile & 1) * 64, kColO, j == w.j0);
          commit(o_done);
          if (j + 1 >= w.j1) commit(o_done + 1);
          commit(empty + S::slot(2 * tile + 1));
        }
        ++n_o[0];
      } else {
        const int end[2] = {w.end_of(p, 0), w.end_of(p, 1)};
        if (!slot_wait(2 * tile)) break;
        tc_fence_after();
        for (int t = 0; t < 2; ++t)
          if (w.j0 < end[t]) scores(t, 2 * tile, t * 128);
        commit(empty + S::slot(2 * tile));
        for (int j = w.j0; j < w.j1 && ok; ++j, ++tile) {
          if (j + 1 >= w.j1) commit(q_empty);
          if (!slot_wait(2 * tile + 1)) break;
          clear_tail(2 * tile + 1, keys - j * kBN);
          const bool more = j + 1 < w.j1;
          for (int t = 0; t < 2 && ok; ++t) {
            if (j >= end[t]) continue;
            if (j == w.j0 && n_o[t] > 0 && !wait(o_free + t, (n_o[t] - 1) & 1, kStatusWaitTmemEmptyTimeout)) break;
            if (!wait(p_ready + t, n_p[t]++ & 1, kStatusWaitTmemFullTimeout)) break;
            tc_fence_after();
            values(2 * tile + 1, t * 128 + kColP, kColO + t * 128, j == w.j0);
            if (j + 1 >= end[t]) {
              commit(o_done + t);
              ++n_o[t];
            }
            if (j + 1 < end[t]) {
              if (!slot_wait(2 * tile + 2)) break;
              tc_fence_after();
              scores(t, 2 * tile + 2, t * 128);
            }
          }
          commit(empty + S::slot(2 * tile + 1));
          if (more) {
            slot_wait(2 * tile + 2);  // where no tile of Q takes part any more, it still counts as read
            commit(empty + S::slot(2 * tile + 2));
          }
        }
      }
    }
  } else if (k8 && warp >= S::kConvWarp) {
    give_registers<S::kShares, 104>();
    // ---------------------------------------------------------------- 8 bits to bf16
    // 16 codes a thread and step. A warp has 8 rows of every 32 (two steps for them if D = 128): eight lanes take four pieces of a row and the other
    // four of the next one, so that their 16-byte writes fall into eight different bank groups. A thread copies the pieces that it will turn into bf16
    // itself, so nobody waits for anybody else's copies, kDepth tiles ahead. (Bulk copies of pages of 16 tokens, 2 KB, took 54 cycles each to issue.)
    const int group = (warp - S::kConvWarp) >> 2, cw = (warp - S::kConvWarp) & 3, tid = cw * 32 + lane;
    constexpr int kGroups = S::kConvGroups > 0 ? S::kConvGroups : 1;
    constexpr int kPerRows = D / 64;             // steps for the same rows
    uint8_t* raw = smem + S::kRawOff + group * S::kDepth * (kBN * D) + tid * 16;
    uint8_t* raw_scale = smem + S::kScaleOff + group * S::kDepth * kBN + cw * 32;
    const int sub = lane >> 2;                   // row of the eight
    Walk a = w;                                  // the copies' walk
    int a_j = a.j0, a_v = group, n_copy = 0, page = 0;
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
        const int slot = n_copy % S::kDepth, bs = p.c.block_size;
        const int valid = unit_keys(p, a.s, a.qb) - a_j * kBN;
        const auto* codes = static_cast<const uint8_t*>(a_v ? p.c.v : p.c.k);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int r = q * 32 + cw * 8 + sub;
          const long long row = (static_cast<long long>(__shfl_sync(0xffffffffu, page, q)) * p.c.Hkv + a.kvh) * bs + ((a_j * kBN + r) & (bs - 1));
#pragma unroll
          for (int h = 0; h < kPerRows; ++h) {
            const int piece = D == 128 ? (lane & 3) + 4 * ((sub & 1) ^ h) : lane & 3;
            cp_async_16(raw + slot * (kBN * D) + (q * kPerRows + h) * 2048, codes + row * D + piece * 16, r < valid);
          }
        }
        // the factors' bytes: four rows a lane
        const int pq = __shfl_sync(0xffffffffu, page, lane >> 1 & 3), r = (lane >> 1 & 3) * 32 + cw * 8 + (lane & 1) * 4;
        if (lane < 8) {
          const long long row = (static_cast<long long>(pq) * p.c.Hkv + a.kvh) * bs + ((a_j * kBN + r) & (bs - 1));
          cp_async_4(raw_scale + slot * kBN + lane * 4, (a_v ? p.c.v_scale : p.c.k_scale) + row, r < valid);
        }
        ++n_copy;
        a_v += kGroups;
        if (a_v > 1) {
          a_v = group;
          if (++a_j == a.j1) {
            a.next(p);
            a_j = a.j0;
          }
          pages();
        }
      }
      cp_async_commit();  // also where nothing is left, so that the waits below name the same tile
    };
    pages();
#pragma unroll 1
    for (int i = 0; i < S::kDepth; ++i) copy();
    int item = group, n = 0;
    bool ok = true;
    for (; w.more() && ok; w.next(p)) {
      for (int j = w.j0; j < w.j1 && ok; ++j) {
        for (int v = group; v < 2 && ok; v += kGroups, item += kGroups, ++n) {
          const int slot = S::slot(item), round = S::round(item), mine = n % S::kDepth;
          cp_async_wait<S::kDepth - 1>();
          __syncwarp();
          // of row 32 (lane / 8) + 8 cw + lane % 8. Behind the last key the codes are zero, and the factor has to be a number
          const int left = unit_keys(p, w.s, w.qb) - j * kBN - cw * 8;
          const Kv8Scale s = kv8_scale((lane >> 3) * 32 + (lane & 7) < left ? raw_scale[mine * kBN + lane] : 0);
          const bool twice = __any_sync(0xffffffffu, s.twice);         // some value above 448 * 2^7
          if (round > 0 && !mbar_wait(empty + slot, (round - 1) & 1)) {
            report_status(status, kStatusWaitEmptyTimeout);
            ok = false;
            break;
          }
          const uint8_t* src = raw + mine * (kBN * D);
          uint8_t* dst = ring + slot * S::kSlotBytes + cw * kGroupBytes<D> + sub * 128;
          const auto convert = [&](auto both) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              Kv8Scale f;
              f.first = __shfl_sync(0xffffffffu, s.first, q * 8 + sub);
              f.second = decltype(both)::value ? __shfl_sync(0xffffffffu, s.second, q * 8 + sub) : 0u;
              f.twice = decltype(both)::value ? __shfl_sync(0xffffffffu, static_cast<int>(s.twice), q * 8 + sub) != 0 : false;
#pragma unroll
              for (int h = 0; h < kPerRows; ++h) {
                const uint4 x = *reinterpret_cast<const uint4*>(src + (q * kPerRows + h) * 2048);
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
    }
    cp_async_wait<0>();
  } else if (warp < S::kSoftWarps) {
    if (S::kShares) asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
    // ---------------------------------------------------------------- softmax, results
    const int t = kFew ? 0 : warp >> 2, quarter = warp & 3;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t tO = tmem + lanes + kColO + t * 128;
    const int r = kFew ? lane : quarter * 32 + lane;  // row of the tile
    const int r_tok = r / p.G, r_head = r - r_tok * p.G;
    int tile = 0, n_o = 0;
    bool ok = true;
    if (kFew) {  // a warp writes its own 32 keys of P: the others stay zero
      uint32_t z[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) z[i] = 0u;
#pragma unroll
      for (int i = 0; i < 8; ++i) tmem_st_32x16(tmem + lanes + kColP + i * 16, z);
      tc_wait_st();
    }
    int n_soft = 0;
    // All softmax warps; bounded as every wait is (a named barrier would wait for a warp that has given up).
    const auto soft_sync = [&] {
      __syncwarp();
      if (lane == 0) mbar_arrive(soft);
      if (ok && !mbar_wait(soft, n_soft++ & 1)) {
        report_status(status, kStatusBarrierTimeout);
        ok = false;
      }
      __syncwarp();
    };
    int4* desc = p.desc + blockIdx.x * 2;
    if (threadIdx.x == 0) desc[0] = make_int4(0, 0, 0, 0);
    int flat = at[5];
    for (; w.more() && ok; flat += w.j1 - w.j0, w.next(p)) {
      const int tok = min(p.tile_tokens, w.tokens(p) - t * p.tile_tokens);  // of this tile
      const int rows = max(tok, 0) * p.G;
      const bool busy = (kFew ? 0 : quarter * 32) < rows;                   // the warp has rows
      const int end = kFew ? w.j1 : w.end_of(p, t);
      const int first_pos = w.s.len - w.s.n + w.qb * p.tokens + t * p.tile_tokens;  // position of the tile's first row
      const int pos = first_pos + r_tok;                                            // the row sees the keys up to its position
      const bool whole = w.j0 == 0 && w.j1 == w.nk;
      float m = -INFINITY;
      float2 l2 = make_float2(0.f, 0.f);
      for (int j = w.j0; j < end; ++j, ++tile) {
        const int buf = kFew ? tile & 1 : t;
        if (!mbar_wait(s_full + buf, (kFew ? tile >> 1 : tile) & 1)) {
          report_status(status, kStatusWaitTmemFullTimeout);
          ok = false;
          break;
        }
        tc_fence_after();
        if (busy) {
          const uint32_t tS = tmem + lanes + buf * 128 + (kFew ? quarter * 32 : 0);
          const int key0 = j * kBN + (kFew ? quarter * 32 : 0);
          const int see = pos - key0;                                         // columns up to this one
          // Rescales O and l where the maximum grew by more than 2^8; the products of the tile before must be complete then.
          const auto raise = [&](float mx) {
            mx *= p.scale_log2;
            float alpha = 1.f;
            if (mx > m + 8.f) {
              alpha = m == -INFINITY ? 0.f : exp2f(m - mx);
              m = mx;
            }
            if (__any_sync(0xffffffffu, alpha != 1.f) && j > w.j0) {
              if (kFew) {
                if (!mbar_wait(o_done, (tile - 1) & 1)) {
                  report_status(status, kStatusWaitTmemFullTimeout);
                  ok = false;
                }
                tc_fence_after();
              }
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
          const auto exponentials = [&](auto diag, const uint32_t (&s)[32], int col, uint32_t dst) {  // 32 columns of P
            const float base = m == -INFINITY ? 0.f : m;
            const float2 sc = make_float2(p.scale_log2, p.scale_log2), neg = make_float2(-base, -base);
            uint32_t pk[16];
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              const float2 z = fma2(make_float2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), sc, neg);
              float2 e = make_float2(exp2f(z.x), exp2f(z.y));
              if (decltype(diag)::value) {
                if (col + i > see) e.x = 0.f;
                if (col + i + 1 > see) e.y = 0.f;
              }
              l2 = add2(l2, e);
              pk[i / 2] = pack_bf16x2(e.x, e.y);
            }
            tmem_st_32x16(dst, pk);
          };
          const auto top = [&](auto diag, const uint32_t (&s)[32], int col, float (&mx)[4]) {
            const auto at = [&](int i) { return decltype(diag)::value && col + i > see ? -INFINITY : __uint_as_float(s[i]); };
#pragma unroll
            for (int i = 0; i < 32; i += 2) mx[i / 2 & 3] = max3(mx[i / 2 & 3], at(i), at(i + 1));
          };
          const auto softmax = [&](auto diag) {  // diag: some row does not see the whole tile
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            if (kFew) {
              uint32_t s[32];
              tmem_ld_32x32(tS, s);
              tc_wait_ld();
              top(diag, s, 0, mx);
              raise(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])));
              exponentials(diag, s, 0, tmem + lanes + kColP + buf * 64 + quarter * 16);
            } else {
              uint32_t s0[32], s1[32];
              tmem_ld_32x32(tS, s0);
              tmem_ld_32x32(tS + 32, s1);
              tc_wait_ld();
              top(diag, s0, 0, mx);
              top(diag, s1, 32, mx);
              tmem_ld_32x32(tS + 64, s0);
              tmem_ld_32x32(tS + 96, s1);
              tc_wait_ld();
              top(diag, s0, 64, mx);
              top(diag, s1, 96, mx);
              raise(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])));
              exponentials(diag, s0, 64, tS + kColP + 32);
              exponentials(diag, s1, 96, tS + kColP + 48);
              tmem_ld_32x32(tS, s0);
              tmem_ld_32x32(tS + 32, s1);
              tc_wait_ld();
              exponentials(diag, s0, 0, tS + kColP);
              exponentials(diag, s1, 32, tS + kColP + 16);
            }
          };
          if (first_pos < key0 + (kFew ? 31 : kBN - 1)) softmax(std::true_type{});
          else softmax(std::false_type{});
          tc_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_ready + buf);
        if (!ok) break;
      }
      if (!ok) break;
      const float l = l2.x + l2.y;
      const bool any = end > w.j0;  // else O holds nothing of this piece
      if (any && !mbar_wait(o_done + (kFew ? 1 : t), n_o++ & 1)) {
        report_status(status, kStatusWaitTmemFullTimeout);
        ok = false;
        break;
      }
      tc_fence_after();
      const int piece = blockIdx.x * 2 + (w.j0 == 0 ? 1 : 0);
      const long long row0 = w.s.row0 + w.qb * p.tokens;
      auto* out = static_cast<__nv_bfloat16*>(p.a.out);
      if (kFew) {
        // the quarters of O: weights by maximum, added through the shared memory of Q, 64 columns at a time
        float2* ml = reinterpret_cast<float2*>(smem);
        ml[quarter * 32 + lane] = make_float2(m, l);
        soft_sync();
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float2 x = ml[q * 32 + lane];
          if (x.y != 0.f) M = fmaxf(M, x.x);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float2 x = ml[q * 32 + lane];
          if (x.y != 0.f) L += x.y * exp2f(x.x - M);
        }
        soft_sync();
        const float weight = l != 0.f ? exp2f(m - M) : 0.f;
        const float scale = !whole ? 1.f : (L != 0.f ? 1.f / L : 0.f);
        constexpr int kPass = D / 2, kVec = kPass / 4;  // columns at a time: what fits into Q's memory
        static_assert(4 * 32 * kPass * 4 <= S::kQBytes, "the quarters of O go through the memory of Q");
        uint8_t* buf = smem;  // [4][32 rows][kVec chunks of 16 bytes], chunk c of a row at c ^ (row & (kVec - 1))
        const auto at_row = [&](int q, int row, int ch) { return reinterpret_cast<float4*>(buf + ((q * 32 + row) * kVec + (ch ^ (row & (kVec - 1)))) * 16); };
#pragma unroll 1
        for (int c0 = 0; c0 < D; c0 += kPass) {
#pragma unroll 1
          for (int h = 0; h < kPass; h += 32) {
            uint32_t o[32];
            tmem_ld_32x32(tO + c0 + h, o);
            tc_wait_ld();
            if (lane < rows) {
              const float f = weight * scale;
#pragma unroll
              for (int i = 0; i < 8; ++i)
                *at_row(quarter, lane, h / 4 + i) =
                    weight == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f)
                                  : make_float4(__uint_as_float(o[4 * i]) * f, __uint_as_float(o[4 * i + 1]) * f, __uint_as_float(o[4 * i + 2]) * f,
                                                __uint_as_float(o[4 * i + 3]) * f);
            }
          }
          soft_sync();
          for (int i = threadIdx.x; i < rows * kVec; i += 128) {
            const int row = i / kVec, ch = i % kVec;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const float4 y = *at_row(q, row, ch);
              x.x += y.x;
              x.y += y.y;
              x.z += y.z;
              x.w += y.w;
            }
            if (whole) {
              const int tk = row / p.G, hd = row - tk * p.G;
              uint2 y;
              y.x = pack_bf16x2(x.x, x.y);
              y.y = pack_bf16x2(x.z, x.w);
              *reinterpret_cast<uint2*>(out + (row0 + tk) * p.a.ldo + static_cast<long long>(w.kvh * p.G + hd) * D + c0 + ch * 4) = y;
            } else {
              *reinterpret_cast<float4*>(p.part_o + (static_cast<long long>(piece) * S::kRows + row) * D + c0 + ch * 4) = x;
            }
          }
          soft_sync();
        }
        if (!whole && quarter == 0 && lane < rows)
          *reinterpret_cast<float2*>(p.part_ml + (static_cast<long long>(piece) * S::kRows + lane) * 2) = make_float2(M, L);
        fence_proxy_async_smem();  // Q comes here next
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(q_empty);
          mbar_arrive(o_free);
        }
      } else {
        const float inv = l != 0.f ? 1.f / l : 0.f;
        const bool valid = r < rows;  // O is read where the tile took part (any) and zero otherwise
        auto* dst = out + (row0 + t * p.tile_tokens + r_tok) * p.a.ldo + static_cast<long long>(w.kvh * p.G + r_head) * D;
        float* part = p.part_o + (static_cast<long long>(piece) * S::kRows + t * 128 + r) * D;
        if (busy) {
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
              for (int i = 0; i < 32; i += 8) {
                uint4 y;
                y.x = pack_bf16x2(__uint_as_float(o[i]) * inv, __uint_as_float(o[i + 1]) * inv);
                y.y = pack_bf16x2(__uint_as_float(o[i + 2]) * inv, __uint_as_float(o[i + 3]) * inv);
                y.z = pack_bf16x2(__uint_as_float(o[i + 4]) * inv, __uint_as_float(o[i + 5]) * inv);
                y.w = pack_bf16x2(__uint_as_float(o[i + 6]) * inv, __uint_as_float(o[i + 7]) * inv);
                *reinterpret_cast<uint4*>(dst + c * 32 + i) = y;
              }
            } else if (valid) {
#pragma unroll
              for (int i = 0; i < 32; i += 4)
                *reinterpret_cast<uint4*>(part + c * 32 + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
            }
          }
          if (valid && !whole) *reinterpret_cast<float2*>(p.part_ml + (static_cast<long long>(piece) * S::kRows + t * 128 + r) * 2) = make_float2(m, l);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0 && any) mbar_arrive(o_free + t);
      }
      // a unit that starts here and ends elsewhere: its parts are those of the CTAs up to the one with its last tile
      if (threadIdx.x == 0 && w.j0 == 0 && w.j1 < w.nk) {
        const long long last = flat + w.nk;  // tiles of the line up to the unit's end
        const int total = at[6];
        desc[0] = make_int4(static_cast<int>(row0), w.tokens(p), w.kvh, static_cast<int>((last * gridDim.x + total - 1) / total) - 1);
        desc[1] = make_int4(total, 0, 0, 0);
      }
    }
  }

  if (S::kShares && warp > S::kLoadWarp && warp < S::kConvWarp) give_registers<S::kShares, 72>();

  tc_fence_before();
  __syncthreads();
  if (warp == S::kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Adds the parts of the units that several CTAs worked on, in the order of the keys. A warp a row.
template <int D, int kRows>
__global__ void __launch_bounds__(256) paged_chunk_combine_kernel(const Params p, int ctas) {
  pdl_wait();
  pdl_launch();
  constexpr int kPer = D / 32;
  const int c = blockIdx.x;
  const int4 u = p.desc[c * 2];
  const int rows = u.y * p.G, last = u.w;
  const int lane = threadIdx.x & 31;
  if (rows == 0) return;
  const long long total = p.desc[c * 2 + 1].x;
  const int per_block = kRows / gridDim.y;
  for (int r = blockIdx.y * per_block + (threadIdx.x >> 5); r < min(rows, (static_cast<int>(blockIdx.y) + 1) * per_block); r += 8) {
    const int tk = r / p.G, hd = r - tk * p.G;
    const int tile = tk / p.tile_tokens;                         // a tile's rows start on 128
    const int slot = r + tile * (128 - p.tile_tokens * p.G);
    float M = -INFINITY, L = 0.f, o[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) o[i] = 0.f;
    for (int k0 = c; k0 <= last; k0 += 32) {
      const int k = k0 + lane;
      const bool on = k <= last && total * k / ctas < total * (k + 1) / ctas;  // the CTA has tiles
      const long long at = (static_cast<long long>(k) * 2 + (k == c ? 1 : 0)) * kRows + slot;
      float2 ml = on ? *reinterpret_cast<const float2*>(p.part_ml + at * 2) : make_float2(-INFINITY, 0.f);
      float mx = ml.y != 0.f ? ml.x : -INFINITY;
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
      const float Mn = fmaxf(M, mx);
      const float keep = M == -INFINITY ? 0.f : exp2f(M - Mn);
      const float wgt = ml.y != 0.f ? exp2f(ml.x - Mn) : 0.f;
      float ls = ml.y * wgt;
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) ls += __shfl_xor_sync(0xffffffffu, ls, off);
      L = L * keep + ls;
      M = Mn;
#pragma unroll
      for (int i = 0; i < kPer; ++i) o[i] *= keep;
      const unsigned have = __ballot_sync(0xffffffffu, wgt != 0.f);
#pragma unroll 4
      for (int i = 0; i < min(32, last - k0 + 1); ++i) {
        const float wi = __shfl_sync(0xffffffffu, wgt, i);
        if (!((have >> i) & 1)) continue;
        const float* src = p.part_o + ((static_cast<long long>(k0 + i) * 2 + (k0 + i == c ? 1 : 0)) * kRows + slot) * D + lane * kPer;
        if (kPer == 4) {
          const float4 x = __ldcg(reinterpret_cast<const float4*>(src));
          o[0] += x.x * wi;
          o[1] += x.y * wi;
          o[2 % kPer] += x.z * wi;
          o[3 % kPer] += x.w * wi;
        } else {
          const float2 x = __ldcg(reinterpret_cast<const float2*>(src));
          o[0] += x.x * wi;
          o[1] += x.y * wi;
        }
      }
    }
    const float inv = L != 0.f ? 1.f / L : 0.f;
    auto* dst = static_cast<__nv_bfloat16*>(p.a.out) + static_cast<long long>(u.x + tk) * p.a.ldo + static_cast<long long>(u.z * p.G + hd) * D + lane * kPer;
    uint32_t y[kPer / 2];
#pragma unroll
    for (int i = 0; i < kPer / 2; ++i) y[i] = pack_bf16x2(o[2 * i] * inv, o[2 * i + 1] * inv);
    if (kPer == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(y[0], y[kPer / 2 - 1]);
    else *reinterpret_cast<uint32_t*>(dst) = y[0];
  }
}

template <int D, bool k8, bool kFew>
void launch(Params p, int num_sms, void* scratch, cudaStream_t s) {
  using S = Shape<D, k8, kFew>;
  p.tile_tokens = (kFew ? 32 : 128) / p.G;
  p.tokens = S::kTiles * p.tile_tokens;
  p.desc = static_cast<int4*>(scratch);
  p.part_ml = reinterpret_cast<float*>(p.desc + 2 * num_sms);
  p.part_o = p.part_ml + static_cast<long long>(num_sms) * 2 * S::kRows * 2;
  const uint64_t dims[3] = {static_cast<uint64_t>(D), static_cast<uint64_t>(p.a.Hq), static_cast<uint64_t>(p.a.Tq)};
  const uint32_t box[3] = {64, static_cast<uint32_t>(p.G), static_cast<uint32_t>(p.tile_tokens)};
  const uint64_t pitch[2] = {static_cast<uint64_t>(D), static_cast<uint64_t>(p.a.ldq)};
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
  auto kernel = paged_chunk_attn_kernel<D, k8, kFew>;
  AGRPO_SET_MAX_DYN_SMEM(kernel, S::kSmem, "paged_chunk_attn smem attr");
  launch_kernel(kernel, dim3(num_sms), dim3(S::kThreads), S::kSmem, s, "paged_chunk_attn", tq, tk, tv, p);
  auto combine = paged_chunk_combine_kernel<D, S::kRows>;
  AGRPO_PREFER_SMEM(combine);
  launch_kernel(combine, dim3(num_sms, kFew ? 4 : 8), dim3(256), 0, s, "paged_chunk_combine", p, num_sms);
}

// Up to 32 rows a sequence on average: the form whose warps share a unit's rows.
bool few_rows(const ChunkAttnArgs& a, const PagedCache& c) { return static_cast<long long>(a.Tq) * (a.Hq / c.Hkv) <= 32ll * a.B; }

}  // namespace

long long paged_chunk_attn_scratch(const ChunkAttnArgs& a, const PagedCache& c, int num_sms) {
  const long long rows = few_rows(a, c) ? 32 : 256;
  return num_sms * (2 * 16 + 2 * rows * (2 + c.D) * 4);
}

void launch_paged_chunk_attn(const ChunkAttnArgs& a, const PagedCache& c, int num_sms, void* scratch, cudaStream_t s) {
  if (a.Tq == 0 || a.B == 0) return;
  Params p = {};
  p.a = a;
  p.c = c;
  p.G = a.Hq / c.Hkv;
  p.scale_log2 = a.softmax_scale * 1.4426950408889634f;
  const auto run = [&](auto d, auto k8) {
    if (few_rows(a, c)) launch<decltype(d)::value, decltype(k8)::value, true>(p, num_sms, scratch, s);
    else launch<decltype(d)::value, decltype(k8)::value, false>(p, num_sms, scratch, s);
  };
  using D128 = std::integral_constant<int, 128>;
  using D64 = std::integral_constant<int, 64>;
  if (c.k_scale != nullptr) c.D == 128 ? run(D128{}, std::true_type{}) : run(D64{}, std::true_type{});
  else c.D == 128 ? run(D128{}, std::false_type{}) : run(D64{}, std::false_type{});
}

}  // namespace agrpo
