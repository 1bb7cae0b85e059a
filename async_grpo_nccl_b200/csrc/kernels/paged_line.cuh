// What the two kernels of paged_chunk_attn share: how a call's work lies in a line, how workers take equal shares of it, and how the parts of a unit
// that several of them worked on are added.
//
// A unit is the rows of some tokens of a sequence under one kv head (row = token * G + query head of the group). All units lie in a line, sequence
// by sequence, kv head by kv head; a unit is as long as it has tiles of kKeys keys to look at. W workers (CTAs or warps; as many as there are, or as many as find
// work for their while) take the tiles [T w / W, T (w + 1) / W) of the T tiles, but for borders that move (below). So one long sequence fills the machine as a batch of
// ragged ones does, and nothing depends on a length that the host would have to know. A worker that has a part of a unit leaves (O, m, l) in the workspace:
// only its first and its last piece can be parts. Parts are added in the order of the keys, so the same call gives the same bits.
//
// Beginning and ending a unit takes a worker as long as some tiles, so a unit's length in the line is that of its tiles and kExtra more, in front of them; a border
// of shares that falls among those moves to the unit's start. (24 prompts in 3 to 13 pieces a CTA took 63 to 99 us a CTA without.) Shares then differ by up to kExtra
// at either end: 25 to 28 for those prompts (kExtra 1), 2 to 11, 7 on average, for 61 sequences of 200 - 4000 tokens in the kernel of few rows (kExtra 4); of 400
// units of 9 tiles there, 512 of 2368 workers get none.
#pragma once
#include <cuda_bf16.h>

#include "../common/ptx.cuh"
#include "../launchers.h"
#include "../launchers_cache.h"

namespace agrpo {

namespace {

struct LineParams {
  ChunkAttnArgs a;
  PagedCache c;
  int G, tokens;      // query heads a kv head; tokens a unit
  int tile_tokens;    // tokens a tile of rows
  int rows;           // rows that a part has room for
  float scale_log2;
  int4* desc;         // [CTAs]: the unit that starts in the CTA and ends in a later one {first row, tokens, kv head, last CTA}
  float* part_ml;     // [CTAs, 2, rows, 2]: parts, [0] of a unit that an earlier CTA starts, [1] of one that starts here
  float* part_o;      // [CTAs, 2, rows, D]
};

struct Seq {
  int row0, n, len;
  bool bad, back;  // does not fit its rows or its table; ends before it starts
};
__device__ __forceinline__ Seq load_seq(const LineParams& p, int b) {
  Seq s;
  s.row0 = p.a.q_starts[b];
  const int end = p.a.q_starts[b + 1];
  s.len = max(p.a.seq_lens[b], 0);
  s.back = end < s.row0;
  s.bad = s.row0 < 0 || s.back || end > p.a.Tq;
  s.n = s.bad ? 0 : end - s.row0;
  if (s.len > p.a.max_blocks * p.c.block_size) {
    s.bad = true;
    s.len = 0;
  }
  return s;
}
// The sequences from a CTA's first one on, in shared memory: a walk that had to load the next one would stop for it.
struct SeqCache {
  int* at;           // {row0, n, len} of each
  int first, room;
  __device__ __forceinline__ void fill(const LineParams& p) const {  // all threads; synchronise after it
    for (int i = threadIdx.x; i < room && first + i < p.a.B; i += blockDim.x) {
      const Seq s = load_seq(p, first + i);
      at[3 * i] = s.row0;
      at[3 * i + 1] = s.n;
      at[3 * i + 2] = s.len;
    }
  }
  __device__ __forceinline__ Seq get(const LineParams& p, int b) const {
    const int i = b - first;
    if (i >= room) return load_seq(p, b);
    return Seq{at[3 * i], at[3 * i + 1], at[3 * i + 2], false, false};
  }
};
// Keys that the last row of unit qb sees, and tiles of them. A unit without keys still has a tile: its rows are zeros to be written.
__device__ __forceinline__ int unit_keys(const LineParams& p, const Seq& s, int qb) { return max(s.len - s.n + min(s.n, (qb + 1) * p.tokens), 0); }
// Keys from here on are hidden from some of a unit's rows. A value there that is infinite or no number would reach those rows by 0 * NaN: the kernels take it
// out of the products, and add it at the end to the rows that see it.
__device__ __forceinline__ int first_hidden(const LineParams& p, const Seq& s, int qb) { return max(s.len - s.n + qb * p.tokens + 1, 0); }
template <int kKeys>
__device__ __forceinline__ int unit_tiles(const LineParams& p, const Seq& s, int qb) {
  return max(1, (unit_keys(p, s, qb) + kKeys - 1) / kKeys);
}
__device__ __forceinline__ int num_units(const LineParams& p, const Seq& s) { return (s.n + p.tokens - 1) / p.tokens; }

// Where a worker's share begins.
struct Share {
  int b, kvh, qb, j;   // sequence, kv head, unit, tile
  int tiles, before;   // of the share, ahead of it
  int total, workers;  // of the line; that have a share
  Seq s;
};

// A worker's walk along its share: one piece (tiles [j0, j1) of a unit) after the other.
template <int kKeys, int kExtra>
struct Walk {
  Seq s;
  SeqCache near;
  int b, kvh, qb, j0, j1, nk, left;

  __device__ __forceinline__ void start(const LineParams& p, const Share& at, const SeqCache& cache) {
    near = cache;
    b = at.b;
    kvh = at.kvh;
    qb = at.qb;
    j0 = at.j;
    left = at.tiles;
    s = at.s;
    if (left > 0) clip(p);
  }
  __device__ __forceinline__ bool more() const { return left > 0; }
  __device__ __forceinline__ void clip(const LineParams& p) {
    nk = unit_tiles<kKeys>(p, s, qb);
    j1 = min(nk, j0 + left - (j0 == 0 ? kExtra : 0));
  }
  __device__ __forceinline__ int length() const { return j1 - j0 + (j0 == 0 ? kExtra : 0); }  // of the piece, in the line
  __device__ __forceinline__ void next(const LineParams& p) {
    left -= length();
    if (left <= 0) return;
    j0 = 0;
    if (++qb == num_units(p, s)) {
      qb = 0;
      if (++kvh == p.c.Hkv) {
        kvh = 0;
        do s = near.get(p, ++b);
        while (s.n == 0);
      }
    }
    clip(p);
  }
  __device__ __forceinline__ int tokens(const LineParams& p) const { return min(p.tokens, s.n - qb * p.tokens); }
  __device__ __forceinline__ bool whole() const { return j0 == 0 && j1 == nk; }
  __device__ __forceinline__ int part(int worker) const { return worker * 2 + (j0 == 0 ? 1 : 0); }
  // Tiles of this piece that tile t of the rows takes part in: [j0, end).
  __device__ __forceinline__ int end_of(const LineParams& p, int t) const {
    const int tok = min(p.tile_tokens * (t + 1), tokens(p));
    if (tok <= p.tile_tokens * t) return j0;
    const int keys = s.len - s.n + qb * p.tokens + tok;
    return max(j0, min(j1, (keys + kKeys - 1) / kKeys));
  }
  // The worker that has the unit's last tile, `flat` of the line being ahead of this piece.
  __device__ __forceinline__ int last_worker(const Share& at, int flat) const {
    const long long end = flat - (j0 == 0 ? 0 : j0 + kExtra) + nk + kExtra;
    return static_cast<int>((end * at.workers + at.total - 1) / at.total) - 1;
  }
};

// The line up to each sequence's end, into `line` (B ints of shared memory). All threads of the CTA; reports sequences that cannot be.
// Starts that go back anywhere leave no line (its end, line[B - 1], is 0). Where they never do, no row belongs to two sequences, and the line is no longer
// than paged_chunk_attn_tiles says; starts like 0, Tq, 0, Tq, .. would give all rows to every second sequence, and the sum could pass 31 bits.
template <int kThreads, int kKeys, int kExtra>
__device__ __forceinline__ void measure_line(const LineParams& p, int* line) {
  const int lane = threadIdx.x & 31;
  for (int base = 0; base < p.a.B; base += kThreads) {
    const int b = base + threadIdx.x;
    Seq s = {0, 0, 0, false, false};
    if (b < p.a.B) s = load_seq(p, b);
    if (s.bad && blockIdx.x == 0) report_status(p.a.status, kStatusBadIndex);
    const int units = num_units(p, s);
    int mine = 0;
    if (units <= 8)
      for (int q = 0; q < units; ++q) mine += unit_tiles<kKeys>(p, s, q) + kExtra;
    for (unsigned big = __ballot_sync(0xffffffffu, units > 8); big != 0; big &= big - 1) {  // the warp together
      const int src = __ffs(big) - 1;
      Seq o = s;
      o.n = __shfl_sync(0xffffffffu, s.n, src);
      o.len = __shfl_sync(0xffffffffu, s.len, src);
      const int total = num_units(p, o);
      int sum = 0;
      for (int q = lane; q < total; q += 32) sum += unit_tiles<kKeys>(p, o, q) + kExtra;
      sum = __reduce_add_sync(0xffffffffu, sum);
      if (lane == src) mine = sum;
    }
    if (b < p.a.B) line[b] = s.back ? -1 : mine * p.c.Hkv;
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    int run = 0;
    bool back = false;
    for (int base = 0; base < p.a.B; base += 32) {
      int v = base + lane < p.a.B ? line[base + lane] : 0;
      back |= v < 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      v += run;
      run = __shfl_sync(0xffffffffu, v, 31);
      if (base + lane < p.a.B) line[base + lane] = v;
    }
    back = __any_sync(0xffffffffu, back);
    __syncwarp();
    if (back && lane == 0) line[p.a.B - 1] = 0;
  }
  __syncthreads();
}

// floor(total * i / n), without a 64-bit division.
__device__ __forceinline__ int share_start(int total, int i, int n) {
  const unsigned per = static_cast<unsigned>(total) / n, rest = static_cast<unsigned>(total) - per * n;
  return static_cast<int>(per * i + rest * i / n);  // i and n are at most a few thousand
}

// The place `x` of the line: sequence, kv head, unit and tile; places among a unit's kExtra are its start. Moves `x` there. All lanes of a warp.
template <int kKeys, int kExtra>
__device__ __forceinline__ void locate(const LineParams& p, const int* line, int& x, Share& at) {
  const int lane = threadIdx.x & 31;
  // The sequence: first the one of up to 32 groups, then within it.
  at.b = 0;
  for (int first = 0, many = p.a.B; many > 1;) {
    const int step = (many + 31) / 32, end = min(first + (lane + 1) * step, first + many);  // lane i: up to the end of group i
    const unsigned past = __ballot_sync(0xffffffffu, line[end - 1] > x);
    const int group = __ffs(past) - 1;
    many = min(step, many - group * step);
    first += group * step;
    at.b = first;
  }
  const int ahead = at.b > 0 ? line[at.b - 1] : 0;
  const int per = (line[at.b] - ahead) / p.c.Hkv;
  int r = x - ahead;
  at.kvh = r / per;
  r -= at.kvh * per;
  at.qb = at.j = 0;
  const Seq s = at.s = load_seq(p, at.b);
  for (int q0 = 0; q0 < num_units(p, s); q0 += 32) {
    const int q = q0 + lane;
    const int nk = q < num_units(p, s) ? unit_tiles<kKeys>(p, s, q) + kExtra : 0;
    int inc = nk;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    const unsigned past = __ballot_sync(0xffffffffu, inc > r);
    if (past != 0) {
      const int src = __ffs(past) - 1;
      const int in = r - __shfl_sync(0xffffffffu, inc - nk, src);
      at.qb = q0 + src;
      at.j = max(in - kExtra, 0);
      if (at.j == 0) x -= in;
      break;
    }
    r -= __shfl_sync(0xffffffffu, inc, 31);
  }
}

// A worker's share, of kLeast tiles at least if there are so many. One warp, all lanes with the same result.
template <int kKeys, int kExtra, int kLeast>
__device__ __forceinline__ Share find_share(const LineParams& p, const int* line, int worker, int workers) {
  Share at = {0, 0, 0, 0, 0, 0, line[p.a.B - 1], 0, {0, 0, 0, false, false}};
  at.workers = min(workers, (at.total + kLeast - 1) / kLeast);
  if (worker >= at.workers) return at;
  int end = share_start(at.total, worker + 1, at.workers);
  if (kExtra > 0 && end < at.total) {
    Share behind;
    locate<kKeys, kExtra>(p, line, end, behind);
  }
  at.before = share_start(at.total, worker, at.workers);
  if (at.before < at.total) locate<kKeys, kExtra>(p, line, at.before, at);
  at.tiles = end - at.before;
  return at;
}

// One row's share of a unit: adds the parts first .. last (the first in place `head` of its pair, the others in 0). A warp; lane i gets dims i D / 32 and on, and
// every lane the row's maximum and sum.
template <int D, bool kShared>
__device__ __forceinline__ void add_parts(const float* part_ml, const float* part_o, int rows, int row, int first, int last, int head, float (&o)[D / 32], float& M,
                                          float& L) {
  constexpr int kPer = D / 32;
  const int lane = threadIdx.x & 31;
  M = -INFINITY;
  L = 0.f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) o[i] = 0.f;
  for (int k0 = first; k0 <= last; k0 += 32) {
    const int k = min(k0 + lane, last);
    const auto* at = reinterpret_cast<const float2*>(part_ml + ((static_cast<long long>(k) * 2 + (k == first ? head : 0)) * rows + row) * 2);
    float2 ml = kShared ? *at : __ldcg(at);
    if (k0 + lane > last) ml.y = 0.f;
    float mx = ml.y != 0.f ? ml.x : -INFINITY;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
    const float Mn = fmaxf(M, mx);
    const float keep = M == -INFINITY ? 0.f : exp2f(M - Mn);
    const float wgt = ml.y != 0.f ? exp2f(ml.x - Mn) : -1.f;  // may be zero where there are keys: then 0 * NaN counts
    float ls = ml.y * wgt;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) ls += __shfl_xor_sync(0xffffffffu, ls, off);
    L = L * keep + ls;
    M = Mn;
#pragma unroll
    for (int i = 0; i < kPer; ++i) o[i] *= keep;
    // eight parts at a time, their loads without a condition between them
    for (int i0 = 0; i0 < min(32, last - k0 + 1); i0 += 8) {
      float x[8][kPer];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int part = min(k0 + i0 + i, last);
        const float* src = part_o + ((static_cast<long long>(part) * 2 + (part == first ? head : 0)) * rows + row) * D + lane * kPer;
        if (kPer == 4) *reinterpret_cast<float4*>(x[i]) = kShared ? *reinterpret_cast<const float4*>(src) : __ldcg(reinterpret_cast<const float4*>(src));
        else *reinterpret_cast<float2*>(x[i]) = kShared ? *reinterpret_cast<const float2*>(src) : __ldcg(reinterpret_cast<const float2*>(src));
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float wi = __shfl_sync(0xffffffffu, wgt, i0 + i);
        if (wi < 0.f) continue;  // no keys: what lies there means nothing
#pragma unroll
        for (int d = 0; d < kPer; ++d) o[d] += x[i][d] * wi;
      }
    }
  }
}
// The finished row of a unit into the output.
template <int D>
__device__ __forceinline__ void store_row(const LineParams& p, int row0, int kvh, int r, const float (&o)[D / 32], float L) {
  constexpr int kPer = D / 32;
  const float inv = L != 0.f ? 1.f / L : 0.f;
  const int tk = r / p.G, hd = r - tk * p.G;
  auto* dst = static_cast<__nv_bfloat16*>(p.a.out) + static_cast<long long>(row0 + tk) * p.a.ldo + static_cast<long long>(kvh * p.G + hd) * D +
              (threadIdx.x & 31) * kPer;
  uint32_t y[kPer / 2];
#pragma unroll
  for (int i = 0; i < kPer / 2; ++i) y[i] = pack_bf16x2(o[2 * i] * inv, o[2 * i + 1] * inv);
  if (kPer == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(y[0], y[kPer / 2 - 1]);
  else *reinterpret_cast<uint32_t*>(dst) = y[0];
}

// Two or three parts of two rows at once, all their loads out before the first is needed.
template <int D, int kParts>
__device__ __forceinline__ void add_few_parts(const LineParams& p, int first, int slot, int rows, float (&o)[2][D / 32], float (&L)[2]) {
  constexpr int kPer = D / 32;
  const int lane = threadIdx.x & 31;
  float2 ml[2][kParts];
  float x[2][kParts][kPer];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
      const long long at = (static_cast<long long>(first + i) * 2 + (i == 0 ? 1 : 0)) * p.rows + min(slot + h, rows - 1);
      ml[h][i] = __ldcg(reinterpret_cast<const float2*>(p.part_ml + at * 2));
      if (kPer == 4) *reinterpret_cast<float4*>(x[h][i]) = __ldcg(reinterpret_cast<const float4*>(p.part_o + at * D + lane * kPer));
      else *reinterpret_cast<float2*>(x[h][i]) = __ldcg(reinterpret_cast<const float2*>(p.part_o + at * D + lane * kPer));
    }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float M = -INFINITY;
#pragma unroll
    for (int i = 0; i < kParts; ++i)
      if (ml[h][i].y != 0.f) M = fmaxf(M, ml[h][i].x);
    L[h] = 0.f;
#pragma unroll
    for (int d = 0; d < kPer; ++d) o[h][d] = 0.f;
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
      if (ml[h][i].y == 0.f) continue;  // no keys: what lies there means nothing
      const float w = exp2f(ml[h][i].x - M);
      L[h] += ml[h][i].y * w;
#pragma unroll
      for (int d = 0; d < kPer; ++d) o[h][d] += x[h][i][d] * w;
    }
  }
}

// Adds the parts of the units that several CTAs had. A warp two rows, 16 rows of a tile a block.
template <int D>
__global__ void __launch_bounds__(256) paged_combine_kernel(const LineParams p) {
  pdl_wait();
  pdl_launch();
  const int c = blockIdx.x;
  const int4 u = p.desc[c];
  if (u.y == 0) return;
  const int slot = blockIdx.y * 16 + (threadIdx.x >> 5) * 2;  // of the part: a tile's rows start on 128
  const int tile = slot / 128, per_tile = p.tile_tokens * p.G;
  const int rows = min(per_tile, u.y * p.G - tile * per_tile) + tile * 128;  // places of this tile end here
  if (slot >= rows) return;
  const int r = slot - tile * (128 - per_tile), parts = u.w - c + 1;
  float o[2][D / 32], L[2];
  if (parts == 2) {
    add_few_parts<D, 2>(p, c, slot, rows, o, L);
  } else if (parts == 3) {
    add_few_parts<D, 3>(p, c, slot, rows, o, L);
  } else {
    float M;
    for (int h = 0; h < 2; ++h) add_parts<D, false>(p.part_ml, p.part_o, p.rows, min(slot + h, rows - 1), c, u.w, 1, o[h], M, L[h]);
  }
  store_row<D>(p, u.x, u.z, r, o[0], L[0]);
  if (slot + 1 < rows) store_row<D>(p, u.x, u.z, r + 1, o[1], L[1]);
}

// Workspace of a launch: what LineParams points to.
inline long long line_scratch(int ctas, int rows, int D) { return static_cast<long long>(ctas) * (32 + 2 * rows * (2 + D) * 4); }
inline void place_scratch(LineParams& p, void* scratch, int ctas, int rows) {
  p.rows = rows;
  p.desc = static_cast<int4*>(scratch);
  p.part_ml = reinterpret_cast<float*>(p.desc + 2 * ctas);  // everything on 32 bytes
  p.part_o = p.part_ml + static_cast<long long>(ctas) * 2 * rows * 2;
}
// Always a dependent launch: its own start overlaps the end of the kernel before it, on whose completion it waits.
template <int D>
inline void launch_combine(const LineParams& p, int ctas, cudaStream_t s) {
  auto combine = paged_combine_kernel<D>;
  AGRPO_PREFER_SMEM(combine);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas, (p.rows + 15) / 16);
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  check_cuda(cudaLaunchKernelEx(&cfg, combine, p), "paged_combine");
}

}  // namespace

}  // namespace agrpo
