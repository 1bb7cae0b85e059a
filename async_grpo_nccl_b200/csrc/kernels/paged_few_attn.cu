// Attention of a few rows a unit over the paged cache: decode steps, drafted tokens. Bound by the cache's bytes.
//
// A warp is a worker (paged_line.cuh) and goes through its keys 16 at a time without ever waiting for another one: keys and values come from memory into the
// registers that the matrix instructions read them from, 8-bit codes are turned into 16-bit numbers there, and the loads of the next 16 keys are out while these
// are worked on. The products are the transposed ones, S^T = K Q^T and O^T += V^T P, so that 16 keys (16 dims) fill an instruction's 16 rows and the query rows are
// its 8 columns: with the query rows as the 16 rows, half of every instruction would be idle for a group of up to 8. At the end a CTA adds the parts of its own
// warps.
//
// Which dim of a head a lane holds is free as long as Q agrees (in S) or the result is put back (in O): a lane has consecutive ones, so that its loads are 16 bytes
// and 4 (K) or 8 (V) lanes read a whole 64 or 128 bytes.
//
// 8 bits: the products are fp16, since one instruction turns two codes into fp16, exactly, and bf16 would take five (moves, masks, a product): 312 -> 240 us for 128
// rows of 40 heads over 1000 - 8000 tokens. fp16's exponents are few, so powers of two are kept apart: a row of Q is scaled to a maximum of 2^14 .. 2^15 (28 binades
// down to fp16's subnormals are exact), a key's own power goes into the fp32 factor of its scores, probabilities are held times 2^13 (at most 2^15; below 2^-37 they
// vanish), and O is held relative to a power of two F that the values of 16 keys may be up to 2^14 below; where they are further below, and after F has grown by
// more than 2^14 (a vanished probability could then have counted), 16 keys take the bf16 products.
//
// mma.sync and not tcgen05: at 8 to 16 rows the products are a hundredth of what tcgen05 could do, and its hand-overs (tile in shared memory, barrier, product,
// barrier, scores from tensor memory, probabilities back, barrier) cost more than the keys' bytes: those rows took 490 us that way.
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include <type_traits>

#include "../common/ptx.cuh"
#include "../launchers.h"
#include "../launchers_cache.h"
#include "kv8.cuh"
#include "paged_line.cuh"

namespace agrpo {

namespace {

constexpr int kKeys = 16;
constexpr int kExtra = 4;          // a unit's beginning and end, in tiles
constexpr int kSeqRoom = 128;      // sequences that a CTA has at hand
constexpr float kNone = -3.0e38f;  // maximum of nothing: finite, so that a difference with it is a number

template <bool half>
__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (half)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// An 8 x 8 matrix of 16-bit values, spread over the warp as a product's result, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float power(int byte) { return __uint_as_float(static_cast<uint32_t>(byte) << 23); }  // 2^(byte - 127)

// kN: query rows / 8 of a unit.
template <int D, bool k8, int kN>
struct Few {
  static constexpr int kRows = 8 * kN;
  static constexpr int kWarps = kN == 1 ? (k8 ? 16 : 12) : (k8 ? 12 : 8);
  static constexpr int kPartBytes = kWarps * 2 * kRows * D * 4;  // shared memory: the warps' parts, then (m, l); before that the line
  static constexpr int kSmem = kPartBytes + kWarps * 2 * kRows * 8;
  static_assert(kSmem >= 32768 && kSmem <= 232448 - 1024 - kSeqRoom * 12, "8192 sequences; shared memory");
};

struct Job {  // a unit whose parts this CTA's warps first .. last have
  int first, last, head;       // head: the place of the first one's part
  int row0, tokens, kvh, end;  // end: the CTA that has the unit's last tile
};

template <int D, bool k8, int kN>
__global__ void __launch_bounds__(Few<D, k8, kN>::kWarps * 32, 1) paged_few_attn_kernel(const __grid_constant__ LineParams p) {
  using F = Few<D, k8, kN>;
  constexpr int kW = F::kWarps;
  constexpr int kSteps = D / 16;            // products of S, tiles of O
  constexpr int kKW = k8 ? D / 16 : D / 8;  // words of a key's dims that a lane holds (K: D / 4 dims)
  constexpr int kVW = k8 ? D / 32 : D / 16; // likewise of V (D / 8 dims)
  constexpr int kRow = k8 ? D : 2 * D;      // bytes of a key
  constexpr float kLift = k8 ? 13.f : 0.f;  // probabilities are held times 2^kLift ...
  constexpr float kSlack = k8 ? 2.f : 8.f;  // ... and relative to a maximum that may have grown by this many binades since

  extern __shared__ __align__(16) uint8_t shared[];
  float* part_o = reinterpret_cast<float*>(shared);
  float* part_ml = reinterpret_cast<float*>(shared + F::kPartBytes);
  __shared__ Job jobs[kW + 1];
  int* line = reinterpret_cast<int*>(shared);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  if (threadIdx.x <= kW) jobs[threadIdx.x].tokens = 0;
  pdl_wait();
  pdl_launch();
  measure_line<kW * 32, kKeys, kExtra>(p, line);
  const int worker = blockIdx.x * kW + warp;
  const Share share = find_share<kKeys, kExtra, 2>(p, line, worker, gridDim.x * kW);
  __shared__ int seqs[3 * kSeqRoom], first_seq;
  if (threadIdx.x == 0) first_seq = share.b;
  __syncthreads();  // the line is read, parts come there
  const SeqCache near = {seqs, first_seq, kSeqRoom};
  near.fill(p);
  __syncthreads();
  Walk<kKeys, kExtra> w;
  w.start(p, share, near);
  if (threadIdx.x == 0) p.desc[blockIdx.x] = make_int4(0, 0, 0, 0);

  const int bs = p.c.block_size, Hkv = p.c.Hkv, G = p.G;
  const auto* k_lane = static_cast<const uint8_t*>(p.c.k) + g * kRow + t * 16;                              // key g, a lane's first dims
  const auto* v_lane = static_cast<const uint8_t*>(p.c.v) + 2 * t * kRow + g * (k8 && D == 64 ? 8 : 16);    // key 2 t
  const auto* ks_lane = p.c.k_scale + g;
  const auto* vs_lane = p.c.v_scale + 2 * t;
  int flat = share.before;

  for (; w.more(); flat += w.length(), w.next(p)) {
    const int keys = unit_keys(p, w.s, w.qb), rows = w.tokens(p) * G;
    const long long row0 = w.s.row0 + w.qb * p.tokens;
    const int first_pos = w.s.len - w.s.n + w.qb * p.tokens;  // position of the unit's first row: it sees the keys up to there
    const int* table = p.a.block_tables + w.b * p.a.table_pitch;

    // The pages of the next 32 tiles, one a lane.
    int pages = 0;
    const auto load_pages = [&](int j) {
      const int key = (j + lane) * kKeys;
      pages = key < keys && j + lane < w.j1 ? table[key / bs] : 0;
      if (pages < 0 || pages >= p.c.num_blocks) {
        report_status(p.a.status, kStatusBadIndex);
        pages = 0;
      }
    };
    const auto row_of = [&](int j) {  // first key of tile j: row of the cache
      return (static_cast<long long>(__shfl_sync(0xffffffffu, pages, (j - w.j0) & 31)) * Hkv + w.kvh) * bs + ((j * kKeys) & (bs - 1));
    };
    uint32_t k[2][kKW];           // keys g and g + 8: a lane's dims
    uint32_t v[4][kVW];           // keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9
    uint32_t k_byte[2], v_byte[2];  // scale bytes: of keys g and g + 8; of keys 2 t and 2 t + 1 (16 bits), 2 t + 8 and 2 t + 9
    // Behind the unit's last key nothing is read: zeros, under a factor that is a number.
    const auto load_k = [&](auto tail, int left, long long row) {
      const uint8_t* src = k_lane + row * kRow;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bool on = !decltype(tail)::value || g + 8 * h < left;
#pragma unroll
        for (int i = 0; i < kKW / 4; ++i) {
          uint4 x = make_uint4(0u, 0u, 0u, 0u);
          if (on) x = __ldg(reinterpret_cast<const uint4*>(src + h * 8 * kRow + i * 64));
          k[h][4 * i] = x.x;
          k[h][4 * i + 1] = x.y;
          k[h][4 * i + 2] = x.z;
          k[h][4 * i + 3] = x.w;
        }
        if (k8) {
          k_byte[h] = 127u;
          if (on) k_byte[h] = __ldg(ks_lane + row + 8 * h);
        }
      }
    };
    const auto load_v = [&](auto tail, int left, long long row) {
      const uint8_t* src = v_lane + row * kRow;
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const int key = (h & 1) + 8 * (h >> 1);
        const bool on = !decltype(tail)::value || 2 * t + key < left;
        if (kVW == 2) {
          uint2 x = make_uint2(0u, 0u);
          if (on) x = __ldg(reinterpret_cast<const uint2*>(src + key * kRow));
          v[h][0] = x.x;
          v[h][1] = x.y;
        } else {
#pragma unroll
          for (int i = 0; i < kVW / 4; ++i) {
            uint4 x = make_uint4(0u, 0u, 0u, 0u);
            if (on) x = __ldg(reinterpret_cast<const uint4*>(src + key * kRow + i * 128));
            v[h][(4 * i) % kVW] = x.x;
            v[h][(4 * i + 1) % kVW] = x.y;
            v[h][(4 * i + 2) % kVW] = x.z;
            v[h][(4 * i + 3) % kVW] = x.w;
          }
        }
      }
      if (k8) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          v_byte[h] = __ldg(reinterpret_cast<const unsigned short*>(vs_lane + row + 8 * h));  // in the page, whatever it holds
          if (decltype(tail)::value) {  // a factor that does not count: the maximum takes care of it
            if (2 * t + 8 * h >= left) v_byte[h] = 0u;
            else if (2 * t + 8 * h + 1 >= left) v_byte[h] = (v_byte[h] & 0xffu) * 0x101u;
          }
        }
      }
    };
    load_pages(w.j0);
    // Q: rows g + 8 n, the dims of this lane's keys. Its loads go out while the pages are on their way.
    uint32_t q[kN][kSteps][2];
    float q_pow[kN][2];            // 8 bits: what rows 8 n + 2 t and 8 n + 2 t + 1 of S are to be multiplied with
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      const int r = g + 8 * n, tk = r / G;
      const auto* src = reinterpret_cast<const uint8_t*>(static_cast<const __nv_bfloat16*>(p.a.q) + (row0 + tk) * p.a.ldq +
                                                         static_cast<long long>(w.kvh * G + r - tk * G) * D);
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const int dim = k8 ? 64 * (s / 4) + 16 * t + 4 * (s % 4) : 32 * (s / 2) + 8 * t + 4 * (s % 2);
        uint2 x = make_uint2(0u, 0u);
        if (r < rows) x = __ldg(reinterpret_cast<const uint2*>(src + dim * 2));
        q[n][s][0] = x.x;
        q[n][s][1] = x.y;
      }
    }
    {
      const long long row = row_of(w.j0);
      const int left = keys - w.j0 * kKeys;
      load_k(std::true_type{}, left, row);
      load_v(std::true_type{}, left, row);
    }
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      if (k8) {
        uint32_t top = 0;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) top = __vmaxu2(top, __vmaxu2(q[n][s][0] & 0x7fff7fffu, q[n][s][1] & 0x7fff7fffu));
        top = max(top & 0xffffu, top >> 16);
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = max(static_cast<int>(top >> 7), 15);             // 2^(e - 127) <= max|q| < 2^(e - 126)
        const float up = power(268 - e);                               // to 2^14 .. 2^15
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            q[n][s][i] = pack_f16x2(__uint_as_float(q[n][s][i] << 16) * up, __uint_as_float(q[n][s][i] & 0xffff0000u) * up);
        const int mine = max(e - 14, 1);
#pragma unroll
        for (int i = 0; i < 2; ++i) q_pow[n][i] = power(__shfl_sync(0xffffffffu, mine, (2 * t + i) * 4)) * p.scale_log2;
      } else {
        q_pow[n][0] = q_pow[n][1] = p.scale_log2;
      }
    }
    // o[n][i] = {(dim 2 i, row 2 t), (dim 2 i, row 2 t + 1), (dim 2 i + 1, row 2 t), (dim 2 i + 1, row 2 t + 1)} of rows 8 n and on; m: maximum less kLift
    float o[kN][kSteps][4], m[kN][2], l[kN][2];
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      m[n][0] = m[n][1] = kNone;
      l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int i = 0; i < kSteps; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
    }
    const int hidden = first_hidden(p, w.s, w.qb);
    bool odd = false;              // a value was taken out of the products
    int v_pow = 0, v_first = 0;    // 8 bits: F + 127, at first; O is held in 2^F

    for (int j = w.j0; j < w.j1; ++j) {
      // ---- S^T: 16 keys x 8 kN rows
      float s[kN][4];
#pragma unroll
      for (int n = 0; n < kN; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
      {
        float s2[4] = {0.f, 0.f, 0.f, 0.f};  // one tile of rows: two chains
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          uint32_t a[4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            a[h] = k8 ? codes_f16x2(k[h][i % kKW], false) : k[h][(2 * i) % kKW];
            a[2 + h] = k8 ? codes_f16x2(k[h][i % kKW], true) : k[h][(2 * i + 1) % kKW];
          }
#pragma unroll
          for (int n = 0; n < kN; ++n) mma16<k8>(kN == 1 && (i & 1) ? s2 : s[n], a[0], a[1], a[2], a[3], q[n][i][0], q[n][i][1]);
        }
        if (kN == 1) {
#pragma unroll
          for (int i = 0; i < 4; ++i) s[0][i] += s2[i];
        }
      }
      // the keys' own factors
      float key_pow[2] = {1.f, 1.f};
      if (k8) {
#pragma unroll
        for (int h = 0; h < 2; ++h) key_pow[h] = k_byte[h] == kKv8NanByte ? __uint_as_float(0x7fffffffu) : power(k_byte[h]);
      }
      const bool more = j + 1 < w.j1;
      const int left = keys - (j + 1) * kKeys;
      long long row = 0;
      if (more) {
        if (((j + 1 - w.j0) & 31) == 0) load_pages(j + 1);
        row = row_of(j + 1);
        if (left >= kKeys) load_k(std::false_type{}, left, row);
        else load_k(std::true_type{}, left, row);
      }
      // ---- softmax: keys j * 16 + g (+ 8) of rows 8 n + 2 t (+ 1)
      float z[kN][4];
#pragma unroll
      for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[n][i] *= k8 ? key_pow[i >> 1] * q_pow[n][i & 1] : q_pow[n][i & 1];
      if (j * kKeys + kKeys - 1 > first_pos) {
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (j * kKeys + g + 8 * (i >> 1) > first_pos + (8 * n + 2 * t + (i & 1)) / G) s[n][i] = -INFINITY;
      }
      float top = -INFINITY;
#pragma unroll
      for (int n = 0; n < kN; ++n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) z[n][i] = s[n][i] - m[n][i & 1];
        top = max3(top, max3(z[n][0], z[n][1], z[n][2]), z[n][3]);
      }
      if (__any_sync(0xffffffffu, top > kSlack + kLift)) {  // some maximum has grown by more than that
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float mx = fmaxf(s[n][i], s[n][i + 2]);
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
            mx -= kLift;
            if (mx > m[n][i]) {
              const float alpha = exp2f(m[n][i] - mx);  // 0 at first
              m[n][i] = mx;
              l[n][i] *= alpha;
#pragma unroll
              for (int d = 0; d < kSteps; ++d) {
                o[n][d][i] *= alpha;
                o[n][d][i + 2] *= alpha;
              }
              z[n][i] = s[n][i] - mx;
              z[n][i + 2] = s[n][i + 2] - mx;
            }
          }
      }
      uint32_t pb[kN][2];   // P: rows 8 n + g, keys 2 t, 2 t + 1 (+ 8)
#pragma unroll
      for (int n = 0; n < kN; ++n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          z[n][i] = exp2f(z[n][i]);
          l[n][i & 1] += z[n][i];
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
          pb[n][h] = transpose8(k8 ? pack_f16x2(z[n][2 * h], z[n][2 * h + 1]) : pack_bf16x2(z[n][2 * h], z[n][2 * h + 1]));
      }
      // ---- O^T += V^T P: tile i has dims 2 i and 2 i + 1 of every lane's; a = {(dim 2 i, keys 2 t and 2 t + 1), (dim 2 i + 1, same), both of keys + 8}
      if (k8) {
        uint32_t f[2] = {__byte_perm(v_byte[0], 0u, 0x4140), __byte_perm(v_byte[1], 0u, 0x4140)};  // a byte a half
        const auto fits = [&] {  // fp16 exponents 1 .. 16 of the factors relative to F
          const uint32_t c = static_cast<uint32_t>(14 - v_pow) * 0x10001u;
          return !__any_sync(0xffffffffu, (((f[0] + c) | (f[1] + c)) & 0xfff0fff0u) != 0u);
        };
        bool good = fits();
        if (!good && hidden < keys && (j + 1) * kKeys > hidden) {
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            const int shift = 16 * (h & 1);
            if (((f[h >> 1] >> shift) & 0xffffu) != kKv8NanByte || j * kKeys + 2 * t + (h & 1) + 8 * (h >> 1) < hidden) continue;
            f[h >> 1] &= 0xffff0000u >> shift;
            odd = true;
#pragma unroll
            for (int i = 0; i < kVW; ++i) v[h][i] = 0u;
          }
        }
        if (!good) {  // another F: the largest byte, without those of NaN
          const auto real = [](uint32_t x) { return x == 255u ? 0u : x; };
          const uint32_t mine = max(max(real(f[0] & 0xffffu), real(f[0] >> 16)), max(real(f[1] & 0xffffu), real(f[1] >> 16)));
          const int most = static_cast<int>(__reduce_max_sync(0xffffffffu, mine));
          if (most > v_pow) {
            const float down = v_pow == 0 ? 0.f : power(max(127 + v_pow - most, 0));
            v_pow = most;
            if (v_first == 0) v_first = most;
#pragma unroll
            for (int n = 0; n < kN; ++n)
#pragma unroll
              for (int i = 0; i < kSteps; ++i)
#pragma unroll
                for (int d = 0; d < 4; ++d) o[n][i][d] *= down;
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {  // keys that are not there
            if ((f[h] & 0xffffu) == 0u) f[h] |= v_pow;
            if ((f[h] >> 16) == 0u) f[h] |= v_pow << 16;
          }
          good = fits();
        }
        if (good && v_pow <= v_first + 14) {
          const uint32_t c = static_cast<uint32_t>(15 - v_pow) * 0x10001u;
          const uint32_t f16[2] = {(f[0] + c) << 10, (f[1] + c) << 10};
#pragma unroll
          for (int i = 0; i < kSteps; ++i) {
            uint32_t a[4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              // codes (dim 2 i: both keys), (dim 2 i + 1: both keys)
              const uint32_t x = __byte_perm(v[2 * h][i / 2], v[2 * h + 1][i / 2], i & 1 ? 0x7362 : 0x5140);
              a[2 * h] = mul_f16x2(codes_f16x2(x, false), f16[h]);
              a[2 * h + 1] = mul_f16x2(codes_f16x2(x, true), f16[h]);
            }
#pragma unroll
            for (int n = 0; n < kN; ++n) mma16<true>(o[n][i], a[0], a[1], a[2], a[3], pb[n][0], pb[n][1]);
          }
        } else {  // values of very different sizes, or a NaN
#pragma unroll
          for (int n = 0; n < kN; ++n) {
            pb[n][0] = transpose8(pack_bf16x2(z[n][0], z[n][1]));
            pb[n][1] = transpose8(pack_bf16x2(z[n][2], z[n][3]));
          }
          Kv8Scale x[2][2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int b0 = f[h] & 0xffffu, b1 = f[h] >> 16;
            x[h][0] = kv8_scale(b0 == kKv8NanByte ? b0 : max(b0 - v_pow + 127, 0));
            x[h][1] = kv8_scale(b1 == kKv8NanByte ? b1 : max(b1 - v_pow + 127, 0));
          }
#pragma unroll
          for (int i = 0; i < kSteps; ++i) {
            uint32_t a[4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              // no factor is above 1 here, so one product does
              const uint2 lo = kv8_decode4(v[2 * h][i / 2], x[h][0]), hi = kv8_decode4(v[2 * h + 1][i / 2], x[h][1]);
              const uint32_t u = i & 1 ? lo.y : lo.x, y = i & 1 ? hi.y : hi.x;
              a[2 * h] = __byte_perm(u, y, 0x5410);
              a[2 * h + 1] = __byte_perm(u, y, 0x7632);
            }
#pragma unroll
            for (int n = 0; n < kN; ++n) mma16<false>(o[n][i], a[0], a[1], a[2], a[3], pb[n][0], pb[n][1]);
          }
        }
      } else {
        if (hidden < keys && (j + 1) * kKeys > hidden) {
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            uint32_t nan = 0u;
#pragma unroll
            for (int i = 0; i < kVW; ++i) nan = times_zero(v[h][i], nan);
            if ((nan & 0x7fff7fffu) == 0u || j * kKeys + 2 * t + (h & 1) + 8 * (h >> 1) < hidden) continue;
            odd = true;
#pragma unroll
            for (int i = 0; i < kVW; ++i) v[h][i] = only_finite(v[h][i]);
          }
        }
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          uint32_t a[4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            a[2 * h] = __byte_perm(v[2 * h][i % kVW], v[2 * h + 1][i % kVW], 0x5410);
            a[2 * h + 1] = __byte_perm(v[2 * h][i % kVW], v[2 * h + 1][i % kVW], 0x7632);
          }
#pragma unroll
          for (int n = 0; n < kN; ++n) mma16<false>(o[n][i], a[0], a[1], a[2], a[3], pb[n][0], pb[n][1]);
        }
      }
      if (more) {
        if (left >= kKeys) load_v(std::false_type{}, left, row);
        else load_v(std::true_type{}, left, row);
      }
    }

    // ---- the piece's end
    if (__any_sync(0xffffffffu, odd)) {
      const int last = min(keys, w.j1 * kKeys);
#pragma unroll 1
      for (int key = max(hidden, w.j0 * kKeys); key < last; ++key) {
        const int page = table[key / bs];
        if (page < 0 || page >= p.c.num_blocks) continue;
        const long long row = (static_cast<long long>(page) * Hkv + w.kvh) * bs + (key & (bs - 1));
        const bool nan = k8 && p.c.v_scale[row] == kKv8NanByte;
        const auto* src = reinterpret_cast<const uint32_t*>(v_lane - 2 * t * kRow + row * kRow);
        const int rows_from = (key - first_pos) * G;  // the rows that see it
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          const uint32_t x = k8 ? (nan ? 0x7fff7fffu : 0u) : src[i % 4 + i / 4 * 32];
#pragma unroll
          for (int n = 0; n < kN; ++n)
#pragma unroll
            for (int d = 0; d < 4; ++d) {
              const uint32_t half = d < 2 ? x << 16 : x & 0xffff0000u;
              if (!is_finite(half >> 16) && 8 * n + 2 * t + (d & 1) >= rows_from) o[n][i][d] += __uint_as_float(half);
            }
        }
      }
    }
    const bool whole = w.whole();
    const int part = w.part(warp) * F::kRows;
    // The lift and F leave one after the other: values are then right from 2^-116 on (F over a sum of 2^13 and more would be below the smallest number) and up
    // to a sum of 2^128, in parts as well.
    const float unit = k8 ? power(v_pow) : 1.f, drop = k8 ? power(127 - static_cast<int>(kLift)) : 1.f;
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = 8 * n + 2 * t + i;
        float sum = l[n][i];
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        if (r >= rows) continue;
        // a lane's dims: D / 8 from D / 8 * g on (8 bits), or 8 from 8 g (+ 64) on
        if (whole) {
          const float f = sum != 0.f ? 1.f / sum : 0.f;
          const auto value = [&](float x) { return x * f * unit; };
          const int tk = r / G;
          auto* dst = static_cast<__nv_bfloat16*>(p.a.out) + (row0 + tk) * p.a.ldo + static_cast<long long>(w.kvh * G + r - tk * G) * D;
#pragma unroll
          for (int i4 = 0; i4 < kSteps / 4; ++i4) {
            uint4 y;
            y.x = pack_bf16x2(value(o[n][4 * i4][i]), value(o[n][4 * i4][i + 2]));
            y.y = pack_bf16x2(value(o[n][4 * i4 + 1][i]), value(o[n][4 * i4 + 1][i + 2]));
            y.z = pack_bf16x2(value(o[n][4 * i4 + 2][i]), value(o[n][4 * i4 + 2][i + 2]));
            y.w = pack_bf16x2(value(o[n][4 * i4 + 3][i]), value(o[n][4 * i4 + 3][i + 2]));
            *reinterpret_cast<uint4*>(dst + (k8 ? D / 8 * g + 8 * i4 : 8 * g + 64 * i4)) = y;
          }
        } else {
          float* dst = part_o + (part + r) * D;
          const auto value = [&](float x) { return x * drop * unit; };
#pragma unroll
          for (int i2 = 0; i2 < kSteps / 2; ++i2) {
            const int dim = k8 ? D / 8 * g + 4 * i2 : 8 * g + 64 * (i2 / 2) + 4 * (i2 % 2);
            *reinterpret_cast<float4*>(dst + dim) =
                make_float4(value(o[n][2 * i2][i]), value(o[n][2 * i2][i + 2]), value(o[n][2 * i2 + 1][i]), value(o[n][2 * i2 + 1][i + 2]));
          }
          if (g == 0) *reinterpret_cast<float2*>(part_ml + (part + r) * 2) = make_float2(m[n][i], sum * drop);
        }
      }
    // A unit that starts in this warp and goes on, or that goes on from the CTA before: its parts in this CTA are added below.
    if (lane == 0 && !whole && (w.j0 == 0 || warp == 0)) {
      const int end = w.last_worker(share, flat);
      Job& job = jobs[w.j0 == 0 ? warp : kW];
      job.first = warp;
      job.last = min(end - static_cast<int>(blockIdx.x) * kW, kW - 1);
      job.head = w.j0 == 0 ? 1 : 0;
      job.row0 = static_cast<int>(row0);
      job.tokens = w.tokens(p);
      job.kvh = w.kvh;
      job.end = end / kW;
    }
  }

  __syncthreads();
  for (int i = warp; i < (kW + 1) * F::kRows; i += kW) {
    const Job& job = jobs[i / F::kRows];
    const int r = i % F::kRows;
    if (r >= job.tokens * G) continue;
    float o[D / 32], M, L;
    add_parts<D, true>(part_ml, part_o, F::kRows, r, job.first, job.last, job.head, o, M, L);
    const bool here = job.end == static_cast<int>(blockIdx.x);
    if (here && job.head == 1) {
      store_row<D>(p, job.row0, job.kvh, r, o, L);
      continue;
    }
    const long long part = (static_cast<long long>(blockIdx.x) * 2 + job.head) * F::kRows + r;
#pragma unroll
    for (int d = 0; d < D / 32; ++d) p.part_o[part * D + lane * (D / 32) + d] = o[d];
    if (lane == 0) {
      *reinterpret_cast<float2*>(p.part_ml + part * 2) = make_float2(M, L);
      if (r == 0 && job.head == 1) p.desc[blockIdx.x] = make_int4(job.row0, job.tokens, job.kvh, job.end);
    }
  }
}

template <int D, bool k8, int kN>
void launch(LineParams p, int num_sms, void* scratch, cudaStream_t s) {
  using F = Few<D, k8, kN>;
  p.tokens = p.tile_tokens = F::kRows / p.G;
  place_scratch(p, scratch, num_sms, F::kRows);
  auto kernel = paged_few_attn_kernel<D, k8, kN>;
  AGRPO_SET_MAX_DYN_SMEM(kernel, F::kSmem, "paged_few_attn smem attr");
  launch_kernel(kernel, dim3(num_sms), dim3(F::kWarps * 32), F::kSmem, s, "paged_few_attn", p);
  launch_combine<D>(p, num_sms, s);
}

}  // namespace

void launch_paged_few_attn(const ChunkAttnArgs& a, const PagedCache& c, int rows, int num_sms, void* scratch, cudaStream_t s) {
  LineParams p = {};
  p.a = a;
  p.c = c;
  p.G = a.Hq / c.Hkv;
  p.scale_log2 = a.softmax_scale * 1.4426950408889634f;
  const auto run = [&](auto d, auto k8) {
    if (rows <= 8) launch<decltype(d)::value, decltype(k8)::value, 1>(p, num_sms, scratch, s);
    else launch<decltype(d)::value, decltype(k8)::value, 2>(p, num_sms, scratch, s);
  };
  using D128 = std::integral_constant<int, 128>;
  using D64 = std::integral_constant<int, 64>;
  if (c.k_scale != nullptr) c.D == 128 ? run(D128{}, std::true_type{}) : run(D64{}, std::true_type{});
  else c.D == 128 ? run(D128{}, std::false_type{}) : run(D64{}, std::false_type{});
}

}  // namespace agrpo
