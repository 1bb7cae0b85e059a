// Launchers of the 8-bit KV cache and of the attention of new tokens over the paged cache (kv8_cache.cu, paged_chunk_attn.cu).
#pragma once
#include <cuda_runtime.h>

namespace agrpo {

// One layer's paged cache: k and v [num_blocks, Hkv, block_size, D], bf16, or e4m3 codes with a scale byte for each vector
// (k_scale, v_scale [num_blocks, Hkv, block_size]; both null for bf16).
struct PagedCache {
  void* k = nullptr;
  void* v = nullptr;
  unsigned char* k_scale = nullptr;
  unsigned char* v_scale = nullptr;
  int num_blocks = 0, Hkv = 0, block_size = 0, D = 0;
};

// Rows of qkv ([T, pitch], k heads from column k_col0, v heads from v_col0) into the slots of an 8-bit cache; slots[t] < 0 skips row t.
void launch_kv8_write(const void* qkv, long long pitch, int k_col0, int v_col0, const int* slots, const PagedCache& c, int T, int* status,
                      cudaStream_t s);
// The other way, for either type of cache: rows of qkv whose slot is negative stay as they are.
void launch_kv_cache_read(const PagedCache& c, const int* slots, void* qkv, long long pitch, int k_col0, int v_col0, int T, int* status,
                          cudaStream_t s);
// Rotates the q and k heads of row b in place (position seq_lens[b] - 1, clamped to the tables) and writes its k and v to the 8-bit cache.
void launch_rope_kv8_write_decode(void* qkv, long long pitch, const float* cos_t, const float* sin_t, int max_pos, const int* block_tables,
                                  long long table_pitch, int max_blocks, const int* seq_lens, const PagedCache& c, int B, int Hq, int* status,
                                  cudaStream_t s);

struct ChunkAttnArgs {
  const void* q;  // bf16 rows, head h at column h * D
  long long ldq;
  void* out;      // bf16 rows, likewise
  long long ldo;
  const int* block_tables;  // [B, table_pitch]
  long long table_pitch;
  int max_blocks;           // entries of a table row
  const int* seq_lens;      // [B]
  const int* q_starts;      // [B + 1]
  int B, Tq, Hq;
  float softmax_scale;
  int* status;
};
// Tiles of keys that the call has at most, if every table is full: has to be below 2^31.
long long paged_chunk_attn_tiles(const ChunkAttnArgs& a, const PagedCache& c);
// `scratch` holds paged_chunk_attn_scratch bytes, 16-byte aligned, and belongs to the call.
long long paged_chunk_attn_scratch(const ChunkAttnArgs& a, const PagedCache& c, int num_sms);
void launch_paged_chunk_attn(const ChunkAttnArgs& a, const PagedCache& c, int num_sms, void* scratch, cudaStream_t s);

// An 8-bit cache in bf16, for the sequences that have rows: block i of sequence b is block b * max_blocks + i of `to` (with its num_blocks set by the caller), which
// is what `table` [B, max_blocks] says afterwards. Blocks behind a sequence's tokens are left as they are.
void launch_kv8_unpack(const ChunkAttnArgs& a, const PagedCache& c, const PagedCache& to, int* table, cudaStream_t s);

// Its form for units of up to 8 or 16 rows (paged_few_attn.cu).
void launch_paged_few_attn(const ChunkAttnArgs& a, const PagedCache& c, int rows, int num_sms, void* scratch, cudaStream_t s);

}  // namespace agrpo
