// How paged decode attention cuts a sequence into chunks, and the partial results of its chunks: what the launcher in attn.cu and the merge kernels agree on.
#pragma once
#include "kernels.cuh"

namespace wf {

constexpr int AT_BLK = 16;                              // tokens per stage
constexpr int AT_D = 128;                               // head_dim (all supported shapes)

// Blocks per chunk of a sequence with `nblocks` 16-token blocks.  The host sizes chunk_blocks from the length HINT of the captured graph
// (a power of two >= the longest sequence); a sequence well below the hint would fill only the first chunks (2049 tokens under a 4096
// hint: chunks of 128 + 1 blocks) — so every (sequence, kv head) pair cuts its own length evenly.  Same value in every CTA of the pair
// and in the merge kernel (it depends on seq_lens only).
__device__ __forceinline__ int chunk_blocks_of(int nblocks, int chunk_blocks, int max_chunks, int min_cb) {
    if (min_cb <= 0 || max_chunks <= 1) return chunk_blocks;
    int c = ((max(nblocks, 1) + max_chunks - 1) / max_chunks + 3) & ~3;
    c = max(c, min_cb);
    return min(c, chunk_blocks);
}

// The chunks' partial results, left unmerged: of chunk c of head h of sequence b, sum of exp2(s - m) v (part_o [B][H][max_chunks][AT_D], float), m and the sum of
// exp2(s - m) (part_ml [B][H][max_chunks][2]), scores s in units of log 2.  A sequence of L tokens has ceil(ceil(L / AT_BLK) / chunk_blocks_of(...)) of them.
struct AttnChunks {
    const float *part_o, *part_ml;
    int max_chunks, chunk_blocks, min_cb;
};
// workspace: attn_chunks_bytes.  beside (bf16 pools): the kernel launched before has waited for all that this part reads, lets the next one start at once and leaves it 64 KB
// of shared memory and 168 x 128 registers of every SM
size_t attn_chunks_bytes(int B, int H, int Hkv, int max_seq);
int attn_decode_chunks(const void* q, const void* pool, int layers, int layer, int Hkv, int page_size, const int32_t* block_table, int max_blocks, const int32_t* seq_lens, int B, int H,
                       float scale, void* ws, size_t ws_bytes, float* kv_scales, bool beside, AttnChunks* out, cudaStream_t s);

// what the decode attention entry points ask of their cache, heads and output (pointers: none of theirs is null)
int check_decode_attn(const wf_kv_layout* kv, int layer, int H, int out_dtype, bool pointers, const char* who);
float* kv_scales_of(const wf_kv_layout* kv);           // scale region of an int8 pool, null for others

}  // namespace wf
