// Device helpers of the paged latent cache: rotary angles, the 4-bit form of a
// latent row, and the row and length lookups of a ragged call.
#pragma once

#include "mla_common.cuh"

namespace mla {

// ---------------------------------------------------------------------------
// The 4-bit form of a latent row: 16 groups of 32 dims, each with a float16 scale
// s; a dim's code n (0..15) stands for (n - 8) s.  Eight consecutive dims d0..d7
// share a 32-bit word whose nibbles, lowest first, are d0 d2 d4 d6 d1 d3 d5 d7, so
// that (word >> 4 j) & 0x000f000f holds dims 2 j and 2 j + 1 as two 16-bit fields.
// ---------------------------------------------------------------------------
constexpr int kI4Group = 32;
constexpr int kI4Groups = kDim / kI4Group;   // scales per row
constexpr int kI4Bytes = kDim / 2;           // code bytes per row

// Codes of dims 2 j, 2 j + 1 (j = 0..3) of word w as (n - 8) in two halves: 0x6400 is
// 1024 in fp16, whose last bit counts ones, so 1024 + n is exact and so is the
// difference.
__device__ __forceinline__ __half2 i4_pair(uint32_t w, int j) {
  const uint32_t v = ((w >> (4 * j)) & 0x000f000fu) | 0x64006400u;
  return __hsub2(*reinterpret_cast<const __half2*>(&v), __half2half2(__ushort_as_half((unsigned short)0x6408u)));
}

// ---------------------------------------------------------------------------
// Rotary angles.  turns = position x frequency / 2 pi in double: position 2^20 and
// the fastest pair make 1.7e5 turns, whose fraction a float would hold to 0.02 of a
// turn only.  The fraction in [-1/2, 1/2] then fits a float (2^-26 of a turn).
// ---------------------------------------------------------------------------
__device__ __forceinline__ float2 rotary_cos_sin(int pos, double turns_per_pos, float gain) {
  double t = (double)pos * turns_per_pos;
  t -= rint(t);
  float s, c;
  sincospif(2.f * (float)t, &s, &c);
  return make_float2(c * gain, s * gain);
}

// ---------------------------------------------------------------------------
// Ragged calls: rows query sequence qs = (s * q_len + t) * kv_heads + kvh attends to,
// the same rule as the tensor-core kernel's: its sequence's length clamped to
// [0, max_len], less the q_len - 1 - t rows the causal mask hides.
// ---------------------------------------------------------------------------
__device__ __forceinline__ int ragged_len(const int* seqlens, int qs, int q_len, int kv_heads, int max_len) {
  int len = max_len;
  if (seqlens != nullptr) {
    len = __ldg(seqlens + qs / (q_len * kv_heads));
    len = len < 0 ? 0 : (len > max_len ? max_len : len);
  }
  len -= q_len - 1 - (qs / kv_heads) % q_len;
  return len < 0 ? 0 : len;
}

// Cache row of row `row` of sequence `seq`: contiguous [batch, seqlen] rows, or a
// page of the block table; -1 when the table names a page the cache does not have
// (such rows read as zeros).
__device__ __forceinline__ long long cache_row(const int* block_table, int max_pages, int page_size, int num_pages,
                                               int seqlen, int seq, int row) {
  if (block_table == nullptr) return (long long)seq * seqlen + row;
  const int pg = __ldg(block_table + (size_t)seq * max_pages + row / page_size);
  return (unsigned)pg < (unsigned)num_pages ? (long long)pg * page_size + row % page_size : -1;
}

// ---------------------------------------------------------------------------
// A decode call over a 4-bit cache (mla_decode_ext_int4kv).
// ---------------------------------------------------------------------------
struct Int4Args {
  const void* q;
  const void* q_pe;
  const uint8_t* codes;     // [rows][kv_heads][256]
  const __half* scales;     // [rows][kv_heads][16]
  const void* k_pe;         // [rows][kv_heads][64]
  const int* block_table;   // [batch][max_pages] or nullptr
  const int* seqlens;       // [batch] or nullptr
  void* out;
  float* lse;               // optional
  float* part_o;
  float* part_lse;
  int batch, q_len, heads, kv_heads, max_seqlen, page_size, num_pages, max_pages, dtype;
  int max_len;              // max_seqlen, or what the block table covers if that is less
  float softmax_scale;
};

// CUDA-core kernel (mla_int4_simt.cu): splits per query sequence, and the launches.
int int4_simt_splits(int qb, int g, int max_len, int asked);
cudaError_t launch_int4_simt(const Int4Args& a, int ns, cudaStream_t stream);

// Warp-level MMA kernel for few query rows (mla_int4_mma.cu): groups of 16 row_tiles
// query rows (row_tiles 1 or 2) of a KV sequence; workspace [status 256 B][info][partial
// LSE][partial O], the status word zero before the first call.
struct Int4MmaPlan {
  int row_tiles, groups, workers;
  long long units;      // (sequence, KV head, row group) triples
  size_t info_off, lse_off, o_off, total;
};
Int4MmaPlan int4_mma_plan(int batch, int q_len, int heads, int kv_heads, int max_len, int row_tiles, int asked);
cudaError_t launch_int4_mma(Int4Args a, const Int4MmaPlan& plan, void* workspace, cudaStream_t stream);

}  // namespace mla
