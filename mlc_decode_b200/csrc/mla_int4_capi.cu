// extern "C" entry points of the decode over a 4-bit latent cache (declared in
// include/mla_decode_b200.h): argument checks, kernel choice and workspace carving.
#include <limits.h>
#include <math.h>

#include "mla_cache.cuh"
#include "mla_sm100.cuh"

namespace mla {
namespace {

inline size_t align_up(size_t x, size_t a) { return (x + a - 1) / a * a; }

enum Int4Kernel { kSimt, kPair, kMma };

// Which of the two tensor-core kernels, by the time each is expected to take in us for
// sequences of the maximal length, the one the host knows (fits to measured calls, one
// B200; rows = query rows per KV head):
//   warp-level, 16 rows a CTA and two CTAs an SM: 16 + 4.0 per round of 64-row tiles;
//   32 rows and one CTA: 16 + 3.1 per round;
//   pair kernel, 128 rows a pair: 30 + 2.9 per round of 128-row tiles, and 15 or 45 to merge
//   sequences cut in many or few pieces, unless each has a pair of its own.
// Measured, warp-level : pair, L2 flushed: b128 s4096, 16 rows 130 : 219, 32 rows 200 : 221, 64
// rows 370 : 223; b64 s8192, 128 rows 693 : 207; b1 s131072, 128 rows 185 : 82, 16 rows
// 54 : 82; b6 s3001, 3 positions x 40 heads 50 : 76; b1 s300, 16 rows 17 : 43.
bool warp_level_is_faster(long long seqs, int q_len, int g, int max_len) {
  const long long rows = (long long)q_len * g;
  const int mt = rows <= 16 ? 1 : 2;
  auto rounds = [](long long n, long long d) { return (double)((n + d - 1) / d); };
  const double mma = 16. + (mt == 1 ? 4.0 : 3.1) * rounds(seqs * ((rows + 16 * mt - 1) / (16 * mt)) * ((max_len + 63) / 64),
                                                          mt == 1 ? 296 : 148);
  const long long vs = seqs * q_len * ((g + 127) / 128), nt = (max_len + 127) / 128;
  const double ranges = rounds(vs * nt, 74), split = 30. + 2.9 * ranges + (nt <= 3 * ranges ? 45. : 15.);
  const double whole = 30. + 2.9 * nt;
  return mma <= (vs <= 74 && whole < split ? whole : split);
}

struct Int4Plan {
  Int4Kernel kernel;
  int splits;       // CUDA-core kernel
  Int4MmaPlan mma;
  size_t lse_off, o_off;
  size_t total;     // workspace bytes
};

int plan_call(const char* fn, int batch, int q_len, int heads, int kv_heads, int max_seqlen_kv, int dtype,
              const MlaCfg* cfg, Int4Plan* p) {
  if (batch < 1 || heads < 1 || max_seqlen_kv < 1 || q_len < 1 || kv_heads < 1 || heads % kv_heads != 0) {
    set_error("%s: batch, q_len, heads, kv_heads and max_seqlen_kv must be >= 1 with heads a multiple of kv_heads "
              "(got %d, %d, %d, %d, %d)", fn, batch, q_len, heads, kv_heads, max_seqlen_kv);
    return MLA_ERR_ARG;
  }
  if (dtype != MLA_DTYPE_F16 && dtype != MLA_DTYPE_BF16) {
    set_error("%s: dtype must be 0 (fp16) or 1 (bf16), got %d", fn, dtype);
    return MLA_ERR_ARG;
  }
  const long long qb = (long long)batch * q_len * kv_heads;
  if (qb > 65535 || (long long)batch * q_len * heads > (1ll << 30) ||
      (long long)batch * max_seqlen_kv > INT_MAX - 256) {
    set_error("%s: shape too large (batch %d, q_len %d, heads %d, kv_heads %d, max_seqlen_kv %d)", fn, batch, q_len,
              heads, kv_heads, max_seqlen_kv);
    return MLA_ERR_UNSUPPORTED;
  }
  const int asked = cfg != nullptr ? cfg->num_split : 0;
  const int kernel = cfg != nullptr ? cfg->kernel : MLA_KERNEL_AUTO;
  if (asked < 0 || asked > 8192 || kernel < MLA_KERNEL_AUTO || kernel > MLA_KERNEL_TC) {
    set_error("%s: num_split must be in [0, 8192] and kernel a MlaKernelKind (got %d, %d)", fn, asked, kernel);
    return MLA_ERR_ARG;
  }
  if (kernel != MLA_KERNEL_SIMT) {
    const int rows = q_len * (heads / kv_heads);
    const bool covered = sm100_supports_ext(batch, q_len, heads, kv_heads, max_seqlen_kv);
    // block_H, query rows per CTA: up to 32 asks for the warp-level kernel, more for the pair kernel
    const int block_h = cfg != nullptr ? cfg->block_H : 0;
    const bool mma = block_h > 0 ? block_h <= 32
                                 : !covered || warp_level_is_faster((long long)batch * kv_heads, q_len,
                                                                    heads / kv_heads, max_seqlen_kv);
    if (mma) {
      p->kernel = kMma;
      p->mma = int4_mma_plan(batch, q_len, heads, kv_heads, max_seqlen_kv, (block_h > 0 ? block_h : rows) <= 16 ? 1 : 2,
                             asked);
      p->total = p->mma.total;
      return MLA_OK;
    }
    if (!covered) {
      set_error("%s: shape outside the pair kernel (batch %d, q_len %d, heads %d, kv_heads %d, max_seqlen_kv %d)", fn,
                batch, q_len, heads, kv_heads, max_seqlen_kv);
      return MLA_ERR_UNSUPPORTED;
    }
    p->kernel = kPair;
    p->total = ext_int4_workspace(fn, batch, q_len, heads, kv_heads, max_seqlen_kv, dtype, cfg);
    return p->total > 0 ? MLA_OK : MLA_ERR_ARG;
  }
  p->kernel = kSimt;
  p->splits = int4_simt_splits((int)qb, heads / kv_heads, max_seqlen_kv, asked);
  const size_t rows = p->splits > 1 ? (size_t)p->splits * batch * q_len * heads : 0;
  // (a status word as in the other kernels' workspaces, which this kernel leaves zero)
  p->lse_off = rows > 0 ? 256 : 0;
  p->o_off = p->lse_off + align_up(rows * sizeof(float), 256);
  p->total = p->o_off + rows * kDim * sizeof(float);
  return MLA_OK;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace
}  // namespace mla

using namespace mla;

extern "C" {

size_t mla_decode_int4kv_workspace_bytes(int32_t batch, int32_t q_len, int32_t heads, int32_t kv_heads,
                                         int32_t max_seqlen_kv, int32_t dtype, const MlaCfg* cfg) {
  set_error("%s", "");
  Int4Plan p;
  if (plan_call("mla_decode_int4kv_workspace_bytes", batch, q_len, heads, kv_heads, max_seqlen_kv, dtype, cfg, &p) !=
      MLA_OK)
    return 0;
  return p.total;
}

int32_t mla_decode_ext_int4kv(const void* q, const void* q_pe, const void* kv_codes, const void* kv_scales,
                              const void* k_pe_cache, const int32_t* block_table, const int32_t* cache_seqlens,
                              void* out, float* lse, void* workspace, size_t workspace_bytes, int32_t batch,
                              int32_t q_len, int32_t heads, int32_t kv_heads, int32_t max_seqlen_kv,
                              int32_t page_size, int32_t num_pages, int32_t max_pages_per_seq, int32_t dtype,
                              const MlaCfg* cfg, void* stream) {
  const char* fn = "mla_decode_ext_int4kv";
  Int4Plan p;
  int rc = plan_call(fn, batch, q_len, heads, kv_heads, max_seqlen_kv, dtype, cfg, &p);
  if (rc != MLA_OK) return rc;
  if (!kv_scales || !aligned16(kv_scales)) {
    set_error(kv_scales ? "%s: tensor pointers must be 16-byte aligned" : "%s: null pointer", fn);
    return MLA_ERR_ARG;
  }
  if (p.kernel == kPair)
    return decode_ext_int4(fn, q, q_pe, kv_codes, kv_scales, k_pe_cache, block_table, cache_seqlens, out, lse,
                           workspace, workspace_bytes, batch, q_len, heads, kv_heads, max_seqlen_kv, page_size,
                           num_pages, max_pages_per_seq, dtype, cfg, stream);
  if (!q || !q_pe || !kv_codes || !k_pe_cache || !out) {
    set_error("%s: null pointer", fn);
    return MLA_ERR_ARG;
  }
  if (!aligned16(q) || !aligned16(q_pe) || !aligned16(kv_codes) || !aligned16(k_pe_cache) || !aligned16(out)) {
    set_error("%s: tensor pointers must be 16-byte aligned", fn);
    return MLA_ERR_ARG;
  }
  if (block_table != nullptr &&
      (page_size < 64 || page_size % 64 != 0 || num_pages < 1 || max_pages_per_seq < 1 ||
       (long long)num_pages * page_size >= (1ll << 31) - 256)) {
    set_error("%s: page_size must be a positive multiple of 64, with num_pages x page_size rows below 2^31 "
              "(page_size %d, num_pages %d, max_pages_per_seq %d)", fn, page_size, num_pages, max_pages_per_seq);
    return MLA_ERR_ARG;
  }
  if (p.total > 0 && (workspace == nullptr || workspace_bytes < p.total ||
                      (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0)) {
    set_error("%s: workspace needs %zu bytes, 256-byte aligned (got %zu at %p)", fn, p.total, workspace_bytes,
              workspace);
    return MLA_ERR_WORKSPACE;
  }
  Int4Args a{};
  a.q = q;
  a.q_pe = q_pe;
  a.codes = static_cast<const uint8_t*>(kv_codes);
  a.scales = static_cast<const __half*>(kv_scales);
  a.k_pe = k_pe_cache;
  a.block_table = block_table;
  a.seqlens = cache_seqlens;
  a.out = out;
  a.lse = lse;
  if (p.kernel == kSimt) {
    a.part_lse = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.lse_off);
    a.part_o = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.o_off);
  }
  a.batch = batch;
  a.q_len = q_len;
  a.heads = heads;
  a.kv_heads = kv_heads;
  a.max_seqlen = max_seqlen_kv;
  a.page_size = block_table != nullptr ? page_size : 0;
  a.num_pages = block_table != nullptr ? num_pages : 0;
  a.max_pages = block_table != nullptr ? max_pages_per_seq : 0;
  a.dtype = dtype;
  a.max_len = max_seqlen_kv;
  if (block_table != nullptr && (long long)max_pages_per_seq * page_size < max_seqlen_kv)
    a.max_len = max_pages_per_seq * page_size;
  a.softmax_scale = (cfg != nullptr && cfg->softmax_scale != 0.f) ? cfg->softmax_scale : 1.0f / sqrtf((float)kQkDim);
  if (!(a.softmax_scale > 0.f) || !isfinite(a.softmax_scale)) {
    set_error("%s: softmax_scale must be finite and > 0", fn);
    return MLA_ERR_ARG;
  }
  const cudaError_t err = p.kernel == kMma ? launch_int4_mma(a, p.mma, workspace, static_cast<cudaStream_t>(stream))
                                           : launch_int4_simt(a, p.splits, static_cast<cudaStream_t>(stream));
  if (err != cudaSuccess) {
    set_error("%s: launch failed: %s", fn, cudaGetErrorString(err));
    return MLA_ERR_CUDA;
  }
  return MLA_OK;
}

}  // extern "C"
