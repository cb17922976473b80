// CUDA-core decode over a 4-bit latent cache: any head count, lengths, paging, query
// positions and KV heads of mla_decode_ext_int4kv.  The cross-check of the tensor-core
// kernel (cfg kernel "simt"), written for clarity: the same online softmax as
// mla_simt.cu over 32-row tiles whose codes are widened to float in shared memory, so
// nothing but P.V's and the scores' float sums rounds.
//
// Grid (splits, groups of 16 heads, query sequences): split z of a query sequence of
// nt tiles takes tiles [z nt / splits, (z + 1) nt / splits) of its own length, so short
// and long sequences are both spread over all splits; the combine launch merges them.
#include <math.h>

#include "mla_cache.cuh"

namespace mla {
namespace {

constexpr int kHeadsPerCta = 16;
constexpr int kTileN = 32;
constexpr int kThreads = 256;
constexpr int kQStride = kQkDim + 1;
constexpr int kKStride = kQkDim + 1;
constexpr int kPStride = kTileN + 1;
constexpr size_t kSmemBytes =
    sizeof(float) * (kHeadsPerCta * kQStride + kTileN * kKStride + kHeadsPerCta * kPStride);

template <typename T>
__global__ void __launch_bounds__(kThreads, 2)
mla_int4_simt_kernel(Int4Args a, int ns, float scale_log2) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  float* sQ = reinterpret_cast<float*>(smem_raw);
  float* sK = sQ + kHeadsPerCta * kQStride;
  float* sP = sK + kTileN * kKStride;

  const int z = blockIdx.x, h0 = blockIdx.y * kHeadsPerCta, qs = blockIdx.z;
  const int g = a.heads / a.kv_heads;   // query heads per KV head
  const int tid = threadIdx.x, hr = tid >> 4, l16 = tid & 15;
  const int nh = min(kHeadsPerCta, g - h0);
  const int seq = qs / (a.q_len * a.kv_heads), kvh = qs % a.kv_heads;
  const int len = ragged_len(a.seqlens, qs, a.q_len, a.kv_heads, a.max_len);
  const int nt = (len + kTileN - 1) / kTileN;
  const int t0 = (int)((long long)z * nt / ns) * kTileN;
  const int t1 = min((int)((long long)(z + 1) * nt / ns) * kTileN, len);

  const T* q = static_cast<const T*>(a.q) + ((size_t)qs * g + h0) * kDim;
  const T* q_pe = static_cast<const T*>(a.q_pe) + ((size_t)qs * g + h0) * kPeDim;
  for (int i = tid; i < kHeadsPerCta * kQkDim; i += kThreads) {
    const int r = i / kQkDim, c = i - r * kQkDim;
    float v = 0.f;
    if (r < nh) v = c < kDim ? Elt<T>::to1(q[r * kDim + c]) : Elt<T>::to1(q_pe[r * kPeDim + (c - kDim)]);
    sQ[r * kQStride + c] = v;
  }

  float m = -INFINITY, l = 0.f, o[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) o[i] = 0.f;

  for (int tt = t0; tt < t1; tt += kTileN) {
    const int nrow = min(kTileN, t1 - tt);
    __syncthreads();   // previous tile fully consumed (and Q staged on entry)
    // eight dims (one code word) or eight rope dims a step; rows past the range as zeros
    for (int i = tid; i < kTileN * (kQkDim / 8); i += kThreads) {
      const int r = i / (kQkDim / 8), w8 = i - r * (kQkDim / 8);
      float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      const long long row =
          r < nrow ? cache_row(a.block_table, a.max_pages, a.page_size, a.num_pages, a.max_seqlen, seq, tt + r) : -1;
      if (row >= 0) {
        const size_t at = (size_t)row * a.kv_heads + kvh;
        if (w8 < kDim / 8) {
          const uint32_t w = __ldg(reinterpret_cast<const uint32_t*>(a.codes + at * kI4Bytes) + w8);
          const float s = __half2float(__ldg(a.scales + at * kI4Groups + w8 / (kI4Group / 8)));
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 n = __half22float2(i4_pair(w, j));
            f[2 * j] = n.x * s;
            f[2 * j + 1] = n.y * s;
          }
        } else {
          const T* pe = static_cast<const T*>(a.k_pe) + at * kPeDim + (w8 - kDim / 8) * 8;
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] = Elt<T>::to1(pe[j]);
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) sK[r * kKStride + 8 * w8 + j] = f[j];
    }
    __syncthreads();

    float s0 = 0.f, s1 = 0.f;   // scores of tokens l16 and l16 + 16 against head row hr
    const float* qr = sQ + hr * kQStride;
    const float* k0 = sK + l16 * kKStride;
    const float* k1 = sK + (l16 + 16) * kKStride;
#pragma unroll 8
    for (int c = 0; c < kQkDim; ++c) {
      s0 = fmaf(qr[c], k0[c], s0);
      s1 = fmaf(qr[c], k1[c], s1);
    }
    if (l16 >= nrow) s0 = -INFINITY;
    if (l16 + 16 >= nrow) s1 = -INFINITY;
    float mx = fmaxf(s0, s1);
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
    const float m_new = fmaxf(m, mx);            // finite: row 0 of a tile is always valid
    const float alpha = exp2f((m - m_new) * scale_log2);
    const float p0 = exp2f((s0 - m_new) * scale_log2);
    const float p1 = exp2f((s1 - m_new) * scale_log2);
    float ps = p0 + p1;
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) ps += __shfl_xor_sync(0xffffffffu, ps, off);
    l = l * alpha + ps;
    m = m_new;
    sP[hr * kPStride + l16] = p0;
    sP[hr * kPStride + l16 + 16] = p1;
    __syncwarp();   // the 16 threads of a head row share one warp
#pragma unroll
    for (int i = 0; i < 32; ++i) o[i] *= alpha;
    for (int j = 0; j < nrow; ++j) {
      const float p = sP[hr * kPStride + j];
      const float* vr = sK + j * kKStride + l16;
#pragma unroll
      for (int k = 0; k < 32; ++k) o[k] = fmaf(p, vr[16 * k], o[k]);
    }
    __syncwarp();
  }

  if (hr >= nh) return;
  const size_t row = (size_t)qs * g + h0 + hr;
  const bool empty = !(t1 > t0);
  const float inv = empty ? 0.f : 1.f / l;
  const float lse_nat = empty ? -INFINITY : (m * scale_log2 + log2f(l)) * kLn2;
  if (ns == 1) {
    T* orow = static_cast<T*>(a.out) + row * kDim;
#pragma unroll
    for (int k = 0; k < 32; ++k) orow[l16 + 16 * k] = Elt<T>::from(o[k] * inv);
    if (a.lse != nullptr && l16 == 0) a.lse[row] = lse_nat;
  } else {
    const size_t prow = (size_t)z * gridDim.z * g + row;
    float* orow = a.part_o + prow * kDim;
#pragma unroll
    for (int k = 0; k < 32; ++k) orow[l16 + 16 * k] = o[k] * inv;
    if (l16 == 0) a.part_lse[prow] = lse_nat;
  }
}

template <typename T>
cudaError_t launch_typed(const Int4Args& a, int ns, cudaStream_t stream) {
  const cudaError_t err = cudaFuncSetAttribute(mla_int4_simt_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (int)kSmemBytes);
  if (err != cudaSuccess) return err;
  const int g = a.heads / a.kv_heads;
  const dim3 grid(ns, (g + kHeadsPerCta - 1) / kHeadsPerCta, a.batch * a.q_len * a.kv_heads);
  mla_int4_simt_kernel<T><<<grid, kThreads, kSmemBytes, stream>>>(a, ns, a.softmax_scale * kLog2e);
  return cudaGetLastError();
}

}  // namespace

// Splits: two resident waves over all SMs, no more than the longest sequence's tiles.
int int4_simt_splits(int qb, int g, int max_len, int asked) {
  const int nt = (max_len + kTileN - 1) / kTileN;
  long long ns = asked;
  if (ns < 1) {
    const long long units = (long long)qb * ((g + kHeadsPerCta - 1) / kHeadsPerCta);
    ns = (148ll * 2 * 2 + units - 1) / units;
  }
  return (int)(ns < nt ? ns : nt);
}

cudaError_t launch_int4_simt(const Int4Args& a, int ns, cudaStream_t stream) {
  cudaError_t err = a.dtype == MLA_DTYPE_F16 ? launch_typed<__half>(a, ns, stream)
                                             : launch_typed<__nv_bfloat16>(a, ns, stream);
  if (err == cudaSuccess && ns > 1)
    err = launch_combine(a.part_lse, a.part_o, ns, a.batch * a.q_len * a.kv_heads, a.heads / a.kv_heads, a.out, a.lse,
                         a.dtype, stream);
  return err;
}

}  // namespace mla
