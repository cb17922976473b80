// Rotary positions (mla_rotary, include/mla_decode_b200.h): pairs (a, b) of a head's
// rotated dims become (a c - b s, a s + b c), c and s the cosine and sine of position x
// frequency times a gain.  Pairs are neighbours (interleaved) or half the rotated width
// apart (halves); the head's other dims are copied.
//
// Bound: bytes, x once in and once out.  A CTA takes a few tokens: its threads first
// fill a shared table of the tokens' cosines and sines (one angle per pair and token
// instead of one per pair, token and head: the angle is a double product and a
// sincospif), then walk the tokens' heads in vectors of 16 bytes, one in flight per
// thread and many threads per SM (two and four per thread, with their registers, were
// slower: 142 us against 170 and 189 at 8192 x 128 x 192, interleaved).
#include "mla_cache.cuh"

namespace mla {
namespace {

constexpr int kThreads = 256;

// Division of n < 2^31 by a run-time constant d >= 1: a 32-bit multiplication and shifts
// (m = floor(2^32 (2^s - d) / d) + 1, s = ceil(log2 d); Granlund and Montgomery).
struct FastDiv {
  uint32_t m, s;
  explicit FastDiv(uint32_t d) {
    s = 0;
    while ((1ull << s) < d) ++s;
    m = (uint32_t)(((1ull << 32) * ((1ull << s) - d)) / d + 1);
  }
  __device__ __forceinline__ int div(int n) const {
    const uint32_t t = __umulhi(m, (uint32_t)n);
    return (int)(((uint64_t)t + (uint32_t)n) >> s);
  }
};

template <typename T>
struct Io {
  static __device__ __forceinline__ float to(T v) { return Elt<T>::to1(v); }
  static __device__ __forceinline__ T from(float v) { return Elt<T>::from(v); }
};
template <>
struct Io<float> {
  static __device__ __forceinline__ float to(float v) { return v; }
  static __device__ __forceinline__ float from(float v) { return v; }
};

struct RotaryArgs {
  const void* x;
  void* out;
  const int* positions;        // [tokens]
  const double* turns;         // [rot / 2] turns per position
  float gain;
  int tokens, heads, head_dim, rot, offset, interleaved;
  long long xs_token, xs_head, os_token, os_head;   // strides in elements
  int tokens_per_cta;
  FastDiv by_items, by_heads;
};

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T e[V];
};

// V elements per access: 16 bytes, or single elements where the layout does not allow
// them (V = 1; interleaved pairs then move as two accesses).
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) mla_rotary_kernel(RotaryArgs a) {
  extern __shared__ float2 s_cs[];   // [tokens_per_cta][rot / 2]
  const int pairs = a.rot / 2;
  const int t0 = blockIdx.x * a.tokens_per_cta;
  const int nt = min(a.tokens_per_cta, a.tokens - t0);
  for (int i = threadIdx.x; i < nt * pairs; i += kThreads) {
    const int t = i / pairs;
    s_cs[i] = rotary_cos_sin(__ldg(a.positions + t0 + t), __ldg(a.turns + (i - t * pairs)), a.gain);
  }
  __syncthreads();
  using W = Vec<T, V>;
  // an item: V rotated elements of a head (interleaved: whole pairs; halves: V pairs, a
  // vector of either half) or V copied ones (only when the result goes elsewhere)
  const int inter = a.interleaved;
  const int rot_items = inter ? (V == 1 ? pairs : a.rot / V) : pairs / V;
  const int items = rot_items + (a.out != a.x ? (a.head_dim - a.rot) / V : 0);
  const int total = nt * a.heads * items;
  constexpr int kInterPairs = V == 1 ? 1 : V / 2;   // pairs of an interleaved item
  for (int i = threadIdx.x; i < total; i += kThreads) {
    const int row = a.by_items.div(i), it = i - row * items;
    const int t = a.by_heads.div(row), h = row - t * a.heads;
    // rotated and copied items load and store at the same places in the code (apart, they
    // would take turns: 174 us against 142)
    const bool rot = it < rot_items;
    int d = (it - rot_items) * V;
    if (rot)
      d = a.offset + (inter ? it * 2 * kInterPairs : it * V);
    else if (d >= a.offset)
      d += a.rot;
    const T* x = static_cast<const T*>(a.x) + (t0 + t) * a.xs_token + h * a.xs_head + d;
    T* o = static_cast<T*>(a.out) + (t0 + t) * a.os_token + h * a.os_head + d;
    const int gap = inter ? 1 : pairs;
    const bool two = rot && (V == 1 || !inter);   // the two elements of a pair in u and v
    W u = *reinterpret_cast<const W*>(x), v = u;
    if (two) v = *reinterpret_cast<const W*>(x + gap);
    if (rot) {
      const float2* cs = s_cs + t * pairs + (inter ? it * kInterPairs : it * V);
      if (V == 1 || !inter) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float p = Io<T>::to(u.e[e]), q = Io<T>::to(v.e[e]);
          u.e[e] = Io<T>::from(p * cs[e].x - q * cs[e].y);
          v.e[e] = Io<T>::from(p * cs[e].y + q * cs[e].x);
        }
      } else {
#pragma unroll
        for (int e = 0; e < V / 2; ++e) {
          const float p = Io<T>::to(u.e[2 * e]), q = Io<T>::to(u.e[2 * e + 1]);
          u.e[2 * e] = Io<T>::from(p * cs[e].x - q * cs[e].y);
          u.e[2 * e + 1] = Io<T>::from(p * cs[e].y + q * cs[e].x);
        }
      }
    }
    if (two) *reinterpret_cast<W*>(o + gap) = v;
    *reinterpret_cast<W*>(o) = u;
  }
}

template <typename T>
cudaError_t launch(RotaryArgs a, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  // 16-byte accesses need every start (base, token, head, the rotated dims and, for
  // halves, their second half) on a vector boundary and whole vectors throughout
  const long long step = a.xs_token | a.xs_head | a.os_token | a.os_head | a.offset | a.head_dim | a.rot |
                         (a.interleaved ? 0 : a.rot / 2);
  const bool wide = ((reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.out)) & 15) == 0 &&
                    step % V == 0;
  const unsigned grid = (unsigned)((a.tokens + a.tokens_per_cta - 1) / a.tokens_per_cta);
  const int v = wide ? V : 1;
  const int items = (a.interleaved && v > 1 ? a.rot / v : a.rot / 2 / v) + (a.out != a.x ? (a.head_dim - a.rot) / v : 0);
  a.by_items = FastDiv((uint32_t)items);
  const size_t smem = (size_t)a.tokens_per_cta * (a.rot / 2) * sizeof(float2);
  if (wide)
    mla_rotary_kernel<T, V><<<grid, kThreads, smem, stream>>>(a);
  else
    mla_rotary_kernel<T, 1><<<grid, kThreads, smem, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace
}  // namespace mla

using namespace mla;

extern "C" int32_t mla_rotary(const void* x, void* out, const int32_t* positions, const double* turns, float gain,
                              int32_t tokens, int32_t heads, int32_t head_dim, int32_t rot_dim, int32_t offset,
                              int32_t interleaved, int64_t x_token_stride, int64_t x_head_stride,
                              int64_t out_token_stride, int64_t out_head_stride, int32_t dtype, void* stream) {
  const char* fn = "mla_rotary";
  if (tokens < 0 || heads < 1 || head_dim < 2 || rot_dim < 2 || rot_dim % 2 != 0 || rot_dim > 1024 || offset < 0 ||
      head_dim > (1 << 20) || offset > head_dim - rot_dim || (long long)heads * head_dim > (1ll << 28)) {
    set_error("%s: bad size (tokens %d, heads %d, head_dim %d, rot_dim %d even and at most 1024, offset %d)", fn,
              tokens, heads, head_dim, rot_dim, offset);
    return MLA_ERR_ARG;
  }
  if (dtype != MLA_DTYPE_F16 && dtype != MLA_DTYPE_BF16 && dtype != MLA_DTYPE_F32) {
    set_error("%s: dtype must be 0, 1 or 2", fn);
    return MLA_ERR_ARG;
  }
  if (x_token_stride < 0 || x_head_stride < 0 || out_token_stride < 0 || out_head_stride < 0) {
    set_error("%s: strides must be >= 0", fn);
    return MLA_ERR_ARG;
  }
  if (tokens == 0) return MLA_OK;
  if (!x || !out || !positions || !turns) {
    set_error("%s: null pointer", fn);
    return MLA_ERR_ARG;
  }
  if (x == out && (x_token_stride != out_token_stride || x_head_stride != out_head_stride)) {
    set_error("%s: in place needs the same strides for x and out", fn);
    return MLA_ERR_ARG;
  }
  const uintptr_t esize = dtype == MLA_DTYPE_F32 ? 4 : 2;
  if (((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(out)) % esize) != 0 ||
      (reinterpret_cast<uintptr_t>(turns) & 7u) != 0) {
    set_error("%s: pointers must be aligned to their elements", fn);
    return MLA_ERR_ARG;
  }
  // tokens per CTA: enough rows to fill its threads when a token has few heads
  int per = 2048 / (heads * head_dim / 8 + 1);
  per = per < 1 ? 1 : (per > 8 ? 8 : per);
  const RotaryArgs a{x, out, positions, turns, gain, tokens, heads, head_dim, rot_dim, offset, interleaved != 0,
                     x_token_stride, x_head_stride, out_token_stride, out_head_stride, per, FastDiv(1),
                     FastDiv((uint32_t)heads)};
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t err = dtype == MLA_DTYPE_F16    ? launch<__half>(a, s)
                          : dtype == MLA_DTYPE_BF16 ? launch<__nv_bfloat16>(a, s)
                                                    : launch<float>(a, s);
  if (err != cudaSuccess) {
    set_error("%s: launch failed: %s", fn, cudaGetErrorString(err));
    return MLA_ERR_CUDA;
  }
  return MLA_OK;
}
