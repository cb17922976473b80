// Rotary positions (mla_rotary, include/mla_decode_b200.h): pairs (a, b) of a head's
// rotated dims become (a c - b s, a s + b c), c and s the cosine and sine of position x
// frequency times a gain.  Pairs are neighbours (interleaved) or half the rotated width
// apart (halves); the head's other dims are copied.
//
// Bound: bytes, x once in and once out.  A CTA takes kTokens tokens: its threads first
// fill a shared table of the tokens' cosines and sines (one angle per pair and token
// instead of one per pair, token and head: the angle is a double product and a
// sincospif), then walk the tokens' heads in vectors of 16 bytes.
#include "mla_cache.cuh"

namespace mla {
namespace {

constexpr int kThreads = 256;

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
  constexpr int VI = V == 1 ? 2 : V;            // interleaved: elements per item (whole pairs)
  const int rot_items = a.interleaved ? a.rot / VI : pairs / V;
  // the copied dims (only when the result goes elsewhere): [0, offset) and [offset + rot, head_dim)
  const bool copy = a.out != a.x;
  const int copy_items = copy ? (a.head_dim - a.rot) / V : 0;
  const int items = rot_items + copy_items;
  const int total = nt * a.heads * items;
  for (int i = threadIdx.x; i < total; i += kThreads) {
    const int row = i / items, it = i - row * items;
    const int t = row / a.heads, h = row - t * a.heads;
    const T* x = static_cast<const T*>(a.x) + (t0 + t) * a.xs_token + h * a.xs_head;
    T* o = static_cast<T*>(a.out) + (t0 + t) * a.os_token + h * a.os_head;
    if (it >= rot_items) {
      int d = (it - rot_items) * V;
      if (d >= a.offset) d += a.rot;
      *reinterpret_cast<W*>(o + d) = *reinterpret_cast<const W*>(x + d);
      continue;
    }
    const float2* cs = s_cs + t * pairs;
    if (a.interleaved) {
      const int d = a.offset + it * VI;
      using WI = Vec<T, V == 1 ? 1 : V>;
      T e[VI];
      if constexpr (V == 1) {
        e[0] = x[d];
        e[1] = x[d + 1];
      } else {
        const WI w = *reinterpret_cast<const WI*>(x + d);
#pragma unroll
        for (int k = 0; k < VI; ++k) e[k] = w.e[k];
      }
#pragma unroll
      for (int k = 0; k < VI / 2; ++k) {
        const float2 c = cs[it * (VI / 2) + k];
        const float u = Io<T>::to(e[2 * k]), v = Io<T>::to(e[2 * k + 1]);
        e[2 * k] = Io<T>::from(u * c.x - v * c.y);
        e[2 * k + 1] = Io<T>::from(u * c.y + v * c.x);
      }
      if constexpr (V == 1) {
        o[d] = e[0];
        o[d + 1] = e[1];
      } else {
        WI w;
#pragma unroll
        for (int k = 0; k < VI; ++k) w.e[k] = e[k];
        *reinterpret_cast<WI*>(o + d) = w;
      }
    } else {
      const int d = a.offset + it * V;
      W u = *reinterpret_cast<const W*>(x + d), v = *reinterpret_cast<const W*>(x + d + pairs);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float2 c = cs[it * V + k];
        const float p = Io<T>::to(u.e[k]), q = Io<T>::to(v.e[k]);
        u.e[k] = Io<T>::from(p * c.x - q * c.y);
        v.e[k] = Io<T>::from(p * c.y + q * c.x);
      }
      *reinterpret_cast<W*>(o + d) = u;
      *reinterpret_cast<W*>(o + d + pairs) = v;
    }
  }
}

template <typename T>
cudaError_t launch(const RotaryArgs& a, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  // 16-byte accesses need every start (base, token, head, the rotated dims and, for
  // halves, their second half) on a vector boundary and whole vectors throughout
  const long long step = a.xs_token | a.xs_head | a.os_token | a.os_head | a.offset | a.head_dim | a.rot |
                         (a.interleaved ? 0 : a.rot / 2);
  const bool wide = ((reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.out)) & 15) == 0 &&
                    step % V == 0;
  const unsigned grid = (unsigned)((a.tokens + a.tokens_per_cta - 1) / a.tokens_per_cta);
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
                     x_token_stride, x_head_stride, out_token_stride, out_head_stride, per};
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
