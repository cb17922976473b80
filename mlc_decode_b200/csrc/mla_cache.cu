// Rows into and out of a latent cache (mla_cache_append, mla_cache_gather,
// include/mla_decode_b200.h): a row's 512 latent dims as they are, as e4m3 codes of one
// per-tensor scale, or in the 4-bit form of mla_cache.cuh, and its 64 rope dims in the
// model's type, rotated on the way in when the call asks for it.
//
// Bound: bytes (a 4-bit append reads 1,152 a row and writes 416).  One warp per row:
// lane l holds dims [8 l, 8 l + 8) and [256 + 8 l, 256 + 8 l + 8) in two 16-byte loads,
// so the four lanes of a 32-dim group find its largest value in two shuffles, each
// lane's eight codes are one 32-bit word and a warp stores whole 128-byte lines; lane l
// also turns rope pair l.  A gather long enough to fill the GPU has the loads of two rows
// in flight per warp (131072 4-bit rows 39 us, 41 with one); an append, which computes
// more, has one row and more warps (37 us for as many, 41 with the rope part turned;
// two and four rows a warp were timed with a slower quantisation only: 62 and 94 against 58).
// As many rotated 16-bit rows take 48 us, e4m3 rows 41, their gathers 48 and 39 (at 6.4 TB/s:
// 47 and 36.5).
#include <cuda_fp8.h>
#include <math.h>
#include <string.h>

#include <type_traits>

#include "mla_cache.cuh"

namespace mla {
namespace {

constexpr int kWarps = 8;
constexpr long long kLongRows = 148ll * 64 * 2;   // a long gather: two rows for every warp slot of the GPU

struct CacheArgs {
  const void* kv;          // append: rows in; gather: unused
  const void* k_pe;
  void* kv_out;            // gather: rows out
  void* k_pe_out;
  const int* slots;        // [tokens] cache rows, outside [0, rows): skipped (append) or zero (gather)
  void* kv_cache;          // [rows][kv_heads][512] (model type or e4m3) or [rows][kv_heads][256] (codes)
  void* scales;            // [rows][kv_heads][16] float16 (4-bit form)
  void* k_pe_cache;        // [rows][kv_heads][64]
  float kv_scale, kv_recip;   // e4m3: the scale, and its reciprocal or 0 (quotient)
  const int* positions;    // rotary: [tokens], else nullptr
  const double* turns;     // [32]
  float gain;
  int interleaved;
  long long tokens, rows;
  int kv_heads;
  long long kv_token, kv_head, pe_token, pe_head;   // strides of the dense rows, in elements
};

template <typename T>
__device__ __forceinline__ void unpack8(uint4 w, float (&f)[8]) {
  const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 p = Elt<T>::to2(v[k]);
    f[2 * k] = p.x;
    f[2 * k + 1] = p.y;
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(Elt<T>::pack2(f[0], f[1]), Elt<T>::pack2(f[2], f[3]), Elt<T>::pack2(f[4], f[5]),
                    Elt<T>::pack2(f[6], f[7]));
}

// rint(f / s) clamped to a code's range, + 8; NaN is 0's code.
__device__ __forceinline__ uint32_t code_of(float f, float s) {
  const float r = rintf(__fdiv_rn(f, s));
  return f == f ? (uint32_t)((int)fminf(fmaxf(r, -8.f), 7.f) + 8) : 8u;
}

// The largest magnitude of eight values; NaN wins.
template <typename T>
__device__ __forceinline__ float max_abs8(uint4 x) {
  using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
  auto abs2 = [](uint32_t w) { return __habs2(*reinterpret_cast<const T2*>(&w)); };
  const T2 m = __hmax2_nan(__hmax2_nan(abs2(x.x), abs2(x.y)), __hmax2_nan(abs2(x.z), abs2(x.w)));
  const float2 f = Elt<T>::to2(*reinterpret_cast<const uint32_t*>(&m));
  return max_nan(f.x, f.y);
}

// This lane's eight dims as codes (low nibble first: dims 0 2 4 6 1 3 5 7) and its
// group's scale.  s = half(max / 7) may round below max / 7, hence the clamp; a group of
// zeros (or one whose scale rounds to zero) has code 8, the value 0; NaN stores as 0 and
// infinities as the largest code.
// max / 7 as a product with 1 / 7, off by 2^-23, rounds to the same half: the maximum has
// at most 11 bits, so max / 7 is no closer than 2^-12 / 7 of itself to the middle of two
// normal halves.  f / s is f times an approximate reciprocal, off by less than 2e-6.  Both have
// at most 11 bits, so 2 f and (2 n + 1) s are multiples of s's last bit and f / s is a
// tie n + 1/2 exactly or at least 2^-12 away from it: rounded to a multiple of 2^-13 first
// (a sum with 1.5 x 2^10) it is the tie again or stays on its side, and a sum with 1.5 x 2^23
// then rounds to the integer as the exact quotient would.  The sums' bits are a constant
// plus the integer; their nibbles are put together as integers, modulo 2^32.  Groups that
// are not finite or whose scale is below fp16's normal range (the only ones whose
// quotients may pass 7.5) are divided.
template <typename T>
__device__ __forceinline__ uint32_t quantise8(uint4 x, __half* scale) {
  float m = max_abs8<T>(x);
  m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 2));
  float f[8];
  unpack8<T>(x, f);
  __half s = __float2half_rn(m * (1.f / 7.f));
  float sf = __half2float(s);
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(sf));
  constexpr float kGrid = 1536.f, kRound = 12582912.f - kGrid;
  constexpr uint32_t kBits = 0x4b400000u;            // of 12582912.f
  constexpr int kOrder[8] = {7, 5, 3, 1, 6, 4, 2, 0};   // dims of the nibbles, highest first
  uint32_t w = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k)
    w = w * 16u + __float_as_uint(__fadd_rn(fmaf(f[kOrder[k]], inv, kGrid), kRound));
  w += 0x88888888u - kBits * 0x11111111u;
  // (the four lanes of a group agree on the scale: all of them or none)
  if (!(sf >= 6.103515625e-5f && sf < INFINITY)) {
    m = 0.f;                                         // the largest of the numbers' magnitudes
#pragma unroll
    for (int k = 0; k < 8; ++k) m = fmaxf(m, fabsf(f[k]));
    const unsigned group = 0xfu << (threadIdx.x & 28);
    m = fmaxf(m, __shfl_xor_sync(group, m, 1));
    m = fmaxf(m, __shfl_xor_sync(group, m, 2));
    s = __float2half_rn(fminf(__fdiv_rn(m, 7.f), 65504.f));
    sf = __half2float(s);
    w = 0x88888888u;
    if (sf > 0.f) {
      w = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) w |= code_of(f[k], sf) << (4 * ((k >> 1) + 4 * (k & 1)));
    }
  }
  *scale = s;
  return w;
}

// e4m3 code pair of (a / s, b / s), each quotient rounded to float32 first: with the
// correctly rounded reciprocal r of s, q = a r and one residual step give the correctly
// rounded quotient (Markstein), unless s's significand is all ones or the numbers leave
// float32's normal range; the host then sets r to zero and the lane divides.  A
// quotient past e4m3's range saturates whatever its last bit.
__device__ __forceinline__ float quotient(float a, float s, float r) {
  if (r == 0.f) return __fdiv_rn(a, s);
  const float q = a * r;
  return fabsf(q) < 1e6f ? fmaf(fmaf(-q, s, a), r, q) : q;
}
__device__ __forceinline__ uint32_t e4m3x2_of(float a, float b, float s, float r) {
  return __nv_cvt_float2_to_fp8x2(make_float2(quotient(a, s, r), quotient(b, s, r)), __NV_SATFINITE, __NV_E4M3);
}

enum Form { kModel = MLA_CACHE_MODEL, kFp8 = MLA_CACHE_FP8, kInt4 = MLA_CACHE_INT4 };

template <typename T, int F>
__global__ void __launch_bounds__(32 * kWarps, 8) mla_cache_append_kernel(CacheArgs a) {
  const int lane = threadIdx.x & 31;
  const long long item = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (item >= a.tokens * a.kv_heads) return;
  const long long t = a.kv_heads == 1 ? item : item / a.kv_heads;
  const int kvh = (int)(item - t * a.kv_heads);
  const int slot = __ldg(a.slots + t);
  const uint4* kv = reinterpret_cast<const uint4*>(static_cast<const T*>(a.kv) + t * a.kv_token + kvh * a.kv_head);
  const uint4 x0 = __ldg(kv + lane), x1 = __ldg(kv + 32 + lane);
  const T* pe = static_cast<const T*>(a.k_pe) + t * a.pe_token + kvh * a.pe_head;
  // rope pair `lane`: two neighbours in one word, or elements lane and lane + 32 (halves)
  const bool words = a.interleaved || a.positions == nullptr;
  uint32_t pair = words ? __ldg(reinterpret_cast<const uint32_t*>(pe) + lane)
                        : __ldg(reinterpret_cast<const unsigned short*>(pe) + lane) |
                              ((uint32_t)__ldg(reinterpret_cast<const unsigned short*>(pe) + 32 + lane) << 16);
  if (a.positions != nullptr) {
    const float2 c = rotary_cos_sin(__ldg(a.positions + t), __ldg(a.turns + lane), a.gain);
    const float2 u = Elt<T>::to2(pair);
    pair = Elt<T>::pack2(u.x * c.x - u.y * c.y, u.x * c.y + u.y * c.x);
  }
  if (slot < 0 || slot >= a.rows) return;
  const long long row = (long long)slot * a.kv_heads + kvh;
  if constexpr (F == kModel) {
    uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(a.kv_cache) + row * kDim);
    dst[lane] = x0;
    dst[32 + lane] = x1;
  } else {
    if constexpr (F == kFp8) {
      float f0[8], f1[8];
      unpack8<T>(x0, f0);
      unpack8<T>(x1, f1);
      uint32_t w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float* f = k < 2 ? f0 + 4 * k : f1 + 4 * (k - 2);
        w[k] = e4m3x2_of(f[0], f[1], a.kv_scale, a.kv_recip) | (e4m3x2_of(f[2], f[3], a.kv_scale, a.kv_recip) << 16);
      }
      uint2* dst = reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.kv_cache) + row * kDim);
      dst[lane] = make_uint2(w[0], w[1]);
      dst[32 + lane] = make_uint2(w[2], w[3]);
    } else {
      __half s0, s1;
      const uint32_t w0 = quantise8<T>(x0, &s0), w1 = quantise8<T>(x1, &s1);
      uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.kv_cache) + row * kI4Bytes);
      dst[lane] = w0;
      dst[32 + lane] = w1;
      if ((lane & 3) == 0) {
        __half* sc = static_cast<__half*>(a.scales) + row * kI4Groups;
        sc[lane >> 2] = s0;
        sc[8 + (lane >> 2)] = s1;
      }
    }
  }
  T* pc = static_cast<T*>(a.k_pe_cache) + row * kPeDim;
  if (words) {
    reinterpret_cast<uint32_t*>(pc)[lane] = pair;
  } else {
    reinterpret_cast<unsigned short*>(pc)[lane] = (unsigned short)pair;
    reinterpret_cast<unsigned short*>(pc)[32 + lane] = (unsigned short)(pair >> 16);
  }
}

template <typename T, int F, int R>
__global__ void __launch_bounds__(32 * kWarps) mla_cache_gather_kernel(CacheArgs a) {
  const int lane = threadIdx.x & 31;
  const long long items = a.tokens * a.kv_heads;
  const long long first = ((long long)blockIdx.x * kWarps + (threadIdx.x >> 5)) * R;
  // what the row's cache form has for this lane: two 16-byte (model), 8-byte (e4m3) or
  // 4-byte (codes) pieces, the pieces' scales and a rope pair
  uint4 y0[R], y1[R];
  uint32_t pe[R];
  __half s0[R], s1[R];
  int slot[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    slot[i] = -1;
    y0[i] = y1[i] = make_uint4(0u, 0u, 0u, 0u);
    pe[i] = 0;
    if (first + i < items) slot[i] = __ldg(a.slots + (a.kv_heads == 1 ? first + i : (first + i) / a.kv_heads));
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (slot[i] < 0 || slot[i] >= a.rows) continue;
    const int kvh = a.kv_heads == 1 ? 0 : (int)((first + i) % a.kv_heads);
    const long long row = (long long)slot[i] * a.kv_heads + kvh;
    pe[i] = __ldg(reinterpret_cast<const uint32_t*>(static_cast<const T*>(a.k_pe_cache) + row * kPeDim) + lane);
    const uint8_t* src = static_cast<const uint8_t*>(a.kv_cache);
    if constexpr (F == kModel) {
      y0[i] = __ldg(reinterpret_cast<const uint4*>(src + row * kDim * 2) + lane);
      y1[i] = __ldg(reinterpret_cast<const uint4*>(src + row * kDim * 2) + 32 + lane);
    } else if constexpr (F == kFp8) {
      const uint2 w0 = __ldg(reinterpret_cast<const uint2*>(src + row * kDim) + lane);
      const uint2 w1 = __ldg(reinterpret_cast<const uint2*>(src + row * kDim) + 32 + lane);
      y0[i] = make_uint4(w0.x, w0.y, 0u, 0u);
      y1[i] = make_uint4(w1.x, w1.y, 0u, 0u);
    } else {
      y0[i].x = __ldg(reinterpret_cast<const uint32_t*>(src + row * kI4Bytes) + lane);
      y1[i].x = __ldg(reinterpret_cast<const uint32_t*>(src + row * kI4Bytes) + 32 + lane);
      const __half* sc = static_cast<const __half*>(a.scales) + row * kI4Groups;
      s0[i] = __ldg(sc + (lane >> 2));
      s1[i] = __ldg(sc + 8 + (lane >> 2));
    }
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (first + i >= items) continue;
    const bool real = slot[i] >= 0 && slot[i] < a.rows;
    uint4 o0 = y0[i], o1 = y1[i];
    if constexpr (F == kFp8) {
      const uint32_t w[4] = {y0[i].x, y0[i].y, y1[i].x, y1[i].y};
      float f[2][8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[k >> 1] >> (16 * (k & 1))), __NV_E4M3);
        f[k >> 2][2 * (k & 3)] = __half2float(__ushort_as_half(h.x)) * a.kv_scale;
        f[k >> 2][2 * (k & 3) + 1] = __half2float(__ushort_as_half(h.y)) * a.kv_scale;
      }
      o0 = pack8<T>(f[0]);
      o1 = pack8<T>(f[1]);
    } else if constexpr (F == kInt4) {
      if (real) {
        const uint32_t w[2] = {y0[i].x, y1[i].x};
        const float s[2] = {__half2float(s0[i]), __half2float(s1[i])};
        float f[2][8];
#pragma unroll
        for (int v = 0; v < 2; ++v)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 n = __half22float2(i4_pair(w[v], j));
            f[v][2 * j] = n.x * s[v];
            f[v][2 * j + 1] = n.y * s[v];
          }
        o0 = pack8<T>(f[0]);
        o1 = pack8<T>(f[1]);
      }
    }
    const long long t = a.kv_heads == 1 ? first + i : (first + i) / a.kv_heads;
    const int kvh = (int)(first + i - t * a.kv_heads);
    uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(a.kv_out) + t * a.kv_token + kvh * a.kv_head);
    dst[lane] = o0;
    dst[32 + lane] = o1;
    reinterpret_cast<uint32_t*>(static_cast<T*>(a.k_pe_out) + t * a.pe_token + kvh * a.pe_head)[lane] = pe[i];
  }
}

template <typename T, int F>
void launch_one(const CacheArgs& a, bool append, cudaStream_t s) {
  const long long items = a.tokens * a.kv_heads;
  const unsigned grid = (unsigned)((items + kWarps - 1) / kWarps);
  if (append)
    mla_cache_append_kernel<T, F><<<grid, 32 * kWarps, 0, s>>>(a);
  else if (items >= kLongRows)
    mla_cache_gather_kernel<T, F, 2><<<(grid + 1) / 2, 32 * kWarps, 0, s>>>(a);
  else
    mla_cache_gather_kernel<T, F, 1><<<grid, 32 * kWarps, 0, s>>>(a);
}

int run(const char* fn, const CacheArgs& a, bool append, int form, int dtype, void* stream) {
  if (a.tokens < 0 || a.rows < 1 || a.kv_heads < 1 || a.rows > INT32_MAX || a.tokens > (1ll << 31) ||
      a.tokens * a.kv_heads > (1ll << 33)) {
    set_error("%s: bad size (tokens %lld, cache rows %lld, kv_heads %d)", fn, a.tokens, a.rows, a.kv_heads);
    return MLA_ERR_ARG;
  }
  if (dtype != MLA_DTYPE_F16 && dtype != MLA_DTYPE_BF16) {
    set_error("%s: dtype must be 0 (fp16) or 1 (bf16), got %d", fn, dtype);
    return MLA_ERR_ARG;
  }
  if (form != MLA_CACHE_MODEL && form != MLA_CACHE_FP8 && form != MLA_CACHE_INT4) {
    set_error("%s: unknown cache form %d", fn, form);
    return MLA_ERR_ARG;
  }
  if (form == MLA_CACHE_FP8 && (!(a.kv_scale > 0.f) || !isfinite(a.kv_scale))) {
    set_error("%s: kv_scale must be finite and > 0", fn);
    return MLA_ERR_ARG;
  }
  if (a.kv_token < 0 || a.kv_head < 0 || a.pe_token < 0 || a.pe_head < 0 || a.kv_token % 8 != 0 ||
      a.kv_head % 8 != 0 || a.pe_token % 8 != 0 || a.pe_head % 8 != 0) {
    set_error("%s: the rows' strides must be >= 0 and multiples of 8 elements (kv %lld, %lld; k_pe %lld, %lld)", fn,
              a.kv_token, a.kv_head, a.pe_token, a.pe_head);
    return MLA_ERR_ARG;
  }
  if (a.tokens == 0) return MLA_OK;
  const void* rows = append ? a.kv : a.kv_out;
  const void* pes = append ? a.k_pe : a.k_pe_out;
  if (!rows || !pes || !a.slots || !a.kv_cache || !a.k_pe_cache || (form == MLA_CACHE_INT4 && !a.scales) ||
      (a.positions != nullptr && !a.turns)) {
    set_error("%s: null pointer", fn);
    return MLA_ERR_ARG;
  }
  const uintptr_t any = reinterpret_cast<uintptr_t>(rows) | reinterpret_cast<uintptr_t>(pes) |
                        reinterpret_cast<uintptr_t>(a.kv_cache) | reinterpret_cast<uintptr_t>(a.k_pe_cache) |
                        (form == MLA_CACHE_INT4 ? reinterpret_cast<uintptr_t>(a.scales) : 0);
  if ((any & 15u) != 0) {
    set_error("%s: tensor pointers must be 16-byte aligned", fn);
    return MLA_ERR_ARG;
  }
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bf = dtype == MLA_DTYPE_BF16;
  if (form == MLA_CACHE_MODEL)
    bf ? launch_one<__nv_bfloat16, kModel>(a, append, s) : launch_one<__half, kModel>(a, append, s);
  else if (form == MLA_CACHE_FP8)
    bf ? launch_one<__nv_bfloat16, kFp8>(a, append, s) : launch_one<__half, kFp8>(a, append, s);
  else
    bf ? launch_one<__nv_bfloat16, kInt4>(a, append, s) : launch_one<__half, kInt4>(a, append, s);
  const cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) {
    set_error("%s: launch failed: %s", fn, cudaGetErrorString(err));
    return MLA_ERR_CUDA;
  }
  return MLA_OK;
}

}  // namespace
}  // namespace mla

using namespace mla;

extern "C" {

int32_t mla_cache_append(const void* kv, const void* k_pe, const int32_t* slots, void* kv_cache, void* kv_scales,
                         void* k_pe_cache, float kv_scale, const int32_t* positions, const double* turns, float gain,
                         int32_t interleaved, int64_t tokens, int32_t kv_heads, int64_t cache_rows,
                         int64_t kv_token_stride, int64_t kv_head_stride, int64_t pe_token_stride,
                         int64_t pe_head_stride, int32_t form, int32_t dtype, void* stream) {
  CacheArgs a{};
  a.kv = kv;
  a.k_pe = k_pe;
  a.slots = slots;
  a.kv_cache = kv_cache;
  a.scales = kv_scales;
  a.k_pe_cache = k_pe_cache;
  a.kv_scale = kv_scale;
  uint32_t bits;
  memcpy(&bits, &kv_scale, sizeof(bits));
  a.kv_recip = kv_scale > 1e-20f && kv_scale < 1e20f && (bits & 0x7fffffu) != 0x7fffffu ? 1.f / kv_scale : 0.f;
  a.positions = positions;
  a.turns = turns;
  a.gain = gain;
  a.interleaved = interleaved;
  a.tokens = tokens;
  a.rows = cache_rows;
  a.kv_heads = kv_heads;
  a.kv_token = kv_token_stride;
  a.kv_head = kv_head_stride;
  a.pe_token = pe_token_stride;
  a.pe_head = pe_head_stride;
  return run("mla_cache_append", a, true, form, dtype, stream);
}

int32_t mla_cache_gather(const int32_t* slots, const void* kv_cache, const void* kv_scales, const void* k_pe_cache,
                         float kv_scale, void* kv, void* k_pe, int64_t tokens, int32_t kv_heads, int64_t cache_rows,
                         int64_t kv_token_stride, int64_t kv_head_stride, int64_t pe_token_stride,
                         int64_t pe_head_stride, int32_t form, int32_t dtype, void* stream) {
  CacheArgs a{};
  a.kv_out = kv;
  a.k_pe_out = k_pe;
  a.slots = slots;
  a.kv_cache = const_cast<void*>(kv_cache);
  a.scales = const_cast<void*>(kv_scales);
  a.k_pe_cache = const_cast<void*>(k_pe_cache);
  a.kv_scale = kv_scale;
  a.tokens = tokens;
  a.rows = cache_rows;
  a.kv_heads = kv_heads;
  a.kv_token = kv_token_stride;
  a.kv_head = kv_head_stride;
  a.pe_token = pe_token_stride;
  a.pe_head = pe_head_stride;
  return run("mla_cache_gather", a, false, form, dtype, stream);
}

}  // extern "C"
