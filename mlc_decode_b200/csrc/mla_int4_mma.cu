// Decode over a 4-bit latent cache for few query rows: warp-level MMAs on operands
// widened in registers.
//
// out = softmax(S) V with S = [q | q_pe] . [V | k_pe]^T, V = (codes - 8) x scales.  With
// at most a few dozen query rows per KV head the tensor-core pair kernel spends a
// tile's time on rows that do not exist; here a tile costs what its rows cost.  The
// query rows of a KV sequence are its q_len positions x query heads per KV head: they
// share every row read.  A CTA takes up to 16 MT of them.
//
// * Codes, scales and rope rows of a 64-row tile come by TMA into a ring of stages
//   (26 KB each), ahead of the math; page lookups are done 32 tiles at a time, one a
//   lane of a warp.
// * The fragments of mma.m16n8k16 are widened straight from the stage's codes: no
//   fp16 copy of the tile exists.  For S a thread's code word (8 dims of one row) is its
//   B fragment of two k-steps, with the dims of Q's A fragment (kept in registers)
//   permuted to match.  The two k-steps are one scale group: their MMAs take the bare
//   codes n - 8 and a float32 product with the scale follows, so the scores have no
//   rounding of the row values (values rounded to fp16 first: 121 us instead of 125 at
//   b128 h16 s4096, and an error of 2e-4 in the log-sum-exp of short sequences).  For P.V the
//   values are rounded to fp16 once, and so are the weights (kI4WeightLog2) of a bf16 call,
//   whose result rounds eight times as coarsely; a fp16 call's weights are two fp16 parts with
//   an MMA each (root-mean-square error 1.25 to 1.38 times the result's own rounding instead of
//   1.40 to 1.52; 145 us instead of 133 at b128 h16 s4096).  The words of
//   two rows are interleaved by 16-bit halves, so that a field pair is one dim of two
//   neighbouring rows; column n of block e is dim 8 n + e of the warp's 64, which leaves
//   each thread with 16 neighbouring output dims.
// * Eight warps: for S two row halves x four quarters of the dims (the quarters' sums
//   meet in shared memory), for P.V 64 output dims each.  The 128-byte TMA swizzle makes
//   both access patterns free of bank conflicts.
// * Workers (two CTAs an SM for MT = 1) take equal ranges of the flattened tile list; a
//   sequence cut by a range's end leaves float32 partials that the combine launch merges.
//   Every CTA sums the lengths itself: no plan launch.
//
// Bound: the issue slots of the widening (13 instructions per 8 codes, once for S and
// once for P.V) with the latencies that 16 warps an SM leave uncovered (issue slots 56 %,
// integer pipe 43 %, tensor pipe 29 % busy at b128 h16 s4096, bf16: 124 us, 1.8 TB/s; the
// fp16 instance spills 40 bytes).
// S of the next tile beside P.V of this one between the same two barriers: no faster.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <math.h>
#include <string.h>

#include <mutex>
#include <type_traits>

#include "mla_cache.cuh"
#include "mla_sm100.cuh"
#include "mla_sm100_ptx.cuh"

namespace mla {
namespace sm100 {   // (mla_sm100.cu)
PFN_cuTensorMapEncodeTiled_v12000 encode_fn();
bool place_map(CUtensorMap* m, const CUtensorMap& form, const void* base);
bool make_map_kv(CUtensorMap* m, const void* base, uint64_t cols, uint64_t kv_heads, uint64_t rows,
                 CUtensorMapDataType dt, uint32_t elem_bytes);
}  // namespace sm100
namespace {

constexpr int kTileR = 64;                 // cache rows per tile
constexpr int kThreads = 256;              // (a ninth warp would cost the other eight their registers)
constexpr int kAhead = 64;                 // tiles whose rows are known ahead (two batches of 32)
constexpr uint32_t kCodeBytes = kTileR * kI4Bytes;          // two swizzled boxes of 64 x 128 bytes
constexpr uint32_t kRopeBytes = kTileR * kPeDim * 2;        // one
constexpr uint32_t kScaleBytes = kTileR * kI4Groups * 2;
constexpr uint32_t kStage = kCodeBytes + kRopeBytes + kScaleBytes;
static_assert(kStage % 1024 == 0, "swizzled boxes start on 1024 bytes");
constexpr int kSPitch = 72, kPPitch = 72;  // elements: rows 8 banks (floats), 4 banks (halves) apart
constexpr float kLazyLog2 = 8.f;           // the running maximum moves when a row's grows by 2^8
constexpr int kMaxWorkers = 512;
constexpr uint32_t kErrLoad = 0x301;
constexpr uint64_t kWaitNs = 2000000000ull;

__device__ __forceinline__ int seq_rows(const Int4Args& a, int s) {
  int len = a.max_len;
  if (a.seqlens != nullptr) {
    len = __ldg(a.seqlens + s);
    len = len < 0 ? 0 : (len > a.max_len ? a.max_len : len);
  }
  return len;
}

// The tiles of a worker's range, in order: tile j of the unit `sub` (KV head and row
// group) of sequence s.
struct Walk {
  int left;   // tiles still to come, this one included
  int s, sub, j, len, nt;
  __device__ __forceinline__ void next(const Int4Args& a, int units_per_seq) {
    --left;
    if (++j < nt || left <= 0) return;
    j = 0;
    if (++sub < units_per_seq) return;
    sub = 0;
    do {
      if (++s >= a.batch) {   // (only if the lengths changed under the call)
        left = 0;
        return;
      }
      len = seq_rows(a, s);
      nt = (len + kTileR - 1) / kTileR;
    } while (nt == 0);
  }
};

template <int MT>
struct Lay {
  static constexpr int kRows = 16 * MT;
  static constexpr int kStages = MT == 1 ? 3 : 5;
  static constexpr int kCtasPerSm = MT == 1 ? 2 : 1;
  static constexpr uint32_t kS = kStages * kStage;                        // [4][rows][kSPitch] float
  static constexpr uint32_t kP = kS + 4 * kRows * kSPitch * 4;            // [2][rows][kPPitch] half: parts of P
  static constexpr uint32_t kAlpha = kP + 2 * kRows * kPPitch * 2;        // [rows] float
  static constexpr uint32_t kInv = kAlpha + kRows * 4;                    // [rows] float
  static constexpr uint32_t kBar = kInv + kRows * 4;                      // a barrier per stage
  static constexpr uint32_t kMisc = kBar + 8 * 8;                         // abort flag, Walk of the lookups
  static_assert(8 + sizeof(Walk) <= 48, "misc block");
  static constexpr uint32_t kBad = kMisc + 48;                            // [2][2] rows of hide_rows, by tile parity
  static constexpr uint32_t kMap = kMisc + 64;                            // [kAhead] first cache row, KV head
  static constexpr uint32_t kBytes = kMap + kAhead * 8 + 1024;            // + alignment slack
};

struct MmaParams {
  CUtensorMap tm_codes;    // [rows][kv_heads][256] bytes, box 64 x 1 x 128
  CUtensorMap tm_scales;   // [rows][kv_heads][16] halves, box 64 x 1 x 16
  CUtensorMap tm_kpe;      // [rows][kv_heads][64], box 64 x 1 x 64
  Int4Args a;
  uint32_t* status;
  int2* info;              // [units] of a split unit: its first piece's slot, its last worker; x < 0: not split
  int g, groups;           // query heads per KV head; groups of 16 MT query rows
  int num_rows;            // rows of the cache
  float sl2;               // softmax scale x log2(e)
};

// Bounded wait; once any wait of the CTA has given up every wait returns at once, so
// that all threads still meet at every barrier and the launch ends.
__device__ __forceinline__ void wait_full(uint32_t bar, uint32_t parity, volatile uint32_t* abort, uint32_t* status,
                                          uint32_t code) {
  if (ptx::mbar_try_wait(bar, parity)) return;
  const uint64_t t0 = ptx::globaltimer();
  for (;;) {
    for (int i = 0; i < 32; ++i)
      if (ptx::mbar_try_wait(bar, parity)) return;
    if (*abort != 0u) return;
    if (ptx::globaltimer() - t0 > kWaitNs) {
      *abort = 1u;
      atomicCAS(status, 0u, code);
      return;
    }
  }
}

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t h2u(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 u2h(uint32_t w) { return *reinterpret_cast<__half2*>(&w); }

// Field pairs 0..3 of a word whose nibbles j and j + 4 are the pair's two codes, as
// n - 8: 1024 + n and 64 + n are exact in fp16, so are the differences.
__device__ __forceinline__ void codes4(uint32_t w, uint32_t (&o)[4]) {
  const uint32_t v = w >> 8;
  const __half2 c0 = u2h(0x64086408u), c1 = u2h(0x54805480u);   // 1032, 72
  o[0] = h2u(__hsub2(u2h((w & 0x000f000fu) | 0x64006400u), c0));
  o[1] = h2u(__hsub2(u2h((w & 0x00f000f0u) | 0x54005400u), c1));
  o[2] = h2u(__hsub2(u2h((v & 0x000f000fu) | 0x64006400u), c0));
  o[3] = h2u(__hsub2(u2h((v & 0x00f000f0u) | 0x54005400u), c1));
}

// The same times s2 (one rounding).
__device__ __forceinline__ void widen4(uint32_t w, __half2 s2, uint32_t (&o)[4]) {
  codes4(w, o);
#pragma unroll
  for (int k = 0; k < 4; ++k) o[k] = h2u(__hmul2(u2h(o[k]), s2));
}

template <typename T>
__device__ __forceinline__ uint32_t to_h2(uint32_t w) {
  if constexpr (std::is_same<T, __half>::value) return w;
  else return Elt<__half>::pack2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// Rows that some of the tile's query rows do not see (a later position's, within the
// length), [first, end) of the tile at `stage`, may hold anything, but their weight 0 times
// a value past fp16 would be NaN.  After the scores are taken, a group with such a value gets the
// scale 0 and its row a bit in `bad`: the query rows that do see it answer NaN instead.
__device__ __noinline__ void hide_rows(uint8_t* stage, uint32_t* bad, int first, int end, int tid) {
  for (int i = first * kI4Groups + tid; i < end * kI4Groups; i += kThreads) {
    const int r = i / kI4Groups, g = i % kI4Groups;
    __half* scale = reinterpret_cast<__half*>(stage + kCodeBytes + kRopeBytes) + i;
    const float s = fabsf(__half2float(*scale));
    if (s * 8.f < 65520.f) continue;   // (65520 and more round to infinity)
    const uint4 w = *reinterpret_cast<const uint4*>(stage + (g >> 3) * (kCodeBytes / 2) + r * 128 +
                                                    (((g & 7) ^ (r & 7)) << 4));
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
    int most = 0;                      // the group's largest |n - 8|
    for (int k = 0; k < kI4Group; ++k) most = max(most, abs((int)((v[k >> 3] >> (4 * (k & 7))) & 15u) - 8));
    if (s * (float)most < 65520.f) continue;
    *scale = __ushort_as_half(0);
    atomicOr(bad + (r >> 5), 1u << (r & 31));
  }
  ptx::fence_proxy_async_smem();
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// kHide: sequences of several positions, whose last rows not all of them see.
template <typename T, int MT, bool kHide>
__global__ void __launch_bounds__(kThreads, Lay<MT>::kCtasPerSm)
mla_int4_mma_kernel(const __grid_constant__ MmaParams p) {
  using L = Lay<MT>;
  constexpr bool kTwoParts = std::is_same<T, __half>::value;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  // (aligned by an offset: a pointer rounded as an integer would make every access generic)
  uint8_t* smem = smem_raw + ((1024u - (ptx::smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t sbase = ptx::smem_u32(smem);
  const Int4Args& a = p.a;
  volatile uint32_t* abort = reinterpret_cast<volatile uint32_t*>(smem + L::kMisc);
  const uint32_t full0 = sbase + L::kBar;
  int2* ahead = reinterpret_cast<int2*>(smem + L::kMap);
  Walk* scout = reinterpret_cast<Walk*>(smem + L::kMisc + 8);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int units_per_seq = a.kv_heads * p.groups;
  const long long me = blockIdx.x;

  // ---- this worker's range: sum the sequences' tiles, find the range's first
  __shared__ long long s_sum[kThreads / 32];
  __shared__ long long s_first[2];   // tile within the flattened list, sequence
  const int per = (a.batch + kThreads - 1) / kThreads;
  const int b0 = min(tid * per, a.batch), b1 = min(b0 + per, a.batch);
  long long mine = 0;
  for (int s = b0; s < b1; ++s) mine += (seq_rows(a, s) + kTileR - 1) / kTileR;
  mine *= units_per_seq;
  long long incl = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const long long o = __shfl_up_sync(0xffffffffu, incl, off);
    if (lane >= off) incl += o;
  }
  if (lane == 31) s_sum[warp] = incl;
  if (tid == 0) {
    *abort = 0u;
    for (int i = 0; i < L::kStages; ++i) ptx::mbar_init(full0 + 8 * i, 1);
    ptx::fence_mbarrier_init();
  }
  __syncthreads();
  long long before = 0, total = 0;
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += s_sum[w];
    total += s_sum[w];
  }
  incl += before;
  // no worker inside a unit may own nothing: as many workers as tiles at most
  const long long workers = max(1ll, min((long long)gridDim.x, total));
  const long long x0 = me < workers ? me * total / workers : total;
  const long long x1 = me < workers ? (me + 1) * total / workers : total;
  if (x0 < x1 && x0 >= incl - mine && x0 < incl) {   // one thread's sequences hold tile x0
    long long at = incl - mine;
    for (int s = b0; s < b1; ++s) {
      const long long n = (long long)((seq_rows(a, s) + kTileR - 1) / kTileR) * units_per_seq;
      if (x0 < at + n) {
        s_first[0] = x0 - at;
        s_first[1] = s;
        break;
      }
      at += n;
    }
  }
  if (tid == 0) ptx::grid_dep_launch();   // the combine launch may be set up
  __syncthreads();
  Walk it{(int)(x1 - x0), 0, 0, 0, 0, 0};
  if (it.left > 0) {
    it.s = (int)s_first[1];
    it.len = seq_rows(a, it.s);
    it.nt = (it.len + kTileR - 1) / kTileR;
    it.sub = (int)(s_first[0] / it.nt);
    it.j = (int)(s_first[0] - (long long)it.sub * it.nt);
  }

  const int n_tiles = it.left;
  // Rows of tiles [32 k, 32 k + 32), one a lane of warp 7 (a chain of dependent loads for
  // all of them instead of one each).
  auto look_ahead = [&](int k) {
    Walk w = *scout;
    int s = -1, j = 0, kvh = 0;
    const int first = 32 * k, n = min(32, n_tiles - first);
    for (int l = 0; l < n; ++l) {
      if (l == lane) {
        s = w.s;
        j = w.j;
        kvh = w.sub / p.groups;
      }
      w.next(a, units_per_seq);
    }
    // a page the cache does not have reads as zeros: past the maps' last row
    const long long r = s < 0 ? -1
                              : cache_row(a.block_table, a.max_pages, a.page_size, a.num_pages, a.max_seqlen, s,
                                          j * kTileR);
    ahead[(first + lane) % kAhead] = make_int2(r >= 0 ? (int)r : p.num_rows, kvh);
    __syncwarp();
    if (lane == 0) *scout = w;
    __syncwarp();
  };
  // Thread 0: tile i into its stage.
  const uint64_t once = ptx::l2_policy_evict_first();
  auto fetch = [&](int i) {
    if (i >= n_tiles || *abort != 0u) return;
    const int2 at = ahead[i % kAhead];
    const int st = i % L::kStages;
    const uint32_t bar = full0 + 8 * st, dst = sbase + st * kStage;
    ptx::mbar_arrive_expect_tx(bar, kStage);
    ptx::tma_load_3d_local_hint(dst, &p.tm_codes, bar, 0, at.y, at.x, once);
    ptx::tma_load_3d_local_hint(dst + kCodeBytes / 2, &p.tm_codes, bar, 128, at.y, at.x, once);
    ptx::tma_load_3d_local_hint(dst + kCodeBytes, &p.tm_kpe, bar, 0, at.y, at.x, once);
    ptx::tma_load_3d_local_hint(dst + kCodeBytes + kRopeBytes, &p.tm_scales, bar, 0, at.y, at.x, once);
  };
  if (warp == 7) {
    if (lane == 0) *scout = it;
    __syncwarp();
    look_ahead(0);
  }
  __syncthreads();
  if (tid == 0)
    for (int i = 0; i < L::kStages; ++i) fetch(i);
  {
    // units without rows: zeros (their query rows see nothing), spread over the workers
    for (long long s = me; s < a.batch; s += gridDim.x) {
      if (seq_rows(a, (int)s) > 0) continue;
      const long long rows = (long long)a.q_len * a.heads;
      for (long long i = tid; i < rows * (kDim * 2 / 16); i += kThreads)
        (static_cast<uint4*>(a.out) + s * rows * (kDim * 2 / 16))[i] = make_uint4(0u, 0u, 0u, 0u);
      if (a.lse != nullptr)
        for (long long i = tid; i < rows; i += kThreads) a.lse[s * rows + i] = -INFINITY;
      for (int i = tid; i < units_per_seq; i += kThreads) p.info[s * units_per_seq + i] = make_int2(-1, -1);
    }
    const int qr = lane >> 2, t = lane & 3;          // fragment row / column group
    const int tq = warp >> 2, dq = warp & 3;         // S: row half, quarter of the dims
    float* sS = reinterpret_cast<float*>(smem + L::kS);
    __half* sP = reinterpret_cast<__half*>(smem + L::kP);
    // A fragment of k-step ks, weights of 16 rows from row `row`
    auto load_p = [&](int row, int ks, uint32_t (&o)[4]) {
      const __half* pr = sP + (row + qr) * kPPitch + 16 * ks + 2 * t;
      o[0] = *reinterpret_cast<const uint32_t*>(pr);
      o[1] = *reinterpret_cast<const uint32_t*>(pr + 8 * kPPitch);
      o[2] = *reinterpret_cast<const uint32_t*>(pr + 8);
      o[3] = *reinterpret_cast<const uint32_t*>(pr + 8 * kPPitch + 8);
    };
    float* sAlpha = reinterpret_cast<float*>(smem + L::kAlpha);
    float* sInv = reinterpret_cast<float*>(smem + L::kInv);
    const int rows_all = a.q_len * p.g;              // query rows of a unit's KV head
    uint32_t qf[MT][8][4], qpf[MT][4];               // Q: latent k-steps of this quarter, rope k-step dq
    float acc[MT][8][4];                             // O: dims 64 warp + 8 n + e
    float m_run[MT], l_run[MT];                      // softmax row (tid / 16) + 16 mt, 4 columns of it
    int row_len[MT];
    long long pos = x0;                              // flattened tile
    int tile = 0;
    // offsets within a stage: granule c of row r of a swizzled box is at c ^ (r & 7), so a
    // thread's other granules are its first one's address with bits 4..6 exclusive-ored
    const uint32_t k_off = (dq >> 1) * (kCodeBytes / 2) + (32 * tq + qr) * 128 + ((((dq & 1) * 4) ^ qr) << 4) + 4 * t;
    const uint32_t r_off = kCodeBytes + (32 * tq + qr) * 128 + (((2 * dq) ^ qr) << 4) + 4 * t;
    // word 8 warp + qr of a row: chunk 2 (warp % 4) + qr / 4 of box warp / 4, scale group 2 warp + qr / 4
    const uint32_t v_off = (warp >> 2) * (kCodeBytes / 2) + 2 * t * 128 +
                           (((2 * (warp & 3) + (qr >> 2)) ^ (2 * t)) << 4) + 4 * (qr & 3);
    const uint32_t vs_off = kCodeBytes + kRopeBytes + 2 * t * 32 + (2 * warp + (qr >> 2)) * 2;
    while (it.left > 0) {
      // ---- a piece: tiles [j0, j1) of unit (s, sub)
      const int s = it.s, sub = it.sub, kvh = sub / p.groups, r_base = (sub % p.groups) * L::kRows;
      const int j0 = it.j, len = it.len, nt = it.nt;
      const int j1 = min(nt, j0 + it.left);
      // query row r of the unit: position r / g, head kvh g + r % g
      auto q_row = [&](int r) -> long long {
        const int pos_t = r / p.g, i = r - pos_t * p.g;
        return ((long long)s * a.q_len + pos_t) * a.heads + kvh * p.g + i;
      };
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = r_base + 16 * mt + 8 * h + qr;
          const bool real = r < rows_all;
          const long long qi = real ? q_row(r) : 0;
          const uint4* q4 = reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + qi * kDim) + 16 * dq + t;
          const uint32_t* pe = reinterpret_cast<const uint32_t*>(static_cast<const T*>(a.q_pe) + qi * kPeDim) + 8 * dq + t;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint4 x = real ? __ldg(q4 + 4 * j) : make_uint4(0u, 0u, 0u, 0u);
            qf[mt][2 * j][h] = to_h2<T>(x.x);
            qf[mt][2 * j][2 + h] = to_h2<T>(x.y);
            qf[mt][2 * j + 1][h] = to_h2<T>(x.z);
            qf[mt][2 * j + 1][2 + h] = to_h2<T>(x.w);
          }
          qpf[mt][h] = real ? __ldg(pe) : 0u;
          qpf[mt][2 + h] = real ? __ldg(pe + 4) : 0u;
        }
        const int r = r_base + 16 * mt + (tid >> 4);
        row_len[mt] = r < rows_all ? len - (a.q_len - 1 - r / p.g) : len;
        m_run[mt] = -INFINITY;
        l_run[mt] = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[mt][e][c] = 0.f;
      }
#pragma unroll 1
      for (int j = j0; j < j1; ++j, ++tile) {
        const int st = tile % L::kStages;
        if ((tile & 31) == 0 && warp == 7) look_ahead(tile / 32 + 1);
        wait_full(full0 + 8 * st, (uint32_t)(tile / L::kStages) & 1u, abort, p.status, kErrLoad);
        const uint32_t stage = st * kStage;
        uint8_t* scales = smem + st * kStage + kCodeBytes + kRopeBytes;
        const int valid = len - j * kTileR;
        // rows of this tile that not every position sees: from its first position's length on
        const int hidden = max(valid - (a.q_len - 1), 0);
        const bool hides = kHide && hidden < kTileR;
        uint32_t* bad = reinterpret_cast<uint32_t*>(smem + L::kBad) + 2 * (tile & 1);
        if (hides && tid < 2) bad[tid] = 0u;
        if (valid < kTileR) {
          // rows past the length: a zero scale makes them zeros whatever the cache holds
          if (tid < 2 * kTileR && (tid >> 1) >= valid)
            reinterpret_cast<uint4*>(scales)[tid] = make_uint4(0u, 0u, 0u, 0u);
          ptx::fence_proxy_async_smem();
          __syncthreads();
        }
        // ---- S, this warp's rows [32 tq, +32) and dims [128 dq, +128) (and 16 rope dims)
#pragma unroll
        for (int nb = 0; nb < 4; ++nb) {
          // the scales of this thread's two columns (rows of the tile), four groups each
          const uint2 sc0 = *reinterpret_cast<const uint2*>(scales + (32 * tq + 8 * nb + 2 * t) * 32 + dq * 8);
          const uint2 sc1 = *reinterpret_cast<const uint2*>(scales + (32 * tq + 8 * nb + 2 * t + 1) * 32 + dq * 8);
          float c[MT][4];
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) c[mt][0] = c[mt][1] = c[mt][2] = c[mt][3] = 0.f;
          const uint32_t r0 = *reinterpret_cast<const uint32_t*>(smem + (stage + r_off) + 1024 * nb);
          const uint32_t r1 = *reinterpret_cast<const uint32_t*>(smem + ((stage + r_off) ^ 16u) + 1024 * nb);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) mma16816<T>(c[mt], qpf[mt], r0, r1);
#pragma unroll
          for (int jj = 0; jj < 4; ++jj) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(smem + ((stage + k_off) ^ (16u * jj)) + 1024 * nb);
            const __half2 a0 = u2h(jj < 2 ? sc0.x : sc0.y), a1 = u2h(jj < 2 ? sc1.x : sc1.y);
            const float s0 = (jj & 1) ? __high2float(a0) : __low2float(a0);
            const float s1 = (jj & 1) ? __high2float(a1) : __low2float(a1);
            uint32_t f[4];
            codes4(w, f);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              float x[4] = {0.f, 0.f, 0.f, 0.f};
              mma16816<__half>(x, qf[mt][2 * jj], f[0], f[1]);
              mma16816<__half>(x, qf[mt][2 * jj + 1], f[2], f[3]);
              c[mt][0] = fmaf(x[0], s0, c[mt][0]);
              c[mt][1] = fmaf(x[1], s1, c[mt][1]);
              c[mt][2] = fmaf(x[2], s0, c[mt][2]);
              c[mt][3] = fmaf(x[3], s1, c[mt][3]);
            }
          }
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            float* dst = sS + (dq * L::kRows + 16 * mt + qr) * kSPitch + 32 * tq + 8 * nb + 2 * t;
            *reinterpret_cast<float2*>(dst) = make_float2(c[mt][0], c[mt][1]);
            *reinterpret_cast<float2*>(dst + 8 * kSPitch) = make_float2(c[mt][2], c[mt][3]);
          }
        }
        __syncthreads();
        // every warp is past the tile before: its stage takes the next load
        if (tid == 0 && tile > 0) fetch(tile - 1 + L::kStages);
        if (hides) hide_rows(smem + stage, bad, hidden, min(valid, kTileR), tid);
        // ---- softmax: thread <-> row tid / 16 (+ 16 mt), columns 4 (tid % 16)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const int row = 16 * mt + (tid >> 4), col = 4 * (tid & 15);
          float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int d = 0; d < 4; ++d) {
            const float4 x = *reinterpret_cast<const float4*>(sS + (d * L::kRows + row) * kSPitch + col);
            v[0] += x.x;
            v[1] += x.y;
            v[2] += x.z;
            v[3] += x.w;
          }
          const int seen = row_len[mt] - j * kTileR - col;
          float mx = -INFINITY;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (e >= seen) v[e] = -INFINITY;
            mx = fmaxf(mx, v[e]);
          }
#pragma unroll
          for (int off = 8; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
          const float m_new = fmaxf(m_run[mt], mx);
          float alpha = 1.f;
          if ((m_new - m_run[mt]) * p.sl2 > kLazyLog2) {   // (also the first rows a query row sees)
            alpha = exp2_approx((m_run[mt] - m_new) * p.sl2);
            m_run[mt] = m_new;
          }
          // a query row that has seen nothing yet: every weight 0
          const float ms = m_run[mt] == -INFINITY ? 0.f : fmaf(m_run[mt], p.sl2, -kI4WeightLog2);
          float ls = 0.f;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            v[e] = exp2_approx(fmaf(v[e], p.sl2, -ms));
            ls += v[e];
          }
          l_run[mt] = fmaf(l_run[mt], alpha, ls);
          const uint2 hi = make_uint2(Elt<__half>::pack2(v[0], v[1]), Elt<__half>::pack2(v[2], v[3]));
          *reinterpret_cast<uint2*>(sP + row * kPPitch + col) = hi;
          if constexpr (kTwoParts) {
            const float2 h0 = Elt<__half>::to2(hi.x), h1 = Elt<__half>::to2(hi.y);
            *reinterpret_cast<uint2*>(sP + (L::kRows + row) * kPPitch + col) =
                make_uint2(Elt<__half>::pack2(v[0] - h0.x, v[1] - h0.y), Elt<__half>::pack2(v[2] - h1.x, v[3] - h1.y));
          }
          if ((tid & 15) == 0) sAlpha[row] = alpha;
        }
        __syncthreads();
        if (hides) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            const int col = 4 * (tid & 15), seen = row_len[mt] - j * kTileR - col;
            const uint32_t mine = bad[col >> 5] >> (col & 31);
            if (seen > 0 && (mine & ((1u << min(seen, 4)) - 1u)) != 0u) l_run[mt] = __int_as_float(0x7fffffff);
          }
        }
        // ---- O += P.V, dims [64 warp, +64)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const float al = sAlpha[16 * mt + qr], ah = sAlpha[16 * mt + 8 + qr];
          if (__any_sync(0xffffffffu, al != 1.f || ah != 1.f)) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              acc[mt][e][0] *= al;
              acc[mt][e][1] *= al;
              acc[mt][e][2] *= ah;
              acc[mt][e][3] *= ah;
            }
          }
        }
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          uint32_t pf[MT][4];
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) load_p(16 * mt, ks, pf[mt]);
          uint32_t f[2][2][4];   // [rows 2 t and 2 t + 8][even, odd dims][pair]
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            // rows 16 ks + 8 h + 2 t and the next
            const int up = 16 * ks + 8 * h;
            const uint32_t w0 = *reinterpret_cast<const uint32_t*>(smem + (stage + v_off) + up * 128);
            const uint32_t w1 = *reinterpret_cast<const uint32_t*>(smem + ((stage + v_off) ^ 16u) + 128 + up * 128);
            const uint32_t sa = *reinterpret_cast<const unsigned short*>(smem + (stage + vs_off) + up * 32);
            const uint32_t sb = *reinterpret_cast<const unsigned short*>(smem + (stage + vs_off) + up * 32 + 32);
            const __half2 s2 = u2h(sa | (sb << 16));
            widen4(__byte_perm(w0, w1, 0x5410), s2, f[h][0]);
            widen4(__byte_perm(w0, w1, 0x7632), s2, f[h][1]);
          }
#pragma unroll
          for (int e = 0; e < 8; ++e)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) mma16816<__half>(acc[mt][e], pf[mt], f[0][e & 1][e >> 1], f[1][e & 1][e >> 1]);
          if constexpr (kTwoParts) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) load_p(L::kRows + 16 * mt, ks, pf[mt]);
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
              for (int mt = 0; mt < MT; ++mt)
                mma16816<__half>(acc[mt][e], pf[mt], f[0][e & 1][e >> 1], f[1][e & 1][e >> 1]);
          }
        }
      }
      // ---- end of the piece: normalise, write the result or a partial
      const bool whole = j0 == 0 && j1 == nt;
      const bool starts = pos == x0;                   // this worker's first piece: slot 0
      const long long slot = 2 * me + (starts ? 0 : 1);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        float l = l_run[mt];
#pragma unroll
        for (int off = 8; off > 0; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
        const int row = 16 * mt + (tid >> 4), r = r_base + row;
        if ((tid & 15) == 0) {
          const float lse = l != 0.f ? (m_run[mt] * p.sl2 + (log2f(l) - kI4WeightLog2)) * kLn2 : -INFINITY;
          sInv[row] = l != 0.f ? 1.f / l : 0.f;
          if (!whole)
            a.part_lse[slot * L::kRows + row] = lse;
          else if (a.lse != nullptr && r < rows_all)
            a.lse[q_row(r)] = lse;
        }
      }
      if (j0 == 0 && tid == 0) {
        // whoever holds a unit's first tile records its workers for the combine launch
        const int last = (int)(((pos + nt) * workers + total - 1) / total - 1);
        p.info[(long long)s * units_per_seq + sub] = whole ? make_int2(-1, -1) : make_int2((int)slot, last);
      }
      __syncthreads();
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int row = 16 * mt + 8 * h + qr, r = r_base + row;
          if (r >= rows_all) continue;
          const float inv = sInv[row];
          // dims 64 warp + 16 t + [0, 8) from column 2 t, + [8, 16) from column 2 t + 1
          if (whole) {
            uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + q_row(r) * kDim + 64 * warp + 16 * t);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              uint32_t o[4];
#pragma unroll
              for (int e = 0; e < 4; ++e)
                o[e] = Elt<T>::pack2(acc[mt][2 * e][2 * h + c] * inv, acc[mt][2 * e + 1][2 * h + c] * inv);
              dst[c] = make_uint4(o[0], o[1], o[2], o[3]);
            }
          } else {
            float4* dst = reinterpret_cast<float4*>(a.part_o + (slot * L::kRows + row) * kDim + 64 * warp + 16 * t);
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                dst[2 * c + e] = make_float4(acc[mt][4 * e][2 * h + c] * inv, acc[mt][4 * e + 1][2 * h + c] * inv,
                                             acc[mt][4 * e + 2][2 * h + c] * inv, acc[mt][4 * e + 3][2 * h + c] * inv);
          }
        }
      }
      pos += j1 - j0;
      it.left -= j1 - j0 - 1;
      it.j = j1 - 1;
      it.next(a, units_per_seq);
    }
    // nothing is in flight here unless the walk ended early (lengths that changed under
    // the call): loads must land before the CTA's shared memory goes away
    for (int i = tile; i < min(n_tiles, max(tile - 1, 0) + L::kStages); ++i)
      wait_full(full0 + 8 * (i % L::kStages), (uint32_t)(i / L::kStages) & 1u, abort, p.status, kErrLoad);
  }
  if (*abort != 0u) {
    // copies in flight land before the CTA's shared memory goes away
    const uint64_t t0 = ptx::globaltimer();
    while (ptx::globaltimer() - t0 < 2000000ull) __nanosleep(1000);
  }
}

// Merge of the units that a range's end cut: one CTA per query row at a time, G groups of
// 128 threads (four dims a thread) taking every G-th piece, eight pieces in flight each;
// their sums meet in shared memory.  The LSE algebra of mla_combine.cu.
template <typename T, int kMergeGroups>
__global__ void __launch_bounds__(128 * kMergeGroups)
mla_int4_mma_combine_kernel(Int4Args a, const int2* __restrict__ info, int g, int groups, int rows, long long items) {
  __shared__ float s_w[kMaxWorkers];
  __shared__ float4 s_acc[kMergeGroups][128];
  const int grp = threadIdx.x >> 7, tid = threadIdx.x & 127, lane = tid & 31;
  const int units_per_seq = a.kv_heads * groups, rows_all = a.q_len * g;
  ptx::grid_dep_wait();
  for (long long i = blockIdx.x; i < items; i += gridDim.x) {
    const long long unit = i / rows;
    const int row = (int)(i - unit * rows);
    const int2 w = __ldcg(info + unit);
    const int s = (int)(unit / units_per_seq), sub = (int)(unit - (long long)s * units_per_seq);
    const int r = (sub % groups) * rows + row;
    if (w.x < 0 || r >= rows_all) continue;      // (the same for every thread)
    const int w0 = w.x >> 1, n = w.y - w0 + 1;   // (at most kMaxWorkers)
    // after the unit's first piece each worker's first
    auto slot = [&](int k) -> long long { return k == 0 ? (long long)w.x : 2ll * (w0 + k); };
    auto piece = [&](int k) -> float4 {
      return k < n ? __ldcg(reinterpret_cast<const float4*>(a.part_o + (slot(k) * rows + row) * kDim) + tid)
                   : make_float4(0.f, 0.f, 0.f, 0.f);
    };
    float4 v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = piece(grp + kMergeGroups * u);
    for (int k = threadIdx.x; k < n; k += 128 * kMergeGroups) s_w[k] = __ldcg(a.part_lse + slot(k) * rows + row);
    __syncthreads();
    // every warp reduces the pieces' LSEs itself
    float mx = -INFINITY;
    for (int k = lane; k < n; k += 32) mx = max_nan(mx, s_w[k]);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, off));
    const bool any = mx != -INFINITY;
    float sum = 0.f;
    if (any)
      for (int k = lane; k < n; k += 32) sum += exp2f((s_w[k] - mx) * kLog2e);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    const float lse = any ? mx + logf(sum) : -INFINITY;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k0 = grp; any && k0 < n; k0 += 8 * kMergeGroups) {
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int k = k0 + kMergeGroups * u;
        if (k >= n) break;
        const float e = exp2f((s_w[k] - lse) * kLog2e);
        acc.x = fmaf(e, v[u].x, acc.x);
        acc.y = fmaf(e, v[u].y, acc.y);
        acc.z = fmaf(e, v[u].z, acc.z);
        acc.w = fmaf(e, v[u].w, acc.w);
      }
      if (k0 + 8 * kMergeGroups < n) {
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = piece(k0 + kMergeGroups * (8 + u));
      }
    }
    if (grp > 0) s_acc[grp][tid] = acc;
    __syncthreads();
    if (grp == 0) {
#pragma unroll
      for (int o = 1; o < kMergeGroups; ++o) {
        const float4 x = s_acc[o][tid];
        acc.x += x.x;
        acc.y += x.y;
        acc.z += x.z;
        acc.w += x.w;
      }
      const int pos_t = r / g;
      const long long qi = ((long long)s * a.q_len + pos_t) * a.heads + (sub / groups) * g + (r - pos_t * g);
      *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + qi * kDim + 4 * tid) =
          make_uint2(Elt<T>::pack2(acc.x, acc.y), Elt<T>::pack2(acc.z, acc.w));
      if (a.lse != nullptr && tid == 0) a.lse[qi] = lse;
    }
    __syncthreads();   // the shared arrays are free for the next row
  }
}

struct DeviceFacts {
  bool ready = false;
  int sms = 0;
};
DeviceFacts g_dev[64];
std::mutex g_mutex;

// SMs of the current device (148 on a host without one: a B200's plan); the kernels'
// shared memory is granted on the first call on a device.
cudaError_t device_facts(int* sms) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) {
    cudaGetLastError();
    *sms = 148;
    return cudaErrorInvalidDevice;
  }
  std::lock_guard<std::mutex> lock(g_mutex);
  DeviceFacts& d = g_dev[dev];
  if (!d.ready) {
    cudaError_t err = cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, dev);
    auto grant = [&](const void* f, uint32_t bytes) {
      if (err == cudaSuccess) err = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    };
    grant(reinterpret_cast<const void*>(mla_int4_mma_kernel<__half, 1, false>), Lay<1>::kBytes);
    grant(reinterpret_cast<const void*>(mla_int4_mma_kernel<__half, 1, true>), Lay<1>::kBytes);
    grant(reinterpret_cast<const void*>(mla_int4_mma_kernel<__nv_bfloat16, 1, false>), Lay<1>::kBytes);
    grant(reinterpret_cast<const void*>(mla_int4_mma_kernel<__nv_bfloat16, 1, true>), Lay<1>::kBytes);
    grant(reinterpret_cast<const void*>(mla_int4_mma_kernel<__half, 2, false>), Lay<2>::kBytes);
    grant(reinterpret_cast<const void*>(mla_int4_mma_kernel<__half, 2, true>), Lay<2>::kBytes);
    grant(reinterpret_cast<const void*>(mla_int4_mma_kernel<__nv_bfloat16, 2, false>), Lay<2>::kBytes);
    grant(reinterpret_cast<const void*>(mla_int4_mma_kernel<__nv_bfloat16, 2, true>), Lay<2>::kBytes);
    if (err != cudaSuccess) return err;
    d.ready = true;
  }
  *sms = d.sms;
  return cudaSuccess;
}

// The tensor maps of a call: encoded for a shape (a thread keeps the last few shapes'),
// then given the call's addresses.
struct Maps {
  CUtensorMap codes, scales, kpe;
};
struct MapKey {
  long long rows;
  int kv_heads, dtype;
};

bool encode_maps(const Int4Args& a, const MapKey& k, Maps* m) {
  const CUtensorMapDataType dt =
      k.dtype == MLA_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  if (!sm100::make_map_kv(&m->codes, a.codes, kI4Bytes, k.kv_heads, k.rows, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1) ||
      !sm100::make_map_kv(&m->kpe, a.k_pe, kPeDim, k.kv_heads, k.rows, dt, 2))
    return false;
  const auto fn = sm100::encode_fn();
  if (fn == nullptr) return false;
  const cuuint64_t dims[3] = {kI4Groups, (cuuint64_t)k.kv_heads, (cuuint64_t)k.rows};
  const cuuint64_t strides[2] = {kI4Groups * 2, (cuuint64_t)k.kv_heads * kI4Groups * 2};
  const cuuint32_t box[3] = {kI4Groups, 1, kTileR};
  const cuuint32_t estr[3] = {1, 1, 1};
  return fn(&m->scales, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<__half*>(a.scales), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool tensor_maps(const Int4Args& a, long long rows, MmaParams* p) {
  const MapKey key{rows, a.kv_heads, a.dtype};
  struct Entry {
    MapKey key;
    Maps maps;
  };
  constexpr int kSlots = 8;
  thread_local Entry cache[kSlots];
  thread_local int filled = 0, next = 0;
  const Maps* m = nullptr;
  for (int i = 0; i < filled && m == nullptr; ++i)
    if (cache[i].key.rows == key.rows && cache[i].key.kv_heads == key.kv_heads && cache[i].key.dtype == key.dtype)
      m = &cache[i].maps;
  if (m == nullptr) {
    Maps made;
    if (!encode_maps(a, key, &made)) return false;
    cache[next] = Entry{key, made};
    m = &cache[next].maps;
    next = (next + 1) % kSlots;
    if (filled < kSlots) ++filled;
  }
  return sm100::place_map(&p->tm_codes, m->codes, a.codes) && sm100::place_map(&p->tm_scales, m->scales, a.scales) &&
         sm100::place_map(&p->tm_kpe, m->kpe, a.k_pe);
}

inline size_t align_up(size_t x, size_t a) { return (x + a - 1) / a * a; }

template <typename T, int MT>
cudaError_t launch_typed(const MmaParams& p, int workers, cudaStream_t stream) {
  using L = Lay<MT>;
  if (p.a.q_len > 1)
    mla_int4_mma_kernel<T, MT, true><<<workers, kThreads, L::kBytes, stream>>>(p);
  else
    mla_int4_mma_kernel<T, MT, false><<<workers, kThreads, L::kBytes, stream>>>(p);
  cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return err;
  const long long items = (long long)p.a.batch * p.a.kv_heads * p.groups * L::kRows;
  cudaLaunchConfig_t cfg{};
  // few rows are cut into many pieces each, many rows into few (b128 h16 s4096, three
  // pieces a row: 16 us more with four groups; b1 h16 s131072, 296 pieces: 18 us less)
  const bool few = items < 148 * 4;
  const long long ctas = few ? items : (items < 148 * 16 ? items : 148 * 16);
  cfg.gridDim = dim3((unsigned)ctas, 1, 1);
  cfg.blockDim = dim3(few ? 512 : 128, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const int2* info = p.info;
  return few ? cudaLaunchKernelEx(&cfg, mla_int4_mma_combine_kernel<T, 4>, p.a, info, p.g, p.groups, L::kRows, items)
             : cudaLaunchKernelEx(&cfg, mla_int4_mma_combine_kernel<T, 1>, p.a, info, p.g, p.groups, L::kRows, items);
}

}  // namespace

Int4MmaPlan int4_mma_plan(int batch, int q_len, int heads, int kv_heads, int max_len, int row_tiles, int asked) {
  Int4MmaPlan p{};
  int sms = 148;
  device_facts(&sms);
  p.row_tiles = row_tiles;
  const int rows = 16 * row_tiles, g = heads / kv_heads;
  p.groups = (q_len * g + rows - 1) / rows;
  p.units = (long long)batch * kv_heads * p.groups;
  const long long tiles = p.units * ((max_len + kTileR - 1) / kTileR);
  long long w = (long long)sms * (row_tiles == 1 ? Lay<1>::kCtasPerSm : Lay<2>::kCtasPerSm);
  if (w > kMaxWorkers) w = kMaxWorkers;
  if (asked > 0 && asked < w) w = asked;
  if (w > tiles) w = tiles;
  p.workers = (int)w;
  p.info_off = 256;
  p.lse_off = p.info_off + align_up((size_t)p.units * sizeof(int2), 256);
  p.o_off = p.lse_off + align_up((size_t)2 * p.workers * rows * sizeof(float), 256);
  p.total = p.o_off + (size_t)2 * p.workers * rows * kDim * sizeof(float);
  return p;
}

cudaError_t launch_int4_mma(Int4Args a, const Int4MmaPlan& plan, void* workspace, cudaStream_t stream) {
  int sms = 0;
  cudaError_t err = device_facts(&sms);
  if (err != cudaSuccess) return err;
  char* base = static_cast<char*>(workspace);
  MmaParams p{};
  a.part_lse = reinterpret_cast<float*>(base + plan.lse_off);
  a.part_o = reinterpret_cast<float*>(base + plan.o_off);
  p.a = a;
  p.status = reinterpret_cast<uint32_t*>(base);
  p.info = reinterpret_cast<int2*>(base + plan.info_off);
  p.g = a.heads / a.kv_heads;
  p.groups = plan.groups;
  p.num_rows = a.block_table != nullptr ? a.num_pages * a.page_size : a.batch * a.max_seqlen;
  p.sl2 = a.softmax_scale * kLog2e;
  if (!tensor_maps(a, p.num_rows, &p)) return cudaErrorInvalidValue;
  const bool bf = a.dtype == MLA_DTYPE_BF16;
  if (plan.row_tiles == 1)
    return bf ? launch_typed<__nv_bfloat16, 1>(p, plan.workers, stream) : launch_typed<__half, 1>(p, plan.workers, stream);
  return bf ? launch_typed<__nv_bfloat16, 2>(p, plan.workers, stream) : launch_typed<__half, 2>(p, plan.workers, stream);
}

}  // namespace mla
