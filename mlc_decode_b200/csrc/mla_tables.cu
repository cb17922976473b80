// Block tables and slots of a paged cache, from request lengths, on the device
// (mla_extend_block_tables, include/mla_decode_b200.h): no host round trip between a
// step's lengths and its decode call.
//
// Request i holds h = ceil(L / page) pages for its L rows and asks for n more rows,
// hence take = ceil((L + n) / page) - h more pages.  Two prefix sums over the
// requests (rows, then pages) give every request its place in the token list and in
// the free list; after that every new row is independent: its request by binary
// search in the row sums, its page from the table (the page its request had begun) or
// from the free list.  The first row of a page also writes the page's table entry.
//
// Bound: a step is a few hundred bytes (latency of one launch); prompts are 8 bytes a
// row written.  A step (up to kSmallBatch requests and kSmallTokens rows) is one CTA
// that keeps the requests' records in shared memory: one launch.  Longer calls take a
// plan launch (one CTA: the sums, the records to the workspace) and a fill launch
// over all SMs.
#include <limits.h>

#include "mla_common.cuh"

namespace mla {
namespace {

constexpr int kThreads = 1024;
constexpr int kSmallBatch = 2048, kSmallTokens = 8192;
constexpr int kFillThreads = 256;

struct TablesArgs {
  int* block_table;          // [batch][max_pages]
  const int* seqlens;        // [batch]
  const int* new_lens;       // [batch]
  const int* free_pages;     // [num_free]
  const int* free_pos;       // [1]
  int* new_seqlens;          // [batch], may be seqlens
  int* new_free_pos;         // [1], may be free_pos
  int* slots;                // [num_tokens]
  int* positions;            // [num_tokens]
  int* cu_new;               // [batch + 1] or nullptr
  int batch, max_pages, page, num_pages, num_free, num_tokens;
  int q_len;                 // 0: rows packed; else request i's rows are the last of [i q_len, (i + 1) q_len)
};

// One request: first row in the packed list, rows held before, rows held after, and
// the free-list index of its first new page.
struct Record {
  int cu, len, end, first;
};

__device__ __forceinline__ int page_count(long long rows, int page) { return (int)((rows + page - 1) / page); }

// Inclusive sum over the CTA's threads of v; every thread calls it.
__device__ long long block_scan(long long v, long long* s_warp) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const long long o = __shfl_up_sync(0xffffffffu, v, off);
    if (lane >= off) v += o;
  }
  __syncthreads();   // s_warp of an earlier scan is free
  if (lane == 31) s_warp[warp] = v;
  __syncthreads();
  long long before = 0;
  for (int w = 0; w < warp; ++w) before += s_warp[w];
  return v + before;
}

// The records of every request, by one CTA; thread t owns requests [t per, (t + 1) per).
// A request's lengths are read and its new length written by the same thread, so
// new_seqlens may be seqlens.
// With kWhole (q_len > 0) a request gets all of its rows or none: one whose table row is too short
// asks for nothing, and one that does not find all its pages takes none; nor do those behind
// it that need any, so that the pages handed out are still a prefix of the sums.
template <bool kWhole>
__device__ void plan(const TablesArgs& a, Record* rec, long long* s_warp) {
  __shared__ int s_taken;   // kWhole: pages handed out
  if (kWhole && threadIdx.x == 0) s_taken = 0;
  const int per = (a.batch + kThreads - 1) / kThreads;
  const int i0 = min((int)threadIdx.x * per, a.batch), i1 = min(i0 + per, a.batch);
  const long long cover = (long long)a.max_pages * a.page;
  const int pos0 = min(max(*a.free_pos, 0), a.num_free);
  auto old_len = [&](int i) { return (int)min((long long)max(a.seqlens[i], 0), cover); };
  auto asked = [&](int i) { return min(max(a.new_lens[i], 0), a.q_len > 0 ? a.q_len : a.num_tokens); };
  // rows: places in the packed list, cut at num_tokens
  long long sum = 0;
  for (int i = i0; i < i1; ++i) sum += asked(i);
  long long at = block_scan(sum, s_warp) - sum;
  auto cut = [&](long long v) { return (int)min(v, (long long)a.num_tokens); };
  long long pages = 0;
  for (int i = i0; i < i1; ++i) {
    const int n = asked(i), cu = cut(at);
    int rows = cut(at + n) - cu;
    at += n;
    const int len = old_len(i);
    if (kWhole && len + (long long)rows > cover) rows = 0;
    rec[i] = Record{cu, len, rows, 0};   // end: the rows asked for, until the pages are known
    pages += page_count(min(len + (long long)rows, cover), a.page) - page_count(len, a.page);
  }
  if (a.cu_new != nullptr && threadIdx.x == kThreads - 1) a.cu_new[a.batch] = cut(at);
  // pages: places in the free list, handed out in request order until it is empty
  const long long incl = block_scan(pages, s_warp);   // (also: every thread has read *free_pos)
  long long taken = incl - pages;
  const long long avail = a.num_free - pos0;
  for (int i = i0; i < i1; ++i) {
    Record r = rec[i];
    const long long want = min(r.len + (long long)r.end, cover);
    const int held = page_count(r.len, a.page);
    const int take = page_count(want, a.page) - held;
    const int got = (int)min(max(avail - taken, 0ll), (long long)take);
    r.first = pos0 + (int)min(taken, avail);
    r.end = (int)min(want, (long long)(held + got) * a.page);
    taken += take;
    if (kWhole) {
      if (got < take)
        r.end = r.len;
      else if (take > 0)
        atomicMax(&s_taken, (int)taken);   // (at most avail)
    }
    rec[i] = r;
    if (a.cu_new != nullptr) a.cu_new[i] = r.cu;
    a.new_seqlens[i] = r.end;
  }
  if (kWhole) __syncthreads();
  if (threadIdx.x == kThreads - 1) *a.new_free_pos = pos0 + (kWhole ? s_taken : (int)min(incl, avail));
}

// Slot and position of row p of request i; p at a page's start also names the page in
// the table (a row past `end` has no place: slot -1).
__device__ __forceinline__ int place(const TablesArgs& a, const Record& r, int i, int p) {
  if (p >= r.end) return -1;
  const int k = p / a.page, off = p - k * a.page, held = page_count(r.len, a.page);
  int* entry = a.block_table + (size_t)i * a.max_pages + k;
  const int id = k < held ? *entry : __ldg(a.free_pages + r.first + (k - held));
  if (k >= held && off == 0) *entry = id;
  return (unsigned)id < (unsigned)a.num_pages ? id * a.page + off : -1;
}

// Rows [k, k + 4) of the token list (thread-sized share of the fill).
__device__ void fill4(const TablesArgs& a, const Record* rec, int k) {
  int slot[4], pos[4];
  int i = 0;
  if (a.q_len == 0) {   // the last request whose rows begin at or before row k
    int lo = 0, hi = a.batch - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (rec[mid].cu <= k) lo = mid; else hi = mid - 1;
    }
    i = lo;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    slot[e] = -1;
    pos[e] = 0;
    const int x = k + e;
    if (x >= a.num_tokens) continue;
    int t, n;   // row t of the request's n
    if (a.q_len > 0) {
      i = x / a.q_len;
      n = min(max(a.new_lens[i], 0), a.q_len);
      t = x - i * a.q_len - (a.q_len - n);
    } else {
      while (i + 1 < a.batch && rec[i + 1].cu <= x) ++i;
      n = min(max(a.new_lens[i], 0), a.num_tokens);
      t = x - rec[i].cu;
    }
    if (t < 0 || t >= n) continue;   // padding
    const long long p = (long long)rec[i].len + t;
    pos[e] = (int)min(p, (long long)INT_MAX);
    slot[e] = place(a, rec[i], i, pos[e]);
  }
  if (a.num_tokens - k >= 4 && ((reinterpret_cast<uintptr_t>(a.slots) | reinterpret_cast<uintptr_t>(a.positions)) & 15) == 0) {
    *reinterpret_cast<int4*>(a.slots + k) = make_int4(slot[0], slot[1], slot[2], slot[3]);
    *reinterpret_cast<int4*>(a.positions + k) = make_int4(pos[0], pos[1], pos[2], pos[3]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (k + e < a.num_tokens) {
        a.slots[k + e] = slot[e];
        a.positions[k + e] = pos[e];
      }
  }
}

template <bool kWhole>
__global__ void __launch_bounds__(kThreads) mla_tables_small_kernel(TablesArgs a) {
  __shared__ Record rec[kSmallBatch];
  __shared__ long long s_warp[kThreads / 32];
  plan<kWhole>(a, rec, s_warp);
  __syncthreads();
  for (int k = 4 * threadIdx.x; k < a.num_tokens; k += 4 * kThreads) fill4(a, rec, k);
}

template <bool kWhole>
__global__ void __launch_bounds__(kThreads) mla_tables_plan_kernel(TablesArgs a, Record* rec) {
  __shared__ long long s_warp[kThreads / 32];
  plan<kWhole>(a, rec, s_warp);
}

__global__ void __launch_bounds__(kFillThreads) mla_tables_fill_kernel(TablesArgs a, const Record* rec) {
  const long long k = 4 * ((long long)blockIdx.x * kFillThreads + threadIdx.x);
  if (k < a.num_tokens) fill4(a, rec, (int)k);
}

bool small(int batch, int num_tokens) { return batch <= kSmallBatch && num_tokens <= kSmallTokens; }


template <bool kWhole>
int extend(const char* fn, const TablesArgs& a, void* workspace, size_t workspace_bytes, void* stream) {
  const int batch = a.batch, max_pages = a.max_pages, page_size = a.page, num_pages = a.num_pages,
            num_free = a.num_free, num_tokens = a.num_tokens, q_len = a.q_len;
  if (batch < 1 || max_pages < 1 || page_size < 1 || num_pages < 1 || num_free < 0 || num_tokens < 0 || q_len < 0) {
    set_error("%s: bad size (batch %d, max_pages %d, page_size %d, num_pages %d, num_free %d, num_tokens %d, "
              "q_len %d)", fn, batch, max_pages, page_size, num_pages, num_free, num_tokens, q_len);
    return MLA_ERR_ARG;
  }
  if ((long long)num_pages * page_size > INT32_MAX || (long long)max_pages * page_size > INT32_MAX) {
    set_error("%s: num_pages x page_size and max_pages x page_size must stay below 2^31 rows (page_size %d, "
              "num_pages %d, max_pages %d)", fn, page_size, num_pages, max_pages);
    return MLA_ERR_ARG;
  }
  if (q_len > 0 && (long long)batch * q_len != num_tokens) {
    set_error("%s: with q_len, num_tokens must be batch x q_len (%d x %d, got %d)", fn, batch, q_len, num_tokens);
    return MLA_ERR_ARG;
  }
  if (!a.block_table || !a.seqlens || !a.new_lens || !a.free_pos || !a.new_seqlens || !a.new_free_pos ||
      (num_free > 0 && !a.free_pages) || (num_tokens > 0 && (!a.slots || !a.positions))) {
    set_error("%s: null pointer", fn);
    return MLA_ERR_ARG;
  }
  const bool one = small(batch, num_tokens);
  if (!one && (workspace == nullptr || workspace_bytes < (size_t)batch * sizeof(Record) ||
               (reinterpret_cast<uintptr_t>(workspace) & 15u) != 0)) {
    set_error("%s: workspace needs %zu bytes, 16-byte aligned (got %zu at %p)", fn, (size_t)batch * sizeof(Record),
              workspace_bytes, workspace);
    return MLA_ERR_WORKSPACE;
  }
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (one) {
    mla_tables_small_kernel<kWhole><<<1, kThreads, 0, s>>>(a);
  } else {
    Record* rec = static_cast<Record*>(workspace);
    mla_tables_plan_kernel<kWhole><<<1, kThreads, 0, s>>>(a, rec);
    const long long quads = ((long long)num_tokens + 3) / 4;
    if (quads > 0)
      mla_tables_fill_kernel<<<(unsigned)((quads + kFillThreads - 1) / kFillThreads), kFillThreads, 0, s>>>(a, rec);
  }
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

size_t mla_block_tables_workspace_bytes(int32_t batch, int32_t num_tokens) {
  set_error("%s", "");
  if (batch < 1 || num_tokens < 0) {
    set_error("mla_block_tables_workspace_bytes: batch must be >= 1 and num_tokens >= 0 (got %d, %d)", batch,
              num_tokens);
    return 0;
  }
  return small(batch, num_tokens) ? 0 : (size_t)batch * sizeof(Record);
}

int32_t mla_extend_block_tables(int32_t* block_table, const int32_t* cache_seqlens, const int32_t* new_lens,
                                const int32_t* free_pages, const int32_t* free_pos, int32_t* new_seqlens,
                                int32_t* new_free_pos, int32_t* slots, int32_t* positions, int32_t* cu_new,
                                void* workspace, size_t workspace_bytes, int32_t batch, int32_t max_pages,
                                int32_t page_size, int32_t num_pages, int32_t num_free, int32_t num_tokens,
                                int32_t q_len, void* stream) {
  const TablesArgs a{block_table, cache_seqlens, new_lens, free_pages, free_pos, new_seqlens, new_free_pos, slots,
                     positions, cu_new, batch, max_pages, page_size, num_pages, num_free, num_tokens, q_len};
  return extend<false>("mla_extend_block_tables", a, workspace, workspace_bytes, stream);
}

int32_t mla_extend_block_tables_whole(int32_t* block_table, const int32_t* cache_seqlens, const int32_t* new_lens,
                                      const int32_t* free_pages, const int32_t* free_pos, int32_t* new_seqlens,
                                      int32_t* new_free_pos, int32_t* slots, int32_t* positions, int32_t* cu_new,
                                      void* workspace, size_t workspace_bytes, int32_t batch, int32_t max_pages,
                                      int32_t page_size, int32_t num_pages, int32_t num_free, int32_t num_tokens,
                                      int32_t q_len, void* stream) {
  const char* fn = "mla_extend_block_tables_whole";
  if (q_len < 1) {
    set_error("%s: q_len must be >= 1, got %d", fn, q_len);
    return MLA_ERR_ARG;
  }
  const TablesArgs a{block_table, cache_seqlens, new_lens, free_pages, free_pos, new_seqlens, new_free_pos, slots,
                     positions, cu_new, batch, max_pages, page_size, num_pages, num_free, num_tokens, q_len};
  return extend<true>(fn, a, workspace, workspace_bytes, stream);
}

}  // extern "C"
