// The tables of one serving step over a paged KV pool, from request lengths
// that live on the GPU: which pages the step's new tokens get, where each
// token's K and V go, and where each request's tokens and keys begin and end.
//
// With n_r = max(new_lens[r], 0), P = page_size, W = the table's width:
//   cu[0] = 0, cu[r+1] = min(cu[r] + n_r, max_tokens)
//   kv[r] = ctx[r] + cu[r+1] - cu[r]
//   have[r] = min(W, ceil(ctx[r] / P)), need[r] = min(W, ceil(kv[r] / P))
//   base[r] = sum over s < r of max(0, need[s] - have[s])
//   table[r, have[r] + j] = free[num_free - 1 - base[r] - j]   (j < need[r] - have[r])
//   slot[t] = table[r, p / P] * P + p % P,  p = ctx[r] + t - cu[r]
//
// Every workgroup scans all requests itself (two prefix sums, a request a
// thread and pass, the results in LDS) and then takes its share of the tokens and
// of the new table entries: a token's new page is worked out from the free list, not
// read back from the table, so workgroups wait for nobody and one launch does
// it all. The work is a few KB; what it costs is the chain of latencies
// (lengths, two scans, a search in LDS, a page id, the store): 32 single tokens
// 3.4 us, 500 requests of up to 128 tokens 5.4 us in the kernel.

#include "jo_device.hpp"
#include "jo_host.hpp"

namespace jo {
namespace {

constexpr int64_t kTabMaxRequests = 4096;  // ctx, cu and base in LDS: 12 bytes a request

struct TablesArgs {
  const int32_t* ctx;
  const int32_t* fresh;  // new tokens of each request
  int32_t* table;
  const int32_t* free_pages;
  const int32_t* num_free;
  int32_t* cu;
  int32_t* kv;
  int64_t* slots;
  int32_t* free_left;
  int64_t table_stride;
  int64_t num_pages;
  uint32_t requests, width, free_capacity, max_tokens;
  FastDiv fd_page;
};

// Sums saturate at 2^32 - 1 (for sums of non-negative numbers the order does
// not matter): lengths past any limit give "no room", never a wrapped sum.
__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) {
  return __builtin_elementwise_add_sat(a, b);
}

// Inclusive prefix sum over the wave, with DPP: shifts within rows of 16 lanes,
// then the rows' totals handed on.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t scan_step(uint32_t v) {
  return add_sat(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL,
                                                                      ROWS, 0xf, false)));
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
  v = scan_step<0x111, 0xf>(v);  // row_shr:1
  v = scan_step<0x112, 0xf>(v);  // row_shr:2
  v = scan_step<0x114, 0xf>(v);  // row_shr:4
  v = scan_step<0x118, 0xf>(v);  // row_shr:8
  v = scan_step<0x142, 0xa>(v);  // row_bcast:15 into rows 1 and 3
  return scan_step<0x143, 0xc>(v);  // row_bcast:31 into rows 2 and 3
}

// Prefix sum over the workgroup's threads (this thread's value left out);
// `total` gets the sum.
template <int WAVES>
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* wave_sums, uint32_t& total) {
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const uint32_t s = wave_scan(v);
  const uint32_t up = __shfl_up(s, 1);
  if (lane == kWave - 1) wave_sums[wave] = s;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    const uint32_t x = wave_sums[w];
    if (w < wave) before = add_sat(before, x);
    all = add_sat(all, x);
  }
  __syncthreads();
  total = all;
  return add_sat(before, lane == 0 ? 0 : up);
}

__device__ __forceinline__ uint32_t pages_of(uint32_t tokens, const TablesArgs& a) {
  // ceil(tokens / P) without the overflow of tokens + P - 1
  const uint32_t p = tokens == 0 ? 0 : fdiv(tokens - 1, a.fd_page) + 1;
  return min(p, a.width);
}

// The page that the list holds for the i-th new page of the step, -1 if it
// holds none there or names none.
__device__ __forceinline__ int32_t take_page(const TablesArgs& a, int64_t available, uint64_t i) {
  const int64_t at = available - 1 - static_cast<int64_t>(i);
  if (at < 0) return -1;
  const int32_t id = a.free_pages[at];
  return id >= 0 && id < a.num_pages ? id : -1;
}

// The last r in [0, n) with key[r] <= x, where key[0] <= x.
__device__ __forceinline__ uint32_t last_not_above(const uint32_t* key, uint32_t n, uint32_t x) {
  uint32_t lo = 0, hi = n;
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (key[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

template <int THREADS>
__global__ __launch_bounds__(THREADS) void paged_tables_kernel(const TablesArgs a) {
  extern __shared__ uint32_t smem[];  // cu [requests + 1], base [requests + 1], ctx [requests]
  __shared__ uint32_t wave_sums[THREADS / kWave];
  uint32_t* cu = smem;
  uint32_t* base = cu + a.requests + 1;
  uint32_t* ctx_of = base + a.requests + 1;
  const uint32_t tid = threadIdx.x;
  const bool first = blockIdx.x == 0;
  const int64_t available = min(max(a.num_free[0], 0), static_cast<int32_t>(a.free_capacity));

  uint32_t tokens = 0, pages = 0;  // of the requests before this pass
  for (uint32_t r0 = 0; r0 < a.requests; r0 += THREADS) {
    const uint32_t r = r0 + tid;
    uint32_t ctx = 0, n = 0;
    if (r < a.requests) {
      ctx = max(a.ctx[r], 0);
      n = max(a.fresh[r], 0);
    }
    uint32_t sum;
    const uint32_t at =
        min(add_sat(tokens, block_scan<THREADS / kWave>(n, wave_sums, sum)), a.max_tokens);
    const uint32_t end = min(add_sat(at, n), a.max_tokens);
    tokens = add_sat(tokens, sum);
    const uint32_t kv = ctx + (end - at);  // below 2^32: both are below 2^31
    const uint32_t have = pages_of(ctx, a), need = pages_of(kv, a);
    const uint32_t mine = block_scan<THREADS / kWave>(need - have, wave_sums, sum);
    if (r < a.requests) {
      ctx_of[r] = ctx;
      cu[r] = at;
      base[r] = add_sat(pages, mine);
      if (first) {
        a.cu[r] = static_cast<int32_t>(at);
        a.kv[r] = static_cast<int32_t>(min(kv, static_cast<uint32_t>(INT32_MAX)));
      }
    }
    pages = add_sat(pages, sum);
  }
  tokens = min(tokens, a.max_tokens);
  if (tid == 0) {
    cu[a.requests] = tokens;
    base[a.requests] = pages;
    if (first) {
      a.cu[a.requests] = static_cast<int32_t>(tokens);
      const int64_t left = available - static_cast<int64_t>(pages);
      a.free_left[0] = static_cast<int32_t>(max(left, static_cast<int64_t>(INT32_MIN)));
    }
  }
  __syncthreads();

  const uint64_t step = static_cast<uint64_t>(gridDim.x) * THREADS;
  const uint64_t me = static_cast<uint64_t>(blockIdx.x) * THREADS + tid;
  for (uint64_t t = me; t < a.max_tokens; t += step) {
    int64_t slot = -1;
    if (t < tokens) {
      const uint32_t r = last_not_above(cu, a.requests, static_cast<uint32_t>(t));
      const uint32_t ctx = ctx_of[r];
      const uint32_t pos = ctx + (static_cast<uint32_t>(t) - cu[r]);
      const uint32_t col = fdiv(pos, a.fd_page);
      if (col < a.width) {
        const uint32_t have = pages_of(ctx, a);
        int32_t page;
        if (col < have) {  // the last page of the cached tokens
          page = a.table[static_cast<int64_t>(r) * a.table_stride + col];
          if (page >= a.num_pages) page = -1;
        } else {
          page = take_page(a, available, static_cast<uint64_t>(base[r]) + (col - have));
        }
        if (page >= 0) slot = static_cast<int64_t>(page) * a.fd_page.d + (pos - col * a.fd_page.d);
      }
    }
    a.slots[t] = slot;
  }
  for (uint64_t i = me; i < pages; i += step) {
    const uint32_t r = last_not_above(base, a.requests, static_cast<uint32_t>(i));
    const uint32_t j = static_cast<uint32_t>(i) - base[r];
    const uint32_t have = pages_of(ctx_of[r], a);
    // (Bounded by the width also where a sum of pages has saturated.)
    if (j < a.width - have)
      a.table[static_cast<int64_t>(r) * a.table_stride + have + j] = take_page(a, available, i);
  }
}

}  // namespace
}  // namespace jo

using namespace jo;

extern "C" int jo_paged_tables(const int32_t* ctx_lens, const int32_t* new_lens, int64_t requests,
                               int32_t* block_table, int64_t table_stride, int64_t table_width,
                               const int32_t* free_pages, int64_t free_capacity,
                               const int32_t* num_free, int64_t page_size, int64_t num_pages,
                               int64_t max_tokens, int32_t* cu_q, int32_t* kv_lens, int64_t* slots,
                               int32_t* free_left, void* stream) {
  const char* op = "paged_tables";
  JO_REQUIRE(requests >= 0 && table_width >= 0 && free_capacity >= 0 && num_pages >= 0 &&
                 max_tokens >= 0,
             "%s: bad shape", op);
  JO_REQUIRE(requests <= kTabMaxRequests, "%s: too many requests (%lld, at most %lld)", op,
             static_cast<long long>(requests), static_cast<long long>(kTabMaxRequests));
  JO_REQUIRE(page_size >= 1 && page_size <= INT32_MAX, "%s: bad page_size", op);
  JO_REQUIRE(table_width <= INT32_MAX && free_capacity <= INT32_MAX && num_pages <= INT32_MAX &&
                 max_tokens <= INT32_MAX,
             "%s: shape too large", op);
  JO_REQUIRE(requests <= 1 || (table_stride >= table_width && table_stride <= int64_t{1} << 40),
             "%s: bad table stride", op);
  JO_REQUIRE(cu_q && free_left && num_free, "%s: null pointer", op);
  JO_REQUIRE(free_left != num_free, "%s: free_left must not be num_free itself", op);
  JO_REQUIRE(requests == 0 || (ctx_lens && new_lens && kv_lens), "%s: null pointer", op);
  JO_REQUIRE(requests == 0 || table_width == 0 || block_table, "%s: null pointer", op);
  JO_REQUIRE((max_tokens == 0 || slots) && (free_capacity == 0 || free_pages), "%s: null pointer",
             op);
  // Each workgroup reads all lengths and its part of the list, and what one has
  // written another may not have read yet: no output lies in an input, not even
  // kv_lens in ctx_lens.
  const struct {
    const void* p;
    int64_t bytes;
  } inputs[] = {{ctx_lens, 4 * requests}, {new_lens, 4 * requests},
                {free_pages, 4 * free_capacity}, {num_free, 4}},
    outputs[] = {{cu_q, 4 * (requests + 1)}, {kv_lens, 4 * requests}, {slots, 8 * max_tokens},
                 {free_left, 4}, {block_table, requests == 0 || table_width == 0 ? 0
                                  : 4 * ((requests - 1) * table_stride + table_width)}};
  for (const auto& o : outputs)
    for (const auto& i : inputs) {
      const uintptr_t x = reinterpret_cast<uintptr_t>(o.p), y = reinterpret_cast<uintptr_t>(i.p);
      JO_REQUIRE(o.bytes == 0 || i.bytes == 0 || x + o.bytes <= y || y + i.bytes <= x,
                 "%s: an output overlaps an input", op);
    }
  TablesArgs a{ctx_lens, new_lens, block_table, free_pages, num_free, cu_q, kv_lens, slots,
               free_left, table_stride, num_pages, static_cast<uint32_t>(requests),
               static_cast<uint32_t>(table_width), static_cast<uint32_t>(free_capacity),
               static_cast<uint32_t>(max_tokens), make_fastdiv(static_cast<uint32_t>(page_size))};
  // Few requests: four waves a workgroup, whose barriers cost less (32 requests in
  // a replayed graph: 3.6 us a call, with 16 waves 4.8). Up to 64 workgroups of a
  // thread a token; beyond them a thread takes more tokens.
  const int64_t threads = requests <= 256 ? 256 : 1024;
  const int64_t want = (max_tokens + threads - 1) / threads;
  const dim3 grid(static_cast<unsigned>(want < 1 ? 1 : want > 64 ? 64 : want));
  const size_t lds = (3 * static_cast<size_t>(requests) + 2) * sizeof(uint32_t);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (threads == 256)
    hipLaunchKernelGGL((paged_tables_kernel<256>), grid, dim3(256), lds, st, a);
  else
    hipLaunchKernelGGL((paged_tables_kernel<1024>), grid, dim3(1024), lds, st, a);
  return launch_status(op);
}
