// Attention of packed query tokens over their request's keys: in a paged pool
// (chunks of new tokens and single tokens) or packed like the queries (whole
// prompts). The formulas and the rules of what a token sees are with
// jo_attention_varlen in joyomni_hip.h.

#include "jo_device.hpp"
#include "jo_host.hpp"

namespace jo {
namespace {

struct AttnArgs {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  int64_t q_ts, q_hs, o_ts, o_hs;    // strides in elements: token, head
  int64_t k_ps, k_ts, k_hs;          // page (paged), token, head
  int64_t v_ps, v_ts, v_hs;
  const int32_t* cu_q;               // [requests + 1]
  const int32_t* cu_k;               // [requests + 1] (packed keys)
  const int32_t* kv_lens;            // [requests] (paged)
  const int32_t* table;              // [requests, width] (paged)
  int64_t table_stride;
  int32_t q_tokens, kv_tokens, requests, width, num_pages;
  int32_t q_heads, kv_heads, group;  // group: query heads a key head
  int32_t capacity;                  // paged: keys that a table row can place
  FastDiv fd_page, fd_group;
  float scale_log2;                  // scale * log2(e): softmax in powers of two
  int32_t causal, fill_rest;
};

// A request's share of the packed arrays, with every bound clamped: what the
// length arrays hold is not trusted to lie inside the tensors.
struct Request {
  int32_t q0, nq;     // query tokens [q0, q0 + nq)
  int32_t k0, keys;   // keys with a place, and (packed) where they begin
  int32_t first_pos;  // position of the first query token: sees keys <= it (causal)
};

template <bool PAGED>
__device__ __forceinline__ Request request(const AttnArgs& a, int r) {
  Request x;
  x.q0 = min(max(a.cu_q[r], 0), a.q_tokens);
  x.nq = min(max(a.cu_q[r + 1], x.q0), a.q_tokens) - x.q0;
  int32_t len;
  if constexpr (PAGED) {
    len = max(a.kv_lens[r], 0);
    x.k0 = 0;
    x.keys = min(len, a.capacity);
  } else {
    x.k0 = min(max(a.cu_k[r], 0), a.kv_tokens);
    len = min(max(a.cu_k[r + 1], x.k0), a.kv_tokens) - x.k0;
    x.keys = len;
  }
  x.first_pos = len - x.nq;
  return x;
}

// Keys [0, n) that the i-th query token of the request may see.
__device__ __forceinline__ int32_t visible(const AttnArgs& a, const Request& x, int32_t i) {
  return a.causal ? max(0, min(x.keys, x.first_pos + i + 1)) : x.keys;
}

// The last r with cu_q[r] <= t (0 if none): the owner of token t, if it has one.
__device__ __forceinline__ int find_request(const AttnArgs& a, int32_t t) {
  int lo = 0, hi = a.requests;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (a.cu_q[mid] <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Element offset of key j's row in a page (K's or V's strides), or -1 if its
// table entry names no page.
__device__ __forceinline__ int32_t page_of(const AttnArgs& a, int r, uint32_t j) {
  const int32_t p = a.table[r * a.table_stride + fdiv(j, a.fd_page)];
  return p < a.num_pages ? p : -1;
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// ---------------------------------------------------------------------------
// One wave a query row, the whole formula in fp32: 64 keys at a time, a key a
// lane for the scores, then D / 64 elements a lane for the sum over v. Only
// keys that the row sees are read.
// ---------------------------------------------------------------------------
template <class Tag, int D, bool PAGED>
__device__ __forceinline__ void attend_row(const AttnArgs& a, int r, const Request& x, int head,
                                           int32_t i, int32_t k_begin, int32_t k_end, float& m_out,
                                           float& l_out, float (&o)[D / 64]) {
  const int lane = threadIdx.x % kWave;
  const int kv_head = fdiv(head, a.fd_group);
  const int64_t q_off = (x.q0 + i) * a.q_ts + head * a.q_hs;
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < D / 64; ++e) o[e] = 0.f;
  for (int32_t base = k_begin; base < k_end; base += kWave) {
    const int32_t j = base + lane;
    bool seen = j < k_end;
    int64_t k_off = 0, v_off = 0;
    if (seen) {
      if constexpr (PAGED) {
        const int32_t page = page_of(a, r, j);
        const uint32_t place = j - fdiv(j, a.fd_page) * a.fd_page.d;
        seen = page >= 0;
        k_off = page * a.k_ps + place * a.k_ts;
        v_off = page * a.v_ps + place * a.v_ts;
      } else {
        k_off = static_cast<int64_t>(x.k0 + j) * a.k_ts;
        v_off = static_cast<int64_t>(x.k0 + j) * a.v_ts;
      }
      k_off += kv_head * a.k_hs;
      v_off += kv_head * a.v_hs;
    }
    float s = -INFINITY;
    if (seen) {
      float dot = 0.f;
      for (int d = 0; d < D; d += 8) {
        const u32x4 qc = ld16(byte_off(a.q, (q_off + d) * Tag::kBytes));
        const u32x4 kc = ld16(byte_off(a.k, (k_off + d) * Tag::kBytes));
#pragma unroll
        for (int e = 0; e < 8; ++e) dot = fmaf(elem<Tag>(qc, e), elem<Tag>(kc, e), dot);
      }
      s = dot * a.scale_log2;
    }
    const float m_new = fmaxf(m, allreduce<64, OpMax>(s));
    const float m_use = m_new == -INFINITY ? 0.f : m_new;
    const float p = seen ? exp2_fast(s - m_use) : 0.f;
    const float fade = exp2_fast(m - m_use);
    l = l * fade + allreduce<64, OpSum>(p);
    m = m_new;
#pragma unroll
    for (int e = 0; e < D / 64; ++e) o[e] *= fade;
    for (int t = 0; t < kWave; ++t) {
      const float pt = __builtin_bit_cast(
          float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, p), t));
      if (pt == 0.f) continue;  // uniform; also every key that is not seen
      const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(v_off), t);
      const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(v_off >> 32), t);
      const int64_t vo = static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo);
#pragma unroll
      for (int e = 0; e < D / 64; ++e)
        o[e] = fmaf(pt, load_elem<Tag>(a.v, vo + e * 64 + lane), o[e]);
    }
  }
  m_out = m;
  l_out = l;
}

template <class Tag, int D, bool PAGED>
__global__ __launch_bounds__(kBlock) void attn_rows_kernel(const AttnArgs a) {
  const int lane = threadIdx.x % kWave;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * (kBlock / kWave) +
                     __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int32_t t = static_cast<int32_t>(id / a.q_heads);
  const int head = static_cast<int>(id - static_cast<int64_t>(t) * a.q_heads);
  if (t >= a.q_tokens) return;
  float o[D / 64] = {}, m, l = 0.f;
  bool owned = false;
  if (a.requests > 0) {
    const int r = find_request(a, t);
    const Request x = request<PAGED>(a, r);
    owned = t >= x.q0 && t < x.q0 + x.nq;
    if (owned)
      attend_row<Tag, D, PAGED>(a, r, x, head, t - x.q0, 0, visible(a, x, t - x.q0), m, l, o);
  }
  if (!owned && !a.fill_rest) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int64_t off = t * a.o_ts + head * a.o_hs;
#pragma unroll
  for (int e = 0; e < D / 64; ++e) store_elem<Tag>(a.out, off + e * 64 + lane, o[e] * inv);
}

template <class Tag, int D, bool PAGED>
int launch_attention(const AttnArgs& a, hipStream_t stream) {
  const int64_t waves = static_cast<int64_t>(a.q_tokens) * a.q_heads;
  hipLaunchKernelGGL((attn_rows_kernel<Tag, D, PAGED>), dim3(static_cast<unsigned>((waves + 3) / 4)),
                     dim3(kBlock), 0, stream, a);
  return launch_status(PAGED ? "attention_paged" : "attention_varlen");
}

template <bool PAGED>
int dispatch_attention(const AttnArgs& a, int64_t head_dim, int dtype, hipStream_t stream) {
  if (dtype == JO_DTYPE_BF16) {
    if (head_dim == 64) return launch_attention<BF16, 64, PAGED>(a, stream);
    if (head_dim == 128) return launch_attention<BF16, 128, PAGED>(a, stream);
    return launch_attention<BF16, 256, PAGED>(a, stream);
  }
  if (head_dim == 64) return launch_attention<F16, 64, PAGED>(a, stream);
  if (head_dim == 128) return launch_attention<F16, 128, PAGED>(a, stream);
  return launch_attention<F16, 256, PAGED>(a, stream);
}

// The arguments that both entry points share. Sets q/out/heads/scale fields of `a`.
int check_attention(const char* op, AttnArgs& a, const void* q, const void* k, const void* v,
                    void* out, int64_t q_tokens, int64_t requests, int64_t q_heads,
                    int64_t kv_heads, int64_t head_dim, const int32_t* cu_q, float scale,
                    int dtype) {
  JO_REQUIRE(dtype == JO_DTYPE_BF16 || dtype == JO_DTYPE_F16, "%s: bf16 or fp16 is needed", op);
  JO_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256, "%s: unsupported head_dim %lld",
             op, static_cast<long long>(head_dim));
  JO_REQUIRE(q_tokens >= 0 && requests >= 0 && q_heads > 0 && kv_heads > 0, "%s: bad shape", op);
  JO_REQUIRE(q_heads % kv_heads == 0, "%s: q_heads %lld is no multiple of kv_heads %lld", op,
             static_cast<long long>(q_heads), static_cast<long long>(kv_heads));
  // Rows (tokens x heads) are counted in 32 bits, with room for the last tiles.
  JO_REQUIRE(q_heads <= 65536 && q_tokens <= (INT32_MAX / 2) / q_heads && requests <= INT32_MAX / 2,
             "%s: shape too large", op);
  JO_REQUIRE(scale > 0.f && scale <= 1e30f, "%s: scale must be positive and finite", op);
  if (q_tokens == 0) return JO_OK;
  JO_REQUIRE(q && out && cu_q, "%s: null pointer", op);
  JO_REQUIRE(aligned(q, 16) && aligned(k, 16) && aligned(v, 16) && aligned(out, 16),
             "%s: tensors must be 16-byte aligned", op);
  JO_REQUIRE(a.q_ts >= 0 && a.q_hs >= 0 && a.k_ps >= 0 && a.k_ts >= 0 && a.k_hs >= 0 &&
                 a.v_ps >= 0 && a.v_ts >= 0 && a.v_hs >= 0 &&
                 (a.q_ts | a.q_hs | a.k_ps | a.k_ts | a.k_hs | a.v_ps | a.v_ts | a.v_hs | a.o_ts |
                  a.o_hs) % 8 == 0,
             "%s: strides must be multiples of 8 elements", op);
  JO_REQUIRE((q_tokens <= 1 || a.o_ts >= head_dim) && (q_heads <= 1 || a.o_hs >= head_dim),
             "%s: rows of out must not overlap", op);
  a.q = q;
  a.k = k;
  a.v = v;
  a.out = out;
  a.cu_q = cu_q;
  a.q_tokens = static_cast<int32_t>(q_tokens);
  a.requests = static_cast<int32_t>(requests);
  a.q_heads = static_cast<int32_t>(q_heads);
  a.kv_heads = static_cast<int32_t>(kv_heads);
  a.group = static_cast<int32_t>(q_heads / kv_heads);
  a.fd_group = make_fastdiv(static_cast<uint32_t>(a.group));
  a.scale_log2 = scale * 1.4426950408889634f;
  return JO_OK;
}

}  // namespace
}  // namespace jo

using namespace jo;

extern "C" int jo_attention_varlen(const void* q, const void* k, const void* v, void* out,
                                   int64_t q_tokens, int64_t kv_tokens, int64_t requests,
                                   int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                                   int64_t q_token_stride, int64_t q_head_stride,
                                   int64_t k_token_stride, int64_t k_head_stride,
                                   int64_t v_token_stride, int64_t v_head_stride,
                                   int64_t out_token_stride, int64_t out_head_stride,
                                   const int32_t* cu_q, const int32_t* cu_k, float scale,
                                   int causal, int fill_rest, int dtype, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
  const char* op = "attention_varlen";
  AttnArgs a{};
  a.q_ts = q_token_stride, a.q_hs = q_head_stride;
  a.k_ts = k_token_stride, a.k_hs = k_head_stride;
  a.v_ts = v_token_stride, a.v_hs = v_head_stride;
  a.o_ts = out_token_stride, a.o_hs = out_head_stride;
  JO_REQUIRE(kv_tokens >= 0 && kv_tokens <= INT32_MAX, "%s: bad shape", op);
  const int st = check_attention(op, a, q, k, v, out, q_tokens, requests, q_heads, kv_heads,
                                 head_dim, cu_q, scale, dtype);
  if (st != JO_OK || q_tokens == 0) return st;
  JO_REQUIRE(cu_k && (kv_tokens == 0 || (k && v)), "%s: null pointer", op);
  a.cu_k = cu_k;
  a.kv_tokens = static_cast<int32_t>(kv_tokens);
  a.causal = causal != 0;
  a.fill_rest = fill_rest != 0;
  return dispatch_attention<false>(a, head_dim, dtype, static_cast<hipStream_t>(stream));
}

extern "C" int jo_attention_paged(const void* q, const void* pages_k, const void* pages_v,
                                  void* out, int64_t q_tokens, int64_t requests, int64_t q_heads,
                                  int64_t kv_heads, int64_t head_dim, int64_t num_pages,
                                  int64_t page_size, int64_t q_token_stride, int64_t q_head_stride,
                                  int64_t k_page_stride, int64_t k_token_stride,
                                  int64_t k_head_stride, int64_t v_page_stride,
                                  int64_t v_token_stride, int64_t v_head_stride,
                                  int64_t out_token_stride, int64_t out_head_stride,
                                  const int32_t* block_table, int64_t table_stride,
                                  int64_t table_width, const int32_t* cu_q, const int32_t* kv_lens,
                                  float scale, int causal, int fill_rest, int dtype,
                                  void* workspace, int64_t workspace_bytes, void* stream) {
  const char* op = "attention_paged";
  AttnArgs a{};
  a.q_ts = q_token_stride, a.q_hs = q_head_stride;
  a.k_ps = k_page_stride, a.k_ts = k_token_stride, a.k_hs = k_head_stride;
  a.v_ps = v_page_stride, a.v_ts = v_token_stride, a.v_hs = v_head_stride;
  a.o_ts = out_token_stride, a.o_hs = out_head_stride;
  JO_REQUIRE(num_pages >= 0 && num_pages <= INT32_MAX && page_size >= 1 && page_size <= INT32_MAX &&
                 table_width >= 0 && table_width <= INT32_MAX,
             "%s: bad shape", op);
  const int st = check_attention(op, a, q, pages_k, pages_v, out, q_tokens, requests, q_heads,
                                 kv_heads, head_dim, cu_q, scale, dtype);
  if (st != JO_OK || q_tokens == 0) return st;
  JO_REQUIRE(requests <= 1 || table_stride >= table_width, "%s: bad table stride", op);
  JO_REQUIRE(requests == 0 || kv_lens, "%s: null pointer", op);
  a.kv_lens = kv_lens;
  a.table = block_table;
  a.table_stride = table_stride;
  a.width = static_cast<int32_t>(table_width);
  a.num_pages = static_cast<int32_t>(num_pages);
  a.fd_page = make_fastdiv(static_cast<uint32_t>(page_size));
  // No pages or no table: no key has a place.
  const int64_t places = num_pages == 0 ? 0 : table_width * page_size;
  JO_REQUIRE(places == 0 || (block_table && pages_k && pages_v), "%s: null pointer", op);
  a.capacity = static_cast<int32_t>(places > INT32_MAX ? INT32_MAX : places);
  a.causal = causal != 0;
  a.fill_rest = fill_rest != 0;
  return dispatch_attention<true>(a, head_dim, dtype, static_cast<hipStream_t>(stream));
}

extern "C" int64_t jo_attention_workspace_bytes(int64_t q_tokens, int64_t requests,
                                                int64_t q_heads, int64_t kv_heads,
                                                int64_t head_dim, int64_t kv_capacity) {
  return 0;
}
