// Attention of packed query tokens over their request's keys: in a paged pool
// (chunks of new tokens and single tokens) or packed like the queries (whole
// prompts). The formulas and the rules of what a token sees are with
// jo_attention_varlen in joyomni_hip.h.

#include <type_traits>

#include "jo_device.hpp"
#include "jo_host.hpp"

namespace jo {
namespace {

// A lambda that is never a call: what it captures stays in registers.
#define JO_INLINE __attribute__((always_inline))

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
  uint32_t k_ps16, k_ts16, v_ps16, v_ts16;  // strides in units of 16 bytes
  uint32_t items;                    // work items launched, a key head each
  uint32_t split_target;             // 0: keys are not split
  FastDiv fd_target;                 // its division
  uint32_t tail_splits, tail_most;   // the last round's splits (1: none), and of how many tiles
  FastDiv fd_round;                  // division by a round's tiles
  float* ws;                         // partial results of split items
};

// Where keys are: packed one behind the other; in pages of a multiple of 16
// keys (the 16 rows of keys 16 i .. 16 i + 15 are then evenly apart, and one
// address serves them); in pages of any other size (an address a lane; two frames
// over three cached ones: pages of 48, 64 or 80 keys 455 us, of 56 or 60 485, of 52
// 507; an address a load, where pages allow it, was within 1% of that).
enum class Keys { kPacked, kPages16, kPages };

// A request's share of the packed arrays, with every bound clamped: what the
// length arrays hold is not trusted to lie inside the tensors.
struct Request {
  int32_t q0, nq;     // query tokens [q0, q0 + nq)
  int32_t k0, keys;   // keys with a place, and (packed) where they begin
  int32_t first_pos;  // position of the first query token: sees keys <= it (causal)
};

struct RawRequest {
  int32_t q0, q1, k0, k1;  // k1: paged, the number of keys
};
template <bool PAGED>
__device__ __forceinline__ RawRequest raw_request(const AttnArgs& a, int r) {
  return RawRequest{a.cu_q[r], a.cu_q[r + 1], PAGED ? 0 : a.cu_k[r],
                    PAGED ? a.kv_lens[r] : a.cu_k[r + 1]};
}
template <bool PAGED>
__device__ __forceinline__ Request request(const AttnArgs& a, const RawRequest& w) {
  Request x;
  x.q0 = min(max(w.q0, 0), a.q_tokens);
  x.nq = min(max(w.q1, x.q0), a.q_tokens) - x.q0;
  int32_t len;
  if constexpr (PAGED) {
    len = max(w.k1, 0);
    x.k0 = 0;
    x.keys = min(len, a.capacity);
  } else {
    x.k0 = min(max(w.k0, 0), a.kv_tokens);
    len = min(max(w.k1, x.k0), a.kv_tokens) - x.k0;
    x.keys = len;
  }
  x.first_pos = len - x.nq;
  return x;
}

// Keys [0, n) that the i-th query token of the request may see.
__device__ __forceinline__ int32_t visible(const AttnArgs& a, const Request& x, int32_t i) {
  return a.causal ? max(0, min(x.keys, x.first_pos + i + 1)) : x.keys;
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

// ---------------------------------------------------------------------------
// Work items. A request's rows are its (token, head of the group) pairs, token
// first: the query heads that share a key head share its K and V tiles. A tile
// is ROWS consecutive rows of one request and one key head; where there are few
// tiles, or requests of very different lengths, a tile's keys are split into
// ranges of `chunk` key blocks of kKeyBlock, a workgroup each, whose partial
// results a second kernel joins.
//
// No host knows the lengths: a workgroup finds its own item from its index.
// With up to kPlanRequests requests each wave scans their lengths (four a lane):
//   cost = sum over requests of tiles x key blocks,
//   chunk = max(kMinChunk, floor(cost / split_target) + 1),
//   splits = ceil(key blocks / chunk), items = tiles x splits, in request order,
// so there are at most tiles + split_target items, which is what is launched.
// With up to 64 requests the longest items go first, in 16 levels of length: a
// long one that starts last is what all others wait for (eight prompts of 200 to
// 3500 tokens 57.6 -> 49.3 us, 20 requests of chunks and single tokens 93 -> 83, 64
// single tokens 148 -> 141). An item's level and place in it come of one count of
// the items in the levels before for every halving of 16, which costs a wave about
// a microsecond and is left out where the order cannot matter.
// Or (tail_splits > 1) all tiles of the rounds that fill the GPU are whole, and
// only those of the last round, `tail` of them, are split:
//   tail = tiles mod round, if that is no more than tail_most (else nothing is),
//   splits = min(tail_splits, key blocks / kMinChunk), for the last `tail` tiles.
// With more requests keys are not split, and request r's tiles begin at index
// floor(cu_q[r] x group / ROWS) + r, which leaves each room for its tiles.
// ---------------------------------------------------------------------------
constexpr int kKeyBlock = 64;
constexpr int kTileRows = 128;  // of attn_tiles_kernel
constexpr int kPlanPerLane = 4;
constexpr int kPlanRequests = kPlanPerLane * kWave;
constexpr int kMinChunk = 4;  // key blocks a split
constexpr int64_t kMaxKeys = INT32_MAX - 4096;  // room for sums of a key index and a block

struct Item {
  Request x;
  int r;               // -1: no work
  int tile;            // rows [tile * ROWS, ...) of the request
  int split, splits;   // this range of the keys, and how many there are
  int chunk;           // key blocks a range
  int index;           // a partial result's place: items in request order, from the first that is
                       // split (in the joining kernel: of the tile's first)
};

// Inclusive prefix sum over the wave (saturating), with DPP: shifts within rows
// of 16 lanes, then the rows' totals handed on.
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
#define JO_SCAN_STEP(ctrl, rows) \
  v = __builtin_elementwise_add_sat( \
      v, static_cast<uint32_t>( \
             __builtin_amdgcn_update_dpp(0, static_cast<int>(v), ctrl, rows, 0xf, false)))
  JO_SCAN_STEP(0x111, 0xf);  // row_shr:1
  JO_SCAN_STEP(0x112, 0xf);  // row_shr:2
  JO_SCAN_STEP(0x114, 0xf);  // row_shr:4
  JO_SCAN_STEP(0x118, 0xf);  // row_shr:8
  JO_SCAN_STEP(0x142, 0xa);  // row_bcast:15 into rows 1 and 3
  JO_SCAN_STEP(0x143, 0xc);  // row_bcast:31 into rows 2 and 3
#undef JO_SCAN_STEP
  return v;
}

__device__ __forceinline__ uint32_t wave_sum(uint32_t v) {
  return __builtin_amdgcn_readlane(wave_scan(v), kWave - 1);
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#define JO_MAX_STEP(ctrl, rows) \
  v = max(v, static_cast<uint32_t>( \
                 __builtin_amdgcn_update_dpp(0, static_cast<int>(v), ctrl, rows, 0xf, false)))
  JO_MAX_STEP(0x111, 0xf);
  JO_MAX_STEP(0x112, 0xf);
  JO_MAX_STEP(0x114, 0xf);
  JO_MAX_STEP(0x118, 0xf);
  JO_MAX_STEP(0x142, 0xa);
  JO_MAX_STEP(0x143, 0xc);
#undef JO_MAX_STEP
  return __builtin_amdgcn_readlane(v, kWave - 1);
}

constexpr uint32_t kNoSplit = 0x40000000u;  // beyond any number of key blocks

// find_item with E requests a lane.
template <int ROWS, bool PAGED, bool TILES, int E>
__device__ __forceinline__ Item plan_item(const AttnArgs& a, uint32_t id) {
  const int lane = threadIdx.x % kWave;
  Item it;
  it.r = -1;
  RawRequest raw[E];
#pragma unroll
  for (int e = 0; e < E; ++e) raw[e] = raw_request<PAGED>(a, min(lane * E + e, a.requests - 1));
  Request x[E];
  uint32_t tiles[E], blocks[E], cost = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    x[e] = request<PAGED>(a, raw[e]);
    tiles[e] = (static_cast<uint32_t>(x[e].nq) * a.group + ROWS - 1) / ROWS;
    if (lane * E + e >= a.requests) tiles[e] = 0;
    blocks[e] = (static_cast<uint32_t>(x[e].keys) + kKeyBlock - 1) / kKeyBlock;
    const uint64_t c = static_cast<uint64_t>(tiles[e]) * blocks[e];
    cost = __builtin_elementwise_add_sat(cost, static_cast<uint32_t>(min(c, uint64_t{UINT32_MAX})));
  }
  uint32_t chunk = kNoSplit;
  if (a.split_target > 0) {
    const uint32_t total = __builtin_amdgcn_readlane(wave_scan(cost), kWave - 1);
    chunk = max(static_cast<uint32_t>(kMinChunk), fdiv(total, a.fd_target) + 1);
    if (total == UINT32_MAX) chunk = kNoSplit;  // a saturated total says too little
  }
  uint32_t splits[E], whole[E], items = 0, units = 0;
  uint32_t full = 0;  // tiles of the rounds before the last, which is split
  if (a.tail_splits > 1) {
    uint32_t mine = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) mine += tiles[e];
    const uint32_t end = wave_scan(mine);
    const uint32_t total = __builtin_amdgcn_readlane(end, kWave - 1);
    const uint32_t tail = total - fdiv(total, a.fd_round) * a.fd_round.d;
    full = tail <= a.tail_most ? total - tail : total;
    uint32_t at = end - mine;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      whole[e] = min(tiles[e], full - min(full, at));
      at += tiles[e];
    }
  }
  auto units_of = [&](int e) JO_INLINE {
    return TILES ? (splits[e] > 1 ? tiles[e] - whole[e] : 0)
                 : whole[e] + (tiles[e] - whole[e]) * splits[e];
  };
  // (One division of 32 bits a request; in fp32 first, blocks and chunk being
  // below 2^24 in any pool that exists, would not hold for all inputs.)
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (a.tail_splits > 1) {
      splits[e] = max(1u, min(a.tail_splits, blocks[e] / kMinChunk));
    } else {
      splits[e] = blocks[e] <= chunk ? 1u : (blocks[e] - 1) / chunk + 1;
      whole[e] = 0;
    }
    items += whole[e] + (tiles[e] - whole[e]) * splits[e];
    units += units_of(e);
  }
  const uint32_t unit_end = wave_scan(units);
  const uint32_t item_end = TILES ? wave_scan(items) : unit_end;
  // The lane whose request it is; in that lane: the index within the lane's.
  uint64_t past = __ballot(unit_end > id);
  uint32_t local = id - (unit_end - units);
  if constexpr (E == 1 && !TILES) {
    const uint32_t parts = (blocks[0] + splits[0] - 1) / splits[0];  // key blocks of a range
    const uint32_t uncut = splits[0] > 1 ? whole[0] : items, cut = items - uncut;
    const uint32_t longest = uncut > 0 ? blocks[0] : cut > 0 ? parts : 0;
    const uint32_t top = wave_max(longest);
    // Items in 16 levels by length: level l has those longer than (15 - l) / 16 of
    // the longest. In order as they are: if all are of the first level, if they all
    // run at once, or of one request.
    const bool shorter = longest + top / 16 < top || (a.causal && uncut > 1);
    if (a.items > a.fd_round.d && a.requests > 1 && __ballot(items > 0 && shorter) != 0) {
      // Of uncut tiles with a causal mask each sees fewer keys than the one behind it,
      // by a tile's share of a block.
      const float step = a.causal ? static_cast<float>(a.group) * kKeyBlock / ROWS : 1e9f;
      const float most = static_cast<float>(uncut);
      auto up_to = [&](uint32_t level) JO_INLINE -> uint32_t {  // items of the levels below
        const uint32_t x = (top >> 4) * (16 - level) + ((top & 15) * (16 - level) >> 4);
        const float n = fminf(static_cast<float>(blocks[0] - x) * step, most);
        const uint32_t u = x < blocks[0] ? min(uncut, static_cast<uint32_t>(n) + 1) : 0u;
        const uint32_t c = x < parts ? cut : 0u;
        return level == 0 ? 0u : level == 16 ? items : u + c;
      };
      uint32_t lo = 0, below = 0;
#pragma unroll
      for (uint32_t half = 8; half > 0; half /= 2) {
        const uint32_t n = wave_sum(up_to(lo + half));
        if (n <= id) lo += half, below = n;
      }
      const uint32_t before = up_to(lo), mine = up_to(lo + 1) - before;
      const uint32_t end = wave_scan(mine);
      past = __ballot(end > id - below);
      local = before + (id - below) - (end - mine);
    }
  }
  if (past == 0) return it;
  const int owner = __builtin_ctzll(past);
  uint32_t first = item_end - items;
  uint32_t e_found = 0, n_splits = splits[0], n_tiles = tiles[0], n_blocks = blocks[0],
           n_whole = whole[0];
  Request y = x[0];
  bool found = local < units_of(0);
#pragma unroll
  for (int e = 1; e < E; ++e) {
    if (!found) {
      local -= units_of(e - 1);
      first += whole[e - 1] + (tiles[e - 1] - whole[e - 1]) * splits[e - 1];
      e_found = e, n_splits = splits[e], n_tiles = tiles[e], n_blocks = blocks[e];
      n_whole = whole[e];
      y = x[e];
      found = local < units_of(e);
    }
  }
  auto of_owner = [&](auto v) {
    return static_cast<decltype(v)>(__builtin_amdgcn_readlane(static_cast<int>(v), owner));
  };
  local = of_owner(local);
  first = of_owner(first);
  n_splits = of_owner(n_splits);
  n_tiles = of_owner(n_tiles);
  n_blocks = of_owner(n_blocks);
  it.x = Request{of_owner(y.q0), of_owner(y.nq), of_owner(y.k0), of_owner(y.keys),
                 of_owner(y.first_pos)};
  it.r = owner * E + of_owner(e_found);
  n_whole = of_owner(n_whole);
  const bool one = n_splits == 1 || (!TILES && local < n_whole);
  it.splits = one ? 1 : n_splits;
  // The ranges of a request are of one length, to a block.
  it.chunk = one ? kNoSplit : (n_blocks - 1) / n_splits + 1;
  const uint32_t rest = TILES ? local : local - n_whole;
  const uint32_t t = one ? local : n_whole + (TILES ? rest : rest / n_splits);
  it.split = one || TILES ? 0 : rest - (t - n_whole) * n_splits;
  // The last tile first: with a causal mask it sees the most keys.
  it.tile = n_tiles - 1 - t;
  it.index = first + (TILES ? n_whole + rest * n_splits : local) - full;
  // (More items than were launched: requests that overlap.)
  if (!one && static_cast<uint32_t>(it.index) >= a.items) it.r = -1;
  return it;
}

// The item of index id (TILES: the split tile of index id, all its splits).
template <int ROWS, bool PAGED, bool TILES>
__device__ __forceinline__ Item find_item(const AttnArgs& a, uint32_t id) {
  if (a.requests <= kWave) return plan_item<ROWS, PAGED, TILES, 1>(a, id);
  if (a.requests <= kPlanRequests) return plan_item<ROWS, PAGED, TILES, kPlanPerLane>(a, id);
  const int lane = threadIdx.x % kWave;
  Item it;
  it.r = -1;
  // 64 ways at a time: the last request whose first index is not above id.
  int lo = 0, n = a.requests;
  while (n > 1) {
    const int step = (n + kWave - 1) / kWave;
    const int r = lo + lane * step;
    bool below = false;
    if (lane * step < n) {
      const uint32_t q0 = min(max(a.cu_q[r], 0), a.q_tokens);
      below = q0 * a.group / ROWS + r <= id;
    }
    const uint64_t mask = __ballot(below);
    const int at = mask == 0 ? 0 : 63 - __builtin_clzll(mask);
    lo += at * step;
    n = min(step, n - at * step);
  }
  it.x = request<PAGED>(a, raw_request<PAGED>(a, lo));
  const uint32_t rows = static_cast<uint32_t>(it.x.nq) * a.group;
  const uint32_t begin = static_cast<uint32_t>(it.x.q0) * a.group / ROWS + lo;
  const uint32_t tiles = (rows + ROWS - 1) / ROWS;
  if (id < begin || id - begin >= tiles) return it;
  it.r = lo;
  it.splits = 1;
  it.split = 0;
  it.chunk = kNoSplit;
  it.index = id;
  it.tile = tiles - 1 - (id - begin);
  return it;
}

// Zeros for the tokens behind the last request, by the workgroups behind the
// items' (part `part` of `parts`).
template <class Tag, int D>
__device__ __forceinline__ void fill_rest(const AttnArgs& a, uint32_t part, uint32_t parts) {
  const int32_t from = a.requests > 0 ? min(max(a.cu_q[a.requests], 0), a.q_tokens) : 0;
  constexpr uint32_t C = D / 8;
  const int64_t pieces = static_cast<int64_t>(a.q_tokens - from) * a.q_heads * C;
  for (int64_t i = static_cast<int64_t>(part) * blockDim.x + threadIdx.x; i < pieces;
       i += static_cast<int64_t>(parts) * blockDim.x) {
    const int64_t row = i / C;
    const int64_t t = row / a.q_heads, h = row - t * a.q_heads;
    st16(byte_off(a.out, ((from + t) * a.o_ts + h * a.o_hs + (i - row * C) * 8) * Tag::kBytes),
         u32x4{0, 0, 0, 0});
  }
}

// ---------------------------------------------------------------------------
// Matrix-core building blocks.
// ---------------------------------------------------------------------------
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

template <class Tag>
__device__ __forceinline__ f32x16 mfma32(const u32x4& a, const u32x4& b, const f32x16& c) {
  if constexpr (std::is_same<Tag, BF16>::value)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <class Tag>
__device__ __forceinline__ f32x4 mfma16(const u32x4& a, const u32x4& b, const f32x4& c) {
  if constexpr (std::is_same<Tag, BF16>::value)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <class Tag>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same<Tag, BF16>::value) return pack_bf16x2(a, b);
  else return pack_f16x2(a, b);
}

// An LDS address held in 32 bits, as a pointer.
#define JO_LDS(type, addr) \
  ((__attribute__((address_space(3))) type*)(static_cast<uintptr_t>(addr)))

__device__ __forceinline__ uint32_t lds_address(char* shared) {
  return static_cast<uint32_t>(
      reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)shared));
}

__device__ __forceinline__ u32x4 lds_read16(uint32_t addr) { return *JO_LDS(u32x4, addr); }

// Two transposing reads: within each 16 lanes, lane i names four consecutive
// elements of row i / 4 and gets column i of the 4 x 16 block: four rows of its
// own column. Rows here are keys, columns places of head_dim.
__device__ __forceinline__ u32x4 lds_read_tr(uint32_t addr0, uint32_t addr1) {
  const u32x2 a =
      __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(JO_LDS(i16x4, addr0)));
  const u32x2 b =
      __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(JO_LDS(i16x4, addr1)));
  return u32x4{a.x, a.y, b.x, b.y};
}

// s_waitcnt limiting only the vector-memory counter to n (n < 64); only the LDS
// counter to 0.
#define JO_WAIT_VM(n) __builtin_amdgcn_s_waitcnt(0x0F70 | ((n) & 15) | (((n) >> 4) << 14))
#define JO_WAIT_LDS0() __builtin_amdgcn_s_waitcnt(0xC07F)
// Keeps memory accesses on their side of it (the compiler does not know what the
// waits above wait for).
#define JO_KEEP_ORDER() asm volatile("" ::: "memory")

// A key row of D elements is D / 8 chunks of 16 bytes; chunk c of row r of a
// tile in LDS sits at chunk position c ^ swz(r). The 32 banks of 8 bytes hold
// 16 chunks: K reads take the same chunk of 16 consecutive rows, which swz_k
// sends to 16 different ones; V's transposing reads take four (32-row tiles) or
// two (16-row tiles) neighbouring chunks of 8 or 16 consecutive rows, which
// swz_v32 / swz_k spread evenly.
template <int D>
__device__ __forceinline__ constexpr int swz_k(int r) {
  return D == 64 ? (r >> 1) & 7 : r & 15;
}
template <int D>
__device__ __forceinline__ constexpr int swz_v32(int r) {
  return D == 64 ? ((r >> 1) & 1) << 2 | ((r >> 2) & 3) : (r & 3) << 2 | ((r >> 2) & 3);
}

// Where the rows of a block of keys lie: the lane's key (base + lane, cut to
// the range's last) as offsets of 16 bytes into K and V, and which keys are there.
struct KeyRows {
  uint32_t k16, v16;
  uint64_t there;  // wave-uniform, bit i: key base + i is in the range and has a page
};

// The first half of key_rows: the page id load, so that it can run ahead.
template <bool PAGED>
__device__ __forceinline__ int32_t key_page(const AttnArgs& a, int r, int32_t base, int32_t end) {
  if constexpr (PAGED) {
    const int32_t j = min(base + static_cast<int32_t>(threadIdx.x % kWave), end - 1);
    return a.table[r * a.table_stride + fdiv(j, a.fd_page)];
  }
  return 0;
}
template <bool PAGED>
__device__ __forceinline__ KeyRows key_rows(const AttnArgs& a, const Request& x, int32_t page,
                                            int32_t base, int32_t end) {
  const int lane = threadIdx.x % kWave;
  const int32_t j = min(base + lane, end - 1);
  KeyRows k;
  bool there = base + lane < end;
  if constexpr (PAGED) {
    const uint32_t place = j - fdiv(j, a.fd_page) * a.fd_page.d;
    const bool has = page >= 0 && page < a.num_pages;
    there = there && has;
    const uint32_t p = has ? page : 0;  // keys without a page read page 0: never used
    k.k16 = p * a.k_ps16 + place * a.k_ts16;
    k.v16 = p * a.v_ps16 + place * a.v_ts16;
  } else {
    k.k16 = static_cast<uint32_t>(x.k0 + j) * a.k_ts16;
    k.v16 = static_cast<uint32_t>(x.k0 + j) * a.v_ts16;
  }
  k.there = __ballot(there);
  return k;
}

// 16 bytes a lane from global memory to LDS at the wave-uniform address `lds` on
// (lane i's at lds + 16 i). In assembly because the compiler, which cannot tell
// the two LDS buffers apart, would wait for the block being loaded before the
// transposing reads of the other one; the waits are where the blocks are used.
// (Of its own loads it then knows too few to be behind them, and waits longer
// than it must, never shorter.) m0, which no compiled code here uses otherwise,
// is set by every load for itself.
__device__ __forceinline__ void load_to_lds(const char* src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
               :
               : "v"(src), "s"(__builtin_amdgcn_readfirstlane(lds))
               : "memory");
}

// A wave-uniform address in scalar registers.
__device__ __forceinline__ const char* uniform(const char* p) {
  const uint64_t v = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<int>(v));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<int>(v >> 32));
  return reinterpret_cast<const char*>(static_cast<uint64_t>(hi) << 32 | lo);
}

// The same from a wave-uniform address and a 32-bit offset a lane.
__device__ __forceinline__ void load_to_lds(const char* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
               :
               : "v"(off), "s"(uniform(base)), "s"(__builtin_amdgcn_readfirstlane(lds))
               : "memory");
}

// Direct global -> LDS loads of ROWS key rows, 16 bytes a lane, written in row
// order from lds_base on: load i of the COUNT that this wave makes fills rows
// first_row + i * (rows a load). SRC: the lanes whose offsets these are.
template <int D, int COUNT, bool V32>
__device__ __forceinline__ void load_rows(const char* base, uint32_t off16, uint32_t lds_base,
                                          int first_row, int lane) {
  constexpr int C = D / 8, PER = kWave / C;  // chunks a row, rows a load
#pragma unroll
  for (int i = 0; i < COUNT; ++i) {
    const int row = first_row + i * PER + lane / C;
    const int sw = V32 ? swz_v32<D>(row) : swz_k<D>(row);
    const uint32_t off = __shfl(off16, row) + ((lane % C) ^ sw);
    load_to_lds(base + (static_cast<uint64_t>(off) << 4),
                lds_base + static_cast<uint32_t>((first_row + i * PER) * D * 2));
  }
}

// Rows whose result came out not finite are worked out again, one by one, from
// the keys they see alone: a tile multiplies every key's v with every row's
// weight, and the zero weight of a key that a row does not see times a NaN or
// an infinity is NaN. What is not finite after that is the definition's.
// `o`, `m`, `l` of the row: lane holds elements e * 64 + lane.
template <class Tag, int D>
__device__ __forceinline__ void store_row(const AttnArgs& a, const Item& it, int kv_head, int row,
                                          int local_row, int rows_per_tile, float m, float l,
                                          const float (&o)[D / 64]) {
  const int lane = threadIdx.x % kWave;
  if (it.splits == 1) {
    const int i = fdiv(row, a.fd_group);
    const int head = kv_head * a.group + row - i * a.group;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int64_t off = (it.x.q0 + i) * a.o_ts + head * a.o_hs;
#pragma unroll
    for (int e = 0; e < D / 64; ++e) store_elem<Tag>(a.out, off + e * 64 + lane, o[e] * inv);
  } else {
    float* part = a.ws + (static_cast<int64_t>(it.index) * a.kv_heads + kv_head) * rows_per_tile *
                             (D + 2);
#pragma unroll
    for (int e = 0; e < D / 64; ++e) part[local_row * D + e * 64 + lane] = o[e];
    if (lane == 0) {
      part[rows_per_tile * D + local_row] = m;
      part[rows_per_tile * (D + 1) + local_row] = l;
    }
  }
}

// max(a, b) that is NaN if either is (v_maximum3_f32, three values an
// instruction; fmaxf would first make a quiet copy of each).
__device__ __forceinline__ float nan_max(float a, float b) {
  return __builtin_elementwise_maximum(a, b);
}

// Largest growth of a row's maximum (as a power of two) that is let pass
// without scaling what is summed so far: the weights then reach 2^8 instead of
// 1, which costs fp32 sums nothing and keeps 16-bit weights in range.
constexpr float kLazyMax = 8.f;

// The kernel's arguments, read again: what only a kernel's end needs of them is
// not held in scalar registers (and spilled) through its loop.
__device__ __forceinline__ AttnArgs args_again() {
#ifdef __HIP_DEVICE_COMPILE__
  auto p = reinterpret_cast<uint64_t>(__builtin_amdgcn_kernarg_segment_ptr());
  asm volatile("" : "+s"(p));
  return *(const __attribute__((address_space(4))) AttnArgs*)(p);
#else
  return AttnArgs{};  // the host's pass over device code
#endif
}

// The end of attn_tiles_kernel: 32 rows from row `first` of the tile on, O^T in o
// (lane: row lane % 32; head_dim 32 d + 8 (e / 4) + 4 (lane / 32) + e % 4), to the
// output or, of a split tile, to the workspace.
template <class Tag, int D, int ROWS, bool PAGED>
__device__ __forceinline__ void store_tile(const AttnArgs a, const Item& it, int kv_head, int first,
                                           int k_begin, int k_end, const f32x16 (&o)[D / 32],
                                           float m, float l) {
  constexpr int DB = D / 32;
  const Request& x = it.x;
  const int lane = threadIdx.x % kWave, half = lane / 32;
  const int rows = x.nq * a.group;
  const int row0 = it.tile * ROWS;
  const int my_row = row0 + first + lane % 32;
  bool fine = finite_bits(l);
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) fine = fine && finite_bits(o[d][e]);
  const uint64_t bad = __ballot(!fine && my_row < rows);
  if (my_row < rows) {
    if (it.splits == 1) {
      const int i = fdiv(my_row, a.fd_group);
      const int head = kv_head * a.group + my_row - i * a.group;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      char* out = static_cast<char*>(a.out) +
                  ((x.q0 + i) * a.o_ts + head * a.o_hs + half * 4) * Tag::kBytes;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          st8(out + (d * 32 + e * 8) * Tag::kBytes,
              u32x2{pack2<Tag>(o[d][4 * e] * inv, o[d][4 * e + 1] * inv),
                    pack2<Tag>(o[d][4 * e + 2] * inv, o[d][4 * e + 3] * inv)});
    } else {
      float* part = a.ws + (static_cast<int64_t>(it.index) * a.kv_heads + kv_head) * ROWS * (D + 2);
      const int row = first + lane % 32;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          *reinterpret_cast<f32x4*>(part + row * D + d * 32 + e * 8 + half * 4) =
              f32x4{o[d][4 * e], o[d][4 * e + 1], o[d][4 * e + 2], o[d][4 * e + 3]};
      if (half == 0) {
        part[ROWS * D + row] = m;
        part[ROWS * (D + 1) + row] = l;
      }
    }
  }
  uint32_t again = static_cast<uint32_t>(bad) | static_cast<uint32_t>(bad >> 32);
  while (again != 0) {
    const int b = __builtin_ctz(again);
    again &= again - 1;
    const int row = row0 + first + b;
    const int i = fdiv(row, a.fd_group);
    float ro[D / 64], rm, rl;
    attend_row<Tag, D, PAGED>(a, it.r, x, kv_head * a.group + row - i * a.group, i, k_begin,
                              min(k_end, visible(a, x, i)), rm, rl, ro);
    store_row<Tag, D>(a, it, kv_head, row, first + b, ROWS, rm, rl, ro);
  }
}

// ---------------------------------------------------------------------------
// Many rows: four waves of 32 rows each over blocks of 64 keys that they share.
//
// Scores are taken transposed, S^T = K Q^T with 32x32x16 products: a lane then
// holds 32 keys' scores of one row (column lane % 32, keys 8 a + 4 (lane / 32)
// + b), so the softmax is arithmetic within a lane but for one exchange between
// the wave's halves, and the weights P^T are in place as the second operand of
// O^T = V^T P^T: a product's 16 key slots may stand for any 16 keys as long as
// V^T's are the same ones, and the transposing LDS reads give a lane four
// consecutive keys of one column of V at a time, just those.
// K and V blocks go straight from global memory to LDS, one block ahead of
// their use; one barrier a block.
//
// Per block and wave (D = 128) the products take 1024 cycles of a matrix unit,
// reading their operands 256 cycles of the CU's LDS (so eight waves' reads take as
// long as all four matrix units do: 32 rows a wave is the least that works, and
// 64 rows a wave leave one wave a SIMD: 761 against 1060 TFLOP/s), the weights
// about 1000 cycles of the vector unit, half of them 32 exponentials. Two
// workgroups share a CU, so one's weights run beside the other's products.
// Measured: a prompt of 16384 tokens, 32 heads over 8 of 128, causal, 2.0 to 2.3
// ms by the card's clock (1.10 to 0.96 PFLOP/s; a plain product of 8192^3 reaches
// 1.21), matrix units busy 61% of the cycles at 1.5 GHz, no bank conflicts: power
// and the LDS bound it. 16384 tokens of 32 over 16 heads of 64: 0.87 PFLOP/s (the
// exponentials); 12000 of 16 over 4 of 256: 0.85 (one workgroup a CU, 128 KB of
// LDS). Dropped: eight waves in two groups a phase apart (1.03 to 1.05), blocks
// of 32 keys with the weights a block behind (1.06, short prompts slower), raised
// wave priority (level), heads grouped by XCD (level; D = 256 slower).
// ---------------------------------------------------------------------------
template <class Tag, int D, Keys KEYS>
__global__ __launch_bounds__(kBlock, D <= 128 ? 2 : 1) void attn_tiles_kernel(const AttnArgs a) {
  constexpr bool PAGED = KEYS != Keys::kPacked;
  constexpr int WAVES = kBlock / kWave, ROWS = kTileRows;
  constexpr int BLOCK = kKeyBlock * D * 2;  // bytes of a K or V block
  constexpr int PER = kWave / (D / 8);      // rows a load
  constexpr int COUNT = kKeyBlock / PER / WAVES;
  constexpr int KK = D / 16, DB = D / 32;
  __shared__ __attribute__((aligned(1024))) char smem[4 * BLOCK];  // K0 K1 V0 V1
  const uint32_t lds = lds_address(smem);
  const int lane = threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const uint32_t id = blockIdx.x;
  const uint32_t work = a.items * a.kv_heads;
  if (id >= work) {
    fill_rest<Tag, D>(a, id - work, gridDim.x - work);
    return;
  }
  const uint32_t item_id = id / a.kv_heads;
  const int kv_head = id - item_id * a.kv_heads;
  const Item it = find_item<ROWS, PAGED, false>(a, item_id);
  if (it.r < 0) return;
  const Request& x = it.x;

  // Rows of the tile; this wave's, cut to the request's last (those are
  // computed again and not stored).
  const int rows = x.nq * a.group;
  const int row0 = it.tile * ROWS;
  const int half = lane / 32;
  const int my_row = row0 + wave * 32 + lane % 32;
  const int my_i = fdiv(min(my_row, rows - 1), a.fd_group);
  const int my_head = kv_head * a.group + min(my_row, rows - 1) - my_i * a.group;
  const int my_end = visible(a, x, my_i);
  const int last_i = fdiv(min(row0 + ROWS, rows) - 1, a.fd_group);
  // Keys of the tile's range, and of the wave's first row.
  const int64_t range0 = static_cast<int64_t>(it.split) * it.chunk * kKeyBlock;
  const int k_end = static_cast<int>(min(static_cast<int64_t>(visible(a, x, last_i)),
                                         range0 + static_cast<int64_t>(it.chunk) * kKeyBlock));
  const int k_begin = static_cast<int>(min(range0, static_cast<int64_t>(k_end)));
  const int first_end = visible(a, x, fdiv(min(row0 + wave * 32, rows - 1), a.fd_group));
  const int wave_end =
      row0 + wave * 32 < rows
          ? min(k_end, visible(a, x, fdiv(min(row0 + wave * 32 + 31, rows - 1), a.fd_group)))
          : 0;

  u32x4 q[KK];
  {
    const char* p = static_cast<const char*>(a.q) +
                    ((x.q0 + my_i) * a.q_ts + my_head * a.q_hs + half * 8) * Tag::kBytes;
#pragma unroll
    for (int k = 0; k < KK; ++k) q[k] = ld16(p + k * 32);
  }

  f32x16 o[DB] = {};
  float m = -INFINITY, l = 0.f;

  const char* kp = static_cast<const char*>(a.k) + kv_head * a.k_hs * Tag::kBytes;
  const char* vp = static_cast<const char*>(a.v) + kv_head * a.v_hs * Tag::kBytes;
  const int n = (k_end - k_begin + kKeyBlock - 1) / kKeyBlock;  // blocks of the range
  const int first_row = wave * (kKeyBlock / WAVES);             // of a block: this wave's loads
  auto base_of = [&](int t) JO_INLINE { return k_begin + t * kKeyBlock; };
  auto page_of_block = [&](int t) JO_INLINE {
    return key_page<PAGED>(a, it.r, min(base_of(t), k_end - 1), k_end);
  };

  // Where the wave's rows of a block are: one address (kPages16, kPacked), or an
  // offset a key (kPages). Rows behind the range's last key read that key.
  struct Rows {
    KeyRows each;          // kPages; `there` in every mode
    int64_t k_off, v_off;  // else: bytes to the row of key `from`
    int from, last;        // of the block: keys from .. last are read by this wave
  };
  auto rows_of = [&](int t, int32_t page) JO_INLINE {
    const int base = base_of(t);
    Rows b;
    if constexpr (KEYS == Keys::kPages) {
      b.each = key_rows<true>(a, x, page, base, k_end);
    } else {
      b.last = min(kKeyBlock, k_end - base) - 1;
      b.from = min(first_row, b.last & ~15);
      uint32_t row = x.k0 + base + b.from;
      int64_t p = 0;
      b.each.there = ~uint64_t{0};
      if constexpr (KEYS == Keys::kPages16) {
        // (Lanes behind the range hold its last key's page.)
        b.each.there = __ballot(page >= 0 && page < a.num_pages);
        const int32_t mine = __builtin_amdgcn_readlane(page, b.from);
        p = mine >= 0 && mine < a.num_pages ? mine : 0;
        row -= fdiv(row, a.fd_page) * a.fd_page.d;
      }
      b.k_off = (p * a.k_ps16 + static_cast<int64_t>(row) * a.k_ts16) << 4;
      b.v_off = (p * a.v_ps16 + static_cast<int64_t>(row) * a.v_ts16) << 4;
      if (b.last < kKeyBlock - 1) b.each.there &= (uint64_t{2} << b.last) - 1;
    }
    return b;
  };
  // This wave's rows of K (V32 false) or V to LDS at `to`.
  auto load_rows_of = [&](const Rows& b, auto v32, uint32_t to) JO_INLINE {
    constexpr bool V32 = decltype(v32)::value;
    if constexpr (KEYS == Keys::kPages) {
      load_rows<D, COUNT, V32>(V32 ? vp : kp, V32 ? b.each.v16 : b.each.k16, to, first_row, lane);
    } else {
#pragma unroll
      for (int i = 0; i < COUNT; ++i) {
        const int row = first_row + i * PER + lane / (D / 8);
        const int chunk = (lane % (D / 8)) ^ (V32 ? swz_v32<D>(row) : swz_k<D>(row));
        const uint32_t off = (min(row, b.last) - b.from) * (V32 ? a.v_ts16 : a.k_ts16) + chunk;
        load_to_lds((V32 ? vp + b.v_off : kp + b.k_off), off << 4,
                    to + (first_row + i * PER) * D * 2);
      }
    }
  };
  auto load_k = [&](const Rows& b, int buf) JO_INLINE {
    load_rows_of(b, std::false_type{}, lds + buf * BLOCK);
  };
  auto load_v = [&](const Rows& b, int buf) JO_INLINE {
    load_rows_of(b, std::true_type{}, lds + (2 + buf) * BLOCK);
  };
  // Lane addresses of the operand reads, one a 16-element step of head_dim (K)
  // and one a 32-column block and half step (V); buffers, key steps and blocks
  // are constants from there.
  uint32_t k_addr[KK], v_addr[DB][2];
#pragma unroll
  for (int k = 0; k < KK; ++k)
    k_addr[k] = lds + (lane % 32) * (D * 2) + (((2 * k + half) ^ swz_k<D>(lane % 32)) << 4);
  // V's transposing reads: key 4 half + i / 4 of an 8-key half step, columns
  // 16 (lane / 16 % 2) + 4 (i % 4) of a 32-column block (i = lane % 16).
  const int v_row = half * 4 + lane % 16 / 4;
  const int v_chunk = (lane / 16 % 2) * 2 + (lane % 4) / 2;
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int h = 0; h < 2; ++h)
      v_addr[d][h] = lds + 2 * BLOCK + (v_row + 8 * h) * (D * 2) + (lane % 2) * 8 +
                     (((d * 4 + v_chunk) ^ swz_v32<D>(v_row + 8 * h)) << 4);

  f32x16 s[2];
  u32x4 p[4];
  auto other_buffer = [&](int buf) JO_INLINE {
    const int step = buf ? -BLOCK : BLOCK;
#pragma unroll
    for (int k = 0; k < KK; ++k) k_addr[k] += step;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int h = 0; h < 2; ++h) v_addr[d][h] += step;
  };
  auto v_read = [&](int k, int d) JO_INLINE {
    return lds_read_tr(v_addr[d][0] + k * 16 * D * 2, v_addr[d][1] + k * 16 * D * 2);
  };
  // Products in groups of four whose operands are read a group ahead: groups 0 ..
  // DB - 1 are V^T P^T (four of the 16-key steps x 32-column blocks each), the
  // KK / 2 groups behind them K Q^T (two steps of head_dim, two key halves).
  auto read_group = [&](u32x4 (&f)[4], int g) JO_INLINE {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      f[e] = g < DB ? v_read((g * 4 + e) / DB, (g * 4 + e) % DB)
                    : lds_read16(k_addr[(g - DB) * 2 + e / 2] + e % 2 * 32 * D * 2);
  };
  auto multiply_group = [&](const u32x4 (&f)[4], int g) JO_INLINE {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (g < DB)
        o[(g * 4 + e) % DB] = mfma32<Tag>(f[e], p[(g * 4 + e) / DB], o[(g * 4 + e) % DB]);
      else
        s[e % 2] = mfma32<Tag>(f[e], q[(g - DB) * 2 + e / 2], s[e % 2]);
    }
  };
  // From scores to weights in two parts: what this row has seen so far is scaled
  // to a larger maximum, and the k-th 16 weights.
  float m_use = 0.f;
  auto new_max = [&](int t, uint64_t there) JO_INLINE {
    const int base = base_of(t);
    if (base + kKeyBlock > first_end || ~there != 0) {  // uniform
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int j = b * 32 + (e / 4) * 8 + half * 4 + e % 4;
          if (base + j >= my_end || !((there >> j) & 1)) s[b][e] = -INFINITY;
        }
    }
    float top = s[0][0];
#pragma unroll
    for (int e = 1; e < 32; ++e) top = nan_max(top, s[e / 16][e % 16]);
    if (__any(top * a.scale_log2 > m + kLazyMax)) {
      const float m_new = fmaxf(m, fmaxf(top, __shfl_xor(top, 32)) * a.scale_log2);
      const float fade = m_new == -INFINITY ? 1.f : exp2_fast(m - m_new);
      m = m_new;
      l *= fade;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] *= fade;
    }
    m_use = m == -INFINITY ? 0.f : m;
  };
  auto weights = [&](int k) JO_INLINE {
    float w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      w[e] = exp2_fast(fmaf(s[k / 2][(k % 2) * 8 + e], a.scale_log2, -m_use));
      l += w[e];
    }
    p[k] = u32x4{pack2<Tag>(w[0], w[1]), pack2<Tag>(w[2], w[3]), pack2<Tag>(w[4], w[5]),
                 pack2<Tag>(w[6], w[7])};
  };
  Rows next;
  int32_t page = 0;
  if (n > 0) {
    next = rows_of(0, page_of_block(0));
    load_k(next, 0);
    load_v(next, 0);
    page = page_of_block(1);
  }
  int buf = 0;
  for (int t = 0; t < n; ++t, buf ^= 1) {
    // This block is in LDS (this wave's loads: the wait; the others': the
    // barrier), and every wave is done with the other buffer.
    JO_KEEP_ORDER();
    JO_WAIT_VM(0);
    JO_WAIT_LDS0();
    __builtin_amdgcn_s_barrier();
    JO_KEEP_ORDER();
    const uint64_t there = next.each.there;
    if (t + 1 < n) {
      next = rows_of(t + 1, page);
      load_k(next, buf ^ 1);
      load_v(next, buf ^ 1);
      page = page_of_block(t + 2);
    }
    if (base_of(t) < wave_end) {  // else the wave's rows see none of these keys (uniform)
      u32x4 f[2][4];
      read_group(f[0], DB);
      s[0] = s[1] = f32x16{};
#pragma unroll
      for (int g = 0; g < KK / 2; ++g) {
        read_group(f[(g + 1) % 2], g + 1 < KK / 2 ? DB + g + 1 : 0);
        __builtin_amdgcn_sched_barrier(0);
        multiply_group(f[g % 2], DB + g);
        __builtin_amdgcn_sched_barrier(0);
      }
      new_max(t, there);
#pragma unroll
      for (int g = 0; g < DB; ++g) {
        if (g + 1 < DB) read_group(f[(KK / 2 + g + 1) % 2], g + 1);
        // (Group g's products take the weights of its 16-key steps.)
#pragma unroll
        for (int k = (g * 4 + DB - 1) / DB; k < ((g + 1) * 4 + DB - 1) / DB; ++k) weights(k);
        multiply_group(f[(KK / 2 + g) % 2], g);
      }
    }
    other_buffer(buf);
  }
  l += __shfl_xor(l, 32);
  store_tile<Tag, D, ROWS, PAGED>(args_again(), it, kv_head, wave * 32, k_begin, k_end, o, m, l);
}

// ---------------------------------------------------------------------------
// Few rows (single tokens): 16 rows a workgroup, its waves sharing the keys, 32
// at a time each, with 16x16x32 products in the same transposed form. Every
// wave loads its own keys into its own part of LDS, a block ahead, and waits for
// no other wave until the waves' results are joined at the end.
//
// Bound by reading the keys once: 64 requests of 100 to 16384 keys, 8 key heads
// of 128, 141 us (5.2 TB/s; a large copy moves 5.15), two of 100000 keys 95 us
// (5.3), 256 of 500 to 2000 211 us (5.3); four of 300 to 2000 keys 11 us, of
// which the joining kernel takes 3 and a launch 4: latency. Two waves a workgroup
// were 4 to 8% slower in full batches, page ids of 32 blocks at a time level; items
// that share an XCD by request instead of by key head: 64 requests 148 -> 203 us.
// ---------------------------------------------------------------------------
template <int D>
struct FewShape {
  static constexpr int kWaves = D == 256 ? 2 : 4;
  static constexpr int kKeys = 32;                 // keys a block
  static constexpr int kBlockBytes = kKeys * D * 2;  // of K or V
  static constexpr int kWaveBytes = 4 * kBlockBytes;
  static constexpr int kRowFloats = D + 4;         // a joined row in LDS
};

template <class Tag, int D, bool PAGED>
__global__ __launch_bounds__(FewShape<D>::kWaves* kWave, 1) void attn_few_kernel(const AttnArgs a) {
  using S = FewShape<D>;
  constexpr int ROWS = 16, W = S::kWaves, BLOCK = S::kBlockBytes;
  constexpr int PER = kWave / (D / 8), COUNT = S::kKeys / PER;
  constexpr int KK = D / 32, DB = D / 16;
  __shared__ __attribute__((aligned(1024))) char smem[W * S::kWaveBytes];
  __shared__ float s_m[W][ROWS], s_l[W][ROWS];
  const uint32_t lds = lds_address(smem);
  const int lane = threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const uint32_t id = blockIdx.x;
  const uint32_t work = a.items * a.kv_heads;
  if (id >= work) {
    fill_rest<Tag, D>(a, id - work, gridDim.x - work);
    return;
  }
  const uint32_t item_id = id / a.kv_heads;
  const int kv_head = id - item_id * a.kv_heads;
  const Item it = find_item<ROWS, PAGED, false>(a, item_id);
  if (it.r < 0) return;
  const Request& x = it.x;

  const int rows = x.nq * a.group;
  const int row0 = it.tile * ROWS;
  const int grp = lane / 16;
  const int my_row = min(row0 + lane % 16, rows - 1);
  const int my_i = fdiv(my_row, a.fd_group);
  const int my_head = kv_head * a.group + my_row - my_i * a.group;
  const int my_end = visible(a, x, my_i);
  const int last_i = fdiv(min(row0 + ROWS, rows) - 1, a.fd_group);
  const int64_t range0 = static_cast<int64_t>(it.split) * it.chunk * kKeyBlock;
  const int k_end = static_cast<int>(min(static_cast<int64_t>(visible(a, x, last_i)),
                                         range0 + static_cast<int64_t>(it.chunk) * kKeyBlock));
  const int k_begin = static_cast<int>(min(range0, static_cast<int64_t>(k_end)));
  const int first_end = visible(a, x, fdiv(row0, a.fd_group));

  u32x4 q[KK];
  {
    const char* p = static_cast<const char*>(a.q) +
                    ((x.q0 + my_i) * a.q_ts + my_head * a.q_hs + grp * 8) * Tag::kBytes;
#pragma unroll
    for (int k = 0; k < KK; ++k) q[k] = ld16(p + k * 64);
  }
  f32x4 o[DB] = {};
  float m = -INFINITY, l = 0.f;

  const char* kp = static_cast<const char*>(a.k) + kv_head * a.k_hs * Tag::kBytes;
  const char* vp = static_cast<const char*>(a.v) + kv_head * a.v_hs * Tag::kBytes;
  const uint32_t mine = lds + wave * S::kWaveBytes;
  auto load_block = [&](const KeyRows& kr, int buf) {
    load_rows<D, COUNT, false>(kp, kr.k16, mine + buf * BLOCK, 0, lane);
    load_rows<D, COUNT, false>(vp, kr.v16, mine + (2 + buf) * BLOCK, 0, lane);
  };
  const int kr_ = lane % 16;
  const uint32_t k_addr = mine + kr_ * (D * 2) + ((grp ^ swz_k<D>(kr_)) << 4);
  const int vi = lane % 16;
  const int v_row = grp * 4 + vi / 4;
  const int v_chunk = (vi % 4) / 2;
  const uint32_t v_addr = mine + 2 * BLOCK + v_row * (D * 2) + (vi % 2) * 8;

  constexpr int STEP = W * S::kKeys;  // a wave's blocks are this far apart
  const int my_begin = k_begin + wave * S::kKeys;
  auto attend = [&](int base, int buf, uint32_t there) JO_INLINE {
    f32x4 s[2] = {};
    const uint32_t ka = k_addr + buf * BLOCK;
#pragma unroll
    for (int k = 0; k < KK; ++k)
#pragma unroll
      for (int b = 0; b < 2; ++b)
        s[b] = mfma16<Tag>(lds_read16((ka ^ (k << 6)) + b * 16 * D * 2), q[k], s[b]);
    if (base + S::kKeys > first_end || ~there != 0) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = b * 16 + grp * 4 + e;
          if (base + j >= my_end || !((there >> j) & 1)) s[b][e] = -INFINITY;
        }
    }
    float top = fmaxf(s[0][0], s[1][0]);
#pragma unroll
    for (int e = 1; e < 4; ++e) top = fmaxf(top, fmaxf(s[0][e], s[1][e]));
    if (__any(top * a.scale_log2 > m + kLazyMax)) {
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      const float m_new = fmaxf(m, top * a.scale_log2);
      const float fade = m_new == -INFINITY ? 1.f : exp2_fast(m - m_new);
      m = m_new;
      l *= fade;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[d][e] *= fade;
    }
    const float m_use = m == -INFINITY ? 0.f : m;
    float w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      w[e] = exp2_fast(fmaf(s[e / 4][e % 4], a.scale_log2, -m_use));
      l += w[e];
    }
    const u32x4 p = {pack2<Tag>(w[0], w[1]), pack2<Tag>(w[2], w[3]), pack2<Tag>(w[4], w[5]),
                     pack2<Tag>(w[6], w[7])};
    const uint32_t va = v_addr + buf * BLOCK;
    const int sw0 = swz_k<D>(v_row), sw1 = swz_k<D>(v_row + 16);
#pragma unroll
    for (int d = 0; d < DB; ++d)
      o[d] = mfma16<Tag>(lds_read_tr(va + (((d * 2 + v_chunk) ^ sw0) << 4),
                                     va + 16 * D * 2 + (((d * 2 + v_chunk) ^ sw1) << 4)),
                         p, o[d]);
  };
  if (my_begin < k_end) {
    // Page ids run two blocks ahead of the loads that they are for: in order with
    // them, a wait for an id is then never a wait for the block just asked for.
    // (Past the range they read its last entry again.)
    auto page_at = [&](int base) { return key_page<PAGED>(a, it.r, min(base, k_end - 1), k_end); };
    KeyRows cur = key_rows<PAGED>(a, x, page_at(my_begin), my_begin, k_end);
    int32_t page1 = page_at(min(my_begin, k_end - STEP) + STEP);
    int32_t page2 = page_at(min(my_begin, k_end - 2 * STEP) + 2 * STEP);
    load_block(cur, 0);
    int buf = 0, base = my_begin;
    for (; base < k_end - STEP; base += STEP, buf ^= 1) {
      const uint32_t there = static_cast<uint32_t>(cur.there);
      cur = key_rows<PAGED>(a, x, page1, base + STEP, k_end);
      page1 = page2;
      page2 = page_at(min(base, k_end - 3 * STEP) + 3 * STEP);
      JO_KEEP_ORDER();
      JO_WAIT_LDS0();  // what was read from the other buffer has arrived
      JO_KEEP_ORDER();
      load_block(cur, buf ^ 1);
      JO_KEEP_ORDER();
      JO_WAIT_VM(2 * COUNT + (PAGED ? 1 : 0));
      JO_KEEP_ORDER();
      attend(base, buf, there);
    }
    JO_KEEP_ORDER();
    JO_WAIT_VM(0);
    JO_KEEP_ORDER();
    attend(base, buf, static_cast<uint32_t>(cur.there));
  }
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);

  // The waves' results, joined: each wave leaves its 16 rows in its part of LDS.
  JO_KEEP_ORDER();
  JO_WAIT_LDS0();
  JO_KEEP_ORDER();
  float* mine_o = reinterpret_cast<float*>(smem + wave * S::kWaveBytes);
#pragma unroll
  for (int d = 0; d < DB; ++d)
    *reinterpret_cast<f32x4*>(mine_o + (lane % 16) * S::kRowFloats + d * 16 + grp * 4) = o[d];
  if (grp == 0) {
    s_m[wave][lane] = m;
    s_l[wave][lane] = l;
  }
  __syncthreads();
  constexpr int TPR = W * kWave / ROWS;  // threads a row
  constexpr int NE = D / TPR / 4;        // pieces of four elements a thread
  const int row = threadIdx.x / TPR, part_of = threadIdx.x % TPR;
  float top = -INFINITY, sum = 0.f;
#pragma unroll
  for (int w = 0; w < W; ++w) top = fmaxf(top, s_m[w][row]);
  f32x4 r[NE] = {};
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const float mw = s_m[w][row];
    const float e = mw == -INFINITY ? (mw == top ? 1.f : 0.f) : exp2_fast(mw - top);
    sum = fmaf(e, s_l[w][row], sum);
    const float* src =
        reinterpret_cast<const float*>(smem + w * S::kWaveBytes) + row * S::kRowFloats;
#pragma unroll
    for (int n = 0; n < NE; ++n) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(src + (n * TPR + part_of) * 4);
#pragma unroll
      for (int c = 0; c < 4; ++c) r[n][c] = fmaf(e, v[c], r[n][c]);
    }
  }
  bool fine = finite_bits(sum);
#pragma unroll
  for (int n = 0; n < NE; ++n)
#pragma unroll
    for (int c = 0; c < 4; ++c) fine = fine && finite_bits(r[n][c]);
  const bool mine_row = row0 + row < rows;
  uint64_t bad = __ballot(!fine && mine_row);
  if (mine_row) {
    if (it.splits == 1) {
      const int i = fdiv(row0 + row, a.fd_group);
      const int head = kv_head * a.group + row0 + row - i * a.group;
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      char* out = static_cast<char*>(a.out) + ((x.q0 + i) * a.o_ts + head * a.o_hs) * Tag::kBytes;
#pragma unroll
      for (int n = 0; n < NE; ++n)
        st8(out + (n * TPR + part_of) * 4 * Tag::kBytes,
            u32x2{pack2<Tag>(r[n][0] * inv, r[n][1] * inv),
                  pack2<Tag>(r[n][2] * inv, r[n][3] * inv)});
    } else {
      float* part = a.ws + (static_cast<int64_t>(it.index) * a.kv_heads + kv_head) * ROWS * (D + 2);
#pragma unroll
      for (int n = 0; n < NE; ++n)
        *reinterpret_cast<f32x4*>(part + row * D + (n * TPR + part_of) * 4) = r[n];
      if (part_of == 0) {
        part[ROWS * D + row] = top;
        part[ROWS * (D + 1) + row] = sum;
      }
    }
  }
  while (bad != 0) {
    const int b = __builtin_ctzll(bad) / TPR;  // the wave's b-th row
    bad &= ~(((TPR == 64 ? 0 : uint64_t{1} << (TPR % 64)) - 1) << (b * TPR));
    const int local = wave * (kWave / TPR) + b;
    const int i = fdiv(row0 + local, a.fd_group);
    float ro[D / 64], rm, rl;
    attend_row<Tag, D, PAGED>(a, it.r, x, kv_head * a.group + row0 + local - i * a.group, i,
                              k_begin, min(k_end, visible(a, x, i)), rm, rl, ro);
    store_row<Tag, D>(a, it, kv_head, row0 + local, local, ROWS, rm, rl, ro);
  }
}

// Joins the partial results of split tiles:
//   out = sum_s e_s o_s / sum_s e_s l_s, e_s = 2^(m_s - max m).
// A workgroup takes EACH times kBlock / (D / 4) / GROUPS rows of a tile and key
// head, four elements a thread, the splits dealt out to GROUPS threads of each
// element whose sums meet in LDS: with few rows there are many splits, and one
// thread would wait for them one after the other.
template <class Tag, int D, int ROWS, bool PAGED, int GROUPS, int EACH>
__global__ __launch_bounds__(kBlock) void attn_join_kernel(const AttnArgs a) {
  constexpr int C = D / 4;                    // threads a row and group
  constexpr int PER = kBlock / C / GROUPS;    // rows a workgroup
  static_assert(GROUPS == 1 || EACH == 1, "the rows' sums in LDS are for one step");
  constexpr int PARTS = ROWS / PER / EACH;
  const uint32_t unit = blockIdx.x / PARTS;
  const int row_begin = (blockIdx.x % PARTS) * PER * EACH;
  const uint32_t tile_id = unit / a.kv_heads;
  const int kv_head = unit - tile_id * a.kv_heads;
  const Item it = find_item<ROWS, PAGED, true>(a, tile_id);
  // (A last item that was not launched: lengths that overlap, nothing to join.)
  if (it.r < 0 || it.splits == 1 || static_cast<uint32_t>(it.index + it.splits) > a.items) return;
  const int rows = min(ROWS, it.x.nq * a.group - it.tile * ROWS);
  const int64_t stride = static_cast<int64_t>(a.kv_heads) * ROWS * (D + 2);
  const float* first =
      a.ws + (static_cast<int64_t>(it.index) * a.kv_heads + kv_head) * ROWS * (D + 2);
  const int c = threadIdx.x % C, group = threadIdx.x / C % GROUPS;
#pragma unroll 1
  for (int row0 = row_begin; row0 < min(rows, row_begin + PER * EACH); row0 += PER) {
    const int row = min(row0 + static_cast<int>(threadIdx.x) / (C * GROUPS), rows - 1);
    float top = -INFINITY, sum = 0.f;
    f32x4 r = {};
#pragma unroll 4
    for (int s = group; s < it.splits; s += GROUPS) {
      const float* p = first + s * stride;
      const float ms = p[ROWS * D + row], ls = p[ROWS * (D + 1) + row];
      const f32x4 v = *reinterpret_cast<const f32x4*>(p + row * D + c * 4);
      const float m_new = fmaxf(top, ms);
      const float m_use = m_new == -INFINITY ? 0.f : m_new;
      const float fade = exp2_fast(top - m_use), e = exp2_fast(ms - m_use);
      top = m_new;
      sum = fmaf(e, ls, sum * fade);
#pragma unroll
      for (int k = 0; k < 4; ++k) r[k] = fmaf(e, v[k], r[k] * fade);
    }
    if constexpr (GROUPS > 1) {
      __shared__ f32x4 s_r[kBlock];
      __shared__ float s_m[kBlock], s_l[kBlock];
      s_r[threadIdx.x] = r;
      s_m[threadIdx.x] = top;
      s_l[threadIdx.x] = sum;
      __syncthreads();
      if (group != 0) return;
      const int at = threadIdx.x;
      float all = top;
#pragma unroll
      for (int g = 1; g < GROUPS; ++g) all = fmaxf(all, s_m[at + g * C]);
      const float use = all == -INFINITY ? 0.f : all;
      sum = 0.f;
      r = f32x4{};
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        const float e = exp2_fast(s_m[at + g * C] - use);
        const f32x4 v = s_r[at + g * C];
        sum = fmaf(e, s_l[at + g * C], sum);
#pragma unroll
        for (int k = 0; k < 4; ++k) r[k] = fmaf(e, v[k], r[k]);
      }
    }
    const int at_row = it.tile * ROWS + row0 + static_cast<int>(threadIdx.x) / (C * GROUPS);
    if (at_row >= it.x.nq * a.group) continue;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int i = fdiv(at_row, a.fd_group);
    const int head = kv_head * a.group + at_row - i * a.group;
    st8(byte_off(a.out, ((it.x.q0 + i) * a.o_ts + head * a.o_hs + c * 4) * Tag::kBytes),
        u32x2{pack2<Tag>(r[0] * inv, r[1] * inv), pack2<Tag>(r[2] * inv, r[3] * inv)});
  }
}

// ---------------------------------------------------------------------------
// Launch plan, from sizes that the host has.
// ---------------------------------------------------------------------------
struct AttnPlan {
  bool few;             // attn_few_kernel
  int64_t tiles;        // at most so many
  int64_t split_target;
  int64_t tail_splits, tail_most, round;
  int64_t items;
  int64_t ws_bytes;
};

constexpr int64_t kComputeUnits = 256;
// Threads that share an element's splits, and steps of rows a workgroup takes.
// (Tiles, 16384 rows a key head and less: two steps 89.3 us, one 91.9, four 90.3
// for 20 requests of chunks and single tokens, the whole call; 62.5, 64.1, 62.1
// for four prompts of 1000 tokens.)
constexpr int kFewJoin = 4, kTileJoin = 1, kTileEach = 2;  // threads that share an element's splits

AttnPlan plan_attention(int64_t q_tokens, int64_t requests, int64_t q_heads, int64_t kv_heads,
                        int64_t head_dim, int64_t kv_capacity, bool causal) {
  AttnPlan p{};
  const int64_t group = q_heads / kv_heads;
  const int64_t all_rows = q_tokens * group;
  p.few = all_rows <= 16 * requests;
  const int64_t rows = p.few ? 16 : kTileRows;
  p.tiles =
      all_rows / rows + (requests < q_tokens || requests > kPlanRequests ? requests : q_tokens);
  if (requests == 0) p.tiles = 0;
  const int64_t blocks = (kv_capacity + kKeyBlock - 1) / kKeyBlock;
  // Workgroups that run at once: LDS and registers let two of the smaller ones
  // share a compute unit.
  const int64_t slots = kComputeUnits * (head_dim <= (p.few ? 64 : 128) ? 2 : 1);
  const int64_t round = (slots + kv_heads - 1) / kv_heads;  // items of one round
  p.split_target = 0;
  // How many tiles there are if the requests are alike.
  const int64_t alike =
      requests == 0 ? 0 : requests * ((q_tokens / requests * group + rows - 1) / rows);
  // Tiles of 128 rows that fill the GPU, with no more than a few keys a token:
  // their ranges would hardly be split, and the joining kernel's launch is saved
  // (four prompts of 1000 tokens, 2.0 rounds: 64.2 -> 59.5 us, eight of 200 to
  // 3500, 2.3 rounds: 62.1 -> 59.3). One request's tiles are alike, all of them
  // where every key is seen. Where keys may be many more than tokens (single tokens
  // over long contexts among chunks), one tile can outlast all others.
  const bool full =
      !p.few && kv_capacity <= 4 * q_tokens &&
      (requests == 1 ? (causal ? 1 : 2) * alike > round : 4 * p.tiles >= 7 * round);
  if (requests > 0 && requests <= kPlanRequests && blocks > kMinChunk && p.tiles < 8 * round &&
      kv_heads <= slots && !full) {
    // A split tile's last range is half full on average: split_target + tiles / 2
    // items come of it. Where tiles are few they are meant to fill one round, or a
    // little less, unequal requests having more tiles (32 requests of 16 tokens 52.9
    // us; with round - tiles 57.3, round - tiles / 2 51.2; 10 of chunks and single
    // tokens 108.7, 108.3, 110.2). Else (single tokens of 48 and 64 requests 112 and
    // 141 us; with one round 113 and 142, with two 117 and 143; of 128 requests 208,
    // 220, 211; chunks beside single tokens: 95.5 us with one round, 98.7 with 0.75,
    // 95.3 with 1.5, 102 with two).
    if (2 * alike <= round) p.split_target = round - 3 * alike / 4;
    else p.split_target = p.few ? 3 * round / 2 : round;
  }
  const int64_t most = p.tiles * (blocks / kMinChunk + 1);
  p.items = p.tiles + p.split_target < most ? p.tiles + p.split_target : most;
  // Tiles that see all keys take equally long, and a last round of a few leaves
  // most of the GPU idle: its tiles are split where that is worth the partial
  // results' way to memory and back. Times in key blocks of a tile: one a CU is
  // 1 us, joining 5 us and 6.5 us a partial result and CU. (Two frames of 1560
  // tokens over three cached ones and themselves, 32 heads: 25 tiles a head, 16 a
  // round; not split 555 us, the last 9 in two 539, three 531, four, as chosen
  // here, 528, six 539, eight 548.)
  int64_t places = p.split_target == 0 ? 0 : p.items;
  p.round = round;
  p.tail_splits = 1;
  if (!p.few && !causal && p.split_target == 0 && requests > 0 && requests <= kPlanRequests &&
      (requests == 1 || p.tiles > round)) {
    const int64_t tail = alike % round;
    auto time = [&](int64_t s) {  // in blocks
      const int64_t n = tail * kv_heads * s;
      const int64_t steps = (n + kComputeUnits - 1) / kComputeUnits;
      return static_cast<double>(steps) * static_cast<double>(blocks) / static_cast<double>(s) +
             (s == 1 ? 0. : 5. + 6.5 * static_cast<double>(n) / kComputeUnits);
    };
    for (int64_t s = 2; s <= 8 && s * kMinChunk <= blocks; ++s)
      if (time(s) < time(p.tail_splits)) p.tail_splits = s;
    if (p.tail_splits > 1) {
      p.tail_most = tail;
      p.items += tail * (p.tail_splits - 1);
      places = tail * p.tail_splits;
    }
  }
  p.ws_bytes = places * kv_heads * rows * (head_dim + 2) * 4;
  return p;
}

template <class Tag, int D, bool PAGED>
int launch_attention(AttnArgs a, int64_t kv_capacity, void* ws, int64_t ws_bytes,
                     hipStream_t stream) {
  const char* op = PAGED ? "attention_paged" : "attention_varlen";
  AttnPlan p =
      plan_attention(a.q_tokens, a.requests, a.q_heads, a.kv_heads, D, kv_capacity, a.causal);
  if (p.ws_bytes > 0 && ws_bytes < p.ws_bytes) {  // none, or one for another call: no splits
    p.split_target = 0;
    p.tail_splits = 1;
    p.items = p.tiles;
  }
  a.split_target = static_cast<uint32_t>(p.split_target);
  a.fd_target = make_fastdiv(a.split_target);
  a.tail_splits = static_cast<uint32_t>(p.tail_splits);
  a.tail_most = static_cast<uint32_t>(p.tail_most);
  a.fd_round = make_fastdiv(static_cast<uint32_t>(p.round));
  a.items = static_cast<uint32_t>(p.items);
  a.ws = static_cast<float*>(ws);
  // Workgroups that clear the rows of no request, 64 KB each if they are all.
  const int64_t bytes = static_cast<int64_t>(a.q_tokens) * a.q_heads * D * 2;
  const int64_t fill = a.fill_rest ? (bytes / 65536 < 256 ? bytes / 65536 + 1 : 256) : 0;
  const int64_t groups = p.items * a.kv_heads + fill;
  JO_REQUIRE(groups <= INT32_MAX / 512, "%s: shape too large", op);
  if (groups == 0) return JO_OK;
  const dim3 grid(static_cast<unsigned>(groups));
  if (p.few)
    hipLaunchKernelGGL((attn_few_kernel<Tag, D, PAGED>), grid, dim3(FewShape<D>::kWaves * kWave), 0,
                       stream, a);
  else if constexpr (!PAGED)
    hipLaunchKernelGGL((attn_tiles_kernel<Tag, D, Keys::kPacked>), grid, dim3(kBlock), 0, stream,
                       a);
  else if (a.fd_page.d % 16 == 0)
    hipLaunchKernelGGL((attn_tiles_kernel<Tag, D, Keys::kPages16>), grid, dim3(kBlock), 0, stream,
                       a);
  else
    hipLaunchKernelGGL((attn_tiles_kernel<Tag, D, Keys::kPages>), grid, dim3(kBlock), 0, stream, a);
  int st = launch_status(op);
  if (st != JO_OK || (p.split_target == 0 && p.tail_splits == 1)) return st;
  // Tiles that are split: the tail's, or no more than split_target, since each has
  // more key blocks than a chunk.
  const int64_t split_tiles = p.tail_splits > 1 ? p.tail_most
                              : p.tiles < p.split_target ? p.tiles
                                                         : p.split_target;
  const int64_t joins = split_tiles * a.kv_heads * (p.few ? 16 : kTileRows) * (D / 4) *
                        (p.few ? kFewJoin : kTileJoin) / kBlock / (p.few ? 1 : kTileEach);
  JO_REQUIRE(joins <= INT32_MAX / 512, "%s: shape too large", op);
  const dim3 join(static_cast<unsigned>(joins));
  if (p.few)
    hipLaunchKernelGGL((attn_join_kernel<Tag, D, 16, PAGED, kFewJoin, 1>), join, dim3(kBlock), 0,
                       stream, a);
  else
    hipLaunchKernelGGL((attn_join_kernel<Tag, D, kTileRows, PAGED, kTileJoin, kTileEach>), join,
                       dim3(kBlock), 0, stream, a);
  return launch_status(op);
}

template <bool PAGED>
int dispatch_attention(const AttnArgs& a, int64_t head_dim, int dtype, int64_t capacity, void* ws,
                       int64_t ws_bytes, hipStream_t s) {
  if (dtype == JO_DTYPE_BF16) {
    if (head_dim == 64) return launch_attention<BF16, 64, PAGED>(a, capacity, ws, ws_bytes, s);
    if (head_dim == 128) return launch_attention<BF16, 128, PAGED>(a, capacity, ws, ws_bytes, s);
    return launch_attention<BF16, 256, PAGED>(a, capacity, ws, ws_bytes, s);
  }
  if (head_dim == 64) return launch_attention<F16, 64, PAGED>(a, capacity, ws, ws_bytes, s);
  if (head_dim == 128) return launch_attention<F16, 128, PAGED>(a, capacity, ws, ws_bytes, s);
  return launch_attention<F16, 256, PAGED>(a, capacity, ws, ws_bytes, s);
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
  // One of out's strides steps over all that the other one reaches.
  auto steps_over = [&](int64_t outer, int64_t n, int64_t inner) {
    return n <= 1 || (outer >= head_dim && (outer - head_dim) / (n - 1) >= inner);
  };
  JO_REQUIRE((q_tokens <= 1 || a.o_ts >= head_dim) && (q_heads <= 1 || a.o_hs >= head_dim) &&
                 (q_tokens <= 1 || q_heads <= 1 || steps_over(a.o_ts, q_heads, a.o_hs) ||
                  steps_over(a.o_hs, q_tokens, a.o_ts)),
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

// Strides of K and V in units of 16 bytes; row offsets are kept in 32 bits of
// them (64 GiB from a tensor's start). rows / pages: the largest index + 1.
int key_offsets(const char* op, AttnArgs& a, int64_t pages, int64_t rows) {
  auto reach = [](int64_t n, int64_t stride) {  // (n - 1) * stride, 2^40 at most
    return n <= 1 || stride == 0 ? 0
           : n - 1 > (int64_t{1} << 40) / stride ? int64_t{1} << 40
                                                 : (n - 1) * stride;
  };
  for (int i = 0; i < 2; ++i) {
    const int64_t ps = i ? a.v_ps : a.k_ps, ts = i ? a.v_ts : a.k_ts;
    JO_REQUIRE((reach(pages, ps) + reach(rows, ts)) / 8 <= INT32_MAX * int64_t{2},
               "%s: K and V rows must lie within 64 GiB", op);
    // (64 rows' offsets in 32 bits of bytes.)
    JO_REQUIRE(ts < (int64_t{1} << 24), "%s: token stride of K or V too large", op);
    (i ? a.v_ps16 : a.k_ps16) = static_cast<uint32_t>(pages > 1 ? ps / 8 : 0);
    (i ? a.v_ts16 : a.k_ts16) = static_cast<uint32_t>(rows > 1 ? ts / 8 : 0);
  }
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
  JO_REQUIRE(kv_tokens >= 0 && kv_tokens <= kMaxKeys, "%s: bad shape", op);
  const int st = check_attention(op, a, q, k, v, out, q_tokens, requests, q_heads, kv_heads,
                                 head_dim, cu_q, scale, dtype);
  if (st != JO_OK || q_tokens == 0) return st;
  JO_REQUIRE(cu_k && (kv_tokens == 0 || (k && v)), "%s: null pointer", op);
  a.cu_k = cu_k;
  a.kv_tokens = static_cast<int32_t>(kv_tokens);
  a.causal = causal != 0;
  a.fill_rest = fill_rest != 0;
  if (const int bad = key_offsets(op, a, 1, kv_tokens); bad != JO_OK) return bad;
  JO_REQUIRE(workspace_bytes >= 0 && aligned(workspace, 16),
             "%s: workspace must be 16-byte aligned", op);
  return dispatch_attention<false>(a, head_dim, dtype, kv_tokens, workspace,
                                   workspace ? workspace_bytes : 0,
                                   static_cast<hipStream_t>(stream));
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
  a.capacity = static_cast<int32_t>(places > kMaxKeys ? kMaxKeys : places);
  a.causal = causal != 0;
  a.fill_rest = fill_rest != 0;
  if (const int bad = key_offsets(op, a, num_pages, page_size); bad != JO_OK) return bad;
  JO_REQUIRE(workspace_bytes >= 0 && aligned(workspace, 16),
             "%s: workspace must be 16-byte aligned", op);
  return dispatch_attention<true>(a, head_dim, dtype, table_width * page_size, workspace,
                                  workspace ? workspace_bytes : 0,
                                  static_cast<hipStream_t>(stream));
}

extern "C" int64_t jo_attention_workspace_bytes(int64_t q_tokens, int64_t requests,
                                                int64_t q_heads, int64_t kv_heads,
                                                int64_t head_dim, int64_t kv_capacity,
                                                int causal) {
  if (q_tokens <= 0 || requests < 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads != 0 ||
      head_dim <= 0 || kv_capacity < 0)
    return 0;
  return plan_attention(q_tokens, requests, q_heads, kv_heads, head_dim, kv_capacity, causal != 0)
      .ws_bytes;
}
