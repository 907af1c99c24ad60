// Device code that the kernels of the paged attention share: waits, copies, the division of the work.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "paged.h"

namespace mononn {
namespace paged {

__device__ __forceinline__ uint32_t smem_address(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void barrier_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
// A barrier of an attention kernel: one arrival too many when it is the one that is to run out.
__device__ __forceinline__ void barrier_init(const AttentionParams& P, AttentionBarrier which, const uint64_t& bar, uint32_t count) {
  barrier_init(smem_address(&bar), count + (P.skewed == which ? 1u : 0u));
}
__device__ __forceinline__ void barrier_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void barrier_arrive_bytes(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool barrier_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0u;
}
__device__ __forceinline__ uint32_t clock_now() {
  uint32_t t;
  asm volatile("mov.u32 %0, %%clock;" : "=r"(t));
  return t;
}
// Bounded: after 2^31 cycles, about a second, the CTA gives up, and so do all its other waits. Inline
// everywhere (a call would hold its caller to the registers of the launch), so it is kept small.
constexpr uint32_t kWaitLimit = 1u << 31;
__device__ __forceinline__ bool barrier_wait(uint32_t bar, uint32_t parity, volatile uint32_t* gave_up) {
  if (barrier_try(bar, parity)) return true;
  const uint32_t t0 = clock_now();
#pragma unroll 1
  while (!barrier_try(bar, parity)) {
    if (*gave_up || clock_now() - t0 >= kWaitLimit) {
      *gave_up = 1u;
      return false;
    }
  }
  return true;
}
// On the way out after that: copies of this CTA that are still in flight, bounded again.
__device__ __forceinline__ void barrier_wait_out(uint32_t bar, uint32_t parity) {
  const uint32_t t0 = clock_now();
#pragma unroll 1
  while (!barrier_try(bar, parity) && clock_now() - t0 < kWaitLimit) {
  }
}
// The whole warp gets the same answer.
__device__ __forceinline__ bool barrier_wait_warp(uint32_t bar, uint32_t parity, volatile uint32_t* gave_up) {
  return __all_sync(0xffffffffu, barrier_wait(bar, parity, gave_up));
}
// Box of 64 elements of a head x `box` token rows of one page.
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, int32_t element, int32_t row,
                                         int32_t head, int32_t page, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(map), "r"(element), "r"(row), "r"(head), "r"(page), "r"(bar)
      : "memory");
}
// Box of 64 elements of the heads of a group x some tokens.
__device__ __forceinline__ void load_queries(uint32_t dst, const CUtensorMap* map, int32_t element, int32_t head,
                                             int32_t token, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(map), "r"(element), "r"(head), "r"(token), "r"(bar)
      : "memory");
}
// The kernels are launched so that the next one's CTAs may be set up while the last one still runs:
// nothing that an earlier kernel wrote is read, and nothing written, before earlier_done.
__device__ __forceinline__ void earlier_done() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_begin() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename T>
struct Pair;
template <>
struct Pair<__half> {
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t v) {
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
  }
};
template <>
struct Pair<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t v) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
  }
};
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void copy_16(uint32_t dst, const void* src, bool wanted) {  // zeros where not
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(wanted ? 16u : 0u) : "memory");
}
// One arrival when the copies that this thread has begun have landed.
__device__ __forceinline__ void arrive_after_copies(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ uint32_t divide(uint32_t n, const Divisor& d) {
  const uint32_t t = __umulhi(n, d.multiplier);
  return (t + ((n - t) >> d.shift1)) >> d.shift2;
}

// ------------------------------------------------------------------ division of the work
struct Sequence {
  int32_t token, n, length;  // first new token, new tokens, keys
};
__device__ __forceinline__ Sequence load_sequence(const AttentionParams& P, uint32_t b) {
  const int32_t tokens = static_cast<int32_t>(P.tokens);
  const int32_t s0 = P.indptr[b], e0 = P.indptr[b + 1], l0 = P.lengths[b];
  const int32_t s = min(max(s0, 0), tokens), e = min(max(e0, s), tokens);
  return Sequence{s, e - s, min(max(l0, 0), static_cast<int32_t>(P.capacity))};
}
struct KeyRange {
  int32_t begin, end;  // keys that some of the tokens see
};
__device__ __forceinline__ KeyRange key_range(const AttentionParams& P, const Sequence& s, uint32_t first, uint32_t last) {
  KeyRange r{0, s.length};
  if (P.causal) {
    const int32_t base = s.length - s.n;
    r.end = max(0, base + static_cast<int32_t>(last) + 1);
    // keys behind position p + 1 - window, where p is the first token's (below zero: it sees nothing)
    const int32_t upto = base + static_cast<int32_t>(first) + 1;
    if (P.window && upto > 0 && static_cast<uint32_t>(upto) > P.window) r.begin = upto - static_cast<int32_t>(P.window);
  }
  return r;
}
__device__ __forceinline__ uint32_t row_tiles(const AttentionParams& P, const Sequence& s) {
  return divide(static_cast<uint32_t>(s.n) * P.group + P.item_rows - 1u, P.by_item_rows);
}
__device__ __forceinline__ KeyRange item_keys(const AttentionParams& P, const Sequence& s, uint32_t tile) {
  const uint32_t first = tile * P.item_rows;
  const uint32_t last = min(first + P.item_rows, static_cast<uint32_t>(s.n) * P.group) - 1u;
  return key_range(P, s, divide(first, P.by_group), divide(last, P.by_group));
}
// Keys from .. to - 1 are those that the token at `position` sees (`length`: keys of its sequence).
__device__ __forceinline__ void seen_keys(const AttentionParams& P, int32_t position, int32_t length, int32_t& from, int32_t& to) {
  to = P.causal ? max(position + 1, 0) : length;
  from = P.causal && P.window && position >= 0 && static_cast<uint32_t>(position) >= P.window
             ? position + 1 - static_cast<int32_t>(P.window) : 0;
}
// What a row's sum is divided by, as a factor: a row that saw nothing becomes zeros. A sum of 0 beside a score means that the
// score left 32 bits when it was scaled: 1 / 0 makes NaN of it.
__device__ __forceinline__ float inverse_of(float top, float sum) {
  return sum == 0.f && top == __int_as_float(0xff800000) ? 0.f : 1.f / sum;
}
__device__ __forceinline__ float log_sum(float top, float sum, float scale) {
  const float ninf = __int_as_float(0xff800000), nan = __int_as_float(0x7fffffff);
  return sum == 0.f ? (top == ninf ? ninf : nan) : top * scale + logf(sum);
}
// Tiles of an item; one that sees no key has one all the same, in which its zeros are written.
template <int KEYS>
__device__ __forceinline__ uint32_t item_tiles(const KeyRange& r) {
  return r.end > r.begin ? (r.end + KEYS - 1) / KEYS - r.begin / KEYS : 1u;
}
// Its units: as many, behind the ones that stand for what an item takes beside its keys (queries, joining the
// warps, the way out); one in all where no item is split.
template <int KEYS>
__device__ __forceinline__ uint32_t item_units(const AttentionParams& P, const Sequence& s, uint32_t tile) {
  return P.whole_items ? 1u : P.item_cost + item_tiles<KEYS>(item_keys(P, s, tile));
}
// Units of one head of a sequence that is the same for the whole warp.
template <int KEYS>
__device__ __forceinline__ uint32_t head_units_warp(const AttentionParams& P, const Sequence& s, uint32_t tiles) {
  uint32_t part = 0;
#pragma unroll 1
  for (uint32_t t = threadIdx.x & 31u; t < tiles; t += 32u) part += item_units<KEYS>(P, s, t);
  return __reduce_add_sync(0xffffffffu, part);
}
// Where a CTA's share begins, how long it is, and how all shares lie: the first `longer` CTAs have
// `each` + 1 units, the others `each`. The host has made sure that units are counted in 31 bits.
struct Share {
  uint32_t units, begin, ctas, each, longer;
  uint32_t sequence, head, row_tile, skip;  // the item that holds the first unit, and its units before that
  Sequence s;
  __device__ __forceinline__ uint32_t cta_of(uint32_t unit) const {
    const uint32_t in_longer = (each + 1u) * longer;
    return unit < in_longer ? unit / (each + 1u) : longer + (unit - in_longer) / each;
  }
};
// Called by all THREADS threads of a CTA; `sums` has an entry for each warp. A warp takes consecutive
// sequences, its lanes too; sequences of many row tiles are summed up by the warp together.
template <int KEYS, int THREADS>
__device__ __forceinline__ void find_share(const AttentionParams& P, uint32_t* sums, Share* share) {
  constexpr uint32_t kWarpsHere = THREADS / 32;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  const uint32_t per_warp = (P.sequences + kWarpsHere - 1) / kWarpsHere, each = (per_warp + 31u) / 32u;
  const uint32_t end = min((warp + 1u) * per_warp, P.sequences);
  const uint32_t b0 = warp * per_warp + lane * each;
  uint32_t mine = 0;
  Sequence s{0, 0, 0};
#pragma unroll 1
  for (uint32_t i = 0; i < each; ++i) {
    s = Sequence{0, 0, 0};
    if (b0 + i < end) s = load_sequence(P, b0 + i);
    const uint32_t tiles = row_tiles(P, s);
    uint32_t u = 0;
    if (tiles <= 2u)
#pragma unroll 1
      for (uint32_t t = 0; t < tiles; ++t) u += item_units<KEYS>(P, s, t);
#pragma unroll 1
    for (uint32_t many = __ballot_sync(0xffffffffu, tiles > 2u); many; many &= many - 1u) {
      const int from = __ffs(many) - 1;
      const Sequence o{0, __shfl_sync(0xffffffffu, s.n, from), __shfl_sync(0xffffffffu, s.length, from)};
      const uint32_t sum = head_units_warp<KEYS>(P, o, __shfl_sync(0xffffffffu, tiles, from));
      if (static_cast<int>(lane) == from) u = sum;
    }
    mine += u * P.kv_heads;
  }
  uint32_t upto = mine;  // inclusive sum over the warp, then over the warps
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t o = __shfl_up_sync(0xffffffffu, upto, d);
    if (lane >= d) upto += o;
  }
  if (lane == 31u) sums[warp] = upto;
  if (threadIdx.x == 0) share->units = 0;
  __syncthreads();
  uint32_t total = 0, before = 0;
#pragma unroll
  for (uint32_t w = 0; w < kWarpsHere; ++w) {
    const uint32_t x = sums[w];
    if (w < warp) before += x;
    total += x;
  }
  const uint32_t ctas = min(gridDim.x, (total + (1u << P.least_shift) - 1u) >> P.least_shift);
  if (blockIdx.x < ctas) {
    const uint32_t share_each = total / ctas, longer = total - share_each * ctas;
    const uint32_t u0 = share_each * blockIdx.x + min(blockIdx.x, longer);
    uint32_t at = before + upto - mine;
    const uint32_t here = __ballot_sync(0xffffffffu, u0 >= at && u0 - at < mine);
    if (here) {  // one lane of one warp; the warp goes on together
      const int from = __ffs(here) - 1;
      at = __shfl_sync(0xffffffffu, at, from);
      uint32_t b = __shfl_sync(0xffffffffu, b0, from);
      s.token = __shfl_sync(0xffffffffu, s.token, from);
      s.n = __shfl_sync(0xffffffffu, s.n, from);
      s.length = __shfl_sync(0xffffffffu, s.length, from);
      uint32_t per_head = 0;
      bool found = false;  // always, where indptr does not decrease; otherwise sums may have wrapped
#pragma unroll 1
      for (; b < end; ++b) {
        if (each > 1u) s = load_sequence(P, b);
        const uint32_t tiles = row_tiles(P, s);
        per_head = tiles == 1u ? item_units<KEYS>(P, s, 0) : head_units_warp<KEYS>(P, s, tiles);
        found = u0 - at < per_head * P.kv_heads;
        if (found) break;
        at += per_head * P.kv_heads;
      }
      const uint32_t head = per_head == 1u ? u0 - at : (u0 - at) / per_head;
      uint32_t left = u0 - at - head * per_head, tile = 0;
      const uint32_t tiles = found ? row_tiles(P, s) : 0u;
      found = found && tiles == 1u;  // nothing to look for then
#pragma unroll 1
      for (uint32_t t0 = 0; !found && t0 < tiles; t0 += 32u) {
        const uint32_t u = t0 + lane < tiles ? item_units<KEYS>(P, s, t0 + lane) : 0u;
        uint32_t sum = u;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const uint32_t o = __shfl_up_sync(0xffffffffu, sum, d);
          if (lane >= d) sum += o;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, left < sum);
        found = past != 0u;
        if (found) {
          const int at_lane = __ffs(past) - 1;
          tile = t0 + at_lane;
          left -= __shfl_sync(0xffffffffu, sum - u, at_lane);
          break;
        }
        left -= __shfl_sync(0xffffffffu, sum, 31);
      }
      if (lane == 0 && found)
        *share = Share{share_each + (blockIdx.x < longer ? 1u : 0u), u0, ctas, share_each, longer, b, head, tile, left, s};
    }
  }
  __syncthreads();
}

// A part of a share that lies in one item: what the loading warp tells the others.
struct Piece {
  int32_t token, n, length;        // of the sequence
  uint32_t head, first_row, rows;  // rows (token x group + head of the group) of the sequence
  int32_t tile, count;             // key tiles tile .. tile + count - 1
  int32_t keys_begin, keys_end;    // that some row of the item sees
  uint32_t begins, ends;           // whether the item begins and ends in it
  uint32_t valid;                  // 0: no more pieces
  uint32_t sequence;
  uint32_t shared, pad;            // many rows: 1 when the two row tiles hold the same rows, for every other key tile each
  int32_t from[2], to[2];          // many rows: the key tiles from .. to - 1 that concern each of the two row tiles
};
// Walks through the pieces of a share; all lanes of the loading warp alike.
template <int KEYS>
struct Walker {
  const AttentionParams& P;
  const Share& share;
  Sequence s;
  uint32_t b, head, tile, skip, left, tiles, at, whole, goes_on;  // goes_on: tiles of the item behind the piece
  Piece piece;
  __device__ __forceinline__ Walker(const AttentionParams& params, const Share& sh)
      : P(params), share(sh), s(sh.s), b(sh.sequence), head(sh.head), tile(sh.row_tile), skip(sh.skip),
        left(sh.units), tiles(0), at(sh.begin), whole(0), goes_on(0), piece{} {
    if (left) tiles = row_tiles(P, s);
  }
  __device__ __forceinline__ bool next() {
    uint32_t units = 0, done = 0;
    KeyRange keys{0, 0};
    for (;;) {
      piece.valid = left != 0;
      if (left == 0) return false;
      if (tile == tiles) {  // on to the next head, or the next sequence that has new tokens
        tile = 0;
        if (++head == P.kv_heads) {
          head = 0;
          do {
            if (++b == P.sequences) {  // not where indptr does not decrease
              left = 0;
              piece.valid = 0;
              return false;
            }
            s = load_sequence(P, b);
          } while (s.n == 0);
          tiles = row_tiles(P, s);
        }
      }
      keys = item_keys(P, s, tile);
      whole = item_tiles<KEYS>(keys);
      if (P.whole_items) {
        units = 1u;
        done = 0;
        piece.count = static_cast<int32_t>(whole);
      } else {
        units = min(P.item_cost + whole - skip, left);
        done = skip > P.item_cost ? skip - P.item_cost : 0u;
        const uint32_t upto = skip + units;
        piece.count = static_cast<int32_t>((upto > P.item_cost ? upto - P.item_cost : 0u) - done);
      }
      left -= units;
      at += units;
      if (piece.count != 0) break;
      // the share ends before the item's first tile: the next CTA begins the item
    }
    piece.sequence = b;
    piece.token = s.token;
    piece.n = s.n;
    piece.length = s.length;
    piece.head = head;
    piece.first_row = tile * P.item_rows;
    piece.rows = min(P.item_rows, static_cast<uint32_t>(s.n) * P.group - piece.first_row);
    piece.tile = static_cast<int32_t>((keys.end > keys.begin ? keys.begin / KEYS : 0u) + done);
    piece.keys_begin = keys.begin;
    piece.keys_end = keys.end;
    piece.begins = done == 0;
    piece.ends = done + piece.count == whole;
    goes_on = whole - done - static_cast<uint32_t>(piece.count);
    ++tile;
    skip = 0;
    return true;
  }
  // Behind the last piece: whether its item goes on, and in how many CTAs.
  __device__ __forceinline__ void write_header() const {
    AttentionHeader h{0, 0, 0, 0, 0, {0, 0, 0}};
    if (share.units != 0 && piece.begins && !piece.ends) {
      const uint32_t last = at + goes_on - 1u;  // the item's last unit
      h = AttentionHeader{min(share.cta_of(last), gridDim.x - 1u) - blockIdx.x, piece.rows, piece.first_row, piece.head,
                          static_cast<uint32_t>(piece.token), {0, 0, 0}};
    }
    P.headers[blockIdx.x] = h;
  }
};
__device__ __forceinline__ void put_piece(Piece* to, const Piece& p, uint32_t lane) {
  if (lane != 0) return;
  int4* d = reinterpret_cast<int4*>(to);
  d[0] = make_int4(p.token, p.n, p.length, static_cast<int>(p.head));
  d[1] = make_int4(static_cast<int>(p.first_row), static_cast<int>(p.rows), p.tile, p.count);
  d[2] = make_int4(p.keys_begin, p.keys_end, static_cast<int>(p.begins), static_cast<int>(p.ends));
  d[3] = make_int4(static_cast<int>(p.valid), static_cast<int>(p.sequence), static_cast<int>(p.shared), 0);
  d[4] = make_int4(p.from[0], p.from[1], p.to[0], p.to[1]);
}

// A warp that loads tiles of keys or values: boxes of one page each, a lane to a box. Page numbers are
// read for 32 boxes at a time, and those one such window ahead.
template <int KEYS, int HALVES>
struct TileLoader {
  const AttentionParams& P;
  const uint32_t lane, boxes, window;  // boxes of a tile, tiles of a window
  uint32_t sequence, first;            // first tile of the present window
  int32_t keys_begin, keys_end;
  int32_t page, row, next_page, next_row;  // row below 0: not wanted
  __device__ __forceinline__ TileLoader(const AttentionParams& params)
      : P(params), lane(threadIdx.x & 31u), boxes(KEYS >> params.box_shift), window((32u << params.box_shift) / KEYS), sequence(0), first(0),
        keys_begin(0), keys_end(0), page(-1), row(-1), next_page(-1), next_row(-1) {}
  __device__ __forceinline__ void look_up(uint32_t tile0, int32_t& page_of, int32_t& row_of) const {
    const int32_t key = static_cast<int32_t>(tile0 * KEYS + (lane << P.box_shift));
    page_of = -1;
    row_of = -1;
    if (key < keys_end && key + (1 << P.box_shift) > keys_begin) {
      const uint32_t p = divide(static_cast<uint32_t>(key), P.by_page_size);
      row_of = key - static_cast<int32_t>(p * P.page_size);
      page_of = P.table[static_cast<int64_t>(sequence) * P.table_stride + p];
    }
  }
  __device__ __forceinline__ void begin(const Piece& piece) {
    sequence = piece.sequence;
    keys_begin = piece.keys_begin;
    // no further than the piece itself goes
    keys_end = min(piece.keys_end, (piece.tile + piece.count) * KEYS);
    first = static_cast<uint32_t>(piece.tile);
    look_up(first, page, row);
  }
  // Loads a tile, the next one of the piece, into `dst` (HALVES blocks of KEYS rows of 128 bytes, swizzled).
  // Boxes without a visible key are left out: what the slot holds there is from earlier.
  __device__ __forceinline__ void load(const CUtensorMap* map, uint32_t tile, uint32_t dst, uint32_t head, uint32_t bar) {
    if (tile - first == window) {
      first = tile;
      page = next_page;
      row = next_row;
    }
    const uint32_t from = (tile - first) * boxes + (lane & (boxes - 1u));
    const int32_t p = __shfl_sync(0xffffffffu, page, from), r = __shfl_sync(0xffffffffu, row, from);
    const bool wanted = lane < boxes && r >= 0;
    const uint32_t count = __popc(__ballot_sync(0xffffffffu, wanted));
    if (lane == 0) barrier_arrive_bytes(bar, (count << P.box_shift) * 128u * HALVES);
    __syncwarp();
    if (wanted) {
#pragma unroll
      for (int h = 0; h < HALVES; ++h)
        load_box(dst + h * KEYS * 128 + (lane << P.box_shift) * 128u, map, h * 64, r, static_cast<int32_t>(head), p, bar);
    }
    if (tile == first) look_up(first + window, next_page, next_row);
  }
};

}  // namespace paged
}  // namespace mononn
