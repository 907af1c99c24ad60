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
__device__ __forceinline__ uint64_t timer_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}
// Bounded: after two seconds the CTA gives up, and so do all its other waits.
constexpr uint64_t kWaitLimitNs = 2000000000ull;
// Inline everywhere: a call would hold its caller to the registers of the launch.
__device__ __forceinline__ bool barrier_wait(uint32_t bar, uint32_t parity, volatile uint32_t* gave_up) {
  if (barrier_try(bar, parity)) return true;
  uint64_t t0 = 0;
#pragma unroll 1
  for (uint32_t it = 1; !barrier_try(bar, parity); ++it) {
    if ((it & 63u) != 0u) continue;
    if (*gave_up) return false;
    const uint64_t now = timer_ns();
    if (t0 == 0) t0 = now;
    if (now - t0 > kWaitLimitNs) {
      *gave_up = 1u;
      return false;
    }
  }
  return true;
}
// On the way out after that: copies of this CTA that are still in flight, bounded again.
__device__ __forceinline__ void barrier_wait_out(uint32_t bar, uint32_t parity) {
  const uint64_t t0 = timer_ns();
  while (!barrier_try(bar, parity) && timer_ns() - t0 <= kWaitLimitNs) {
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

// ------------------------------------------------------------------ division of the work
struct Sequence {
  int32_t token, n, length;  // first new token, new tokens, keys
};
__device__ __forceinline__ Sequence load_sequence(const AttentionParams& P, uint32_t b) {
  const int32_t tokens = static_cast<int32_t>(P.tokens);
  const int32_t s = min(max(P.indptr[b], 0), tokens);
  const int32_t e = min(max(P.indptr[b + 1], s), tokens);
  const int32_t l = min(max(P.lengths[b], 0), static_cast<int32_t>(P.capacity));
  return Sequence{s, e - s, l};
}
struct KeyRange {
  int32_t begin, end;  // keys that some row of an item sees
};
template <int ROWS>
__device__ __forceinline__ KeyRange key_range(const AttentionParams& P, const Sequence& s, uint32_t row_tile) {
  KeyRange r{0, s.length};
  if (P.causal) {
    const uint32_t first = row_tile * ROWS;
    const uint32_t last = min(first + ROWS, static_cast<uint32_t>(s.n) * P.group) - 1u;
    const int32_t base = s.length - s.n;
    r.end = max(0, base + static_cast<int32_t>(last / P.group) + 1);
    if (P.window) {
      const int64_t b = static_cast<int64_t>(base) + first / P.group + 1 - static_cast<int64_t>(P.window);
      r.begin = static_cast<int32_t>(max(static_cast<int64_t>(0), b));
    }
  }
  return r;
}
// Tiles of an item; one that sees no key has one all the same, in which its zeros are written.
template <int KEYS>
__device__ __forceinline__ uint32_t item_tiles(const KeyRange& r) {
  return r.end > r.begin ? (r.end + KEYS - 1) / KEYS - r.begin / KEYS : 1u;
}
// Its units: as many, or one where no item is split.
template <int KEYS>
__device__ __forceinline__ uint32_t item_units(const AttentionParams& P, const KeyRange& r) {
  return P.whole_items ? 1u : item_tiles<KEYS>(r);
}
template <int ROWS>
__device__ __forceinline__ uint32_t row_tiles(const AttentionParams& P, const Sequence& s) {
  return (static_cast<uint32_t>(s.n) * P.group + ROWS - 1) / ROWS;
}
template <int ROWS, int KEYS>
__device__ __forceinline__ uint64_t head_units(const AttentionParams& P, const Sequence& s) {
  uint64_t u = 0;
  const uint32_t tiles = row_tiles<ROWS>(P, s);
  if (P.whole_items) return tiles;
  for (uint32_t t = 0; t < tiles; ++t) u += item_units<KEYS>(P, key_range<ROWS>(P, s, t));
  return u;
}
// Where a CTA's share begins, how long it is, and how all shares lie.
struct Share {
  uint64_t total;     // units of the call
  uint64_t begin;     // first unit of this CTA
  uint32_t units;     // units of this CTA
  uint32_t ctas;      // CTAs that have a share
  uint32_t sequence, head, row_tile, skip;  // the item that holds the first unit, and its units before it
};
__device__ __forceinline__ uint64_t share_begin(uint64_t total, uint32_t ctas, uint32_t cta) {
  return total * cta / ctas;
}
// Called by all THREADS threads of a CTA; `sums` has THREADS entries.
template <int ROWS, int KEYS, int THREADS>
__device__ __forceinline__ void find_share(const AttentionParams& P, uint64_t* sums, Share* share) {
  const uint32_t t = threadIdx.x;
  // sequences of this thread
  const uint32_t each = (P.sequences + THREADS - 1) / THREADS;
  const uint32_t b0 = min(t * each, P.sequences), b1 = min(b0 + each, P.sequences);
  uint64_t mine = 0;
  for (uint32_t b = b0; b < b1; ++b) mine += head_units<ROWS, KEYS>(P, load_sequence(P, b)) * P.kv_heads;
  uint64_t upto = mine;  // inclusive sum over the warp, then over the warps
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint64_t o = __shfl_up_sync(0xffffffffu, upto, d);
    if ((t & 31u) >= d) upto += o;
  }
  if ((t & 31u) == 31u) sums[t >> 5] = upto;
  if (t == 0) share->units = 0;
  __syncthreads();
  uint64_t total = 0;
#pragma unroll
  for (uint32_t w = 0; w < THREADS / 32; ++w) {
    const uint64_t s = sums[w];
    if (w < (t >> 5)) upto += s;
    total += s;
  }
  const uint64_t want = (total + P.min_units - 1) / P.min_units;
  const uint32_t ctas = want < gridDim.x ? static_cast<uint32_t>(want) : gridDim.x;
  if (blockIdx.x < ctas) {
    const uint64_t u0 = share_begin(total, ctas, blockIdx.x), u1 = share_begin(total, ctas, blockIdx.x + 1);
    uint64_t at = upto - mine;
    if (u0 >= at && u0 < upto) {  // exactly one thread
      uint32_t b = b0;
      Sequence s = load_sequence(P, b);
      uint64_t per_head = head_units<ROWS, KEYS>(P, s);
      while (u0 >= at + per_head * P.kv_heads) {
        at += per_head * P.kv_heads;
        s = load_sequence(P, ++b);
        per_head = head_units<ROWS, KEYS>(P, s);
      }
      const uint64_t head = (u0 - at) / per_head;
      uint64_t left = u0 - at - head * per_head;
      uint32_t tile = 0;
      for (;;) {
        const uint32_t u = item_units<KEYS>(P, key_range<ROWS>(P, s, tile));
        if (left < u) break;
        left -= u;
        ++tile;
      }
      share->total = total;
      share->begin = u0;
      share->ctas = ctas;
      share->sequence = b;
      share->head = static_cast<uint32_t>(head);
      share->row_tile = tile;
      share->skip = static_cast<uint32_t>(left);
      share->units = static_cast<uint32_t>(u1 - u0);
    }
  }
  __syncthreads();
}
// Walks through the pieces of a share: what every role of a CTA does by itself.
template <int ROWS, int KEYS>
struct Pieces {
  const AttentionParams& P;
  Sequence s;
  uint32_t b, head, tile, skip, left, tiles;
  uint64_t at;
  // the piece
  KeyRange keys;
  uint32_t first_tile, count, whole;  // key tiles first_tile .. first_tile + count - 1 of the item's `whole`

  __device__ __forceinline__ Pieces(const AttentionParams& params, const Share& share)
      : P(params), b(share.sequence), head(share.head), tile(share.row_tile), skip(share.skip),
        left(share.units), at(share.begin) {
    if (left) {
      s = load_sequence(P, b);
      tiles = row_tiles<ROWS>(P, s);
    }
  }
  __device__ __forceinline__ bool next() {
    if (left == 0) return false;
    if (tile == tiles) {  // on to the next head, or the next sequence that has new tokens
      tile = 0;
      if (++head == P.kv_heads) {
        head = 0;
        do {
          s = load_sequence(P, ++b);
        } while (s.n == 0);
        tiles = row_tiles<ROWS>(P, s);
      }
    }
    keys = key_range<ROWS>(P, s, tile);
    whole = item_tiles<KEYS>(keys);
    first_tile = (keys.end > keys.begin ? keys.begin / KEYS : 0u) + skip;
    count = P.whole_items ? whole : min(whole - skip, left);
    return true;
  }
  __device__ __forceinline__ bool begins() const { return skip == 0; }
  __device__ __forceinline__ bool ends() const { return skip + count == whole; }
  __device__ __forceinline__ uint32_t rows() const {
    return min(static_cast<uint32_t>(ROWS), static_cast<uint32_t>(s.n) * P.group - tile * ROWS);
  }
  // CTAs behind this one that have more of the piece's item
  __device__ __forceinline__ uint32_t more(const Share& share) const {
    const uint64_t last = at + (whole - skip) - 1;  // the item's last unit
    const uint64_t cta = ((last + 1) * share.ctas - 1) / share.total;
    return static_cast<uint32_t>(cta) - blockIdx.x;
  }
  __device__ __forceinline__ void done() {
    const uint32_t units = P.whole_items ? 1u : count;
    left -= units;
    at += units;
    ++tile;
    skip = 0;
  }
};

// The warp that loads: boxes of a tile of keys, one lane each; page numbers are read a tile ahead.
template <int KEYS, int HALVES>
struct TileLoader {
  const AttentionParams& P;
  const uint32_t lane;
  const uint32_t boxes;
  int32_t page, row;
  bool wanted;
  __device__ __forceinline__ TileLoader(const AttentionParams& params)
      : P(params), lane(threadIdx.x & 31u), boxes(KEYS / params.box) {}
  __device__ __forceinline__ void look_up(uint32_t b, const KeyRange& keys, uint32_t tile) {
    const int32_t key = static_cast<int32_t>(tile * KEYS + lane * P.box);
    wanted = lane < boxes && key < keys.end && key + static_cast<int32_t>(P.box) > keys.begin;
    page = -1;
    row = 0;
    if (wanted) {
      const uint32_t p = static_cast<uint32_t>(key) / P.page_size;
      row = key - static_cast<int32_t>(p * P.page_size);
      page = P.table[static_cast<int64_t>(b) * P.table_stride + p];
    }
  }
  // Loads the tile of this look-up into `dst` (HALVES blocks of KEYS rows of 128 bytes, swizzled).
  // Boxes without a visible key are left out: what the slot holds there is from earlier.
  __device__ __forceinline__ void load(const CUtensorMap* map, uint32_t dst, uint32_t head, uint32_t bar) const {
    const uint32_t count = __popc(__ballot_sync(0xffffffffu, wanted));
    if (lane == 0) barrier_arrive_bytes(bar, count * P.box * 128u * HALVES);
    __syncwarp();
    if (wanted) {
#pragma unroll
      for (int h = 0; h < HALVES; ++h)
        load_box(dst + h * KEYS * 128 + lane * P.box * 128u, map, h * 64, row, static_cast<int32_t>(head), page, bar);
    }
  }
};

}  // namespace paged
}  // namespace mononn
