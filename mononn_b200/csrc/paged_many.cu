// Attention over a paged cache for many rows: prompts, chunks of prompts, drafts of wide groups.
//
// The same one pass over the keys as the kernel for few rows, on the fifth-generation tensor cores. An item has
// up to 256 rows, two tiles of 128; a unit is 128 keys, loaded once for both. Roles of a CTA (one per SM):
//   warps 0-3, 4-7  the softmax of one row tile each, a thread to a row: scores from tensor memory,
//                   running maximum, probabilities back to tensor memory, row sums in registers
//   warp 8          issues the matrix products: S = Q K^T (both operands in shared memory), O += P V (P in
//                   tensor memory, in the place of the scores it was made from)
//   warp 9          loads keys and values, page by page, into a ring of tiles
// While one row tile's softmax runs, the tensor cores work on the other's products.
// O stays in tensor memory. It is rescaled only when a row's maximum has risen by more than
// 2^8 since its reference was set: until then probabilities are above 1, by 2^8 at most, which costs no accuracy.
#include "paged_device.h"

namespace mononn {
namespace paged {

constexpr int kTileRows = 128;
constexpr int kRows = static_cast<int>(kManyRows), kKeys = static_cast<int>(kManyKeys);
constexpr int kThreadsMany = 384;
constexpr int kMmaWarp = 8, kLoadWarp = 9;  // 10 and 11 only make up the group whose registers go to the others
constexpr uint32_t kSoftmaxRegisters = 200, kOtherRegisters = 104, kLaunchRegisters = 168;
static_assert(256 * kSoftmaxRegisters + 128 * kOtherRegisters <= kThreadsMany * kLaunchRegisters, "register split");
constexpr float kRise = 8.0f;  // in powers of two

template <int DIM>
struct ManySmem {
  static constexpr int kTileBytes = kTileRows * DIM * 2;  // of queries, keys or values
  static constexpr int kSlots = DIM == 64 ? 8 : 5;
  static constexpr int kRing = 2 * kTileBytes;
  static constexpr int kControl = kRing + kSlots * kTileBytes;
  static constexpr int kBytes = kControl + 512;
};
struct ManyControl {
  uint64_t full[8], empty[8];
  uint64_t scores[2], probabilities[2], queries[2], outputs[2], drained;
  uint64_t sums[12];
  Share share;
  uint32_t gave_up, tmem;
};
static_assert(sizeof(ManyControl) <= 512, "control block");

__device__ __forceinline__ void after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void shared_to_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ bool elected() {
  uint32_t pred;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(pred)::"memory");
  return pred != 0u;
}
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// 128-byte swizzled operand: groups of eight 128-byte rows 1024 bytes apart; `leading` is the distance of
// the next 64 elements of a row (in 16-byte units), where the rows run along the contraction.
__device__ __forceinline__ uint64_t operand(uint32_t address, uint32_t leading) {
  return static_cast<uint64_t>((address & 0x3ffffu) >> 4) | (static_cast<uint64_t>(leading) << 16) | (64ull << 32) |
         (1ull << 46) | (2ull << 61);
}
// f16 or bf16 operands, f32 accumulator, M = 128
template <typename T>
__device__ __forceinline__ constexpr uint32_t instruction(uint32_t n, bool b_along_n) {
  const uint32_t type = sizeof(T) && __is_same(T, __nv_bfloat16) ? 1u : 0u;
  return (1u << 4) | (type << 7) | (type << 10) | (b_along_n ? 1u << 16 : 0u) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}
__device__ __forceinline__ void product_shared(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(add))
      : "memory");
}
__device__ __forceinline__ void product_tensor(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(add))
      : "memory");
}
#define MONONN_R8(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7])
#define MONONN_P8(r, i) "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7])
#define MONONN_I8(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), "r"(r[i + 5]), "r"(r[i + 6]), "r"(r[i + 7])
// 32 columns of this warp's 32 rows. The values are there after loads_done on the same registers.
__device__ __forceinline__ void load_columns(uint32_t address, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : MONONN_R8(r, 0), MONONN_R8(r, 8), MONONN_R8(r, 16), MONONN_R8(r, 24)
      : "r"(address)
      : "memory");
}
__device__ __forceinline__ void loads_done(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : MONONN_P8(r, 0), MONONN_P8(r, 8), MONONN_P8(r, 16), MONONN_P8(r, 24)::"memory");
}
// the same for 16 columns
__device__ __forceinline__ void load_columns_16(uint32_t address, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : MONONN_R8(r, 0), MONONN_R8(r, 8)
      : "r"(address)
      : "memory");
}
__device__ __forceinline__ void loads_done_16(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : MONONN_P8(r, 0), MONONN_P8(r, 8)::"memory");
}
__device__ __forceinline__ void store_columns_16(uint32_t address, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::MONONN_I8(r, 0),
      MONONN_I8(r, 8), "r"(address)
      : "memory");
}
__device__ __forceinline__ void stores_done() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Columns that the row does not see: before `to`, and from `from` on.
__device__ __forceinline__ void hide(uint32_t* s, int first, int32_t to, int32_t from) {
#pragma unroll
  for (int j = 0; j < 32; ++j)
    if (first + j < to || first + j >= from) s[j] = 0xff800000u;
}

// What a row tile of a piece has to do: units from .. to - 1 hold keys that some of its rows see.
struct TileRange {
  int32_t from, to;
  __device__ __forceinline__ bool has(int32_t unit) const { return unit >= from && unit < to; }
};
__device__ __forceinline__ TileRange tile_range(const AttentionParams& P, const Pieces<kRows, kKeys>& piece, uint32_t t) {
  TileRange r{0, 0};
  if (t * kTileRows >= piece.rows()) return r;
  const KeyRange k = key_range<kTileRows>(P, piece.s, piece.tile * 2 + t);
  if (k.end <= k.begin) return r;
  r.from = max(static_cast<int32_t>(piece.first_tile), k.begin / kKeys);
  r.to = min(static_cast<int32_t>(piece.first_tile + piece.count), (k.end + kKeys - 1) / kKeys);
  if (r.to < r.from) r.to = r.from;
  return r;
}

template <typename T, int DIM>
__global__ void __launch_bounds__(kThreadsMany, 1) many_rows_kernel(const __grid_constant__ AttentionParams P) {
  extern __shared__ uint8_t raw[];
  using M = ManySmem<DIM>;
  constexpr int kHalves = DIM / 64, kSlots = M::kSlots;
  uint8_t* smem = raw + ((1024u - (smem_address(raw) & 1023u)) & 1023u);
  ManyControl& C = *reinterpret_cast<ManyControl*>(smem + M::kControl);
  const uint32_t base = smem_address(smem), ring = base + M::kRing;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kSlots; ++i) {
      barrier_init(smem_address(&C.full[i]), 1);
      barrier_init(smem_address(&C.empty[i]), 1);
    }
    for (int t = 0; t < 2; ++t) {
      barrier_init(smem_address(&C.scores[t]), 1);
      barrier_init(smem_address(&C.probabilities[t]), 4);
      barrier_init(smem_address(&C.queries[t]), 4);
      barrier_init(smem_address(&C.outputs[t]), 1);
    }
    barrier_init(smem_address(&C.drained), 1);
    C.gave_up = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&P.k_map));
    asm volatile("prefetch.tensormap [%0];" ::"l"(&P.v_map));
  }
  let_next_begin();
  earlier_done();
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_address(&C.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    before_sync();
  }
  find_share<kRows, kKeys, kThreadsMany>(P, C.sums, &C.share);  // barriers of the CTA within
  after_sync();
  const uint32_t tmem = *const_cast<volatile uint32_t*>(&C.tmem);
  const Share& share = C.share;
  Pieces<kRows, kKeys> piece(P, share);
  AttentionHeader header{0, 0, 0, 0, 0, {0, 0, 0}};
  uint32_t fills = 0;
  bool fine = true;

  if (warp >= kMmaWarp)
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegisters));
  else
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegisters));

  if (warp == kLoadWarp) {
    TileLoader<kKeys, kHalves> loader(P);
    while (fine && piece.next()) {
      loader.look_up(piece.b, piece.keys, piece.first_tile);
      for (uint32_t u = 0; fine && u < piece.count; ++u) {
        const TileLoader<kKeys, kHalves> now = loader;
        if (u + 1 < piece.count) loader.look_up(piece.b, piece.keys, piece.first_tile + u + 1);
        for (int kv = 0; kv < 2; ++kv) {
          const uint32_t slot = fills % kSlots;
          fine = fine && barrier_wait_warp(smem_address(&C.empty[slot]), ((fills / kSlots) & 1u) ^ 1u, &C.gave_up);
          if (!fine) break;
          now.load(kv ? &P.v_map : &P.k_map, ring + slot * M::kTileBytes, piece.head, smem_address(&C.full[slot]));
          ++fills;
        }
      }
      piece.done();
    }
  } else if (warp == kMmaWarp) {
    uint32_t used = 0;               // ring slots taken before this piece
    uint32_t query_phase[2] = {0, 0}, probability_phase[2] = {0, 0};
    const bool issuer = elected();
    constexpr uint32_t kScores = instruction<T>(kKeys, false), kOutput = instruction<T>(DIM, true);
    while (fine && piece.next()) {
      const TileRange range[2] = {tile_range(P, piece, 0), tile_range(P, piece, 1)};
      const int32_t first = static_cast<int32_t>(piece.first_tile), end = first + static_cast<int32_t>(piece.count);
      // step u: O += P V of unit u, then the scores of unit u + 1, for one row tile after the other
      for (int32_t u = first - 1; fine && u < end; ++u) {
        const uint32_t v_fill = used + 2u * static_cast<uint32_t>(u - first) + 1u, k_fill = v_fill + 1u;
        if (u >= first) {
          const uint32_t slot = v_fill % kSlots;
          fine = barrier_wait_warp(smem_address(&C.full[slot]), (v_fill / kSlots) & 1u, &C.gave_up);
          if (!fine) break;
          // value rows that no row sees may hold anything: 0 x NaN is not 0
          const int32_t key0 = u * kKeys;
          if (key0 < piece.keys.begin || key0 + kKeys > piece.keys.end) {
            const int32_t from = piece.keys.begin - key0, to = piece.keys.end - key0;
            uint8_t* const tile = smem + M::kRing + slot * M::kTileBytes;
            for (uint32_t i = lane; i < kKeys * DIM / 8; i += 32) {
              const int32_t r = static_cast<int32_t>((i >> 3) % kKeys);  // a row has 128 bytes of each 64 elements
              if (r < from || r >= to) *reinterpret_cast<uint4*>(tile + i * 16) = make_uint4(0, 0, 0, 0);
            }
            shared_to_async();
            __syncwarp();
          }
        }
        if (u + 1 < end) {
          fine = barrier_wait_warp(smem_address(&C.full[k_fill % kSlots]), (k_fill / kSlots) & 1u, &C.gave_up);
          if (!fine) break;
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const uint32_t s = tmem + t * 128, o = tmem + 256 + t * 128;
          if (u >= first && range[t].has(u)) {
            fine = fine && barrier_wait_warp(smem_address(&C.probabilities[t]), probability_phase[t], &C.gave_up);
            if (!fine) break;
            probability_phase[t] ^= 1u;
            after_sync();
            if (issuer) {
              const uint64_t v = operand(ring + (v_fill % kSlots) * M::kTileBytes, kKeys * 128 / 16);
#pragma unroll
              for (int k = 0; k < kKeys / 16; ++k)
                product_tensor(o, s + k * 8, v + k * (16 * 128 / 16), kOutput, k > 0 || u > range[t].from);
              if (u + 1 == range[t].to) commit(smem_address(&C.outputs[t]));
            }
            __syncwarp();
          }
          if (range[t].has(u + 1)) {
            if (u + 1 == range[t].from) {
              fine = fine && barrier_wait_warp(smem_address(&C.queries[t]), query_phase[t], &C.gave_up);
              if (!fine) break;
              query_phase[t] ^= 1u;
              after_sync();
            }
            if (issuer) {
              const uint64_t q = operand(base + t * M::kTileBytes, 1);
              const uint64_t k_tile = operand(ring + (k_fill % kSlots) * M::kTileBytes, 1);
#pragma unroll
              for (int k = 0; k < DIM / 16; ++k) {
                const uint32_t at = (k >> 2) * (kTileRows * 128 / 16) + (k & 3) * 2;
                product_shared(s, q + at, k_tile + at, kScores, k > 0);
              }
              commit(smem_address(&C.scores[t]));
            }
            __syncwarp();
          }
        }
        if (issuer && fine) {
          if (u >= first) commit(smem_address(&C.empty[v_fill % kSlots]));
          if (u + 1 < end) commit(smem_address(&C.empty[k_fill % kSlots]));
        }
        __syncwarp();
      }
      used += 2u * piece.count;
      piece.done();
    }
    if (!fine) {
      if (issuer) commit(smem_address(&C.drained));
      barrier_wait_out(smem_address(&C.drained), 0);
    }
  } else if (warp < kMmaWarp) {
    const uint32_t t = warp >> 2, thread = threadIdx.x & 127u;
    const uint32_t lanes = (warp & 3u) << 21;  // this warp's rows of tensor memory: lane 32 x (warp & 3), bits 16 up
    const uint32_t s_at = tmem + t * 128 + lanes, o_at = tmem + 256 + t * 128 + lanes;
    const float ninf = __int_as_float(0xff800000);
    uint32_t score_phase = 0, output_phase = 0;
    while (fine && piece.next()) {
      const TileRange range = tile_range(P, piece, t);
      const uint32_t rows = piece.rows();
      const uint32_t r = t * kTileRows + thread;  // row of the item
      const bool valid = r < rows;
      const uint32_t g = piece.tile * kRows + r;
      const uint32_t token = g / P.group, head = piece.head * P.group + g % P.group;
      float m = ninf, l = 0.f;
      if (range.to > range.from) {
        // queries: consecutive lanes take consecutive parts of a row
        uint8_t* const q_tile = smem + t * M::kTileBytes;
        constexpr uint32_t kParts = DIM / 8;
#pragma unroll 4
        for (uint32_t i = thread; i < kTileRows * kParts; i += 128) {
          const uint32_t row = i / kParts, part = i % kParts;
          const uint32_t gr = piece.tile * kRows + t * kTileRows + row;
          uint4 v = make_uint4(0, 0, 0, 0);
          if (t * kTileRows + row < rows && part * 8 < P.head_dim) {
            const uint32_t tok = gr / P.group;
            v = *reinterpret_cast<const uint4*>(static_cast<const T*>(P.q) + (piece.s.token + static_cast<int64_t>(tok)) * P.q_token +
                                                static_cast<int64_t>(piece.head * P.group + gr - tok * P.group) * P.q_head + part * 8);
          }
          *reinterpret_cast<uint4*>(q_tile + (part >> 3) * (kTileRows * 128) + row * 128 + (((part & 7u) ^ (row & 7u)) << 4)) = v;
        }
        shared_to_async();
        __syncwarp();
        if (lane == 0) barrier_arrive(smem_address(&C.queries[t]));

        const int32_t position = piece.s.length - piece.s.n + static_cast<int32_t>(token);
        int32_t see_from = 0, see_to = 0x7fffffff;
        if (valid) {
          see_to = P.causal ? max(position + 1, 0) : piece.s.length;
          if (P.causal && P.window)
            see_from = static_cast<int32_t>(max(static_cast<int64_t>(0), position + 1 - static_cast<int64_t>(P.window)));
        }
        const int32_t all_from = __reduce_max_sync(0xffffffffu, see_from);
        const int32_t all_to = __reduce_min_sync(0xffffffffu, see_to);

        for (int32_t u = range.from; u < range.to; ++u) {
          fine = barrier_wait_warp(smem_address(&C.scores[t]), score_phase, &C.gave_up);
          if (!fine) break;
          score_phase ^= 1u;
          after_sync();
          const int32_t key0 = u * kKeys;
          const bool tested = key0 < all_from || key0 + kKeys > all_to;
          const int32_t hide_to = see_from - key0, hide_from = see_to - key0;
          // The scores are read twice, a part at a time: once for the maximum, once for the probabilities.
          // All 128 of them in registers spill.
          float top = ninf;
          {
            uint32_t s[2][32];
            load_columns(s_at, s[0]);
#pragma unroll
            for (int i = 0; i < kKeys; i += 32) {
              uint32_t* now = s[(i >> 5) & 1];
              loads_done(now);
              if (i + 32 < kKeys) load_columns(s_at + i + 32, s[((i >> 5) + 1) & 1]);
              if (tested) hide(now, i, hide_to, hide_from);
              float part[4] = {__uint_as_float(now[0]), __uint_as_float(now[1]), __uint_as_float(now[2]), __uint_as_float(now[3])};
#pragma unroll
              for (int j = 4; j < 32; ++j) part[j & 3] = fmaxf(part[j & 3], __uint_as_float(now[j]));
              top = fmaxf(top, fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])));
            }
          }
          if (u == range.from) {
            m = top;
          } else {
            // the scores of this unit are there, so the last unit's O is complete
            const bool rise = (top - m) * P.scale_log2 > kRise;
            if (__any_sync(0xffffffffu, rise)) {
              const float f = rise ? exp2_fast((m - top) * P.scale_log2) : 1.f;
              if (rise) m = top;
              l *= f;
#pragma unroll 1
              for (int i = 0; i < DIM; i += 16) {
                uint32_t o[16];
                load_columns_16(o_at + i, o);
                loads_done_16(o);
#pragma unroll
                for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
                store_columns_16(o_at + i, o);
              }
              stores_done();
            }
          }
          const float shift = m == ninf ? 0.f : m * P.scale_log2;
          float sum[4] = {0.f, 0.f, 0.f, 0.f};
          {
            uint32_t s[2][32];
            load_columns(s_at, s[0]);
#pragma unroll
            for (int i = 0; i < kKeys; i += 32) {
              uint32_t* now = s[(i >> 5) & 1];
              loads_done(now);
              if (i + 32 < kKeys) load_columns(s_at + i + 32, s[((i >> 5) + 1) & 1]);
              if (tested) hide(now, i, hide_to, hide_from);
              uint32_t p[16];
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                const float a = exp2_fast(fmaf(__uint_as_float(now[2 * j]), P.scale_log2, -shift));
                const float b = exp2_fast(fmaf(__uint_as_float(now[2 * j + 1]), P.scale_log2, -shift));
                sum[j & 3] += a + b;
                p[j] = Pair<T>::pack(a, b);  // one rounding to the values' type
              }
              store_columns_16(s_at + i / 2, p);  // over scores that have been read
            }
          }
          l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
          stores_done();
          before_sync();
          __syncwarp();
          if (lane == 0) barrier_arrive(smem_address(&C.probabilities[t]));
        }
        if (!fine) break;
        fine = barrier_wait_warp(smem_address(&C.outputs[t]), output_phase, &C.gave_up);
        if (!fine) break;
        output_phase ^= 1u;
        after_sync();
      }
      const bool any = range.to > range.from;
      const bool complete = piece.begins() && piece.ends();
      if (t * kTileRows < rows) {
        const int64_t at = piece.s.token + static_cast<int64_t>(token);
        const float inverse = l == 0.f ? 0.f : 1.f / l;
        float* slot = complete ? nullptr
                               : P.partial + (2u * blockIdx.x + (piece.begins() ? 1u : 0u)) *
                                                 static_cast<size_t>(kRows * (2 + DIM));
        if (valid) {
          if (!complete)
            *reinterpret_cast<float2*>(slot + r * 2) = make_float2(m, l);
          else if (P.lse)
            P.lse[at * P.kv_heads * P.group + head] = l == 0.f ? ninf : m * P.scale + logf(l);
        }
#pragma unroll 1
        for (int i = 0; i < DIM; i += 32) {
          uint32_t o[32];
          if (any) {
            load_columns(o_at + i, o);
            loads_done(o);
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = 0u;
          }
          if (!valid) continue;
          if (complete) {
            T* to = static_cast<T*>(P.out) + at * P.out_token + static_cast<int64_t>(head) * P.out_head + i;
#pragma unroll
            for (int j = 0; j < 32; j += 8)
              if (static_cast<uint32_t>(i + j) < P.head_dim) {
                uint4 v;
                v.x = Pair<T>::pack(__uint_as_float(o[j]) * inverse, __uint_as_float(o[j + 1]) * inverse);
                v.y = Pair<T>::pack(__uint_as_float(o[j + 2]) * inverse, __uint_as_float(o[j + 3]) * inverse);
                v.z = Pair<T>::pack(__uint_as_float(o[j + 4]) * inverse, __uint_as_float(o[j + 5]) * inverse);
                v.w = Pair<T>::pack(__uint_as_float(o[j + 6]) * inverse, __uint_as_float(o[j + 7]) * inverse);
                *reinterpret_cast<uint4*>(to + j) = v;
              }
          } else {
            uint4* to = reinterpret_cast<uint4*>(slot + kRows * 2 + r * DIM + i);
#pragma unroll
            for (int j = 0; j < 32; j += 4) to[j / 4] = make_uint4(o[j], o[j + 1], o[j + 2], o[j + 3]);
          }
        }
        before_sync();
      }
      if (piece.begins() && !piece.ends())
        header = AttentionHeader{piece.more(share), rows, piece.tile * kRows, piece.head,
                                 static_cast<uint32_t>(piece.s.token), {0, 0, 0}};
      piece.done();
    }
    if (threadIdx.x == 0 && P.headers) P.headers[blockIdx.x] = header;
  }
  before_sync();
  __syncthreads();
  after_sync();
  if (C.gave_up && warp == kLoadWarp) {
    for (uint32_t f = fills > kSlots ? fills - kSlots : 0u; f < fills; ++f)
      barrier_wait_out(smem_address(&C.full[f % kSlots]), (f / kSlots) & 1u);
    if (lane == 0) atomicExch(P.status, 1u);
  }
  if (warp == kMmaWarp)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

}  // namespace paged

size_t many_rows_smem(uint32_t padded_dim) {
  return 1024 + (padded_dim == 64 ? paged::ManySmem<64>::kBytes : paged::ManySmem<128>::kBytes);
}
namespace {
template <typename T, int DIM>
cudaError_t prepare() {
  // setmaxnreg.inc would wait for good if the launch brought fewer registers than its warps share out
  cudaFuncAttributes a;
  const cudaError_t e = cudaFuncGetAttributes(&a, paged::many_rows_kernel<T, DIM>);
  if (e != cudaSuccess) return e;
  if (a.numRegs < static_cast<int>(paged::kLaunchRegisters)) return cudaErrorInvalidDeviceFunction;
  return cudaFuncSetAttribute(paged::many_rows_kernel<T, DIM>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              static_cast<int>(many_rows_smem(DIM)));
}
template <typename T, int DIM>
cudaError_t launch(const AttentionParams& p, const AttentionPlan& plan, cudaStream_t stream) {
  return launch_dependent(paged::many_rows_kernel<T, DIM>, dim3(plan.ctas), paged::kThreadsMany, many_rows_smem(DIM), p,
                          stream);
}
}  // namespace
cudaError_t prepare_many_rows() {
  for (cudaError_t e : {prepare<__half, 64>(), prepare<__half, 128>(), prepare<__nv_bfloat16, 64>(),
                        prepare<__nv_bfloat16, 128>()})
    if (e != cudaSuccess) return e;
  return cudaSuccess;
}
cudaError_t launch_many_rows(const AttentionParams& p, const AttentionPlan& plan, bool bf16, cudaStream_t stream) {
  if (bf16)
    return plan.padded_dim == 64 ? launch<__nv_bfloat16, 64>(p, plan, stream) : launch<__nv_bfloat16, 128>(p, plan, stream);
  return plan.padded_dim == 64 ? launch<__half, 64>(p, plan, stream) : launch<__half, 128>(p, plan, stream);
}

}  // namespace mononn
