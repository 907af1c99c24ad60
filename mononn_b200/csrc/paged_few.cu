// Attention over a paged cache for few rows: single tokens, a few drafted ones, grouped heads.
//
// o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m), s_j = scale q.k_j, in one pass over the keys with the
// running maximum m and sum of every row. The rows of an item (new tokens x query heads that share a key
// head) fill one 16-row matrix instruction; each of four warps takes a quarter of every unit's keys (64, or 128 of 64-wide
// heads: 16 KB) and keeps a maximum, a sum and an output of its own, which are added up when the item ends.
// The keys are read once, and that bounds it: two loading warps keep 32 to 64 KB of each CTA on their way, two CTAs an SM. The
// rows are far too few for the 128 of a tensor-memory product, and the 16-row instruction needs no round trip
// through it. 32 sequences of 500 to 8000 keys, 8 key heads of 128: 558 MB in 92 us (0.93 of what a copy reaches; with the
// join); 48 of 60 to 2000 keys, 32 heads of 64: 406 MB in 70 us; one of 150001 keys: 307 MB in 56 us; the rest are some 7 us
// at the begin and the end (launch, shares, first keys, join): a single sequence of 300 keys takes 6.9 us.
#include "paged_device.h"

namespace mononn {
namespace paged {

constexpr int kWarps = 4;   // that compute
constexpr int kThreadsFew = (kWarps + 2) * 32;  // one more that loads keys, one that loads values
constexpr int kPieces = 2;  // told ahead
constexpr int kRows = static_cast<int>(kFewRows);

template <int DIM>
struct FewShape {
  static constexpr int kKeys = static_cast<int>(few_keys(DIM));  // of a unit; 16 KB of keys
  static constexpr int kEach = kKeys / kWarps;                   // of a warp
  static constexpr int kSlotBytes = kKeys * DIM * 2;
  static constexpr int kSlots = 4;        // 0, 2: keys, 1, 3: values of a unit
  static constexpr int kPitch = DIM + 8;  // floats between rows of the warps' outputs: no bank conflicts
  static constexpr int kQueries = kSlots * kSlotBytes, kQueryBytes = kRows * DIM * 2;
  static constexpr int kOutputs = kQueries + kPieces * kQueryBytes;
  static constexpr int kControl = kOutputs + kWarps * kRows * kPitch * 4;
  static constexpr int kSmem = 1024 + kControl + 1280;
};
struct FewControl {
  uint64_t full[4], empty[4], told[kPieces], queries[kPieces], taken[kPieces], meeting;
  alignas(16) Piece pieces[kPieces];
  Share share;
  uint32_t sums[kWarps + 2];
  uint32_t gave_up;
  float maxima[kWarps][kRows], totals[kWarps][kRows];
};
static_assert(sizeof(FewControl) <= 1280, "control block");
static_assert(FewShape<128>::kSmem <= 113 * 1024 && FewShape<64>::kSmem <= 113 * 1024, "two CTAs share an SM");

__device__ __forceinline__ void matrices_4(uint32_t address, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(address)
               : "memory");
}
__device__ __forceinline__ void matrices_4_transposed(uint32_t address, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(address)
               : "memory");
}
template <typename T>
__device__ __forceinline__ void multiply(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void multiply<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void multiply<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The warps that compute, bounded like every other wait.
__device__ __forceinline__ bool warps_meet(uint32_t bar, uint32_t& phase, volatile uint32_t* gave_up) {
  __syncwarp();
  if ((threadIdx.x & 31u) == 0u) barrier_arrive(bar);
  const bool fine = barrier_wait_warp(bar, phase, gave_up);
  phase ^= 1u;
  return fine;
}

template <typename T, int DIM>
__global__ void __launch_bounds__(kThreadsFew, 2) few_rows_kernel(const __grid_constant__ AttentionParams P) {
  extern __shared__ uint8_t raw[];
  using S = FewShape<DIM>;
  constexpr int kHalves = DIM / 64, kSteps = DIM / 16, kSlots = S::kSlots, kKeys = S::kKeys, kEach = S::kEach;
  uint8_t* smem = raw + ((1024u - (smem_address(raw) & 1023u)) & 1023u);
  FewControl& C = *reinterpret_cast<FewControl*>(smem + S::kControl);
  const uint32_t slots = smem_address(smem);
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kSlots; ++i) {
      barrier_init(P, kBarrierFull, C.full[i], 1);
      barrier_init(P, kBarrierEmpty, C.empty[i], kWarps);
    }
    for (int i = 0; i < kPieces; ++i) {
      barrier_init(P, kBarrierTold, C.told[i], 1);
      barrier_init(P, kBarrierQueries, C.queries[i], 32);
      barrier_init(P, kBarrierTaken, C.taken[i], kWarps + 1);
    }
    barrier_init(P, kBarrierMeeting, C.meeting, kWarps);
    C.gave_up = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&P.k_map));
    asm volatile("prefetch.tensormap [%0];" ::"l"(&P.v_map));
  }
  let_next_begin();
  earlier_done();
  find_share<kKeys, kThreadsFew>(P, C.sums, &C.share);  // barriers of the CTA within
  // Slots 0, 2, .. hold keys, 1, 3, .. values.
  constexpr uint32_t kPairs = kSlots / 2;
  uint32_t fills = 0;  // of this loading warp

  if (warp == kWarps) {
    TileLoader<kKeys, kHalves> loader(P);
    Walker<kKeys> walk(P, C.share);
    bool fine = true;
    for (uint32_t i = 0; fine; ++i) {
      const bool some = walk.next();
      if (some) loader.begin(walk.piece);
      const uint32_t at = i % kPieces;
      fine = barrier_wait_warp(smem_address(&C.taken[at]), ((i / kPieces) & 1u) ^ 1u, &C.gave_up);
      if (!fine) break;
      put_piece(&C.pieces[at], walk.piece, lane);
      if (lane == 0) barrier_arrive(smem_address(&C.told[at]));
      __syncwarp();
      if (!some) break;
      for (int32_t u = 0; u < walk.piece.count; ++u) {
        const uint32_t slot = fills % kPairs * 2u;
        fine = barrier_wait_warp(smem_address(&C.empty[slot]), ((fills / kPairs) & 1u) ^ 1u, &C.gave_up);
        if (!fine) break;
        loader.load(&P.k_map, walk.piece.tile + u, slots + slot * S::kSlotBytes, walk.piece.head, smem_address(&C.full[slot]));
        ++fills;
        if (u == 0) {  // the queries, behind the first keys: consecutive lanes along a row
          constexpr uint32_t kParts = DIM / 8;
          const uint32_t tile = slots + S::kQueries + at * S::kQueryBytes;
#pragma unroll 4
          for (uint32_t j = lane; j < kRows * kParts; j += 32) {
            const uint32_t row = j / kParts, part = j % kParts, g = walk.piece.first_row + row, token = divide(g, P.by_group);
            const bool wanted = row < walk.piece.rows && part * 8 < P.head_dim;
            const T* src = static_cast<const T*>(P.q);
            if (wanted)
              src += (walk.piece.token + static_cast<int64_t>(token)) * P.q_token +
                     static_cast<int64_t>(walk.piece.head * P.group + g - token * P.group) * P.q_head + part * 8;
            copy_16(tile + (part >> 3) * (kRows * 128) + row * 128 + (((part & 7u) ^ (row & 7u)) << 4), src, wanted);
          }
          arrive_after_copies(smem_address(&C.queries[at]));
        }
      }
    }
    if (lane == 0 && P.headers) walk.write_header();
  } else if (warp == kWarps + 1) {
    TileLoader<kKeys, kHalves> loader(P);
    bool fine = true;
    for (uint32_t i = 0; fine; ++i) {
      const uint32_t at = i % kPieces;
      fine = barrier_wait_warp(smem_address(&C.told[at]), (i / kPieces) & 1u, &C.gave_up);
      const Piece& piece = C.pieces[at];
      if (!fine || piece.valid == 0) break;
      const int32_t tile = piece.tile, count = piece.count;
      const uint32_t head = piece.head;
      loader.begin(piece);
      __syncwarp();
      if (lane == 0) barrier_arrive(smem_address(&C.taken[at]));
      for (int32_t u = 0; u < count; ++u) {
        const uint32_t slot = fills % kPairs * 2u + 1u;
        fine = barrier_wait_warp(smem_address(&C.empty[slot]), ((fills / kPairs) & 1u) ^ 1u, &C.gave_up);
        if (!fine) break;
        loader.load(&P.v_map, tile + u, slots + slot * S::kSlotBytes, head, smem_address(&C.full[slot]));
        ++fills;
      }
    }
  } else {
    const float ninf = __int_as_float(0xff800000);
    uint32_t slot = 0, parity = 0, meetings = 0;
    float* const outputs = reinterpret_cast<float*>(smem + S::kOutputs);
    // ldmatrix addresses: lanes 0-7, 8-15, .. point at the rows of the four 8 x 8 matrices
    const uint32_t key_row = warp * kEach + (lane & 7u) + ((lane >> 4) << 3), key_chunk = (lane >> 3) & 1u;
    const uint32_t val_row = warp * kEach + (lane & 15u), val_chunk = lane >> 4;
    const uint32_t query_row = lane & 15u, query_chunk = lane >> 4;
    for (uint32_t n = 0;; ++n) {
      const uint32_t at = n % kPieces;
      if (!barrier_wait_warp(smem_address(&C.told[at]), (n / kPieces) & 1u, &C.gave_up)) break;
      const Piece& piece = C.pieces[at];
      if (piece.valid == 0) break;
      const int32_t count = piece.count, tile0 = piece.tile, keys_begin = piece.keys_begin, keys_end = piece.keys_end;
      if (!barrier_wait_warp(smem_address(&C.queries[at]), (n / kPieces) & 1u, &C.gave_up)) break;
      const uint32_t queries = slots + S::kQueries + at * S::kQueryBytes + query_row * 128;
      uint32_t q[kSteps][4];
#pragma unroll
      for (int k = 0; k < kSteps; ++k)
        matrices_4(queries + (k >> 2) * (kRows * 128) + ((((k & 3) * 2 + query_chunk) ^ (query_row & 7u)) << 4), q[k]);
      int32_t see_from[2], see_to[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t r = (lane >> 2) + 8 * i;
        const bool valid = r < piece.rows;
        const int32_t position = piece.length - piece.n + static_cast<int32_t>(divide(piece.first_row + r, P.by_group));
        see_from[i] = 0;
        see_to[i] = 0x7fffffff;
        if (valid) seen_keys(P, position, piece.length, see_from[i], see_to[i]);
      }
      // keys that every row sees need no test
      const int32_t all_from = __reduce_max_sync(0xffffffffu, max(see_from[0], see_from[1]));
      const int32_t all_to = __reduce_min_sync(0xffffffffu, min(see_to[0], see_to[1]));

      float acc[kSteps * 2][4];
#pragma unroll
      for (int i = 0; i < kSteps * 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
      float m[2] = {ninf, ninf}, l[2] = {0.f, 0.f};

      for (int32_t u = 0; u < count; ++u) {
        const int32_t key0 = (tile0 + u) * kKeys + static_cast<int32_t>(warp) * kEach;
        const bool any = key0 < keys_end && key0 + kEach > keys_begin;
        const bool tested = key0 < all_from || key0 + kEach > all_to;
        float s[kEach / 8][4];
#pragma unroll
        for (int i = 0; i < kEach / 8; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
        if (!barrier_wait_warp(smem_address(&C.full[slot]), parity, &C.gave_up)) break;
        if (any) {
          const uint32_t base = slots + slot * S::kSlotBytes + key_row * 128;
#pragma unroll
          for (int k = 0; k < kSteps; ++k)
#pragma unroll
            for (int i = 0; i < kEach / 16; ++i) {
              uint32_t b[4];
              const uint32_t chunk = (k & 3) * 2 + key_chunk;
              matrices_4(base + (k >> 2) * kKeys * 128 + i * 16 * 128 + ((chunk ^ (key_row & 7u)) << 4), b);
              multiply<T>(s[2 * i], q[k], b[0], b[1]);
              multiply<T>(s[2 * i + 1], q[k], b[2], b[3]);
            }
        }
        __syncwarp();
        if (lane == 0) barrier_arrive(smem_address(&C.empty[slot]));
        if (++slot == kSlots) slot = 0, parity ^= 1u;

        uint32_t p[kEach / 16][4];
        if (any) {
          if (tested) {
#pragma unroll
            for (int i = 0; i < kEach / 8; ++i)
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const int32_t key = key0 + i * 8 + (lane & 3u) * 2 + (j & 1);
                if (key < see_from[j >> 1] || key >= see_to[j >> 1]) s[i][j] = ninf;
              }
          }
          float top[2];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            top[r] = m[r];
#pragma unroll
            for (int i = 0; i < kEach / 8; ++i) top[r] = fmaxf(top[r], fmaxf(s[i][r * 2], s[i][r * 2 + 1]));
            top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
            top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
          }
          if (__any_sync(0xffffffffu, top[0] != m[0] || top[1] != m[1])) {
            float f[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              f[r] = top[r] == m[r] ? 1.f : exp2_fast((m[r] - top[r]) * P.scale_log2);
              m[r] = top[r];
              l[r] *= f[r];
            }
#pragma unroll
            for (int i = 0; i < kSteps * 2; ++i) {
              acc[i][0] *= f[0];
              acc[i][1] *= f[0];
              acc[i][2] *= f[1];
              acc[i][3] *= f[1];
            }
          }
          // a row that has seen nothing yet: exp2(-inf - 0) = 0
          const float shift[2] = {m[0] == ninf ? 0.f : m[0] * P.scale_log2, m[1] == ninf ? 0.f : m[1] * P.scale_log2};
#pragma unroll
          for (int i = 0; i < kEach / 8; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              s[i][j] = exp2_fast(fmaf(s[i][j], P.scale_log2, -shift[j >> 1]));
              l[j >> 1] += s[i][j];
            }
            // the probabilities take the values' type for the product: one rounding of half a step each
            p[i / 2][(i & 1) * 2] = Pair<T>::pack(s[i][0], s[i][1]);
            p[i / 2][(i & 1) * 2 + 1] = Pair<T>::pack(s[i][2], s[i][3]);
          }
        }
        if (!barrier_wait_warp(smem_address(&C.full[slot]), parity, &C.gave_up)) break;
        if (any) {
          const uint32_t base = slots + slot * S::kSlotBytes + val_row * 128;
          // value rows that no row of the item sees may hold anything: 0 x NaN is not 0
          const bool clear = key0 < keys_begin || key0 + kEach > keys_end;
#pragma unroll
          for (int i = 0; i < kEach / 16; ++i) {
            uint32_t keep[2] = {0xffffffffu, 0xffffffffu};
            if (clear) {
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                const int32_t key = key0 + i * 16 + j * 8 + (lane & 3u) * 2;
                const bool a = key >= keys_begin && key < keys_end;
                const bool b = key + 1 >= keys_begin && key + 1 < keys_end;
                keep[j] = (a ? 0xffffu : 0u) | (b ? 0xffff0000u : 0u);
              }
            }
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
              uint32_t b[4];
              const uint32_t chunk = (k & 3) * 2 + val_chunk;
              matrices_4_transposed(base + (k >> 2) * kKeys * 128 + i * 16 * 128 + ((chunk ^ (val_row & 7u)) << 4), b);
              multiply<T>(acc[k * 2], p[i], b[0] & keep[0], b[1] & keep[1]);
              multiply<T>(acc[k * 2 + 1], p[i], b[2] & keep[0], b[3] & keep[1]);
            }
          }
        }
        __syncwarp();
        if (lane == 0) barrier_arrive(smem_address(&C.empty[slot]));
        if (++slot == kSlots) slot = 0, parity ^= 1u;
      }

      // the four warps' results
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      }
      const uint32_t rows = piece.rows;
      if (!warps_meet(smem_address(&C.meeting), meetings, &C.gave_up)) break;  // the last piece's have been read
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint32_t row = (lane >> 2) + 8 * r;
        if (row < rows) {
          if ((lane & 3u) == 0) {
            C.maxima[warp][row] = m[r];
            C.totals[warp][row] = l[r];
          }
          float* to = outputs + (warp * kRows + row) * S::kPitch + (lane & 3u) * 2;
#pragma unroll
          for (int i = 0; i < kSteps * 2; ++i)
            *reinterpret_cast<float2*>(to + i * 8) = make_float2(acc[i][r * 2], acc[i][r * 2 + 1]);
        }
      }
      if (!warps_meet(smem_address(&C.meeting), meetings, &C.gave_up)) break;
      const bool complete = piece.begins && piece.ends;
      float* slot_out = nullptr;
      if (!complete)
        slot_out = P.partial + (2u * blockIdx.x + (piece.begins ? 1u : 0u)) * static_cast<size_t>(kRows * (2 + DIM));
      for (uint32_t i = threadIdx.x; i < rows * (DIM / 8); i += kWarps * 32) {
        const uint32_t row = i / (DIM / 8), d = (i % (DIM / 8)) * 8;
        float top = C.maxima[0][row];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) top = fmaxf(top, C.maxima[w][row]);
        float sum = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float mw = C.maxima[w][row];
          const float f = mw == ninf ? 0.f : exp2_fast((mw - top) * P.scale_log2);
          sum += f * C.totals[w][row];
          const float4* from = reinterpret_cast<const float4*>(outputs + (w * kRows + row) * S::kPitch + d);
          const float4 a = from[0], b = from[1];
          o[0] += f * a.x; o[1] += f * a.y; o[2] += f * a.z; o[3] += f * a.w;
          o[4] += f * b.x; o[5] += f * b.y; o[6] += f * b.z; o[7] += f * b.w;
        }
        if (complete) {
          const uint32_t g = piece.first_row + row;
          const uint32_t of = divide(g, P.by_group);
          const int64_t token = piece.token + static_cast<int64_t>(of);
          const uint32_t head = piece.head * P.group + (g - of * P.group);
          const float inverse = inverse_of(top, sum);
          if (d < P.head_dim) {
            uint4 v;
            v.x = Pair<T>::pack(o[0] * inverse, o[1] * inverse);
            v.y = Pair<T>::pack(o[2] * inverse, o[3] * inverse);
            v.z = Pair<T>::pack(o[4] * inverse, o[5] * inverse);
            v.w = Pair<T>::pack(o[6] * inverse, o[7] * inverse);
            *reinterpret_cast<uint4*>(static_cast<T*>(P.out) + token * P.out_token +
                                      static_cast<int64_t>(head) * P.out_head + d) = v;
          }
          if (d == 0 && P.lse)
            P.lse[token * P.kv_heads * P.group + head] = log_sum(top, sum, P.scale);
        } else {
          if (d == 0) {
            slot_out[row * 2] = top;
            slot_out[row * 2 + 1] = sum;
          }
          float4* to = reinterpret_cast<float4*>(slot_out + kRows * 2 + row * DIM + d);
          to[0] = make_float4(o[0], o[1], o[2], o[3]);
          to[1] = make_float4(o[4], o[5], o[6], o[7]);
        }
      }
      __syncwarp();
      if (lane == 0) barrier_arrive(smem_address(&C.taken[at]));
    }
  }
  __syncthreads();
  if (C.gave_up && warp >= kWarps) {
    asm volatile("cp.async.wait_all;" ::: "memory");
    for (uint32_t f = fills > kPairs ? fills - kPairs : 0u; f < fills; ++f)
      barrier_wait_out(smem_address(&C.full[f % kPairs * 2u + (warp - kWarps)]), (f / kPairs) & 1u);
    if (lane == 0) atomicExch(P.status, 1u);
  }
}

// Joins the pieces of the items that span CTAs: o = sum_i f_i o_i / sum_i f_i l_i, f_i = exp(m_i - m),
// in the order of the keys. Block (CTA, y): rows y, y + the number of blocks, .. (in groups of the rows that a block
// takes at once) of the item that begins in that CTA. A warp for each row, or, where items are few and cut into many
// pieces, all of a block with a part of the pieces each.
constexpr int kJoinWarps = 8;
// Blocks of a CTA's item. Few rows: 16 rows are rare, and blocks without any cost (decode of 32 sequences, 4 rows: 90.3 us
// with 4 blocks, 91.3 with 16; one long document, 8 rows: 60.0 and 58.6); many rows: one for each 8 (2 us less than 8 blocks).
constexpr uint32_t kJoinBlocksFew = 8, kJoinBlocksMany = kManyRows / kJoinWarps;
template <typename T, int DIM, int ROWS, int PARTS>
__global__ void __launch_bounds__(kJoinWarps * 32) join_kernel(const __grid_constant__ AttentionParams P) {
  constexpr uint32_t kRowsHere = kJoinWarps / PARTS;
  constexpr int kEach = DIM / 32;  // consecutive elements of a lane
  __shared__ float sums[PARTS > 1 ? kJoinWarps : 1][DIM];
  __shared__ float tops[kJoinWarps], totals[kJoinWarps];
  earlier_done();
  const AttentionHeader h = P.headers[blockIdx.x];
  if (h.more == 0) return;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, part = warp % PARTS;
  const float ninf = __int_as_float(0xff800000);
  constexpr size_t kSlot = static_cast<size_t>(ROWS) * (2 + DIM);
  const uint32_t pieces = h.more + 1u;
  const uint32_t first = pieces * part / PARTS, last = pieces * (part + 1u) / PARTS;
#pragma unroll 1
  for (uint32_t row0 = blockIdx.y * kRowsHere; row0 < h.rows; row0 += gridDim.y * kRowsHere) {
    const uint32_t row = row0 + warp / PARTS;
    const bool valid = row < h.rows;
    float top = ninf, total = 0.f, o[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) o[i] = 0.f;
    if (valid) {
#pragma unroll 4
      for (uint32_t i = first; i < last; ++i) {
        const float* slot = P.partial + (2u * (blockIdx.x + i) + (i == 0 ? 1u : 0u)) * kSlot;
        const float2 ml = *reinterpret_cast<const float2*>(slot + row * 2);
        const float* from = slot + ROWS * 2 + row * DIM + lane * kEach;
        float v[kEach];
        if constexpr (kEach == 4) {
          const float4 a = *reinterpret_cast<const float4*>(from);
          v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        } else {
          const float2 a = *reinterpret_cast<const float2*>(from);
          v[0] = a.x; v[1] = a.y;
        }
        const float next = fmaxf(top, ml.x);
        const float keep = top == next ? 1.f : exp2_fast((top - next) * P.scale_log2);
        const float f = ml.x == next ? (next == ninf ? 0.f : 1.f) : exp2_fast((ml.x - next) * P.scale_log2);
        top = next;
        total = total * keep + f * ml.y;
#pragma unroll
        for (int j = 0; j < kEach; ++j) o[j] = o[j] * keep + f * v[j];
      }
    }
    if constexpr (PARTS > 1) {
      if (lane == 0) tops[warp] = top, totals[warp] = total;
#pragma unroll
      for (int j = 0; j < kEach; ++j) sums[warp][lane * kEach + j] = o[j];
      __syncthreads();
      if (part == 0) {
#pragma unroll
        for (int p = 1; p < PARTS; ++p) top = fmaxf(top, tops[warp + p]);
        total = 0.f;
#pragma unroll
        for (int j = 0; j < kEach; ++j) o[j] = 0.f;
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
          const float mp = tops[warp + p];
          const float f = mp == ninf ? 0.f : exp2_fast((mp - top) * P.scale_log2);
          total += f * totals[warp + p];
#pragma unroll
          for (int j = 0; j < kEach; ++j) o[j] += f * sums[warp + p][lane * kEach + j];
        }
      }
      __syncthreads();
    }
    if (part != 0 || !valid) continue;
    const uint32_t g = h.first_row + row;
    const uint32_t of = divide(g, P.by_group);
    const int64_t token = static_cast<int64_t>(h.token) + of;
    const uint32_t head = h.head * P.group + (g - of * P.group);
    const float inverse = inverse_of(top, total);
    const uint32_t d = lane * kEach;
    if (d < P.head_dim) {
      uint32_t* to = reinterpret_cast<uint32_t*>(static_cast<T*>(P.out) + token * P.out_token +
                                                 static_cast<int64_t>(head) * P.out_head + d);
#pragma unroll
      for (int j = 0; j < kEach; j += 2) to[j / 2] = Pair<T>::pack(o[j] * inverse, o[j + 1] * inverse);
    }
    if (lane == 0 && P.lse)
      P.lse[token * P.kv_heads * P.group + head] = log_sum(top, total, P.scale);
  }
}

}  // namespace paged

static __device__ uint32_t g_status;
cudaError_t paged_status_word(uint32_t** out) { return cudaGetSymbolAddress(reinterpret_cast<void**>(out), g_status); }

namespace {
template <typename T, int DIM>
cudaError_t prepare() {
  cudaFuncAttributes a;
  for (cudaError_t e : {cudaFuncGetAttributes(&a, paged::join_kernel<T, DIM, static_cast<int>(kFewRows), paged::kJoinWarps>),
                        cudaFuncGetAttributes(&a, paged::join_kernel<T, DIM, static_cast<int>(kManyRows), 1>)})
    if (e != cudaSuccess) return e;
  return cudaFuncSetAttribute(paged::few_rows_kernel<T, DIM>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              paged::FewShape<DIM>::kSmem);
}
template <typename T, int DIM>
cudaError_t launch(const AttentionParams& p, const AttentionPlan& plan, cudaStream_t stream) {
  return launch_dependent(paged::few_rows_kernel<T, DIM>, dim3(plan.ctas), paged::kThreadsFew, paged::FewShape<DIM>::kSmem, p,
                          stream);
}
template <typename T, int DIM>
cudaError_t join(const AttentionParams& p, const AttentionPlan& plan, cudaStream_t stream) {
  if (plan.many)
    return launch_dependent(paged::join_kernel<T, DIM, static_cast<int>(kManyRows), 1>,
                            dim3(plan.ctas, paged::kJoinBlocksMany), paged::kJoinWarps * 32, 0, p, stream);
  return launch_dependent(paged::join_kernel<T, DIM, static_cast<int>(kFewRows), paged::kJoinWarps>,
                          dim3(plan.ctas, paged::kJoinBlocksFew), paged::kJoinWarps * 32, 0, p, stream);
}
}  // namespace

cudaError_t prepare_few_rows() {
  for (cudaError_t e : {prepare<__half, 64>(), prepare<__half, 128>(), prepare<__nv_bfloat16, 64>(),
                        prepare<__nv_bfloat16, 128>()})
    if (e != cudaSuccess) return e;
  return cudaSuccess;
}
cudaError_t launch_few_rows(const AttentionParams& p, const AttentionPlan& plan, bool bf16, cudaStream_t stream) {
  if (bf16)
    return plan.padded_dim == 64 ? launch<__nv_bfloat16, 64>(p, plan, stream) : launch<__nv_bfloat16, 128>(p, plan, stream);
  return plan.padded_dim == 64 ? launch<__half, 64>(p, plan, stream) : launch<__half, 128>(p, plan, stream);
}
cudaError_t launch_join(const AttentionParams& p, const AttentionPlan& plan, bool bf16, cudaStream_t stream) {
  if (bf16) return plan.padded_dim == 64 ? join<__nv_bfloat16, 64>(p, plan, stream) : join<__nv_bfloat16, 128>(p, plan, stream);
  return plan.padded_dim == 64 ? join<__half, 64>(p, plan, stream) : join<__half, 128>(p, plan, stream);
}

}  // namespace mononn
