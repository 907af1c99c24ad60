// Attention over a paged cache for many rows: prompts, chunks of prompts, drafts of wide groups.
//
// o = sum_j p_j v_j / sum_j p_j, p_j = exp2(c (s_j - r)), s_j = q.k_j, c = scale log2(e): any reference r of a row gives
// the same o, so r need not be the maximum, only near enough that no p_j is too large. One pass over the keys, on
// the fifth-generation tensor cores. An item has up to 256 rows, two tiles of 128; a unit is 128 keys, loaded once
// for both. Roles of a CTA (one per SM):
//   warps 4-7, 8-11 the softmax of one row tile each, a thread to a row: scores from tensor memory, probabilities
//                   back to tensor memory, row sums in registers
//   warp 0          issues the matrix products: S = Q K^T (both operands in shared memory), O += P V (P in
//                   tensor memory: in the place of the scores it was made from, or beside them for 64-wide heads)
//   warps 1, 2      load keys (and queries) and values, page by page, into a ring of tiles
// While one row tile's softmax runs, the tensor cores work on the other's products. O stays in tensor memory. It is
// rescaled only when a probability may be above 2^8: until then they are above 1, which costs no accuracy.
//
// 8192 queries x 8192 keys x 8 heads of 128: 222 us, 1240 TFLOP/s (0.76 of what a large matrix product reaches in such a
// short run; the tensor cores are active in 0.66 of the cycles). 32 heads of 64: 680 us, 810 TFLOP/s. What bounds it is the
// chain of a row tile: scores, softmax of 128 of them a thread (about 1600 of some 3300 cycles a unit), product with the
// values, next scores, which have no other place with 128-wide heads (all 512 columns are used). It does not get
// shorter by halving the units (next scores early, but products of 64 keys read 1.5 times as much shared memory: 228), by two
// issuing warps (279), or by handing over the probabilities in halves (238); more exponentials by polynomial: 234. 64-wide
// heads: exponentials and the 8 warps' other instructions, 0.55 of the special-function units' rate. Drafts: the keys, read at
// 5.5 to 6 TB/s once they are on their way; 16 of 3 to 8 tokens over 700 to 6000 keys 55 us.
#include "paged_device.h"

namespace mononn {
namespace paged {

constexpr int kRows = static_cast<int>(kManyRows), kKeys = static_cast<int>(kManyKeys);
constexpr int kThreadsMany = 384;
// The warps that issue and load come first: the scheduler prefers them, and they are on everybody's path. Warp 3 only makes
// up the group whose registers go to the others.
constexpr int kMmaWarp = 0, kKeyWarp = 1, kValueWarp = 2, kSoftmaxWarp = 4;
constexpr int kPieces = 4;                  // told ahead
constexpr uint32_t kSoftmaxRegisters = 216, kOtherRegisters = 72, kLaunchRegisters = 168;
static_assert(256 * kSoftmaxRegisters + 128 * kOtherRegisters <= kThreadsMany * kLaunchRegisters, "register split");
constexpr float kRise = 8.0f;  // 64-wide heads: how far a maximum may be above the reference, in powers of two
// Heads of 65 to 128: of the probabilities of a unit, by the reference that their row has. Above, the unit is done again by a
// higher one. A sum is there anyway, and no probability is above it, so the maxima are left out: they are on the chain from
// one unit's scores to the next one's (8192 x 8192 x 8 heads of 128: 236 us with them, 222 without). 64-wide heads keep them: their
// scores would make room only when the sum is known (6 prompts of 2048, 32 heads: 179 us with the maxima, 185 without).
constexpr float kMostSum = 256.0f;

template <int DIM>
struct ManySmem {
  static constexpr int kTileBytes = static_cast<int>(kTileRows) * DIM * 2;  // of queries, keys or values
  // A slot of the ring holds the values of one unit and the keys of the next: what one step of the products needs.
  static constexpr int kPairs = DIM == 64 ? 4 : 2;
  static constexpr int kRing = 2 * kTileBytes;
  static constexpr int kStage = kRing + 2 * kPairs * kTileBytes;  // 4 KB of each softmax warp, for its rows' way out
  static constexpr int kControl = kStage + 8 * 4096;
  static constexpr int kBytes = kControl + 1024;
  // Tensor memory, 512 columns: 128 of scores and DIM of outputs for each row tile. The probabilities (64
  // columns) have a place of their own where DIM leaves one, otherwise that of the scores.
  static constexpr bool kApart = DIM == 64;
  static __device__ __forceinline__ uint32_t score_column(uint32_t t) { return t * 128; }
  static __device__ __forceinline__ uint32_t probability_column(uint32_t t) { return kApart ? 256 + t * 64 : t * 128; }
  static __device__ __forceinline__ uint32_t output_column(uint32_t t) { return kApart ? 384 + t * 64 : 256 + t * 128; }
};
struct ManyControl {
  uint64_t full[4], empty[4];  // of pairs
  uint64_t scores[2], scores_read[2], probabilities[2], outputs[2], queries[2], queries_free[2];  // of row tiles
  uint64_t told[kPieces], taken[kPieces], drained;
  uint64_t other_done, other_read;  // of two row tiles that hold the same rows, the second
  alignas(16) Piece pieces[kPieces], deferred;
  Share share;
  uint32_t sums[12];
  uint32_t gave_up, tmem;
};
static_assert(sizeof(ManyControl) <= 1024, "control block");
static_assert(ManySmem<128>::kBytes + 1024 <= 227 * 1024, "shared memory");

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
// The registers of a load that an earlier wait covered: nothing that uses them moves before it.
__device__ __forceinline__ void loaded(uint32_t* r) {
  asm volatile("" : MONONN_P8(r, 0), MONONN_P8(r, 8), MONONN_P8(r, 16), MONONN_P8(r, 24)::"memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ void store_columns(uint32_t address, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::MONONN_I8(r, 0),
      MONONN_I8(r, 8), MONONN_I8(r, 16), MONONN_I8(r, 24), "r"(address)
      : "memory");
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
__device__ __forceinline__ void hide(uint32_t (&s)[32], int32_t to, int32_t from) {
  const uint32_t seen = (to <= 0 ? 0xffffffffu : to >= 32 ? 0u : 0xffffffffu << to) &
                        (from <= 0 ? 0u : from >= 32 ? 0xffffffffu : ~(0xffffffffu << from));
#pragma unroll
  for (int j = 0; j < 32; ++j)
    if (!(seen & (1u << j))) s[j] = 0xff800000u;
}
// Highest of 32 scores in four parts.
__device__ __forceinline__ void highest_32(const uint32_t* s, float (&part)[4]) {
#pragma unroll
  for (int j = 0; j < 32; j += 8)
#pragma unroll
    for (int i = 0; i < 4; ++i) part[i] = max3(part[i], __uint_as_float(s[j + 2 * i]), __uint_as_float(s[j + 2 * i + 1]));
}
__device__ __forceinline__ uint64_t two(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 apart(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t multiply_add_two(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add_two(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t multiply_two(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float at_least(float x, float low) {  // NaN stays NaN
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(low));
  return r;
}
__device__ __forceinline__ float within(float x, float low, float high) {  // NaN stays NaN
  float r;
  asm("{\n\t.reg .f32 t;\n\tmax.NaN.f32 t, %1, %2;\n\tmin.NaN.f32 %0, t, %3;\n\t}" : "=f"(r) : "f"(x), "f"(low), "f"(high));
  return r;
}
// Kept in its order, which is that of the loop below: the exponentials of one group beside the sums of the last.
__device__ __forceinline__ float exp2_in_order(float x) {
  float y;
  asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 2^x for two x on the arithmetic pipes: 2^n from the integer nearest to x, times a polynomial of degree
// 4 on -1/2 .. 1/2 (smallest largest relative error, 2.6e-6, found by exchange of its extrema). Below -126.5
// it is 0, as for a key that is hidden; from 127.5 on it is infinite.
template <bool BOUNDED>
__device__ __forceinline__ float2 exp2_polynomial(uint64_t x) {
  const float2 v = apart(x);
  x = BOUNDED ? two(at_least(v.x, -127.f), at_least(v.y, -127.f))
              : two(within(v.x, -127.f, 128.f), within(v.y, -127.f, 128.f));
  const uint64_t moved = add_two(x, two(12582912.f, 12582912.f));  // 1.5 x 2^23: the integer is in the low bits
  const uint64_t whole = add_two(moved, two(-12582912.f, -12582912.f));
  const uint64_t f = multiply_add_two(whole, two(-1.f, -1.f), x);
  uint64_t y = two(0.00957010191f, 0.00957010191f);
  y = multiply_add_two(y, f, two(0.0559178603f, 0.0559178603f));
  y = multiply_add_two(y, f, two(0.240247448f, 0.240247448f));
  y = multiply_add_two(y, f, two(0.693121815f, 0.693121815f));
  y = multiply_add_two(y, f, two(0.999999261f, 0.999999261f));
  const float2 n = apart(moved);
  return apart(multiply_two(y, two(__uint_as_float((__float_as_uint(n.x) << 23) + 0x3f800000u),
                                   __uint_as_float((__float_as_uint(n.y) << 23) + 0x3f800000u))));
}
// The probabilities exp2(scale x s + shift) of 32 scores, rounded to T once, in pairs, and their sum.
// The special-function units take 8 cycles for the exponentials of a warp and bound this loop: one of eight goes to
// the arithmetic pipes instead, which have time left.
// BOUNDED: none of them is above 2^127.
template <typename T, bool BOUNDED>
__device__ __forceinline__ void probabilities(uint32_t (&s)[32], uint32_t* p, uint64_t scales, uint64_t shifts,
                                              uint64_t (&sum)[2]) {
#pragma unroll
  for (int g = 0; g <= 4; ++g) {
    if (g < 4) {
#pragma unroll
      for (int j = g * 8; j < g * 8 + 8; j += 2) {
        const uint64_t x = multiply_add_two(two(__uint_as_float(s[j]), __uint_as_float(s[j + 1])), scales, shifts);
        float2 e = apart(x);
        if (j % 16 == 14) {
          e = exp2_polynomial<BOUNDED>(x);
        } else {
          e.x = exp2_in_order(e.x);
          e.y = exp2_in_order(e.y);
        }
        s[j] = __float_as_uint(e.x);
        s[j + 1] = __float_as_uint(e.y);
      }
    }
    if (g > 0) {
      const int h = g - 1;
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const float a = __uint_as_float(s[h * 8 + j]), b = __uint_as_float(s[h * 8 + j + 1]);
        sum[(j >> 1) & 1] = add_two(sum[(j >> 1) & 1], two(a, b));
        p[h * 4 + j / 2] = Pair<T>::pack(a, b);
      }
    }
  }
}
// The key tiles of a piece that hold keys which some row of row tile t sees. Where the rows fill no more than one tile, both
// hold them, and take turns with the key tiles: the chain of a row tile (see above) is then half as long.
template <bool TURNS>
__device__ __forceinline__ void set_ranges(const AttentionParams& P, Piece& p) {
  const uint32_t half = P.item_rows / 2;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    p.from[t] = p.to[t] = 0;
    if (t * half >= p.rows) continue;
    const uint32_t first = p.first_row + t * half, last = p.first_row + min((t + 1) * half, p.rows) - 1u;
    const KeyRange k = key_range(P, Sequence{p.token, p.n, p.length}, divide(first, P.by_group), divide(last, P.by_group));
    if (k.end <= k.begin) continue;
    p.from[t] = max(p.tile, k.begin / kKeys);
    p.to[t] = max(p.from[t], min(p.tile + p.count, (k.end + kKeys - 1) / kKeys));
  }
  p.shared = TURNS && p.rows <= half && p.to[0] > p.from[0] + 1 ? 1u : 0u;
  if (p.shared) {  // `to` is one behind the last tile of a turn
    p.from[1] = p.from[0] + 1;
    p.to[1] = p.from[1] + ((p.to[0] - p.from[1] - 1) & ~1) + 1;
    p.to[0] = p.from[0] + ((p.to[0] - p.from[0] - 1) & ~1) + 1;
  }
}

// TURNS: whether row tiles may take turns, which costs the issuing warp some code.
template <typename T, int DIM, bool TURNS>
__global__ void __launch_bounds__(kThreadsMany, 1) many_rows_kernel(const __grid_constant__ AttentionParams P) {
  extern __shared__ uint8_t raw[];
  using M = ManySmem<DIM>;
  constexpr int kHalves = DIM / 64;
  constexpr bool kApart = M::kApart;
  uint8_t* smem = raw + ((1024u - (smem_address(raw) & 1023u)) & 1023u);
  ManyControl& C = *reinterpret_cast<ManyControl*>(smem + M::kControl);
  const uint32_t base = smem_address(smem), ring = base + M::kRing;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;

  if (threadIdx.x == 0) {
    for (int i = 0; i < M::kPairs; ++i) {
      barrier_init(P, kBarrierFull, C.full[i], 2);
      barrier_init(P, kBarrierEmpty, C.empty[i], 1);
    }
    for (int t = 0; t < 2; ++t) {
      barrier_init(P, kBarrierScores, C.scores[t], 1);
      barrier_init(P, kBarrierScoresRead, C.scores_read[t], 4);
      barrier_init(P, kBarrierProbabilities, C.probabilities[t], 4);
      barrier_init(P, kBarrierQueries, C.queries[t], 1);
      barrier_init(P, kBarrierQueriesFree, C.queries_free[t], 1);
      barrier_init(P, kBarrierOutputs, C.outputs[t], 1);
    }
    for (int i = 0; i < kPieces; ++i) {
      barrier_init(P, kBarrierTold, C.told[i], 1);
      barrier_init(P, kBarrierTaken, C.taken[i], 10);  // all but the warp that tells
    }
    barrier_init(smem_address(&C.drained), 1);
    barrier_init(P, kBarrierOtherDone, C.other_done, 4);
    barrier_init(P, kBarrierOtherRead, C.other_read, 4);
    C.gave_up = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&P.k_map));
    asm volatile("prefetch.tensormap [%0];" ::"l"(&P.v_map));
    asm volatile("prefetch.tensormap [%0];" ::"l"(&P.q_map));
  }
  let_next_begin();
  earlier_done();
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_address(&C.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    before_sync();
  }
  find_share<kKeys, kThreadsMany>(P, C.sums, &C.share);  // barriers of the CTA within
  after_sync();
  const uint32_t tmem = *const_cast<volatile uint32_t*>(&C.tmem);
  constexpr uint32_t kPairs = M::kPairs;
  uint32_t fills = 0;  // of this loading warp
  bool fine = true;
  // Each group of warps within its own branch: code behind a meeting of both is held to the fewer registers.
  if (warp < kSoftmaxWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegisters));
    if (warp == kKeyWarp) {
      TileLoader<kKeys, kHalves> loader(P);
      Walker<kKeys> walk(P, C.share);
      const uint32_t half = P.item_rows / 2, half_tokens = divide(half, P.by_group);
      uint32_t query_loads[2] = {0, 0};
      // A share that begins within an item takes that item's rest last: CTAs whose items see the same keys then go through
      // them at about the same time, and most reads find them in L2.
      bool deferred = false, last = false;
      for (uint32_t i = 0; fine; ++i) {
        bool some = walk.next();
        if (i == 0 && some && !walk.piece.begins && walk.left != 0u) {
          if (lane == 0) C.deferred = walk.piece;
          __syncwarp();
          deferred = true;
          some = walk.next();
        }
        if (!some && !last) {  // behind the last piece in order
          last = true;
          if (lane == 0 && P.headers) walk.write_header();
          if (deferred) {
            walk.piece = C.deferred;
            some = true;
          }
        }
        if (some) {
          loader.begin(walk.piece);
          set_ranges<TURNS>(P, walk.piece);
        }
        const uint32_t at = i % kPieces;
        fine = barrier_wait_warp(smem_address(&C.taken[at]), ((i / kPieces) & 1u) ^ 1u, &C.gave_up);
        if (!fine) break;
        put_piece(&C.pieces[at], walk.piece, lane);
        if (lane == 0) barrier_arrive(smem_address(&C.told[at]));
        __syncwarp();
        if (!some) break;
        for (int32_t u = 0; u <= walk.piece.count; ++u) {
          const uint32_t slot = fills % kPairs, full = smem_address(&C.full[slot]);
          fine = barrier_wait_warp(smem_address(&C.empty[slot]), ((fills / kPairs) & 1u) ^ 1u, &C.gave_up);
          if (!fine) break;
          ++fills;
          if (u == walk.piece.count) {  // the last values come alone
            if (lane == 0) barrier_arrive(full);
            __syncwarp();
            break;
          }
          loader.load(&P.k_map, walk.piece.tile + u, ring + slot * 2u * M::kTileBytes, walk.piece.head, full);
          if (u == 0) {  // the queries, behind the first keys: whole tokens, some of the next sequence perhaps
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              if (walk.piece.to[t] <= walk.piece.from[t]) continue;
              fine = fine && barrier_wait_warp(smem_address(&C.queries_free[t]), (query_loads[t] & 1u) ^ 1u, &C.gave_up);
              if (!fine) break;
              ++query_loads[t];
              if (lane == 0) {
                const uint32_t bar = smem_address(&C.queries[t]);
                barrier_arrive_bytes(bar, half * 128u * kHalves);
                const uint32_t from_token =
                    divide(walk.piece.first_row, P.by_group) + (TURNS && walk.piece.shared ? 0u : t * half_tokens);
                const int32_t token = walk.piece.token + static_cast<int32_t>(from_token);
#pragma unroll
                for (int h = 0; h < kHalves; ++h)
                  load_queries(base + t * M::kTileBytes + h * (kTileRows * 128), &P.q_map, h * 64,
                               static_cast<int32_t>(walk.piece.head * P.group), token, bar);
              }
              __syncwarp();
            }
            if (!fine) break;
          }
        }
      }
      if (!last && lane == 0 && P.headers) walk.write_header();  // on the way out after a wait that gave up
      for (int t = 0; t < 2; ++t)  // where all goes well they landed long ago
        if (query_loads[t]) barrier_wait_out(smem_address(&C.queries[t]), (query_loads[t] - 1u) & 1u);
    } else if (warp == kValueWarp) {
      TileLoader<kKeys, kHalves> loader(P);
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
        for (int32_t u = -1; u < count; ++u) {
          const uint32_t slot = fills % kPairs, full = smem_address(&C.full[slot]);
          fine = barrier_wait_warp(smem_address(&C.empty[slot]), ((fills / kPairs) & 1u) ^ 1u, &C.gave_up);
          if (!fine) break;
          ++fills;
          if (u < 0) {  // the first keys come alone
            if (lane == 0) barrier_arrive(full);
            __syncwarp();
          } else {
            loader.load(&P.v_map, tile + u, ring + (slot * 2u + 1u) * M::kTileBytes, head, full);
          }
        }
      }
    } else if (warp == kMmaWarp) {
      uint32_t step = 0;  // slots of the ring taken so far
      uint32_t query_phase[2] = {0, 0}, probability_phase[2] = {0, 0}, read_phase[2] = {1, 1};
      const bool issuer = elected();
      constexpr uint32_t kScores = instruction<T>(kKeys, false), kOutput = instruction<T>(DIM, true);
      for (uint32_t n = 0; fine; ++n) {
        const uint32_t at = n % kPieces;
        fine = barrier_wait_warp(smem_address(&C.told[at]), (n / kPieces) & 1u, &C.gave_up);
        const Piece& piece = C.pieces[at];
        if (!fine || piece.valid == 0) break;
        const int32_t first = piece.tile, end = first + piece.count;
        const int32_t from[2] = {piece.from[0], piece.from[1]}, to[2] = {piece.to[0], piece.to[1]};
        const int32_t keys_begin = piece.keys_begin, keys_end = piece.keys_end;
        const int32_t turns = TURNS ? static_cast<int32_t>(piece.shared) : 0;
        // step u: O += P V of unit u, then the scores of unit u + 1, for one row tile after the other
        for (int32_t u = first - 1; fine && u < end; ++u) {
          const uint32_t slot = step % kPairs;
          const uint32_t k_at = ring + slot * 2u * M::kTileBytes, v_at = k_at + M::kTileBytes;
          fine = barrier_wait_warp(smem_address(&C.full[slot]), (step / kPairs) & 1u, &C.gave_up);
          if (!fine) break;
          ++step;
          // value rows that no row sees may hold anything: 0 x NaN is not 0
          const int32_t key0 = u * kKeys;
          if (u >= first && (key0 < keys_begin || key0 + kKeys > keys_end)) {
            uint8_t* const tile = smem + (v_at - base);
            for (uint32_t i = lane; i < kKeys * DIM / 8; i += 32) {
              const int32_t r = static_cast<int32_t>((i >> 3) % kKeys);  // a row has 128 bytes of each 64 elements
              if (key0 + r < keys_begin || key0 + r >= keys_end) *reinterpret_cast<uint4*>(tile + i * 16) = make_uint4(0, 0, 0, 0);
            }
            shared_to_async();
            __syncwarp();
          }
          auto weigh = [&](int t) {  // O += P V of unit u; false after a wait that gave up
            if (u < from[t] || u >= to[t] || ((u - from[t]) & turns)) return true;
            if (!barrier_wait_warp(smem_address(&C.probabilities[t]), probability_phase[t], &C.gave_up)) return false;
            probability_phase[t] ^= 1u;
            after_sync();
            if (issuer) {
              const uint64_t v = operand(v_at, kKeys * 128 / 16);
#pragma unroll
              for (int k = 0; k < kKeys / 16; ++k)
                product_tensor(tmem + M::output_column(t), tmem + M::probability_column(t) + k * 8, v + k * (16 * 128 / 16),
                               kOutput, k > 0 || u > from[t]);
              if (kApart || u + 1 == to[t]) commit(smem_address(&C.outputs[t]));
            }
            return true;
          };
          auto score = [&](int t) {  // S of unit u + 1
            if (u + 1 < from[t] || u + 1 >= to[t] || ((u + 1 - from[t]) & turns)) return true;
            if (kApart) {
              if (!barrier_wait_warp(smem_address(&C.scores_read[t]), read_phase[t], &C.gave_up)) return false;
              read_phase[t] ^= 1u;
            }
            if (u + 1 == from[t]) {
              if (!barrier_wait_warp(smem_address(&C.queries[t]), query_phase[t], &C.gave_up)) return false;
              query_phase[t] ^= 1u;
            }
            if (kApart || u + 1 == from[t]) after_sync();
            if (issuer) {
              const uint64_t q = operand(base + t * M::kTileBytes, 1);
              const uint64_t k_tile = operand(k_at, 1);
#pragma unroll
              for (int k = 0; k < DIM / 16; ++k) {
                const uint32_t part = (k >> 2) * (static_cast<int>(kTileRows) * 128 / 16) + (k & 3) * 2;
                product_shared(tmem + M::score_column(t), q + part, k_tile + part, kScores, k > 0);
              }
              commit(smem_address(&C.scores[t]));
              if (u + 2 == to[t]) commit(smem_address(&C.queries_free[t]));
            }
            return true;
          };
          // Where scores and probabilities have places of their own the next scores come first, as soon as the last
          // ones have been read; otherwise behind the product that reads the probabilities in their place.
          // Tiles that take turns: the second one's scores need not wait for the first one's probabilities.
          if (turns) fine = score(1);
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const bool scored = t == 1 && turns;
            fine = fine && (kApart ? (scored || score(t)) && weigh(t) : weigh(t) && (scored || score(t)));
          }
          if (issuer && fine) commit(smem_address(&C.empty[slot]));
        }
        if (lane == 0) barrier_arrive(smem_address(&C.taken[at]));
      }
      if (!fine) {
        if (issuer) commit(smem_address(&C.drained));
        barrier_wait_out(smem_address(&C.drained), 0);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegisters));
    const uint32_t t = (warp - kSoftmaxWarp) >> 2, thread = threadIdx.x & 127u;
    const uint32_t lanes = (warp & 3u) << 21;  // this warp's rows of tensor memory: lane 32 x (warp & 3), bits 16 up
    const uint32_t s_at = tmem + M::score_column(t) + lanes, p_at = tmem + M::probability_column(t) + lanes,
                   o_at = tmem + M::output_column(t) + lanes;
    const float ninf = __int_as_float(0xff800000);
    uint32_t score_phase = 0, output_phase = 0, other_phase = 0;
    const uint32_t half = P.item_rows / 2;
    uint8_t* const stage = smem + M::kStage + (warp - kSoftmaxWarp) * 4096;
    for (uint32_t n = 0;; ++n) {
      const uint32_t at = n % kPieces;
      fine = barrier_wait_warp(smem_address(&C.told[at]), (n / kPieces) & 1u, &C.gave_up);
      const Piece& piece = C.pieces[at];
      if (!fine || piece.valid == 0) break;
      const bool shared = TURNS && piece.shared != 0;
      const uint32_t r = (shared ? 0u : t * half) + thread;  // row of the item
      const bool valid = thread < half && r < piece.rows;
      const uint32_t g = piece.first_row + r;
      const int32_t from = piece.from[t], to = piece.to[t];
      float m = ninf, l = 0.f;
      if (to > from) {
        int32_t see_from = 0, see_to = 0x7fffffff;
        if (valid)
          seen_keys(P, piece.length - piece.n + static_cast<int32_t>(divide(g, P.by_group)), piece.length, see_from, see_to);
        const int32_t all_from = __reduce_max_sync(0xffffffffu, see_from);
        const int32_t all_to = __reduce_min_sync(0xffffffffu, see_to);

        for (int32_t u = from; u < to; u += shared ? 2 : 1) {
          fine = barrier_wait_warp(smem_address(&C.scores[t]), score_phase, &C.gave_up);
          if (!fine) break;
          score_phase ^= 1u;
          after_sync();
          if constexpr (!kApart) {
            const int32_t key0 = u * kKeys;
            const bool tested = key0 < all_from || key0 + kKeys > all_to;
            uint32_t s[32], other[32], p[64];
            const uint64_t scales = two(P.scale_log2, P.scale_log2);
            uint64_t shifts, sum[2] = {two(0.f, 0.f), two(0.f, 0.f)};
            bool again = __any_sync(0xffffffffu, valid && m == ninf);  // a row that has seen nothing has no reference
            if (!again) {
              const float shift = m * P.scale_log2;
              shifts = two(-shift, -shift);
              load_columns(s_at, s);
              load_columns(s_at + 32, other);
              loads_done(s);
              loaded(other);
              if (tested) hide(s, see_from - key0, see_to - key0), hide(other, see_from - key0 - 32, see_to - key0 - 32);
              probabilities<T, false>(s, p, scales, shifts, sum);
              load_columns(s_at + 64, s);
              probabilities<T, false>(other, p + 16, scales, shifts, sum);
              loads_done(s);
              load_columns(s_at + 96, other);
              if (tested) hide(s, see_from - key0 - 64, see_to - key0 - 64);
              probabilities<T, false>(s, p + 32, scales, shifts, sum);
              loads_done(other);
              if (tested) hide(other, see_from - key0 - 96, see_to - key0 - 96);
              probabilities<T, false>(other, p + 48, scales, shifts, sum);
              const float2 sums = apart(add_two(sum[0], sum[1]));
              // no probability is above their sum
              again = __any_sync(0xffffffffu, valid && !(sums.x + sums.y <= kMostSum));
            }
            if (again) {
              float part[4] = {m, m, m, m};
#pragma unroll 1
              for (int i = 0; i < kKeys; i += 32) {
                load_columns(s_at + i, s);
                loads_done(s);
                if (tested) hide(s, see_from - key0 - i, see_to - key0 - i);
                highest_32(s, part);
              }
              const float top = fmaxf(max3(part[0], part[1], part[2]), part[3]);
              if (u != from) {
                // the scores of this unit are there, so the last unit's O is complete
                const float f = top == m ? 1.f : exp2_fast((m - top) * P.scale_log2);
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
              }
              m = top;
              const float shift = m == ninf ? 0.f : m * P.scale_log2;
              shifts = two(-shift, -shift);
              sum[0] = sum[1] = two(0.f, 0.f);
#pragma unroll 1
              for (int i = 0; i < kKeys; i += 32) {
                load_columns(s_at + i, s);
                loads_done(s);
                if (tested) hide(s, see_from - key0 - i, see_to - key0 - i);
                probabilities<T, false>(s, p, scales, shifts, sum);
                store_columns_16(p_at + i / 2, p);
              }
            } else {
              store_columns(p_at, p);
              store_columns(p_at + 32, p + 32);
            }
            const float2 sums = apart(add_two(sum[0], sum[1]));
            l += sums.x + sums.y;
          } else {
            const int32_t key0 = u * kKeys;
            const bool tested = key0 < all_from || key0 + kKeys > all_to;
            // The code of a unit is kept small (it is run by eight warps beside four others' that differ): the scores are
            // read twice, for the maximum and for the probabilities, and hidden ones are put back as such.
            float part[4] = {ninf, ninf, ninf, ninf};
            uint32_t s[32], other[32];
            if (tested) {
#pragma unroll 1
              for (int i = kKeys - 32; i >= 0; i -= 32) {
                load_columns(s_at + i, s);
                loads_done(s);
                hide(s, see_from - key0 - i, see_to - key0 - i);
                highest_32(s, part);
                store_columns(s_at + i, s);
              }
              stores_done();
            } else {
              uint32_t rest[64];
              load_columns(s_at, s);
              load_columns(s_at + 32, other);
              load_columns(s_at + 64, rest);
              load_columns(s_at + 96, rest + 32);
              loads_done(s);
              loaded(other);
              loaded(rest);
              loaded(rest + 32);
              highest_32(s, part);
              highest_32(other, part);
              highest_32(rest, part);
              highest_32(rest + 32, part);
            }
            const float top = fmaxf(max3(part[0], part[1], part[2]), part[3]);
            if (u != from) {  // the last unit's probabilities have been used
              fine = barrier_wait_warp(smem_address(&C.outputs[t]), output_phase, &C.gave_up);
              if (!fine) break;
              output_phase ^= 1u;
              after_sync();
            }
            if (u == from) {
              m = top;
            } else {
              // the scores of this unit are there, so the last unit's O is complete
              const bool rise = valid && (top - m) * P.scale_log2 > kRise;
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
            const uint64_t scales = two(P.scale_log2, P.scale_log2), shifts = two(-shift, -shift);
            uint64_t sum[2] = {two(0.f, 0.f), two(0.f, 0.f)};
#pragma unroll 1
            for (int i = 0; i < kKeys; i += 64) {
              load_columns(s_at + i + 32, other);
              uint32_t p[16];
              probabilities<T, true>(s, p, scales, shifts, sum);
              store_columns_16(p_at + i / 2, p);  // over scores that have been read
              loads_done(other);
              if (i == 0) {
                load_columns(s_at + 64, s);
              } else {  // the next scores may come
                before_sync();
                __syncwarp();
                if (lane == 0) barrier_arrive(smem_address(&C.scores_read[t]));
              }
              probabilities<T, true>(other, p, scales, shifts, sum);
              store_columns_16(p_at + i / 2 + 16, p);
              loads_done(s);
            }
            const float2 sums = apart(add_two(sum[0], sum[1]));
            l += sums.x + sums.y;
          }
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
      // Two tiles of the same rows: the second leaves its references and sums in its stage, the first takes these and
      // the second's O, which is in its own lanes of tensor memory.
      float keep = 1.f, take = 0.f;
      if (shared) {
        float2* const other = reinterpret_cast<float2*>(smem + M::kStage + ((warp - kSoftmaxWarp) | 4u) * 4096);
        if (t == 1) {
          other[lane] = make_float2(m, l);
          before_sync();
          __syncwarp();
          if (lane == 0) barrier_arrive(smem_address(&C.other_done));
          fine = barrier_wait_warp(smem_address(&C.other_read), other_phase, &C.gave_up);
        } else {
          fine = barrier_wait_warp(smem_address(&C.other_done), other_phase, &C.gave_up);
          after_sync();
          const float2 o = other[lane];
          const float top = fmaxf(m, o.x);
          keep = m == top ? 1.f : exp2_fast((m - top) * P.scale_log2);
          take = o.x == top ? 1.f : exp2_fast((o.x - top) * P.scale_log2);
          m = top;
          l = l * keep + o.y * take;
        }
        if (!fine) break;
        other_phase ^= 1u;
      }
      if (shared ? t == 0 : t * half < piece.rows) {
        const bool any = to > from, complete = piece.begins && piece.ends;
        const uint32_t token = divide(g, P.by_group), head = piece.head * P.group + (g - token * P.group);
        const int64_t row_of = piece.token + static_cast<int64_t>(token);
        const float inverse = !complete ? 1.f : inverse_of(m, l);
        uint64_t row_at;  // where this thread's row goes
        if (complete) {
          row_at = reinterpret_cast<uint64_t>(static_cast<T*>(P.out) + row_of * P.out_token +
                                              static_cast<int64_t>(head) * P.out_head);
          if (valid && P.lse) P.lse[row_of * P.kv_heads * P.group + head] = log_sum(m, l, P.scale);
        } else {
          float* slot = P.partial + (2u * blockIdx.x + (piece.begins ? 1u : 0u)) * static_cast<size_t>(kRows * (2 + DIM));
          row_at = reinterpret_cast<uint64_t>(slot + kRows * 2 + r * DIM);
          if (valid) *reinterpret_cast<float2*>(slot + r * 2) = make_float2(m, l);
        }
        // 32 columns at a time through this warp's stage, so that eight lanes write 128 bytes of a row together
        const uint32_t rows_here = __popc(__ballot_sync(0xffffffffu, valid));  // the first ones
#pragma unroll 1
        for (int i = 0; i < DIM; i += 32) {
          uint32_t o[32];
          if (shared) {
            uint32_t other[32];
            load_columns(o_at + i, o);
            load_columns(tmem + M::output_column(1) + lanes + i, other);
            loads_done(o);
            loaded(other);
#pragma unroll
            for (int j = 0; j < 32; ++j)
              o[j] = __float_as_uint(__uint_as_float(o[j]) * keep + __uint_as_float(other[j]) * take);
          } else if (any) {
            load_columns(o_at + i, o);
            loads_done(o);
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = 0u;
          }
          uint8_t* const mine = stage + lane * 128;
          if (complete) {  // 64 bytes: two turns fill a row of the stage
#pragma unroll
            for (int j = 0; j < 32; j += 8) {
              uint4 v;
              v.x = Pair<T>::pack(__uint_as_float(o[j]) * inverse, __uint_as_float(o[j + 1]) * inverse);
              v.y = Pair<T>::pack(__uint_as_float(o[j + 2]) * inverse, __uint_as_float(o[j + 3]) * inverse);
              v.z = Pair<T>::pack(__uint_as_float(o[j + 4]) * inverse, __uint_as_float(o[j + 5]) * inverse);
              v.w = Pair<T>::pack(__uint_as_float(o[j + 6]) * inverse, __uint_as_float(o[j + 7]) * inverse);
              const uint32_t part = (i & 32) / 8 + j / 8;
              *reinterpret_cast<uint4*>(mine + ((part ^ (lane & 7u)) << 4)) = v;
            }
            if ((i & 32) == 0) continue;
          } else {
#pragma unroll
            for (int j = 0; j < 32; j += 4)
              *reinterpret_cast<uint4*>(mine + ((static_cast<uint32_t>(j / 4) ^ (lane & 7u)) << 4)) =
                  make_uint4(o[j], o[j + 1], o[j + 2], o[j + 3]);
          }
          __syncwarp();
          const uint32_t part = lane & 7u;
          const uint32_t element = complete ? static_cast<uint32_t>(i - 32) + part * 8 : static_cast<uint32_t>(i) + part * 4;
          const uint32_t offset = complete ? element * 2 : element * 4;
          uint64_t to_row[8];
          uint4 v[8];
#pragma unroll
          for (uint32_t j = 0; j < 8; ++j) {
            const uint32_t row = j * 4 + (lane >> 3);
            to_row[j] = __shfl_sync(0xffffffffu, row_at, row);
            v[j] = *reinterpret_cast<const uint4*>(stage + row * 128 + ((part ^ (row & 7u)) << 4));
          }
          const bool wanted = !complete || element < P.head_dim;
#pragma unroll
          for (uint32_t j = 0; j < 8; ++j)
            if (wanted && j * 4 + (lane >> 3) < rows_here) *reinterpret_cast<uint4*>(to_row[j] + offset) = v[j];
          __syncwarp();
        }
        before_sync();
        if (shared) {
          __syncwarp();
          if (lane == 0) barrier_arrive(smem_address(&C.other_read));
        }
      }
      if (lane == 0) barrier_arrive(smem_address(&C.taken[at]));
    }
  }
  before_sync();
  __syncthreads();
  after_sync();
  if (C.gave_up && (warp == kKeyWarp || warp == kValueWarp)) {  // each its own fills: either may be ahead of the other
    for (uint32_t f = fills > kPairs ? fills - kPairs : 0u; f < fills; ++f)
      barrier_wait_out(smem_address(&C.full[f % kPairs]), (f / kPairs) & 1u);
    if (lane == 0) atomicExch(P.status, 1u);
  }
  if (warp == kMmaWarp)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

}  // namespace paged

namespace {
template <typename T, int DIM, bool TURNS>
cudaError_t prepare() {
  // setmaxnreg.inc would wait for good if the launch brought fewer registers than its warps share out
  cudaFuncAttributes a;
  const cudaError_t e = cudaFuncGetAttributes(&a, paged::many_rows_kernel<T, DIM, TURNS>);
  if (e != cudaSuccess) return e;
  if (a.numRegs < static_cast<int>(paged::kLaunchRegisters)) return cudaErrorInvalidDeviceFunction;
  return cudaFuncSetAttribute(paged::many_rows_kernel<T, DIM, TURNS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              1024 + paged::ManySmem<DIM>::kBytes);
}
template <typename T, int DIM>
cudaError_t launch(const AttentionParams& p, const AttentionPlan& plan, cudaStream_t stream) {
  return launch_dependent(plan.turns ? paged::many_rows_kernel<T, DIM, true> : paged::many_rows_kernel<T, DIM, false>,
                          dim3(plan.ctas), paged::kThreadsMany, 1024 + paged::ManySmem<DIM>::kBytes, p, stream);
}
}  // namespace
cudaError_t prepare_many_rows() {
  for (cudaError_t e : {prepare<__half, 64, false>(), prepare<__half, 128, false>(), prepare<__nv_bfloat16, 64, false>(),
                        prepare<__nv_bfloat16, 128, false>(), prepare<__half, 64, true>(), prepare<__half, 128, true>(),
                        prepare<__nv_bfloat16, 64, true>(), prepare<__nv_bfloat16, 128, true>()})
    if (e != cudaSuccess) return e;
  return cudaSuccess;
}
cudaError_t launch_many_rows(const AttentionParams& p, const AttentionPlan& plan, bool bf16, cudaStream_t stream) {
  if (bf16)
    return plan.padded_dim == 64 ? launch<__nv_bfloat16, 64>(p, plan, stream) : launch<__nv_bfloat16, 128>(p, plan, stream);
  return plan.padded_dim == 64 ? launch<__half, 64>(p, plan, stream) : launch<__half, 128>(p, plan, stream);
}

}  // namespace mononn
