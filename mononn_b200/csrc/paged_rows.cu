// Rotation of positions, and the append of new keys and values to a paged cache with the rotation on the way.
//
// (a, b) -> m (a cos t - b sin t, b cos t + a sin t) for the pairs of the leading rotary_dim elements of
// a head, t = position x f_i. The angle is taken in 64 bits as a share of a full turn (position x f_i / 2 pi, of
// which only the fraction matters), so that positions of any size keep it to 32 bits; sine and
// cosine of that share, and the products, are 32-bit. Bound by memory: every element is read once and written once.
// 8192 tokens x 40 heads of 128 to another tensor (168 MB): 32 us, 5.2 TB/s, in place 33; append of 11.6k tokens x 32 heads of 64 (191 MB):
// 34 us, 5.6 TB/s, 0.86 of what a copy reaches. One token: 3.0 us, the launch. A block takes a few tokens, so that
// the angles and places, worked out once for all of their heads, are few beside the elements.
#include "paged_device.h"

namespace mononn {
namespace paged {

constexpr int kRowsThreads = 256;
constexpr uint32_t kRowsTokens = 8, kRowsAngles = 512;  // of a block, at most

// V elements at once, of type T
template <typename T, int V>
struct Vector;
template <typename T>
struct Vector<T, 8> {
  uint4 v;
  __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<uint4*>(p) = v; }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 a = Pair<T>::unpack(w[i]);
      f[2 * i] = a.x;
      f[2 * i + 1] = a.y;
    }
  }
  __device__ __forceinline__ void set(const float (&f)[8]) {
    v = make_uint4(Pair<T>::pack(f[0], f[1]), Pair<T>::pack(f[2], f[3]), Pair<T>::pack(f[4], f[5]),
                   Pair<T>::pack(f[6], f[7]));
  }
};
template <typename T>
struct Vector<T, 1> {
  T v;
  __device__ __forceinline__ void load(const T* p) { v = *p; }
  __device__ __forceinline__ void store(T* p) const { *p = v; }
  __device__ __forceinline__ void get(float (&f)[1]) const { f[0] = static_cast<float>(v); }
  __device__ __forceinline__ void set(const float (&f)[1]) { v = static_cast<T>(f[0]); }
};

// Number of entries of indptr[1 .. n] that are at most `token`: the sequence of a token. The warp looks
// at 32 places of the range at a time.
__device__ __forceinline__ uint32_t sequence_of(const int32_t* indptr, uint32_t n, int32_t token) {
  const uint32_t lane = threadIdx.x & 31u;
  uint32_t low = 0, high = n;  // the answer is in low .. high
  while (low < high) {
    const uint32_t step = (high - low + 31u) / 32u;
    const uint32_t i = low + (lane + 1u) * step;  // entry i: the answer is at least i when it is at most `token`
    const uint32_t below = __ballot_sync(0xffffffffu, i <= high && indptr[min(i, high)] <= token);
    const uint32_t k = __popc(below);
    const uint32_t next = low + k * step;
    high = min(high, next + step - 1u);
    low = next;
    if (step == 1u) break;
  }
  return low;
}

// What a block knows of its tokens.
struct RowsShared {
  alignas(16) float cosines[kRowsAngles], sines[kRowsAngles];  // token by token
  int64_t page_at[kRowsTokens];  // of the token's row in the pages, in elements; below 0: none
  int32_t position[kRowsTokens];
  bool member[kRowsTokens];      // of some sequence
};
enum RowsMode { kCopy, kPairs, kNeighbours };

// The vectors `first` .. `first` + each - 1 of every head of every token of a block, a thread to a vector: consecutive
// threads along a head, then along heads and tokens. 64 bytes of each thread are on their way at a time.
template <typename T, int V, RowsMode MODE>
__device__ __forceinline__ void move_rows(const RowsSource& s, const RowsShared& S, uint32_t token0, uint32_t tokens,
                                          bool to_pages, uint32_t first, uint32_t each, uint32_t rd) {
  if (each == 0 || s.heads == 0) return;
  for (uint32_t j0 = 0; j0 < each; j0 += kRowsThreads) {
    const uint32_t wide = min(each - j0, static_cast<uint32_t>(kRowsThreads));
    const uint32_t step = kRowsThreads / wide;  // rows at once
    if (threadIdx.x >= step * wide) continue;
    const uint32_t j = j0 + threadIdx.x % wide;
    // element of the vector, and of its partner
    const uint32_t d0 = MODE == kCopy ? first + j * V : MODE == kPairs ? j * V : (V == 8 ? j * V : 2 * j);
    const uint32_t d1 = MODE == kPairs ? rd / 2 + j * V : 2 * j + 1;
    constexpr bool kTwo = MODE == kPairs || (MODE == kNeighbours && V == 1);
    uint32_t t = threadIdx.x / wide / s.heads, h = threadIdx.x / wide % s.heads;
    const uint32_t step_t = step / s.heads, step_h = step % s.heads;
    constexpr int kAtOnce = kTwo ? 2 : 4;
    while (t < tokens) {
      Vector<T, V> a[kAtOnce], b[kAtOnce];
      T* to[kAtOnce];
      uint32_t of[kAtOnce];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        to[u] = nullptr;
        of[u] = t;
        if (t < tokens && (to_pages ? S.page_at[t] >= 0 : S.member[t])) {
          const int64_t token = token0 + t;
          const T* from = static_cast<const T*>(s.src) + token * s.src_token + h * s.src_head;
          to[u] = static_cast<T*>(s.dst) + (to_pages ? S.page_at[t] : token * s.dst_token) + h * s.dst_head;
          a[u].load(from + d0);
          if (kTwo) b[u].load(from + d1);
        }
        t += step_t;
        h += step_h;
        if (h >= s.heads) h -= s.heads, ++t;
      }
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        if (to[u] == nullptr) continue;
        const float* cosines = S.cosines + of[u] * (rd / 2);
        const float* sines = S.sines + of[u] * (rd / 2);
        if constexpr (MODE == kNeighbours && V == 8) {
          float x[V], y[V];
          a[u].get(x);
          const float4 c = *reinterpret_cast<const float4*>(cosines + j * 4), n = *reinterpret_cast<const float4*>(sines + j * 4);
          const float cs[4] = {c.x, c.y, c.z, c.w}, ns[4] = {n.x, n.y, n.z, n.w};
#pragma unroll
          for (int i = 0; i < V; i += 2) {
            y[i] = x[i] * cs[i / 2] - x[i + 1] * ns[i / 2];
            y[i + 1] = x[i + 1] * cs[i / 2] + x[i] * ns[i / 2];
          }
          a[u].set(y);
        } else if constexpr (kTwo) {
          float x[V], y[V], p[V], q[V];
          a[u].get(x);
          b[u].get(y);
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float c = cosines[j * V + i], n = sines[j * V + i];
            p[i] = x[i] * c - y[i] * n;
            q[i] = y[i] * c + x[i] * n;
          }
          a[u].set(p);
          b[u].set(q);
          b[u].store(to[u] + d1);
        }
        a[u].store(to[u] + d0);
      }
    }
  }
}

// Six blocks an SM leave 40 registers a thread, and the form for vectors spills 108 bytes of each thread. That costs nothing where
// memory bounds the call (8192 x 40 x 128, half turned: 31.2 us, with five blocks and no spills 31.2, with four 33.8; append of
// 11.7k tokens, 32 heads of 64: 32.6, 33.0, 34.5), and up to a sixth in smaller ones (2048 x 12 heads of 64: 6.7, 6.2, 5.6).
template <typename T, int V>
__global__ void __launch_bounds__(kRowsThreads, 6) rows_kernel(const __grid_constant__ RowsParams P) {
  __shared__ RowsShared S;
  let_next_begin();
  earlier_done();
  const uint32_t token0 = blockIdx.x * P.block_tokens, tokens = min(P.block_tokens, P.tokens - token0);
  const uint32_t warp = threadIdx.x >> 5;
  if (warp < tokens) {  // a warp to a token
    const uint32_t token = token0 + warp;
    int64_t page_at = -1;
    int32_t position = 0;
    bool member = true;
    if (P.indptr) {
      const uint32_t b = sequence_of(P.indptr, P.sequences, static_cast<int32_t>(token));
      member = b < P.sequences;
      if (member) {
        const int32_t begin = P.indptr[b], end = P.indptr[b + 1], length = P.lengths[b];
        member = begin <= static_cast<int32_t>(token);
        const int64_t at = static_cast<int64_t>(length) - (static_cast<int64_t>(end) - begin) +
                           (static_cast<int64_t>(token) - begin);
        position = static_cast<int32_t>(at);
        if (member && at >= 0 && at < static_cast<int64_t>(P.max_pages) * P.page_size) {
          const uint32_t n = divide(static_cast<uint32_t>(at), P.by_page_size);
          const int32_t page = P.table[static_cast<int64_t>(b) * P.table_stride + n];
          if (page >= 0 && static_cast<uint32_t>(page) < P.num_pages)
            page_at = page * P.page_stride + static_cast<int64_t>(static_cast<uint32_t>(at) - n * P.page_size) * P.k.dst_token;
        }
      }
    }
    if (P.positions) position = P.positions[token];
    if ((threadIdx.x & 31u) == 0u) {
      S.page_at[warp] = page_at;
      S.position[warp] = position;
      S.member[warp] = member;
    }
  }
  __syncthreads();
  const uint32_t rd = P.rotary_dim, pairs = rd / 2;
  if (rd) {
    for (uint32_t i = threadIdx.x; i < tokens * 128; i += kRowsThreads) {
      const uint32_t t = i >> 7, p = i & 127u;
      if (p >= pairs) continue;
      const double turns = S.position[t] * P.turns[p];
      float s, c;
      sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &s, &c);
      S.cosines[t * pairs + p] = c * P.magnitude;
      S.sines[t * pairs + p] = s * P.magnitude;
    }
    __syncthreads();
    if (P.interleaved) {
      const uint32_t n = V == 8 ? rd / 8 : pairs;
      move_rows<T, V, kNeighbours>(P.q, S, token0, tokens, false, 0, n, rd);
      move_rows<T, V, kNeighbours>(P.k, S, token0, tokens, true, 0, n, rd);
    } else {
      move_rows<T, V, kPairs>(P.q, S, token0, tokens, false, 0, pairs / V, rd);
      move_rows<T, V, kPairs>(P.k, S, token0, tokens, true, 0, pairs / V, rd);
    }
  }
  if (rd < P.head_dim) {
    move_rows<T, V, kCopy>(P.q, S, token0, tokens, false, rd, (P.head_dim - rd) / V, rd);
    move_rows<T, V, kCopy>(P.k, S, token0, tokens, true, rd, (P.head_dim - rd) / V, rd);
  }
  move_rows<T, V, kCopy>(P.v, S, token0, tokens, true, 0, P.head_dim / V, rd);
}

}  // namespace paged

cudaError_t prepare_rows() {
  cudaFuncAttributes a;
  for (cudaError_t e : {cudaFuncGetAttributes(&a, paged::rows_kernel<__half, 1>),
                        cudaFuncGetAttributes(&a, paged::rows_kernel<__half, 8>),
                        cudaFuncGetAttributes(&a, paged::rows_kernel<__nv_bfloat16, 1>),
                        cudaFuncGetAttributes(&a, paged::rows_kernel<__nv_bfloat16, 8>)})
    if (e != cudaSuccess) return e;
  return cudaSuccess;
}
// One token a block until there are four blocks for each SM, then up to four tokens a block (one and four, 32 heads of 128: 100
// tokens 3.7 and 5.2 us, 300 4.5 and 5.3, 592 5.6 and 4.7, 4000 16.0 and 12.7): as many as take the fewest turns of move_rows
// a token, so that few threads stay idle in a last turn (8192 tokens of 40 heads, half of each turned: three tokens 32.0 us, four, in
// two turns of which the second is a quarter full, 34.6, two 35.5; append of 32 heads of 64, no turn: 35.1, 34.4, 39.6).
// With few heads up to eight (12 heads of the same bytes in all: 36 us instead of 46 with four).
// 16-byte vectors where everything is aligned to them, otherwise single elements: 2.7 and 4.2 us for one token, 9.5 and 21.4
// for 2048, 26 and 55 for 8192 x 40 heads (in L2).
cudaError_t launch_rows(const RowsParams& params, bool bf16, bool vectors, int sm_count, cudaStream_t stream) {
  RowsParams p = params;
  p.block_tokens = 1;
  if (p.tokens >= 4u * static_cast<unsigned>(sm_count)) {
    const uint32_t v = vectors ? 8 : 1, rest = (p.head_dim - p.rotary_dim) / v;
    const bool two = !p.interleaved || v == 1;  // a thread turns two vectors
    const uint32_t turned = p.interleaved && !two ? p.rotary_dim / 8 : p.rotary_dim / 2 / (p.interleaved ? 1 : v);
    auto turns = [&](uint32_t tokens, uint32_t vectors_each, uint32_t heads, uint32_t at_once) {
      const uint64_t each = static_cast<uint64_t>(paged::kRowsThreads) * at_once;
      return (static_cast<uint64_t>(tokens) * heads * vectors_each + each - 1) / each;
    };
    auto all_turns = [&](uint32_t t) {
      uint64_t sum = turns(t, p.head_dim / v, p.v.heads, 4);
      for (uint32_t heads : {p.q.heads, p.k.heads}) sum += turns(t, turned, heads, two ? 2 : 4) + turns(t, rest, heads, 4);
      return sum;
    };
    p.block_tokens = 4;
    for (uint32_t t : {3, 2})  // fewer turns a token
      if (all_turns(t) * p.block_tokens < all_turns(p.block_tokens) * t) p.block_tokens = t;
    while (p.block_tokens >= 4 && p.block_tokens < paged::kRowsTokens && all_turns(p.block_tokens + 1) == all_turns(1) &&
           (p.block_tokens + 1) * (p.rotary_dim / 2) <= paged::kRowsAngles)
      ++p.block_tokens;  // as long as one turn is enough
  }
  const dim3 grid((p.tokens + p.block_tokens - 1) / p.block_tokens);
  auto launch = [&](auto kernel) { return launch_dependent(kernel, grid, paged::kRowsThreads, 0, p, stream); };
  if (bf16) return vectors ? launch(paged::rows_kernel<__nv_bfloat16, 8>) : launch(paged::rows_kernel<__nv_bfloat16, 1>);
  return vectors ? launch(paged::rows_kernel<__half, 8>) : launch(paged::rows_kernel<__half, 1>);
}

}  // namespace mononn
