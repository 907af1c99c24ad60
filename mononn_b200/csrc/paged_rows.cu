// Rotation of positions, and the append of new keys and values to a paged cache with the rotation on the way.
//
// (a, b) -> m (a cos t - b sin t, b cos t + a sin t) for the pairs of the leading rotary_dim elements of
// a head, t = position x f_i. The angle is taken in 64 bits as a share of a full turn (position x f_i / 2 pi, of
// which only the fraction matters), so that positions of any size keep it to 32 bits; sine and
// cosine of that share, and the products, are 32-bit. Bound by memory: every element is read once and written once.
#include "paged_device.h"

namespace mononn {
namespace paged {

constexpr int kRowsThreads = 256;

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

template <typename T, int V>
__device__ __forceinline__ void rotate_heads(const RowsSource& s, const T* src, T* dst, uint32_t rd, uint32_t dim,
                                             bool interleaved, const float* cosines, const float* sines) {
  // of each head: pieces that are rotated, then pieces that are copied
  const uint32_t turned = interleaved ? (V == 8 ? rd / 8 : rd / 2) : rd / 2 / V;
  const uint32_t each = turned + (dim - rd) / V;
  if (each == 0) return;
  if (threadIdx.x >= each * (kRowsThreads / each) && each <= kRowsThreads) return;
  const uint32_t step = each <= kRowsThreads ? kRowsThreads / each : 1u;
  const uint32_t head0 = each <= kRowsThreads ? threadIdx.x / each : 0u;
  for (uint32_t j = each <= kRowsThreads ? threadIdx.x % each : threadIdx.x; j < each; j += kRowsThreads) {
    if (j >= turned) {
      const uint32_t d = rd + (j - turned) * V;
      for (uint32_t h = head0; h < s.heads; h += step) {
        Vector<T, V> a;
        a.load(src + h * s.src_head + d);
        a.store(dst + h * s.dst_head + d);
      }
    } else if (interleaved && V == 8) {
      for (uint32_t h = head0; h < s.heads; h += step) {
        Vector<T, V> a;
        a.load(src + h * s.src_head + j * V);
        float x[V], y[V];
        a.get(x);
#pragma unroll
        for (int i = 0; i + 1 < V; i += 2) {
          const float c = cosines[j * (V / 2) + i / 2], n = sines[j * (V / 2) + i / 2];
          y[i] = x[i] * c - x[i + 1] * n;
          y[i + 1] = x[i + 1] * c + x[i] * n;
        }
        a.set(y);
        a.store(dst + h * s.dst_head + j * V);
      }
    } else {
      const uint32_t d0 = interleaved ? 2 * j : j * V, d1 = interleaved ? 2 * j + 1 : rd / 2 + j * V;
      for (uint32_t h = head0; h < s.heads; h += step) {
        Vector<T, V> a, b;
        a.load(src + h * s.src_head + d0);
        b.load(src + h * s.src_head + d1);
        float x[V], y[V], u[V], w[V];
        a.get(x);
        b.get(y);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float c = cosines[j * V + i], n = sines[j * V + i];
          u[i] = x[i] * c - y[i] * n;
          w[i] = y[i] * c + x[i] * n;
        }
        a.set(u);
        b.set(w);
        a.store(dst + h * s.dst_head + d0);
        b.store(dst + h * s.dst_head + d1);
      }
    }
  }
}

template <typename T, int V>
__global__ void __launch_bounds__(kRowsThreads) rows_kernel(const __grid_constant__ RowsParams P) {
  __shared__ float cosines[128], sines[128];
  let_next_begin();
  earlier_done();
  const uint32_t token = blockIdx.x;
  int64_t page_at = -1;  // of the token's row, in elements
  int32_t position = 0;
  bool member = true;
  if (P.indptr) {
    const uint32_t b = sequence_of(P.indptr, P.sequences, static_cast<int32_t>(token));
    member = b < P.sequences && P.indptr[b] <= static_cast<int32_t>(token);
    if (member) {
      const int32_t begin = P.indptr[b], end = P.indptr[b + 1];
      const int64_t at = static_cast<int64_t>(P.lengths[b]) - (static_cast<int64_t>(end) - begin) + (token - begin);
      position = static_cast<int32_t>(at);
      if (at >= 0 && at < static_cast<int64_t>(P.max_pages) * P.page_size) {
        const uint32_t n = static_cast<uint32_t>(at) / P.page_size;
        const int32_t page = P.table[static_cast<int64_t>(b) * P.table_stride + n];
        if (page >= 0 && static_cast<uint32_t>(page) < P.num_pages)
          page_at = page * P.page_stride + static_cast<int64_t>(static_cast<uint32_t>(at) - n * P.page_size) * P.k.dst_token;
      }
    }
  }
  if (!member) return;
  if (P.rotary_dim) {
    if (P.positions) position = P.positions[token];
    if (threadIdx.x < P.rotary_dim / 2) {
      const double turns = position * P.turns[threadIdx.x];
      const float part = static_cast<float>(2.0 * (turns - rint(turns)));
      float s, c;
      sincospif(part, &s, &c);
      cosines[threadIdx.x] = c * P.magnitude;
      sines[threadIdx.x] = s * P.magnitude;
    }
    __syncthreads();
  }
  if (P.q.heads)
    rotate_heads<T, V>(P.q, static_cast<const T*>(P.q.src) + token * P.q.src_token,
                       static_cast<T*>(P.q.dst) + token * P.q.dst_token, P.rotary_dim, P.head_dim, P.interleaved != 0,
                       cosines, sines);
  if (page_at >= 0) {
    rotate_heads<T, V>(P.k, static_cast<const T*>(P.k.src) + token * P.k.src_token, static_cast<T*>(P.k.dst) + page_at,
                       P.rotary_dim, P.head_dim, P.interleaved != 0, cosines, sines);
    rotate_heads<T, V>(P.v, static_cast<const T*>(P.v.src) + token * P.v.src_token, static_cast<T*>(P.v.dst) + page_at,
                       0, P.head_dim, false, cosines, sines);
  }
}

}  // namespace paged

cudaError_t launch_rows(const RowsParams& p, bool bf16, bool vectors, int, cudaStream_t stream) {
  auto launch = [&](auto kernel) { return launch_dependent(kernel, dim3(p.tokens), paged::kRowsThreads, 0, p, stream); };
  if (bf16) return vectors ? launch(paged::rows_kernel<__nv_bfloat16, 8>) : launch(paged::rows_kernel<__nv_bfloat16, 1>);
  return vectors ? launch(paged::rows_kernel<__half, 8>) : launch(paged::rows_kernel<__half, 1>);
}

}  // namespace mononn
