// Operators behind a prompt: what their host side (paged.cc) and their kernels share.
//
// A call's work is divided in units: one tile of keys for one item, an item being the queries of one
// row tile (rows = new tokens x query heads of one key head) of one sequence. Sequences differ in
// length by orders of magnitude and their lengths are on the device only, so every CTA adds up the
// units of the whole call itself and takes an equal, contiguous share of them: the shares differ by
// one unit at most whatever the lengths are. A share may begin or end within an item; such pieces
// go to the workspace with their row maxima and sums, and a second, small kernel joins
// them in the order of the keys.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace mononn {

// Division by a number that the host knows, by multiplication (Granlund and Montgomery 1994): exact for every
// 32-bit dividend, four instructions instead of some twenty.
struct Divisor {
  uint32_t multiplier, shift1, shift2;
};
inline Divisor make_divisor(uint32_t d) {  // d > 0
  uint32_t l = 0;
  while (l < 32 && (1ull << l) < d) ++l;
  const uint64_t m = ((1ull << 32) * ((1ull << l) - d)) / d + 1;
  return Divisor{static_cast<uint32_t>(m), l < 1 ? l : 1u, l > 0 ? l - 1 : 0u};
}

// ------------------------------------------------------------- rotation and append
struct RowsSource {  // tokens x heads x head_dim
  const void* src;
  void* dst;
  int64_t src_token, src_head, dst_token, dst_head;
  uint32_t heads;
};
struct RowsParams {
  RowsSource q, k, v;    // q and k are rotated; k and v go into pages when `table` is set
  const int32_t* positions;
  const int32_t* indptr;
  const int32_t* lengths;
  const int32_t* table;
  int64_t table_stride, page_stride;
  uint32_t tokens, head_dim, sequences, max_pages, num_pages, page_size;
  uint32_t rotary_dim, interleaved, block_tokens;
  Divisor by_page_size;
  float magnitude;
  double turns[128];
};
cudaError_t prepare_rows();
cudaError_t launch_rows(const RowsParams& p, bool bf16, bool vectors, int sm_count, cudaStream_t stream);

// ------------------------------------------------------------------------ attention
// The kernel for few rows takes items of 16 rows, and as many keys a unit as fill 16 KB; the one for many rows two
// tiles of up to 128 rows (whole tokens), and 128 keys.
constexpr uint32_t kFewRows = 16;
constexpr uint32_t few_keys(uint32_t padded_dim) { return 8192 / padded_dim; }
constexpr uint32_t kTileRows = 128, kManyRows = 2 * kTileRows, kManyKeys = 128;

// Barriers of the attention kernels. A launch can be told to wait for one arrival more than there will be on one of them:
// how the tests let a bounded wait run out.
enum AttentionBarrier : uint32_t {
  kBarrierNone, kBarrierFull, kBarrierEmpty, kBarrierTold, kBarrierTaken, kBarrierQueries,
  kBarrierMeeting,                                                       // few rows only
  kBarrierScores, kBarrierScoresRead, kBarrierProbabilities, kBarrierOutputs, kBarrierQueriesFree,  // many rows only
  kBarrierOtherDone, kBarrierOtherRead, kBarriers
};
struct AttentionHeader {  // one per CTA: the item that begins in it and goes on in the next `more` CTAs
  uint32_t more;          // 0: none
  uint32_t rows;
  uint32_t first_row;     // within the sequence's (token, head of the group) rows
  uint32_t head;          // key head
  uint32_t token;         // first new token of the sequence
  uint32_t pad[3];
};
struct AttentionParams {
  CUtensorMap k_map, v_map, q_map;  // q_map: many rows only
  const void* q;
  void* out;
  float* lse;
  int64_t q_token, q_head, out_token, out_head, table_stride;
  const int32_t* table;
  const int32_t* lengths;
  const int32_t* indptr;
  AttentionHeader* headers;
  float* partial;           // slots 2 * CTA (an item begun earlier) and 2 * CTA + 1 (one that goes on)
  uint32_t* status;
  uint32_t sequences, tokens, kv_heads, group, head_dim, page_size, capacity, box_shift, item_rows, item_cost;
  uint32_t causal, window, least_shift, whole_items;
  uint32_t skewed;          // AttentionBarrier
  Divisor by_group, by_item_rows, by_page_size;
  float scale, scale_log2;  // of the scores; scale * log2(e)
};
struct AttentionPlan {  // how a call is launched: the same for every content of its device arrays
  bool many, turns;     // the kernel for many rows; with row tiles that may take turns
  uint32_t rows, keys, padded_dim, ctas, least_units;  // rows: of a slot of the workspace
  uint32_t item_rows;   // rows of an item, at most `rows`
  uint32_t item_cost;   // units that stand for an item's work beside its keys
  uint32_t box;         // token rows that one copy brings
  bool joins;           // an item may span CTAs: workspace and the second kernel are needed
  size_t workspace;
};
// Floats of one slot: row maximum and row sum, then the rows.
inline size_t attention_slot_floats(const AttentionPlan& p) {
  return static_cast<size_t>(p.rows) * (2 + p.padded_dim);
}
cudaError_t prepare_few_rows();
cudaError_t launch_few_rows(const AttentionParams& p, const AttentionPlan& plan, bool bf16, cudaStream_t stream);
cudaError_t prepare_many_rows();
cudaError_t launch_many_rows(const AttentionParams& p, const AttentionPlan& plan, bool bf16, cudaStream_t stream);
cudaError_t launch_join(const AttentionParams& p, const AttentionPlan& plan, bool bf16, cudaStream_t stream);
cudaError_t paged_status_word(uint32_t** out);

// A launch whose CTAs may be set up while the kernel before it still runs (they wait for its end
// before they read or write anything; see earlier_done).
template <typename K, typename Params>
cudaError_t launch_dependent(K kernel, dim3 grid, uint32_t threads, size_t smem, const Params& p, cudaStream_t stream) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

}  // namespace mononn
