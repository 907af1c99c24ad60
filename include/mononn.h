/* C ABI of libmononn_b200.so: the B200 (sm_100a) backend for the MonoNN hot path
 * "XLA HLO module in -> one persistent kernel -> one launch per inference".
 *
 * Conventions
 *   - every function returns 0 on success and a negative MONONN_ERR_* code on failure;
 *     nothing here aborts the process (the reference LOG(FATAL)s instead) and there is
 *     no CPU fallback: without a usable sm_100 device the calls fail.
 *   - pointers are borrowed for the duration of the call unless the parameter is `out`.
 *   - different modules may be used from different threads; one module from one
 *     thread at a time. Launches of one module must be ordered on the GPU (one stream, or
 *     streams chained by events): a module owns one barrier counter and one stage table.
 *   - every call runs on the module's device and restores the caller's current device.
 */
#ifndef MONONN_B200_H_
#define MONONN_B200_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum {
  MONONN_OK = 0,
  MONONN_ERR_INVALID_ARGUMENT = -1,
  MONONN_ERR_PARSE = -2,           /* HLO text or spec JSON is malformed */
  MONONN_ERR_UNSUPPORTED = -3,     /* op / dtype / layout / pattern outside the supported set */
  MONONN_ERR_CUDA = -4,            /* a CUDA runtime or driver call failed */
  MONONN_ERR_NO_DEVICE = -5,       /* no sm_100 device */
  MONONN_ERR_BARRIER_TIMEOUT = -6, /* a bounded wait inside the kernel expired */
  MONONN_ERR_CONSTANT = -7,        /* unknown constant name or wrong size */
  MONONN_ERR_IO = -8,              /* spec / dump directory I/O */
  MONONN_ERR_NOT_READY = -9,       /* launch before all constants were set */
  MONONN_ERR_TOO_LARGE = -10       /* size beyond a documented maximum */
};

typedef struct mononn_module mononn_module; /* opaque; free with mononn_destroy */

/* Replaces the environment + Config singleton of the reference
 * (mononn_engine/config/config.h:19-53, EnvVars.md:4-16). NULL strings fall back to the
 * environment variables TF_MONONN_DUMP_DIR / TF_MONONN_EXISTING_TUNING_SPEC_DIR /
 * TF_MONONN_THREADPOOL_SIZE. */
typedef struct {
  int device;                   /* CUDA device ordinal (the reference hard-codes 0) */
  const char* dump_dir;         /* where tune() writes specs and reports */
  const char* spec_dir;         /* existing tuning spec to load instead of tuning */
  int threadpool_size;          /* host threads that re-pack weights into tiles whenever a plan is
                                   (re)loaded, i.e. per tuning candidate; 0 = all cores */
  int tuning_level;             /* what mononn_tune searches: 0 nothing (times the heuristic spec),
                                   1 stage structure (qkv_fusion, row_fusion) and per-GEMM-class
                                   tiles timed on their own stage, 2 + the number of CTAs */
  unsigned barrier_timeout_us;  /* bound on every in-kernel wait, any value up to 2^32 - 1; 0 = 2 000 000 */
} mononn_options;

typedef struct {
  int index;        /* position in the kernel argument list */
  size_t bytes;
  int kind;         /* 0 parameter, 1 live-out, 2 temp */
  int param_number; /* HLO parameter_number for kind 0, live-out ordinal for kind 1 */
} mononn_arg_desc;

/* Parse -> fuse -> (load spec | heuristics) -> stage table.
 * Replaces IRParserFused::from_hlo_module_unique + OptimizationRunner::run_group_* +
 * GraphCodegen::generate as driven by MonoNNModule::generate_code
 * (mononn_engine/module/mononn_module.cc:39-159) and the spec-loading side of the
 * TF_MONONN_EXISTING_TUNING_SPEC_DIR hook (README.md:145-149). */
int mononn_compile_hlo_text(const char* hlo_text, size_t len, const char* kernel_name,
                            const mononn_options* options, mononn_module** out);

/* Standalone path: build the fused graph of an encoder family from a JSON configuration
 * instead of an HLO dump, e.g. {"model":"bert","layers":12,"hidden":768,"heads":12,
 * "ffn":3072,"vocab":30522,"max_pos":512,"types":2,"batch":1,"seq":128,"eps":1e-12,
 * "act":"gelu_erf"}. The model definitions are those the reference exports in
 * examples/utils/save_model.py:44-110; constants are named "embeddings.word",
 * "layer<i>.attn.q.w", ... (mononn_constant_info lists them). */
int mononn_compile_encoder_json(const char* config_json, const char* kernel_name,
                                const mononn_options* options, mononn_module** out);

/* Kernel argument list: parameters by parameter_number, live-outs, then temp
 * (mononn_engine/module/mononn_module.cc:91-143, README.md:186-200). */
int mononn_module_args(const mononn_module* m, const mononn_arg_desc** descs, int* n);

/* grid_dim, block_dim, dynamic shared memory: GraphSpecification.cuda_context.
 * cuda_runtime_context (mononn_engine/core/context/cuda_runtime_context.cc:32-55). */
int mononn_module_launch_config(const mononn_module* m, unsigned grid[3], unsigned block[3],
                                unsigned* smem_bytes);

/* Non-scalar HLO constants (the frozen weights). Replaces the
 * `__device__ uint8_t buffer_for_<name>[bytes]` module globals the TF side fills
 * (mononn_engine/codegen/graph_codegen.cc:71-86). `host` is row-major in the HLO shape. */
int mononn_set_constant(mononn_module* m, const char* hlo_constant_name, const void* host,
                        size_t bytes);
/* Number of constants and the i-th constant's name / byte size. */
int mononn_constant_count(const mononn_module* m, int* n);
int mononn_constant_info(const mononn_module* m, int i, const char** name, size_t* bytes);

/* Exactly one kernel launch on `cuda_stream` (a cudaStream_t), asynchronous.
 * Mirrors the launch sequence of mononn_engine/module/mononn_module_tuner.cc:99-150.
 * device_args[i] follows mononn_module_args order. The first launch with a new set of
 * argument pointers also uploads the re-bound stage table on the same stream. */
int mononn_launch(mononn_module* m, void* const* device_args, int n, void* cuda_stream);

/* One inference from and to HOST memory, the shape of the reference's user-facing call
 * (`sess.run` on host tensors, examples/run_mononn.py:72-84): copies host_inputs[k] (one per
 * parameter, by parameter number) into device_args, launches once, copies every live-out
 * into host_outputs[j], reads the kernel's status word and waits for `cuda_stream`. Pinned
 * host buffers make the copies asynchronous. Where device_args[i] IS the host buffer (pinned
 * memory is device-addressable under unified addressing) no copy is issued: the kernel reads
 * the parameter from, or writes the live-out to, host memory directly. Returns MONONN_ERR_BARRIER_TIMEOUT (and restores
 * the module) when a bounded wait expired in the kernel. */
int mononn_infer_host(mononn_module* m, const void* const* host_inputs, int n_inputs,
                      void* const* host_outputs, int n_outputs, void* const* device_args, int n,
                      void* cuda_stream);

/* Synchronises the device, then reports the kernel's status word: 0, or
 * MONONN_ERR_BARRIER_TIMEOUT with the stage and CTA that gave up. */
int mononn_last_status(mononn_module* m, int* stage, int* cta);

/* Search tile shapes on the device (MonoNNModuleTuner::tune,
 * mononn_engine/module/mononn_module_tuner.cc:620-991): per-GEMM candidates timed in
 * isolation with the allow-list mechanism, best ones merged, end-to-end pick. Needs all
 * constants set and a full argument list. Writes dump_dir/<cluster>/ when set. */
int mononn_tune(mononn_module* m, void* const* device_args, int n, void* cuda_stream);

/* Writes <dir>/<cluster_N>/best_tuning_spec.json (+ performance_report.csv when known):
 * the layout of mononn_engine/module/mononn_module_tuner.cc:584-603. */
int mononn_save_spec(const mononn_module* m, const char* dir);
/* JSON of the current spec; the pointer stays valid until the next call on `m`. */
int mononn_spec_json(mononn_module* m, const char** json);

/* Per-stage device time of the last profiled launch (performance_report.csv,
 * mononn_engine/module/mononn_module_tuner.cc:422-448): launches once with in-kernel
 * %globaltimer stamps, synchronises, fills up to `cap` entries of microseconds and sets
 * *n_stages. names[i] points into module storage. */
int mononn_profile_stages(mononn_module* m, void* const* device_args, int n, void* cuda_stream,
                          double* us, const char** names, int cap, int* n_stages);

/* Inspection. mononn_plan_json: the lowered stage table (stages, operators with tiles,
 * tensor placements, constant bindings) of a module; stands in for the `<context>_src/`
 * dump of the reference (mononn_engine/module/mononn_module_tuner.cc:560-575), since the
 * table is the artefact. mononn_describe lowers without touching a device (kind "hlo" or
 * "encoder", optional spec JSON, SM count) and returns {"plan":..,"spec":..} in a string
 * the caller frees with mononn_free_string. */
int mononn_plan_json(mononn_module* m, const char** json);
int mononn_describe(const char* kind, const char* text, size_t len, const char* spec_json,
                    unsigned sm_count, char** out_json);
void mononn_free_string(char* s);

/* Runs only stages [stage_begin, stage_end) in one launch: the single-node isolation of
 * the reference's codegen_allow_list (mononn_engine/tuning/tuning_space_generator.cc:405-414)
 * used for per-stage timing and for checking intermediate tensors. */
int mononn_launch_stages(mononn_module* m, void* const* device_args, int n, void* cuda_stream,
                         unsigned stage_begin, unsigned stage_end);

/* Per-CTA event trace of one launch: out[(cta * n_stages + stage) * 16 + event] in
 * nanoseconds since the earliest event (0 = event did not occur). Events: 0 epilogue warps
 * passed the previous barrier, 1 finished the stage's items, 2 arrived at the barrier,
 * 3 activation producer passed the barrier, 4 issued its last activation load, 5 MMA issuer
 * saw its first operands, 6 committed its last MMA, 7 weight producer issued its last load,
 * 8..15 finer marks inside the epilogue / row-wise code.
 * This is how the barrier's share of kernel time is measured without a profiler
 * (the reference's performance_report.csv isolates nodes instead,
 * mononn_engine/module/mononn_module_tuner.cc:422-448). cap counts doubles. */
int mononn_trace_stages(mononn_module* m, void* const* device_args, int n, void* cuda_stream,
                        double* out, size_t cap, int* grid, int* n_stages);

/* Test aid (host-side fault injection, no GPU fault involved): the next launch waits for
 * `missing_arrivals` grid-barrier arrivals that no CTA will make, so its first bounded wait
 * expires after barrier_timeout_us; the kernel then drains, returns, and
 * mononn_last_status reports MONONN_ERR_BARRIER_TIMEOUT and restores the module. */
int mononn_debug_skew_barrier(mononn_module* m, unsigned missing_arrivals);

/* Measurement aid: cycles per tcgen05.mma (128 x n x 16, f16 in, f32 accumulate) issued from
 * operands resident in shared memory, on `ctas` CTAs (one per SM) at once: `count` instructions
 * cycling through `accumulators` TMEM buffers, one commit at the end. mode bits (each mode is a
 * separately compiled kernel, so that no run-time test sits in the timed loop):
 *   0  a commit after every four instructions
 *   1  a satisfied mbarrier wait + tcgen05 fence before every four (bits 0 and 1 together are the
 *      bookkeeping of the kernel's main loop)
 *   2  M = 64 instead of 128
 *   3  the A operand is read from tensor memory instead of shared memory
 *   4  the instruction is written without the optional disable-output-lane vector
 *   5  the whole warp runs the loop converged and one elected lane issues (otherwise one lane
 *      runs it alone, diverged from the other 31)
 *   6  the operand descriptors are rebuilt for every group of four from a ring-slot index
 * cycles_per_mma covers first issue .. commit observed, issue_cycles_per_mma the issuing
 * thread alone. The issue loop of the kernel's MMA role and the GEMM tile menu of the tuner are
 * designed from this table; the reference times whole CUTLASS tiles instead
 * (mononn_engine/core/op_impl/gemm_impl.cc:505-566). */
int mononn_debug_mma_issue(int device, unsigned n, unsigned count, unsigned accumulators,
                           unsigned mode, unsigned ctas, double* cycles_per_mma,
                           double* issue_cycles_per_mma, double* ns_per_mma);

/* Algorithmic bytes and FLOPs of one inference (weights once + gathered rows + I/O). */
int mononn_module_cost(const mononn_module* m, double* bytes, double* flops);

/* Allocation-free attention (no counterpart in the reference, which leaves every buffer to
 * XLA's allocator and never allocates on its own).
 *
 * For hosts where this library must not call cudaMalloc: under TensorFlow/XLA the framework's
 * allocator normally owns the whole GPU, so an allocation made by a plug-in can fail or
 * fragment the pool, and serving threads avoid cudaMalloc because it synchronises the device.
 * The call runs one attention stage of the persistent kernel,
 *     out[b, s, h*64:(h+1)*64] = softmax(scale * Q_h K_h^T + (1 - mask) * mask_scale) V_h,
 * on caller-owned f16 buffers and keeps everything else the kernel needs (stage table, tensor
 * maps, barrier counter, status word, the f32 additive mask) in a static device array of
 * 2 KB + 4 * MONONN_NOALLOC_MAX_TOKENS bytes that every GPU loading the library holds until exit.
 *   q, k   f16 [batches*seq, ld_qk], head h in columns h*64 .. h*64+63
 *   v_t    f16 [batches*heads*64, ld_vt]: V transposed per batch (row = b*heads*64 + h*64 + d,
 *          column = key position)
 *   mask   int32 [batches, seq] or NULL;  out  f16 [batches*seq, ld_out]
 * Limits: seq <= 128, head dimension 64, batches*seq <= MONONN_NOALLOC_MAX_TOKENS (larger
 * sizes return MONONN_ERR_TOO_LARGE); base addresses and row pitches multiples of 16 bytes.
 * The call is asynchronous on `cuda_stream` and allocates nothing. All calls on a device
 * share the static array and rewrite it: calls that overlap on the GPU (other streams or
 * threads) race, so serialise them. The first call on a device does the one-time set-up
 * (device address of the array, kernel attributes) and should come before any stream capture.
 * Every call stages a small table from host memory, so a stream that is being captured is
 * refused with MONONN_ERR_INVALID_ARGUMENT. `out` and the row pitches must be 16-byte aligned;
 * a misaligned one is refused on the host, nothing is launched. */
#define MONONN_NOALLOC_MAX_TOKENS 16384
int mononn_attention_noalloc(const void* q, const void* k, const void* v_t, const int32_t* mask,
                             void* out, unsigned batches, unsigned heads, unsigned seq,
                             unsigned ld_qk, unsigned ld_vt, unsigned ld_out, float scale,
                             float mask_scale, int causal, void* cuda_stream);
/* Waits for `cuda_stream`, then reads the status word the kernel keeps in the same static array
 * (no allocation): MONONN_OK, or MONONN_ERR_BARRIER_TIMEOUT when a bounded wait expired during
 * the last mononn_attention_noalloc on this device, in which case `out` is incomplete. Like the
 * entry point itself it has no counterpart in the reference, whose kernels spin without a bound
 * (mononn_engine/core/gpu/synchronization.cc:45-97). */
int mononn_attention_noalloc_status(void* cuda_stream);

/* Operators behind a prompt: positions by rotation, a key/value cache of pages, attention of new
 * tokens over it (no counterpart in the reference, whose decoder graphs end with the prompt). They
 * work on caller-owned device memory, allocate nothing, launch on `cuda_stream` without waiting for it
 * and may be captured into a CUDA graph; pointers and sizes are those of the call, what indptr,
 * lengths, page_table and positions hold is read on the device at each launch. Every call runs on the device that owns
 * its first buffer (a stream of another device is refused) and restores the caller's current device.
 * What a call writes may not overlap what it reads or writes otherwise, but for what an entry point allows.
 * dtype: MONONN_F16 or MONONN_BF16 for every tensor of a call; sums, softmax and rotations are
 * computed in 32 bits (angles in 64). Strides count elements. */
enum { MONONN_F16 = 0, MONONN_BF16 = 1 };

/* How the turning rates of a rotary embedding follow from its configuration. Pair i of r / 2 turns
 * by f_i = theta^(-2i/r) radians a position, and with a longer context of `factor` times the
 * `original_length` by
 *   LINEAR  f_i / factor
 *   BASE    the same with theta * factor^(r/(r-2)) instead of theta
 *   RAMP    a blend that goes from f_i to f_i / factor over the pair's index, between the pairs that
 *           make `high` and `low` turns within original_length (defaults 32 and 1); values are
 *           multiplied by 0.1 ln(factor) + 1
 *   BANDS   the same blend over the number of turns itself, from f_i at `high` (default 4) or more
 *           to f_i / factor at `low` (default 1) or fewer. */
enum {
  MONONN_ROTARY_PLAIN = 0,
  MONONN_ROTARY_LINEAR = 1,
  MONONN_ROTARY_BASE = 2,
  MONONN_ROTARY_RAMP = 3,
  MONONN_ROTARY_BANDS = 4
};
#define MONONN_MAX_ROTARY_PAIRS 128
typedef struct {
  unsigned rotary_dim;    /* leading elements of a head that are rotated: even, 2 .. 256 */
  int interleaved;        /* pairs (2i, 2i+1); 0: pairs (i, i + rotary_dim/2) */
  int scaling;            /* MONONN_ROTARY_* */
  double theta;           /* 0 = 10000 */
  double factor;          /* of the scalings, > 0 */
  double original_length; /* RAMP and BANDS: positions the model was trained on */
  double low, high;       /* RAMP and BANDS: 0 = the defaults above */
  double magnitude;       /* what rotated values are multiplied by; 0 = 1, RAMP: 0.1 ln(factor) + 1
                             (1 for a factor of 1 or less) */
} mononn_rotary_config;
/* What the kernels read, a plain value owned by the caller: made once by mononn_rotary_init, or filled by hand. */
typedef struct {
  unsigned rotary_dim;
  int interleaved;
  double magnitude;
  double turns[MONONN_MAX_ROTARY_PAIRS]; /* f_i / 2 pi */
} mononn_rotary;
int mononn_rotary_init(const mononn_rotary_config* config, mononn_rotary* out);

/* out[t, h, :] = x[t, h, :] with its leading rotary_dim elements rotated by positions[t] (any int32);
 * the rest is copied. `out` may be `x` itself (same strides); other overlaps are not allowed.
 * head_dim up to 256. Without alignment to 16 bytes (addresses, strides, and 8 | head_dim; rotary_dim a
 * multiple of 16, interleaved of 8) a slower form of the kernel runs, element by element. */
typedef struct {
  const void* x;
  void* out;
  int64_t x_token_stride, x_head_stride, out_token_stride, out_head_stride;
  const int32_t* positions; /* [tokens] */
  unsigned tokens, heads, head_dim;
  int dtype;
} mononn_rotary_args;
int mononn_rotary_apply(const mononn_rotary* rotary, const mononn_rotary_args* args, void* cuda_stream);

/* A cache of keys and values in pages of page_size tokens. Element (token row r, head h, d) of page p is at
 * p * page_stride + r * token_stride + h * head_stride + d in k_pages and v_pages alike, so pages may be
 * token-major or head-major. Sequence b's keys 0 .. lengths[b]-1 are in the pages page_table[b *
 * table_stride + key / page_size]. Attention counts a length beyond max_pages * page_size as that; the append
 * writes no token at a position beyond it. Sequences may share pages. A page number outside of 0 ..
 * num_pages-1 is never followed: its tokens are not written, and read as zeros. New tokens are packed: sequence
 * b has the rows indptr[b] .. indptr[b+1]-1 of the token tensors (indptr: [sequences + 1], not decreasing), and
 * they are its LAST positions: row indptr[b] + i is at position lengths[b] - (indptr[b+1] - indptr[b]) + i, so
 * `lengths` counts them.
 * Rows outside of every sequence (behind indptr[sequences]) are left as they were. */
typedef struct {
  void* k_pages;
  void* v_pages;
  int64_t page_stride, token_stride, head_stride;
  const int32_t* page_table;
  int64_t table_stride;
  const int32_t* lengths;
  unsigned sequences, max_pages, num_pages, page_size, kv_heads, head_dim;
  int dtype;
} mononn_paged_cache;

/* Writes the new tokens' keys and values into their pages, the keys rotated by their position on
 * the way (rotary NULL: as they are), and rotates the queries of the same tokens in the same launch
 * (q NULL: none; q_out may be q itself). positions: what is rotated by instead of the position in
 * the cache, or NULL. A token without a place (a negative position, a page number out of range) is not
 * written; its query is rotated all the same. Two tokens that fall on one place of a
 * shared page leave a mixture there, each element one of the two (so equal tokens may share it). k, v and q are
 * not themselves in the pages, and no element is at once in a written page of k_pages and in one of v_pages
 * (within one page that is refused). Alignment as mononn_rotary_apply. */
typedef struct {
  const void *k, *v;
  int64_t k_token_stride, k_head_stride, v_token_stride, v_head_stride;
  const void* q;
  void* q_out;
  int64_t q_token_stride, q_head_stride, q_out_token_stride, q_out_head_stride;
  const int32_t* indptr;
  const int32_t* positions;
  unsigned tokens, q_heads; /* rows of the token tensors */
} mononn_paged_append_args;
int mononn_paged_append(const mononn_paged_cache* cache, const mononn_rotary* rotary,
                        const mononn_paged_append_args* args, void* cuda_stream);

/* out[t, h, :] = sum_j p_j v_j,  p = softmax over the visible keys j of scale * q[t, h] . k_j,
 * where head h reads key head h / (q_heads / kv_heads). A token at position p sees the keys j <= p
 * (causal; otherwise all of its sequence), and with window > 0 (causal only) of those the ones with
 * j > p - window. A row that sees nothing becomes zeros (lse: minus infinity), as one whose scores are all minus infinity;
 * one whose scores, times scale and log2 e, leave 32 bits becomes NaN. lse: natural
 * logarithm of the sum of the exponentials, f32 [tokens, q_heads], or NULL. Keys that no row
 * of a sequence sees and page rows behind a length may hold anything, NaN too; an infinity or NaN among the values
 * that some of a sequence's new tokens see may reach those of its new tokens that do not (its weight there is zero).
 * max_new: at most how many new tokens a sequence has, as a hint that chooses between the kernel for
 * few rows (single tokens, drafts) and the one for many; 0 = unknown. Results are right whatever it says. The other
 * thing that a launch is planned by is the table's width, max_pages, since lengths are on the device: in a table that is much
 * wider than its sequences items are split although they are short, which costs a workspace and the launch that joins them
 * (a table of 131072 keys: 1 to 4 us a call). A chunk of a prompt beside many sequences' single tokens takes less time
 * as two calls.
 * The same arguments and contents give the same bits again. No gradients.
 * Limits: head_dim a multiple of 8 up to 128; page_size a multiple of 8; q_heads / kv_heads whole (up to 128 have
 * a kernel for many rows; above, every 16 rows read the keys again); addresses of pages, q and out, and all their
 * strides, multiples of 16 bytes (lse, indptr: 4); new tokens x keys such that the tiles of both, with max_pages *
 * page_size keys for every sequence, count below 2^31. The first call of these operators on a device loads their
 * kernels: make it before a stream is captured. */
typedef struct {
  const void* q;
  void* out;
  float* lse;
  int64_t q_token_stride, q_head_stride, out_token_stride, out_head_stride;
  const int32_t* indptr;
  unsigned tokens, q_heads;
  float scale; /* > 0; 0 = 1 / sqrt(head_dim) */
  int causal;
  unsigned window;
  unsigned max_new;
  void* workspace; /* of mononn_paged_attention_workspace bytes, 16-byte aligned; needs no initial
                      state; calls that overlap on the GPU need one each */
  size_t workspace_bytes;
} mononn_paged_attention_args;
int mononn_paged_attention(const mononn_paged_cache* cache, const mononn_paged_attention_args* args,
                           void* cuda_stream);
/* Bytes for calls with this cache and these arguments (0: none), whatever the device arrays hold. */
int mononn_paged_attention_workspace(const mononn_paged_cache* cache, const mononn_paged_attention_args* args,
                                     size_t* bytes);
/* Waits for `cuda_stream`, then reports and clears the status word that the attention kernels of its
 * device share: MONONN_OK, or MONONN_ERR_BARRIER_TIMEOUT when a bounded wait expired in one of them
 * since the last report (its output is incomplete). A null stream is the default one of the current device. */
int mononn_paged_attention_status(void* cuda_stream);
/* Test aid, as mononn_debug_skew_barrier: this thread's next mononn_paged_attention waits for one arrival that
 * nobody makes on the given barriers of its kernel, so that a bounded wait there runs out; its output is
 * incomplete, and mononn_paged_attention_status reports it. 1: keys or values landed, 2: their slot free, 3: a
 * piece of work told, 4: taken, 5: queries landed; kernel for few rows 6: its warps' meeting; kernel for many rows 7:
 * scores made, 8: read (64-wide heads), 9: probabilities made, 10: outputs made, 11: queries used, 12 and 13: the second of two
 * row tiles that take turns done, and read. 0: none. A call that has no wait on the barrier is an ordinary one. */
int mononn_debug_paged_skew(unsigned barrier);

void mononn_destroy(mononn_module* m);
const char* mononn_strerror(int code);
/* Message of the last failing call on this thread. */
const char* mononn_last_error(void);

/* TF_MONONN_ENABLED is truthy for "True", "true" or "1"
 * (mononn_engine/helpers/env_variable.cc:20-26); the host shim does not call in otherwise. */
int mononn_enabled(void);

#ifdef __cplusplus
}
#endif
#endif /* MONONN_B200_H_ */
