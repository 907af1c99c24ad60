// C entry points of the operators behind a prompt (declared in include/mononn.h): checks of arguments,
// tensor maps, the division into kernels and workspaces. No device memory is read or allocated here.
#include "paged.h"

#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>
#include <cstdio>
#include <initializer_list>
#include <mutex>
#include <numeric>
#include <string>
#include <utility>

#include "../../include/mononn.h"
#include "runtime.h"

using namespace mononn;

namespace {

// Nothing is thrown across the C entry points: a message that finds no memory is left out.
int fail(int code, const char* msg, const char* more = "") {
  try {
    set_last_error(std::string(msg) + more);
  } catch (...) {
  }
  return code;
}
int invalid(const char* msg) { return fail(MONONN_ERR_INVALID_ARGUMENT, msg); }

#define PG_TRY(expr)                                                                         \
  do {                                                                                       \
    cudaError_t e__ = (expr);                                                                \
    if (e__ != cudaSuccess) return fail(MONONN_ERR_CUDA, #expr ": ", cudaGetErrorString(e__)); \
  } while (0)

// A launch on a stream of another device than the kernel's ends in this error (the stream itself cannot be
// asked for its device while it is captured).
int launched(cudaError_t e) {
  if (e == cudaSuccess) return MONONN_OK;
  cudaGetLastError();
  if (e == cudaErrorInvalidResourceHandle)
    return invalid("the stream belongs to another device than the buffers, or to none");
  return fail(MONONN_ERR_CUDA, "kernel launch: ", cudaGetErrorString(e));
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

constexpr int kMaxDevices = 64;
struct Device {
  bool ready = false;
  int sm_count = 0;
  uint32_t* status = nullptr;
};
Device g_devices[kMaxDevices];
std::mutex g_mutex;
EncodeTiledFn g_encode = nullptr;
thread_local uint32_t t_skewed = kBarrierNone;  // of this thread's next attention call

// One-time set-up of the current device.
int set_up(int dev, const Device** out) {
  std::lock_guard<std::mutex> lock(g_mutex);
  Device& d = g_devices[dev];
  if (!d.ready) {
    int major = 0;
    PG_TRY(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev));
    if (major != 10) return fail(MONONN_ERR_NO_DEVICE, "the kernels are built for sm_100a only");
    PG_TRY(cudaDeviceGetAttribute(&d.sm_count, cudaDevAttrMultiProcessorCount, dev));
    PG_TRY(paged_status_word(&d.status));
    // every kernel is loaded here, none during a capture later
    PG_TRY(prepare_rows());
    PG_TRY(prepare_few_rows());
    PG_TRY(prepare_many_rows());
    if (!g_encode) {
      cudaDriverEntryPointQueryResult q;
      void* fn = nullptr;
      PG_TRY(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q));
      if (q != cudaDriverEntryPointSuccess || !fn)
        return fail(MONONN_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
      g_encode = reinterpret_cast<EncodeTiledFn>(fn);
    }
    d.ready = true;
  }
  *out = &d;
  return MONONN_OK;
}

// The device of a call is the one that owns its first buffer; the caller's current one comes back at the end.
class OnDeviceOf {
 public:
  ~OnDeviceOf() {
    if (previous_ >= 0) cudaSetDevice(previous_);
  }
  int enter(const void* buffer, const Device** out) {
    int count = 0;
    if (cudaGetDeviceCount(&count) != cudaSuccess || count == 0) {
      cudaGetLastError();
      return fail(MONONN_ERR_NO_DEVICE, "no CUDA device");
    }
    cudaPointerAttributes a;
    PG_TRY(cudaPointerGetAttributes(&a, buffer));
    if (a.type != cudaMemoryTypeDevice && a.type != cudaMemoryTypeManaged)
      return invalid("buffers have to be in device memory");
    if (a.device < 0 || a.device >= kMaxDevices) return invalid("device ordinal out of range");
    int current = 0;
    PG_TRY(cudaGetDevice(&current));
    if (current != a.device) {
      PG_TRY(cudaSetDevice(a.device));
      previous_ = current;
    }
    return set_up(a.device, out);
  }

 private:
  int previous_ = -1;
};

bool aligned(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
bool whole8(int64_t stride) { return (stride & 7) == 0; }

// Strides that no tensor of this size can have are refused, so that the kernels' 64-bit offsets never wrap.
bool stride_in_range(int64_t s) { return s >= 0 && s < (1ll << 39); }

// Whether no two elements share a place (what is written would depend on an order): by growing stride, each
// dimension has to reach over all that the smaller ones span.
using Dimension = std::pair<uint32_t, int64_t>;  // size, stride
bool apart(uint32_t head_dim, std::initializer_list<Dimension> dims) {
  Dimension sorted[3];  // as many as any caller has
  size_t n = 0;
  for (const Dimension& d : dims)
    if (d.first > 1) sorted[n++] = d;
  std::sort(sorted, sorted + n, [](const Dimension& a, const Dimension& b) { return a.second < b.second; });
  unsigned __int128 span = head_dim;
  for (size_t i = 0; i < n; ++i) {
    if (static_cast<uint64_t>(sorted[i].second) < span) return false;
    span += static_cast<unsigned __int128>(sorted[i].first - 1) * static_cast<uint64_t>(sorted[i].second);
  }
  return true;
}

int check_dtype(int dtype) {
  if (dtype != MONONN_F16 && dtype != MONONN_BF16)
    return fail(MONONN_ERR_UNSUPPORTED, "dtype must be MONONN_F16 or MONONN_BF16");
  return MONONN_OK;
}
int check_rotary(const mononn_rotary& r, unsigned head_dim) {
  if (r.rotary_dim == 0 || (r.rotary_dim & 1u) || r.rotary_dim > 2 * MONONN_MAX_ROTARY_PAIRS || r.rotary_dim > head_dim)
    return invalid("rotary_dim must be even, at least 2 and at most head_dim");
  // the kernel takes the magnitude in 32 bits, and the angle of the farthest position in 64
  if (!(std::fabs(r.magnitude) <= FLT_MAX)) return invalid("rotary magnitude must be finite in 32 bits");
  for (unsigned i = 0; i < r.rotary_dim / 2; ++i)
    if (!std::isfinite(r.turns[i] * 2147483648.0))
      return invalid("rotary rates must be finite, and so the angles of all 32-bit positions");
  return MONONN_OK;
}
int check_cache(const mononn_paged_cache& c) {
  if (!c.k_pages || !c.v_pages || !c.page_table || !c.lengths) return invalid("cache: null pointer");
  if (int rc = check_dtype(c.dtype)) return rc;
  if (c.page_size == 0 || c.kv_heads == 0 || c.head_dim == 0 || c.max_pages == 0 || c.num_pages == 0)
    return invalid("cache: a size is zero");
  if (c.num_pages > INT_MAX || c.kv_heads > 65536 || c.head_dim > 256 || c.sequences > (1u << 24))
    return fail(MONONN_ERR_TOO_LARGE, "cache: num_pages < 2^31, kv_heads <= 65536, head_dim <= 256, sequences <= 2^24");
  if (static_cast<uint64_t>(c.max_pages) * c.page_size > (1u << 30))
    return fail(MONONN_ERR_TOO_LARGE, "cache: max_pages * page_size exceeds 2^30 keys");
  if (!stride_in_range(c.page_stride) || !stride_in_range(c.token_stride) || !stride_in_range(c.head_stride) ||
      c.table_stride < c.max_pages || !stride_in_range(c.table_stride))
    return invalid("cache: strides must be in 0 .. 2^39, table_stride at least max_pages");
  if (!aligned(c.page_table, 4) || !aligned(c.lengths, 4) || !aligned(c.k_pages, 2) || !aligned(c.v_pages, 2))
    return invalid("cache: misaligned pointer");
  const int64_t d = c.head_dim;
  if ((c.page_size > 1 && c.token_stride < d) || (c.kv_heads > 1 && c.head_stride < d) ||
      (c.num_pages > 1 && c.page_stride < d))
    return invalid("cache: strides are smaller than the heads they hold");
  return MONONN_OK;
}

// Elements of 16-byte vectors are read and written whole where everything is aligned to them.
bool rows_by_vectors(const RowsParams& p) {
  bool ok = p.head_dim % 8 == 0 && p.rotary_dim % (p.interleaved ? 8 : 16) == 0 && whole8(p.page_stride);
  for (const RowsSource* s : {&p.q, &p.k, &p.v})
    if (s->heads)
      ok = ok && aligned(s->src, 16) && aligned(s->dst, 16) && whole8(s->src_token) && whole8(s->src_head) &&
           whole8(s->dst_token) && whole8(s->dst_head);
  return ok;
}
void set_rotation(RowsParams* p, const mononn_rotary& r) {
  p->rotary_dim = r.rotary_dim;
  p->interleaved = r.interleaved != 0;
  p->magnitude = static_cast<float>(r.magnitude);
  for (unsigned i = 0; i < r.rotary_dim / 2; ++i) p->turns[i] = r.turns[i];
}

int encoded(CUresult r, const char* what) {
  if (r == CUDA_SUCCESS) return MONONN_OK;
  char detail[64];
  std::snprintf(detail, sizeof(detail), ": cuTensorMapEncodeTiled failed (CUresult %d)", static_cast<int>(r));
  return fail(MONONN_ERR_CUDA, what, detail);
}
// Elements are 16 bits wide. One box is 64 elements of a head x `box` rows of one page; elements behind
// head_dim, rows and pages out of range arrive as zeros.
int encode_pages(CUtensorMap* map, const mononn_paged_cache& c, const void* base, uint32_t box, const char* what) {
  const cuuint64_t dims[4] = {c.head_dim, c.page_size, c.kv_heads, c.num_pages};
  // the stride of a dimension of one element is never used, but has to be valid
  auto stride = [&](int64_t s, unsigned n) { return static_cast<cuuint64_t>(n > 1 ? s : (c.head_dim + 7) / 8 * 8) * 2; };
  const cuuint64_t strides[3] = {stride(c.token_stride, c.page_size), stride(c.head_stride, c.kv_heads),
                                 stride(c.page_stride, c.num_pages)};
  const cuuint32_t boxes[4] = {64, box, 1, 1}, steps[4] = {1, 1, 1, 1};
  const CUresult r = g_encode(map, c.dtype == MONONN_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                              4, const_cast<void*>(base), dims, strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return encoded(r, what);
}

// One box is 64 elements of the heads of a group x the tokens of a row tile.
int encode_queries(CUtensorMap* map, const mononn_paged_cache& c, const mononn_paged_attention_args& a, const AttentionPlan& plan) {
  const uint32_t group = a.q_heads / c.kv_heads;
  const cuuint64_t dims[3] = {c.head_dim, a.q_heads, a.tokens};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(a.q_heads > 1 ? a.q_head_stride : c.head_dim) * 2,
                                 static_cast<cuuint64_t>(a.tokens > 1 ? a.q_token_stride : c.head_dim) * 2};
  const cuuint32_t boxes[3] = {64, group, plan.item_rows / 2 / group}, steps[3] = {1, 1, 1};
  const CUresult r = g_encode(map, c.dtype == MONONN_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                              3, const_cast<void*>(a.q), dims, strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return encoded(r, "q");
}

int check_attention(const mononn_paged_cache* cache, const mononn_paged_attention_args* a) {
  if (int rc = check_cache(*cache)) return rc;
  const mononn_paged_cache& c = *cache;
  if (c.head_dim % 8 || c.head_dim > 128)
    return fail(MONONN_ERR_UNSUPPORTED, "attention: head_dim must be a multiple of 8 up to 128");
  if (c.page_size % 8) return fail(MONONN_ERR_UNSUPPORTED, "attention: page_size must be a multiple of 8");
  if (!a->q || !a->out || !a->indptr) return invalid("attention: null pointer");
  if (a->q_heads == 0 || a->q_heads % c.kv_heads) return invalid("attention: q_heads must be a multiple of kv_heads");
  if (a->q_heads > 65536 || static_cast<uint64_t>(a->tokens) * (a->q_heads / c.kv_heads) > INT_MAX)
    return fail(MONONN_ERR_TOO_LARGE, "attention: q_heads <= 65536, tokens * q_heads / kv_heads < 2^31");
  if (!stride_in_range(a->q_token_stride) || !stride_in_range(a->q_head_stride) ||
      !stride_in_range(a->out_token_stride) || !stride_in_range(a->out_head_stride))
    return invalid("attention: strides must be in 0 .. 2^39");
  const int64_t d = c.head_dim;
  if ((a->q_heads > 1 && a->q_head_stride < d) || (a->tokens > 1 && a->q_token_stride < d))
    return invalid("attention: strides of q are smaller than the heads they hold");
  if (!apart(c.head_dim, {{a->tokens, a->out_token_stride}, {a->q_heads, a->out_head_stride}}))
    return invalid("attention: strides put elements of out into one place");
  if (!aligned(c.k_pages, 16) || !aligned(c.v_pages, 16) || !whole8(c.page_stride) || !whole8(c.token_stride) ||
      !whole8(c.head_stride) || !aligned(a->q, 16) || !whole8(a->q_token_stride) || !whole8(a->q_head_stride) ||
      !aligned(a->out, 16) || !whole8(a->out_token_stride) || !whole8(a->out_head_stride))
    return invalid("attention: addresses and strides of pages, q and out must be multiples of 16 bytes");
  if (!aligned(a->lse, 4) || !aligned(a->indptr, 4)) return invalid("attention: lse and indptr must be 4-byte aligned");
  if (!std::isfinite(a->scale * 2.f) || a->scale < 0.f) return invalid("attention: scale must be positive and finite, or 0");
  if (a->window && !a->causal) return invalid("attention: a window needs causal attention");
  return MONONN_OK;
}

// Which kernel, how many CTAs, and whether an item may span them. Only sizes count that the host knows.
// What an item takes beside its keys counts as units, too: with one instead of two for many rows, 8 prompts of 1000 and 2000
// tokens take 103.8 and 286 us instead of 99.2 and 278 (three: 102.4 and 284); few rows: no difference between one and two.
int plan_attention(const mononn_paged_cache& c, const mononn_paged_attention_args& a, int sm_count, AttentionPlan* p) {
  const uint32_t group = a.q_heads / c.kv_heads;
  const uint64_t capacity = static_cast<uint64_t>(c.max_pages) * c.page_size;
  const uint64_t new_tokens = a.max_new ? a.max_new : (static_cast<uint64_t>(a.tokens) + c.sequences - 1) / c.sequences;
  const uint64_t most_rows = static_cast<uint64_t>(a.tokens) * group;
  // a row tile for each `rows` rows at most, and a ragged one for each sequence
  auto items = [&](uint32_t rows) { return (most_rows / rows + std::min<uint64_t>(c.sequences, a.tokens)) * c.kv_heads; };
  auto tiles = [&](uint32_t keys) { return (capacity + keys - 1) / keys; };
  constexpr uint64_t kMostUnits = 1ull << 31;
  const uint64_t rows = std::min<uint64_t>(new_tokens * group, most_rows);
  p->padded_dim = c.head_dim <= 64 ? 64 : 128;
  const uint32_t few = few_keys(p->padded_dim);
  const uint32_t whole_tokens = group <= kTileRows ? kTileRows / group * group : 0;  // rows of a row tile of the other
  // More than 16 rows: the kernel for many, which takes 53, 55, 56, 57 and 62 us for 16, 32, 48, 64 and 128 rows of 16 sequences
  // of 3350 keys (8 key heads of 128), where the one for few takes 46, 62, 114, 146 and 252 (keys read again). But
  // calls that leave most of the GPU idle are done as soon or sooner by the one for few, which starts and ends faster and has
  // twice the CTAs: up to an item for each of those and seven units in all (8 key heads, 64 rows, few and many: a sequence of
  // 2000 keys 16.1 and 16.1 us, four 27.4 and 21.2; eight of 500 keys 14.5 and 14.9, of 1000 30.0 and 22.0;
  // 128 rows, eight of 250 keys: 16.6 and 12.5).
  const uint64_t few_ctas = 2 * static_cast<uint64_t>(static_cast<unsigned>(sm_count));
  const uint64_t few_items =
      std::min<uint64_t>(c.sequences, a.tokens) * c.kv_heads * ((new_tokens * group + kFewRows - 1) / kFewRows);
  const bool idle = few_items <= few_ctas && few_items * tiles(few) <= 7 * few_ctas;
  p->many = whole_tokens && ((rows > kFewRows && !idle) || items(kFewRows) * (tiles(few) + 2) >= kMostUnits);
  // Where an item's rows fill no more than one row tile, that tile and the other take turns with the keys: 16 drafts of 3 to 8
  // tokens over 700 to 6000 keys (8 x 5 heads of 128) 53 us instead of 58, 48 of 32 tokens over 2000 keys (8 x 4) 101 instead
  // of 105, 16 of 128 over 8000 (12 heads of 64) 121 instead of 129. The code for it costs prompts 1 to 4 %, so it is another form.
  p->turns = p->many && new_tokens * group <= whole_tokens;
  p->rows = p->many ? kManyRows : kFewRows;
  p->item_rows = p->many ? 2 * whole_tokens : kFewRows;
  p->keys = p->many ? kManyKeys : few;
  // Units of a CTA's share, at least: joining takes longer than they do otherwise (many rows, 32 of them over 1000 keys,
  // 8 key heads: 14.9 us with shares of one unit, 15.2 of two, 18.0 of four, 23.9 of eight; 400 rows: 20.9, 18.6, 20.4, 27.4;
  // single tokens over 1000 keys: 8.6 with one unit, 9.1 with two, 13.1 with eight).
  p->least_units = p->many ? 2 : 1;
  p->box = std::gcd(c.page_size, p->keys);
  p->item_cost = p->many ? 2 : 1;
  const uint64_t most_units = items(p->item_rows) * (tiles(p->keys) + p->item_cost);
  if (most_units >= kMostUnits)
    return fail(MONONN_ERR_TOO_LARGE, "attention: so many new tokens over so many keys count 2^31 units of work or more");
  const uint64_t most = static_cast<uint64_t>(p->many ? 1 : 2) * static_cast<unsigned>(sm_count);
  // Short caches: no item is split, and the join not needed. One sequence and 8 key heads: 250 keys 7.8 us whole and 8.6
  // split, 500 keys 10.6 and 8.0 (4 and 8 units); 64 sequences: 13.8 and 16.7, 26.7 and 29.4; a prompt of 500 tokens 16.6 and 27.8.
  const bool whole = tiles(p->keys) <= 4 || (!p->many && tiles(p->keys) <= 8 && 2 * items(p->item_rows) >= most);
  const uint64_t wanted = whole ? items(p->item_rows) : (most_units + p->least_units - 1) / p->least_units;
  p->ctas = static_cast<uint32_t>(std::max<uint64_t>(1, std::min(wanted, most)));
  p->joins = !whole && p->ctas > 1;
  p->workspace = 0;
  if (p->joins) {
    const size_t headers = (p->ctas * sizeof(AttentionHeader) + 255) / 256 * 256;
    p->workspace = headers + 2 * static_cast<size_t>(p->ctas) * attention_slot_floats(*p) * sizeof(float);
  }
  return MONONN_OK;
}
}  // namespace

extern "C" {

int mononn_rotary_init(const mononn_rotary_config* config, mononn_rotary* out) {
  if (!config || !out) return invalid("null argument");
  const mononn_rotary_config& c = *config;
  const unsigned r = c.rotary_dim;
  if (r == 0 || (r & 1u) || r > 2 * MONONN_MAX_ROTARY_PAIRS) return invalid("rotary_dim must be even, 2 .. 256");
  if (c.scaling < MONONN_ROTARY_PLAIN || c.scaling > MONONN_ROTARY_BANDS) return invalid("unknown rotary scaling");
  double theta = c.theta == 0.0 ? 10000.0 : c.theta;
  if (!(theta > 1.0) || !std::isfinite(theta)) return invalid("rotary theta must be finite and above 1");
  const double s = c.scaling == MONONN_ROTARY_PLAIN ? 1.0 : c.factor;
  if (!(s > 0.0) || !std::isfinite(s)) return invalid("rotary factor must be positive and finite");
  const bool blended = c.scaling == MONONN_ROTARY_RAMP || c.scaling == MONONN_ROTARY_BANDS;
  const double low = c.low == 0.0 ? 1.0 : c.low;
  const double high = c.high == 0.0 ? (c.scaling == MONONN_ROTARY_RAMP ? 32.0 : 4.0) : c.high;
  if (blended && !(c.original_length > 0.0 && std::isfinite(c.original_length)))
    return invalid("rotary original_length must be positive and finite");
  if (blended && !(low > 0.0 && high > low && std::isfinite(high))) return invalid("rotary turns: 0 < low < high");
  if (!std::isfinite(c.magnitude) || c.magnitude < 0.0) return invalid("rotary magnitude must be finite and not negative");
  const double two_pi = 6.283185307179586476925286766559;
  if (c.scaling == MONONN_ROTARY_BASE && r > 2) theta *= std::pow(s, static_cast<double>(r) / (r - 2.0));
  double first = 0.0, last = 0.0;
  if (c.scaling == MONONN_ROTARY_RAMP) {
    auto pair = [&](double turns) {
      return r * std::log(c.original_length / (turns * two_pi)) / (2.0 * std::log(theta));
    };
    first = std::max(0.0, std::floor(pair(high)));
    last = std::min(r - 1.0, std::ceil(pair(low)));
  }
  mononn_rotary made{};
  made.rotary_dim = r;
  made.interleaved = c.interleaved != 0;
  made.magnitude = c.magnitude != 0.0 ? c.magnitude
                   : c.scaling == MONONN_ROTARY_RAMP && s > 1.0 ? 0.1 * std::log(s) + 1.0 : 1.0;
  for (unsigned i = 0; i < r / 2; ++i) {
    double f = std::pow(theta, -2.0 * i / r);
    auto blend = [&](double slow) { f = (1.0 - slow) * f + slow * f / s; };
    auto clamp = [](double x) { return std::min(1.0, std::max(0.0, x)); };
    if (c.scaling == MONONN_ROTARY_LINEAR) f /= s;
    if (c.scaling == MONONN_ROTARY_RAMP) blend(clamp((i - first) / std::max(last - first, 0.001)));
    if (c.scaling == MONONN_ROTARY_BANDS) blend(1.0 - clamp((c.original_length * f / two_pi - low) / (high - low)));
    made.turns[i] = f / two_pi;
  }
  if (int rc = check_rotary(made, r)) return rc;
  *out = made;
  return MONONN_OK;
}

int mononn_rotary_apply(const mononn_rotary* rotary, const mononn_rotary_args* args, void* cuda_stream) {
  if (!rotary || !args) return invalid("null argument");
  const mononn_rotary_args& a = *args;
  if (a.tokens == 0 || a.heads == 0) return MONONN_OK;
  if (int rc = check_dtype(a.dtype)) return rc;
  if (a.head_dim == 0 || a.head_dim > 256 || a.heads > 65536)
    return fail(MONONN_ERR_TOO_LARGE, "rotary: head_dim in 1 .. 256, heads <= 65536");
  if (int rc = check_rotary(*rotary, a.head_dim)) return rc;
  if (!stride_in_range(a.x_token_stride) || !stride_in_range(a.x_head_stride) ||
      !stride_in_range(a.out_token_stride) || !stride_in_range(a.out_head_stride))
    return invalid("rotary: strides must be in 0 .. 2^39");
  if (a.tokens > INT_MAX) return fail(MONONN_ERR_TOO_LARGE, "rotary: tokens < 2^31");
  if (!a.x || !a.out || !a.positions) return invalid("rotary: null pointer");
  if (!aligned(a.x, 2) || !aligned(a.out, 2) || !aligned(a.positions, 4)) return invalid("rotary: misaligned pointer");
  if (!apart(a.head_dim, {{a.tokens, a.out_token_stride}, {a.heads, a.out_head_stride}}))
    return invalid("rotary: strides put elements of out into one place");
  if (a.x == a.out && (a.x_token_stride != a.out_token_stride || a.x_head_stride != a.out_head_stride))
    return invalid("rotary: in place, x and out have the same strides");
  OnDeviceOf guard;
  const Device* dev = nullptr;
  if (int rc = guard.enter(a.out, &dev)) return rc;
  RowsParams p{};
  p.q = RowsSource{a.x, a.out, a.x_token_stride, a.x_head_stride, a.out_token_stride, a.out_head_stride, a.heads};
  p.positions = a.positions;
  p.tokens = a.tokens;
  p.head_dim = a.head_dim;
  set_rotation(&p, *rotary);
  return launched(launch_rows(p, a.dtype == MONONN_BF16, rows_by_vectors(p), dev->sm_count,
                              static_cast<cudaStream_t>(cuda_stream)));
}

int mononn_paged_append(const mononn_paged_cache* cache, const mononn_rotary* rotary,
                        const mononn_paged_append_args* args, void* cuda_stream) {
  if (!cache || !args) return invalid("null argument");
  if (args->tokens == 0 || cache->sequences == 0) return MONONN_OK;
  if (int rc = check_cache(*cache)) return rc;
  const mononn_paged_cache& c = *cache;
  const mononn_paged_append_args& a = *args;
  if (rotary)
    if (int rc = check_rotary(*rotary, c.head_dim)) return rc;
  if (!a.k || !a.v || !a.indptr) return invalid("append: null pointer");
  if ((a.q == nullptr) != (a.q_out == nullptr)) return invalid("append: q and q_out go together");
  if (a.q && a.q_heads == 0) return invalid("append: q without heads");
  if (a.tokens > INT_MAX || a.q_heads > 65536)
    return fail(MONONN_ERR_TOO_LARGE, "append: tokens < 2^31, q_heads <= 65536");
  if (!stride_in_range(a.k_token_stride) || !stride_in_range(a.k_head_stride) || !stride_in_range(a.v_token_stride) ||
      !stride_in_range(a.v_head_stride) || !stride_in_range(a.q_token_stride) || !stride_in_range(a.q_head_stride) ||
      !stride_in_range(a.q_out_token_stride) || !stride_in_range(a.q_out_head_stride))
    return invalid("append: strides must be in 0 .. 2^39");
  if (!aligned(a.k, 2) || !aligned(a.v, 2) || !aligned(a.q, 2) || !aligned(a.q_out, 2) || !aligned(a.indptr, 4) ||
      !aligned(a.positions, 4))
    return invalid("append: misaligned pointer");
  const uintptr_t k_at = reinterpret_cast<uintptr_t>(c.k_pages), v_at = reinterpret_cast<uintptr_t>(c.v_pages);
  const uint64_t between = (k_at < v_at ? v_at - k_at : k_at - v_at) / 2;
  if (between > INT64_MAX / 2 || !apart(c.head_dim, {{c.page_size, c.token_stride}, {c.kv_heads, c.head_stride},
                                                     {2, static_cast<int64_t>(between)}}))
    return invalid("append: keys and values of a page go to the same places");
  if (!apart(c.head_dim, {{c.page_size, c.token_stride}, {c.kv_heads, c.head_stride}, {c.num_pages, c.page_stride}}))
    return invalid("append: strides put elements of pages into one place");
  if (a.q && !apart(c.head_dim, {{a.tokens, a.q_out_token_stride}, {a.q_heads, a.q_out_head_stride}}))
    return invalid("append: strides put elements of q_out into one place");
  if (a.q && a.q == a.q_out &&
      (a.q_token_stride != a.q_out_token_stride || a.q_head_stride != a.q_out_head_stride))
    return invalid("append: in place, q and q_out have the same strides");
  OnDeviceOf guard;
  const Device* dev = nullptr;
  if (int rc = guard.enter(c.k_pages, &dev)) return rc;
  RowsParams p{};
  if (a.q)
    p.q = RowsSource{a.q, a.q_out, a.q_token_stride, a.q_head_stride, a.q_out_token_stride, a.q_out_head_stride, a.q_heads};
  p.k = RowsSource{a.k, c.k_pages, a.k_token_stride, a.k_head_stride, c.token_stride, c.head_stride, c.kv_heads};
  p.v = RowsSource{a.v, c.v_pages, a.v_token_stride, a.v_head_stride, c.token_stride, c.head_stride, c.kv_heads};
  p.positions = a.positions;
  p.indptr = a.indptr;
  p.lengths = c.lengths;
  p.table = c.page_table;
  p.table_stride = c.table_stride;
  p.page_stride = c.page_stride;
  p.tokens = a.tokens;
  p.head_dim = c.head_dim;
  p.sequences = c.sequences;
  p.max_pages = c.max_pages;
  p.num_pages = c.num_pages;
  p.page_size = c.page_size;
  p.by_page_size = make_divisor(c.page_size);
  if (rotary) set_rotation(&p, *rotary);
  return launched(launch_rows(p, c.dtype == MONONN_BF16, rows_by_vectors(p), dev->sm_count,
                              static_cast<cudaStream_t>(cuda_stream)));
}

int mononn_paged_attention_workspace(const mononn_paged_cache* cache, const mononn_paged_attention_args* args,
                                     size_t* bytes) {
  if (!bytes || !cache || !args) return invalid("null argument");
  *bytes = 0;
  if (args->tokens == 0 || cache->sequences == 0) return MONONN_OK;
  if (int rc = check_attention(cache, args)) return rc;
  OnDeviceOf guard;
  const Device* dev = nullptr;
  if (int rc = guard.enter(cache->k_pages, &dev)) return rc;
  AttentionPlan plan;
  if (int rc = plan_attention(*cache, *args, dev->sm_count, &plan)) return rc;
  *bytes = plan.workspace;
  return MONONN_OK;
}

int mononn_paged_attention(const mononn_paged_cache* cache, const mononn_paged_attention_args* args,
                           void* cuda_stream) {
  const uint32_t skewed = std::exchange(t_skewed, kBarrierNone);
  if (!cache || !args) return invalid("null argument");
  if (args->tokens == 0 || cache->sequences == 0) return MONONN_OK;
  if (int rc = check_attention(cache, args)) return rc;
  const mononn_paged_cache& c = *cache;
  const mononn_paged_attention_args& a = *args;
  OnDeviceOf guard;
  const Device* dev = nullptr;
  if (int rc = guard.enter(c.k_pages, &dev)) return rc;
  AttentionPlan plan;
  if (int rc = plan_attention(c, a, dev->sm_count, &plan)) return rc;
  if (plan.workspace && (!a.workspace || a.workspace_bytes < plan.workspace || !aligned(a.workspace, 16))) {
    char detail[64];
    std::snprintf(detail, sizeof(detail), "%zu bytes, 16-byte aligned", plan.workspace);
    return fail(MONONN_ERR_INVALID_ARGUMENT, "attention: needs a workspace of ", detail);
  }
  AttentionParams p{};
  if (int rc = encode_pages(&p.k_map, c, c.k_pages, plan.box, "k_pages")) return rc;
  if (int rc = encode_pages(&p.v_map, c, c.v_pages, plan.box, "v_pages")) return rc;
  if (plan.many)
    if (int rc = encode_queries(&p.q_map, c, a, plan)) return rc;
  p.q = a.q;
  p.out = a.out;
  p.lse = a.lse;
  p.q_token = a.q_token_stride;
  p.q_head = a.q_head_stride;
  p.out_token = a.out_token_stride;
  p.out_head = a.out_head_stride;
  p.table_stride = c.table_stride;
  p.table = c.page_table;
  p.lengths = c.lengths;
  p.indptr = a.indptr;
  if (plan.joins) {
    p.headers = static_cast<AttentionHeader*>(a.workspace);
    p.partial = reinterpret_cast<float*>(static_cast<char*>(a.workspace) +
                                         (plan.ctas * sizeof(AttentionHeader) + 255) / 256 * 256);
  }
  p.status = dev->status;
  p.sequences = c.sequences;
  p.tokens = a.tokens;
  p.kv_heads = c.kv_heads;
  p.group = a.q_heads / c.kv_heads;
  p.head_dim = c.head_dim;
  p.page_size = c.page_size;
  p.capacity = c.max_pages * c.page_size;
  while ((1u << p.box_shift) < plan.box) ++p.box_shift;  // a power of two, as the keys of a unit are
  p.item_rows = plan.item_rows;
  p.item_cost = plan.item_cost;
  p.causal = a.causal != 0;
  p.window = a.window;
  p.by_group = make_divisor(p.group);
  p.by_item_rows = make_divisor(p.item_rows);
  p.by_page_size = make_divisor(c.page_size);
  p.whole_items = !plan.joins;
  p.skewed = skewed;
  p.least_shift = plan.joins && plan.least_units == 2 ? 1 : 0;
  p.scale = a.scale > 0.f ? a.scale : 1.0f / std::sqrt(static_cast<float>(c.head_dim));
  p.scale_log2 = p.scale * 1.4426950408889634f;
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  const bool bf16 = c.dtype == MONONN_BF16;
  if (int rc = launched(plan.many ? launch_many_rows(p, plan, bf16, stream) : launch_few_rows(p, plan, bf16, stream))) return rc;
  return plan.joins ? launched(launch_join(p, plan, bf16, stream)) : MONONN_OK;
}

int mononn_debug_paged_skew(unsigned barrier) {
  if (barrier >= kBarriers) return invalid("no such barrier");
  t_skewed = barrier;
  return MONONN_OK;
}

int mononn_paged_attention_status(void* cuda_stream) {
  int count = 0;
  if (cudaGetDeviceCount(&count) != cudaSuccess || count == 0) {
    cudaGetLastError();
    return fail(MONONN_ERR_NO_DEVICE, "no CUDA device");
  }
  int current = 0, of_stream = 0;
  PG_TRY(cudaGetDevice(&current));
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  of_stream = current;
  if (cuda_stream && cuda_stream != cudaStreamLegacy && cuda_stream != cudaStreamPerThread)
    PG_TRY(cudaStreamGetDevice(stream, &of_stream));
  struct Back {
    int to;
    ~Back() {
      if (to >= 0) cudaSetDevice(to);
    }
  } back{-1};
  if (of_stream != current) {
    PG_TRY(cudaSetDevice(of_stream));
    back.to = current;
  }
  if (of_stream < 0 || of_stream >= kMaxDevices) return invalid("device ordinal out of range");
  const Device* dev = nullptr;
  if (int rc = set_up(of_stream, &dev)) return rc;
  uint32_t status = 0;
  PG_TRY(cudaMemcpyAsync(&status, dev->status, sizeof(status), cudaMemcpyDeviceToHost, stream));
  PG_TRY(cudaStreamSynchronize(stream));
  if (status == 0) return MONONN_OK;
  PG_TRY(cudaMemsetAsync(dev->status, 0, sizeof(uint32_t), stream));
  PG_TRY(cudaStreamSynchronize(stream));
  return fail(MONONN_ERR_BARRIER_TIMEOUT, "a bounded wait expired in a paged attention kernel; its output is incomplete");
}

}  // extern "C"
