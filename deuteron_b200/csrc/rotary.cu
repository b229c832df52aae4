// Rotary positions, and the same rotation fused with the write of keys and values into the pages of a cache.
//
// Pair i of a head (elements (i, i + r/2) in the half layout, (2i, 2i + 1) interleaved) is turned by the angle p * w_i:
//   (a, b) -> amplitude * (a cos - b sin, b cos + a sin),
// the other elements are copied. The transpose of that map, which the backward pass applies to the gradient, is the same
// with the sine's sign turned.
//
// The angle is p * w_i / 2 pi turns in 64 bits, reduced to a fraction of a turn there (at position 10^6 a 32-bit angle would
// already be off by 0.03 radians) and only then rounded to 32 bits: sincospif of that fraction is off by about 1e-7. One
// sine and cosine per token and pair serves every head of the token, so the 64-bit work is a few instructions per 40 or
// more vectors moved; the kernels are bound by memory (each value is read and written once).
#include "paged.cuh"

namespace dtn {

// One of the three streams of heads: queries (rotated to an output), keys (rotated into pages), values (copied into pages).
struct HeadStream {
  const void* src;
  int64_t token_stride, head_stride;   // elements
  int heads;
};

struct RotaryParams {
  HeadStream q, k, v;
  void* q_out;
  int64_t q_out_token_stride, q_out_head_stride;
  void *k_pages, *v_pages;
  int64_t page_stride, page_head_stride;   // elements, of both pools; a page's rows of one head are dense
  const int* tables;
  int64_t table_stride;
  const int* rows;
  int64_t sequences, pages;
  int64_t capacity;                        // tokens that a row of the tables covers
  int page_size;
  const void* positions;
  int positions_64;
  const double* frequencies;
  int pairs, dim;
  float amplitude, sign;
  int64_t tokens;
  int* status;
};

__device__ __forceinline__ int64_t position_of(const RotaryParams& p, int64_t token) {
  return p.positions_64 ? static_cast<const int64_t*>(p.positions)[token] : (int64_t) static_cast<const int*>(p.positions)[token];
}

// amplitude * (cos, sin) of position * frequency.
__device__ __forceinline__ float2 turn(const RotaryParams& p, int64_t position, int pair) {
  const double turns = (double)position * p.frequencies[pair] * 0.15915494309189533577;   // 1 / (2 pi)
  const float half_turns = (float)(2.0 * (turns - rint(turns)));
  float s, c;
  sincospif(half_turns, &s, &c);
  return make_float2(c * p.amplitude, s * (p.amplitude * p.sign));
}

// Offset in elements of a token's row of head 0 in the pools, or -1 when the token is not stored.
__device__ __forceinline__ int64_t page_offset(const RotaryParams& p, int64_t token) {
  const int row = p.rows[token];
  if (row < 0) return -1;
  const int64_t position = position_of(p, token);
  if (row >= p.sequences || position < 0 || position >= p.capacity) {
    paged_report(p.status, PAGED_STATUS_APPEND);
    return -1;
  }
  const int64_t index = position / p.page_size;
  const int page = p.tables[row * p.table_stride + index];
  if (page < 0 || page >= p.pages) {
    paged_report(p.status, PAGED_STATUS_APPEND);
    return -1;
  }
  return page * p.page_stride + (position - index * p.page_size) * p.dim;
}

// Where head `head` (counted over queries, keys, values) of a token is read and written; false: nothing to write.
template <typename T>
__device__ __forceinline__ bool head_places(const RotaryParams& p, int64_t token, int head, int64_t offset, const T*& src, T*& dst, bool& rotated) {
  rotated = true;
  if (head < p.q.heads) {
    src = static_cast<const T*>(p.q.src) + token * p.q.token_stride + head * p.q.head_stride;
    dst = static_cast<T*>(p.q_out) + token * p.q_out_token_stride + head * p.q_out_head_stride;
    return true;
  }
  head -= p.q.heads;
  const bool value = head >= p.k.heads;
  if (value) head -= p.k.heads;
  rotated = !value;
  const HeadStream& from = value ? p.v : p.k;
  src = static_cast<const T*>(from.src) + token * from.token_stride + head * from.head_stride;
  dst = static_cast<T*>(value ? p.v_pages : p.k_pages) + offset + head * p.page_head_stride;
  return offset >= 0;
}

// Any layout, any pair count, any alignment: a warp stages one head in shared memory (so that an output that is the input
// itself is safe), then writes element by element with its partner read from there.
constexpr int R_MAX_DIM = 1024;
constexpr int R_WARPS = 4;

template <typename T, bool INTERLEAVED>
__global__ void __launch_bounds__(R_WARPS * 32) rotary_staged_kernel(const RotaryParams p) {
  __shared__ float2 turns[R_MAX_DIM / 2];
  __shared__ T staged[R_WARPS][R_MAX_DIM];
  const int64_t token = blockIdx.x;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  for (int i = threadIdx.x; i < p.pairs; i += blockDim.x) turns[i] = turn(p, position_of(p, token), i);
  __shared__ int64_t offset;
  if (threadIdx.x == 0) offset = p.k.heads + p.v.heads > 0 ? page_offset(p, token) : -1;
  __syncthreads();
  const int heads = p.q.heads + p.k.heads + p.v.heads;
  for (int head = warp + R_WARPS * blockIdx.y; head < heads; head += R_WARPS * gridDim.y) {
    const T* src;
    T* dst;
    bool rotated;
    if (!head_places(p, token, head, offset, src, dst, rotated)) continue;
    for (int d = lane; d < p.dim; d += 32) staged[warp][d] = src[d];
    __syncwarp();
    for (int d = lane; d < p.dim; d += 32) {
      T y = staged[warp][d];
      if (rotated && d < 2 * p.pairs) {
        const int pair = INTERLEAVED ? d / 2 : (d < p.pairs ? d : d - p.pairs);
        const bool first = INTERLEAVED ? d % 2 == 0 : d < p.pairs;
        const int partner = INTERLEAVED ? d ^ 1 : (first ? d + p.pairs : d - p.pairs);
        const float x = to_float(y), z = to_float(staged[warp][partner]);
        const float2 cs = turns[pair];
        y = from_float<T>(first ? fmaf(x, cs.x, -z * cs.y) : fmaf(x, cs.x, z * cs.y));
      }
      dst[d] = y;
    }
    __syncwarp();
  }
}

template <typename T>
static int rotary_launch_t(const RotaryParams& p, int interleaved, cudaStream_t s) {
  const int heads = p.q.heads + p.k.heads + p.v.heads;
  const int by = (heads + R_WARPS - 1) / R_WARPS;
  // few tokens: a block per four heads; many: a block walks the heads of its token
  const int64_t wanted = (2 * (int64_t)sm_count() + p.tokens - 1) / p.tokens;
  dim3 grid((unsigned)p.tokens, (unsigned)(wanted < by ? (wanted < 1 ? 1 : wanted) : by));
  if (interleaved)
    rotary_staged_kernel<T, true><<<grid, R_WARPS * 32, 0, s>>>(p);
  else
    rotary_staged_kernel<T, false><<<grid, R_WARPS * 32, 0, s>>>(p);
  DTN_LAUNCH_CHECK("rotary_staged_kernel");
  return DTN_OK;
}

static int rotary_launch(const RotaryParams& p, int interleaved, int storage, cudaStream_t s) {
  if (p.tokens == 0 || p.dim == 0 || p.q.heads + p.k.heads + p.v.heads == 0) return DTN_OK;
  if (storage == DTN_STORAGE_F32) return rotary_launch_t<float>(p, interleaved, s);
  if (storage == DTN_STORAGE_F16) return rotary_launch_t<__half>(p, interleaved, s);
  return rotary_launch_t<__nv_bfloat16>(p, interleaved, s);
}

}  // namespace dtn

extern "C" {

int dtn_rotary(const void* x, void* out, const void* positions, int positions_64, const double* frequencies, int64_t tokens, int64_t heads,
               int64_t dim, int64_t pairs, int64_t x_token_stride, int64_t x_head_stride, int64_t out_token_stride, int64_t out_head_stride,
               int interleaved, int transpose, float amplitude, int storage, void* stream) {
  using namespace dtn;
  DTN_REQUIRE(tokens >= 0 && heads >= 0 && dim >= 0 && pairs >= 0, DTN_ERR_INVALID, "rotary: negative extent");
  DTN_REQUIRE(paged_storage_known(storage), DTN_ERR_INVALID, "rotary: unknown storage %d", storage);
  DTN_REQUIRE(2 * pairs <= dim, DTN_ERR_INVALID, "rotary: %lld pairs do not fit a head of %lld", (long long)pairs, (long long)dim);
  DTN_REQUIRE(dim <= R_MAX_DIM && heads < (1 << 20) && tokens < (1LL << 31), DTN_ERR_UNSUPPORTED,
              "rotary: heads of at most %d elements, fewer than 2^31 tokens", R_MAX_DIM);
  if (tokens == 0 || heads == 0 || dim == 0) return DTN_OK;
  DTN_REQUIRE(x && out && positions && (frequencies || pairs == 0), DTN_ERR_INVALID, "rotary: null pointer");
  RotaryParams p = {};
  p.q = {x, x_token_stride, x_head_stride, (int)heads};
  p.q_out = out;
  p.q_out_token_stride = out_token_stride;
  p.q_out_head_stride = out_head_stride;
  p.positions = positions;
  p.positions_64 = positions_64;
  p.frequencies = frequencies;
  p.pairs = (int)pairs;
  p.dim = (int)dim;
  p.amplitude = amplitude;
  p.sign = transpose ? -1.f : 1.f;
  p.tokens = tokens;
  return rotary_launch(p, interleaved, storage, as_stream(stream));
}

int dtn_paged_append(const void* k, const void* v, void* k_pages, void* v_pages, const int* tables, const int* rows, const void* positions,
                     int positions_64, int64_t tokens, int64_t kv_heads, int64_t dim, int64_t k_token_stride, int64_t k_head_stride,
                     int64_t v_token_stride, int64_t v_head_stride, int64_t pages, int64_t page_size, int64_t page_stride,
                     int64_t page_head_stride, int64_t sequences, int64_t pages_per_sequence, int64_t table_stride, const double* frequencies,
                     int64_t pairs, int interleaved, float amplitude, const void* q, void* q_out, int64_t q_heads, int64_t q_token_stride,
                     int64_t q_head_stride, int64_t q_out_token_stride, int64_t q_out_head_stride, int storage, void* stream) {
  using namespace dtn;
  DTN_REQUIRE(tokens >= 0 && kv_heads >= 0 && dim >= 0 && pairs >= 0 && q_heads >= 0 && pages >= 0 && sequences >= 0 && pages_per_sequence >= 0,
              DTN_ERR_INVALID, "paged append: negative extent");
  DTN_REQUIRE(page_size >= 1 && page_size < (1LL << 31), DTN_ERR_INVALID, "paged append: page size %lld", (long long)page_size);
  DTN_REQUIRE(paged_storage_known(storage), DTN_ERR_INVALID, "paged append: unknown storage %d", storage);
  DTN_REQUIRE(2 * pairs <= dim, DTN_ERR_INVALID, "paged append: %lld pairs do not fit a head of %lld", (long long)pairs, (long long)dim);
  DTN_REQUIRE(dim <= R_MAX_DIM && kv_heads < (1 << 20) && q_heads < (1 << 20) && tokens < (1LL << 31) && pages < (1LL << 31), DTN_ERR_UNSUPPORTED,
              "paged append: heads of at most %d elements, fewer than 2^31 tokens and pages", R_MAX_DIM);
  if (tokens == 0 || dim == 0 || kv_heads + q_heads == 0) return DTN_OK;
  DTN_REQUIRE(k && v && rows && positions && (frequencies || pairs == 0), DTN_ERR_INVALID, "paged append: null pointer");
  DTN_REQUIRE((k_pages && v_pages) || pages == 0, DTN_ERR_INVALID, "paged append: null pool");
  DTN_REQUIRE(tables || sequences == 0 || pages_per_sequence == 0, DTN_ERR_INVALID, "paged append: null tables");
  DTN_REQUIRE(q_heads == 0 || (q && q_out), DTN_ERR_INVALID, "paged append: null queries");
  RotaryParams p = {};
  p.q = {q, q_token_stride, q_head_stride, (int)q_heads};
  p.k = {k, k_token_stride, k_head_stride, (int)kv_heads};
  p.v = {v, v_token_stride, v_head_stride, (int)kv_heads};
  p.q_out = q_out;
  p.q_out_token_stride = q_out_token_stride;
  p.q_out_head_stride = q_out_head_stride;
  p.k_pages = k_pages;
  p.v_pages = v_pages;
  p.page_stride = page_stride;
  p.page_head_stride = page_head_stride;
  p.tables = tables;
  p.table_stride = table_stride;
  p.rows = rows;
  p.sequences = sequences;
  p.pages = pages;
  p.capacity = pages_per_sequence * page_size;
  p.page_size = (int)page_size;
  p.positions = positions;
  p.positions_64 = positions_64;
  p.frequencies = frequencies;
  p.pairs = (int)pairs;
  p.dim = (int)dim;
  p.amplitude = amplitude;
  p.sign = 1.f;
  p.tokens = tokens;
  p.status = device_status_word_unless_capturing(as_stream(stream));
  return rotary_launch(p, interleaved, storage, as_stream(stream));
}

}  // extern "C"
