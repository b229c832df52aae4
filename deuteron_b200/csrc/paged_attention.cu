// Attention of one new token per sequence over a paged key-value cache.
#include "paged.cuh"

namespace dtn {

struct PagedAttentionParams {
  const void *q, *k_pages, *v_pages;
  void* out;
  const int *tables, *lengths, *rows;   // rows may be null: sequence i uses row i
  int64_t count, sequences, pages, table_stride, capacity;
  int64_t q_token_stride, q_head_stride, out_token_stride, out_head_stride;
  int64_t page_stride, page_head_stride;
  int q_heads, kv_heads, group, dim, page_size;
  int64_t window;
  float scale_log2e;
  int out_f32;
  int* status;
};

// One warp per (sequence, query head): the running maximum and sum of a softmax over the tokens, in order.
template <typename T, int PER_LANE>
__global__ void __launch_bounds__(128) paged_attention_simple_kernel(const PagedAttentionParams p) {
  const int64_t item = (int64_t)blockIdx.x * 4 + threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  if (item >= p.count * p.q_heads) return;
  const int64_t sequence = item / p.q_heads;
  const int head = (int)(item % p.q_heads), kv_head = head / p.group;
  int64_t row = p.rows ? p.rows[sequence] : sequence;
  int64_t length = row >= 0 && row < p.sequences ? p.lengths[row] : 0;
  if (row >= p.sequences || length > p.capacity) {
    paged_report(p.status, PAGED_STATUS_ATTENTION);
    length = length > p.capacity ? p.capacity : length;
  }
  int64_t first = p.window > 0 && length > p.window ? length - p.window : 0;
  float q[PER_LANE], acc[PER_LANE], m = -INFINITY, l = 0.f;
  const T* query = static_cast<const T*>(p.q) + sequence * p.q_token_stride + head * p.q_head_stride;
  for (int i = 0; i < PER_LANE; ++i) {
    const int d = lane + 32 * i;
    q[i] = d < p.dim ? to_float(query[d]) : 0.f;
    acc[i] = 0.f;
  }
  bool bad = false;
  for (int64_t t = first; t < length; ++t) {
    const int64_t index = t / p.page_size;
    int page = p.tables[row * p.table_stride + index];
    if (page < 0 || page >= p.pages) {
      bad = true;
      continue;
    }
    const int64_t at = page * p.page_stride + kv_head * p.page_head_stride + (t - index * p.page_size) * p.dim;
    const T *k = static_cast<const T*>(p.k_pages) + at, *v = static_cast<const T*>(p.v_pages) + at;
    float s = 0.f;
    for (int i = 0; i < PER_LANE; ++i) s = fmaf(q[i], lane + 32 * i < p.dim ? to_float(k[lane + 32 * i]) : 0.f, s);
    s = warp_sum(s) * p.scale_log2e;
    const float top = fmaxf(m, s), base = top == -INFINITY ? 0.f : top;
    const float alpha = ex2_approx(m - base), pr = ex2_approx(s - base);
    l = fmaf(l, alpha, pr);
    for (int i = 0; i < PER_LANE; ++i) acc[i] = fmaf(acc[i], alpha, pr * (lane + 32 * i < p.dim ? to_float(v[lane + 32 * i]) : 0.f));
    m = top;
  }
  if (bad && lane == 0) paged_report(p.status, PAGED_STATUS_ATTENTION);
  if (bad) l = __int_as_float(0x7fffffff);   // NaN: a page that does not exist is no zero
  for (int i = 0; i < PER_LANE; ++i) {
    const int d = lane + 32 * i;
    if (d >= p.dim) continue;
    const float y = first < length ? acc[i] / l : 0.f;
    const int64_t to = sequence * p.out_token_stride + head * p.out_head_stride + d;
    if (p.out_f32)
      static_cast<float*>(p.out)[to] = y;
    else
      static_cast<T*>(p.out)[to] = from_float<T>(y);
  }
}

template <typename T>
static int paged_attention_launch_t(const PagedAttentionParams& p, cudaStream_t s) {
  const int64_t items = p.count * p.q_heads;
  paged_attention_simple_kernel<T, 8><<<(unsigned)((items + 3) / 4), 128, 0, s>>>(p);
  DTN_LAUNCH_CHECK("paged_attention_simple_kernel");
  return DTN_OK;
}

}  // namespace dtn

extern "C" int dtn_paged_attention(const void* q, const void* k_pages, const void* v_pages, const int* tables, const int* lengths, const int* rows,
                                   void* out, int64_t count, int64_t q_heads, int64_t kv_heads, int64_t dim, int64_t q_token_stride,
                                   int64_t q_head_stride, int64_t out_token_stride, int64_t out_head_stride, int64_t pages, int64_t page_size,
                                   int64_t page_stride, int64_t page_head_stride, int64_t sequences, int64_t pages_per_sequence,
                                   int64_t table_stride, float scale, int64_t window, int storage, int out_f32, void* stream) {
  using namespace dtn;
  DTN_REQUIRE(count >= 0 && q_heads >= 0 && kv_heads >= 0 && dim >= 0 && pages >= 0 && sequences >= 0 && pages_per_sequence >= 0 && window >= 0,
              DTN_ERR_INVALID, "paged attention: negative extent");
  DTN_REQUIRE(page_size >= 1 && page_size < (1LL << 31), DTN_ERR_INVALID, "paged attention: page size %lld", (long long)page_size);
  DTN_REQUIRE(paged_storage_known(storage), DTN_ERR_INVALID, "paged attention: unknown storage %d", storage);
  if (count == 0 || q_heads == 0 || dim == 0) return DTN_OK;
  DTN_REQUIRE(kv_heads > 0 && q_heads % kv_heads == 0, DTN_ERR_INVALID, "paged attention: query heads must be a multiple of kv heads");
  DTN_REQUIRE(dim <= 256, DTN_ERR_UNSUPPORTED, "paged attention: heads of at most 256 elements");
  DTN_REQUIRE(q && out && (rows || count <= sequences), DTN_ERR_INVALID, "paged attention: null pointer");
  DTN_REQUIRE((k_pages && v_pages) || pages == 0, DTN_ERR_INVALID, "paged attention: null pool");
  DTN_REQUIRE(sequences == 0 || (lengths && (tables || pages_per_sequence == 0)), DTN_ERR_INVALID, "paged attention: null tables");
  DTN_REQUIRE(pages < (1LL << 31) && count * q_heads < (1LL << 31), DTN_ERR_UNSUPPORTED, "paged attention: too many rows for one launch");
  cudaStream_t s = as_stream(stream);
  PagedAttentionParams p = {};
  p.q = q;
  p.k_pages = k_pages;
  p.v_pages = v_pages;
  p.out = out;
  p.tables = tables;
  p.lengths = lengths;
  p.rows = rows;
  p.count = count;
  p.sequences = sequences;
  p.pages = pages;
  p.table_stride = table_stride;
  p.capacity = pages_per_sequence * page_size;
  p.q_token_stride = q_token_stride;
  p.q_head_stride = q_head_stride;
  p.out_token_stride = out_token_stride;
  p.out_head_stride = out_head_stride;
  p.page_stride = page_stride;
  p.page_head_stride = page_head_stride;
  p.q_heads = (int)q_heads;
  p.kv_heads = (int)kv_heads;
  p.group = (int)(q_heads / kv_heads);
  p.dim = (int)dim;
  p.page_size = (int)page_size;
  p.window = window;
  p.scale_log2e = scale * 1.4426950408889634f;
  p.out_f32 = out_f32;
  p.status = device_status_word_unless_capturing(s);
  if (storage == DTN_STORAGE_F32) return paged_attention_launch_t<float>(p, s);
  if (storage == DTN_STORAGE_F16) return paged_attention_launch_t<__half>(p, s);
  return paged_attention_launch_t<__nv_bfloat16>(p, s);
}
