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

// How the work is laid out: a block has `tokens` tokens and `heads` heads (counted over queries, keys, values), a head `units`
// units. The multipliers divide small numbers: n / d = umulhi(n, ceil(2^32 / d)) while n * d < 2^32.
struct RotaryLayout {
  int tokens, heads, units;
  uint32_t units_mul, heads_mul;
};

__device__ __forceinline__ int small_divide(int n, int d, uint32_t mul) { return d == 1 ? n : (int)__umulhi((uint32_t)n, mul); }

// Where head `head` of a token is read.
template <typename T>
__device__ __forceinline__ const T* head_source(const RotaryParams& p, int64_t token, int head) {
  if (head < p.q.heads) return static_cast<const T*>(p.q.src) + token * p.q.token_stride + head * p.q.head_stride;
  head -= p.q.heads;
  if (head < p.k.heads) return static_cast<const T*>(p.k.src) + token * p.k.token_stride + head * p.k.head_stride;
  head -= p.k.heads;
  return static_cast<const T*>(p.v.src) + token * p.v.token_stride + head * p.v.head_stride;
}
// Where it is written (offset: the token's place in the pools, or -1); null: nowhere. Values are not rotated.
template <typename T>
__device__ __forceinline__ T* head_target(const RotaryParams& p, int64_t token, int head, int64_t offset, bool& rotated) {
  rotated = true;
  if (head < p.q.heads) return static_cast<T*>(p.q_out) + token * p.q_out_token_stride + head * p.q_out_head_stride;
  if (offset < 0) return nullptr;
  head -= p.q.heads;
  if (head < p.k.heads) return static_cast<T*>(p.k_pages) + offset + head * p.page_head_stride;
  rotated = false;
  return static_cast<T*>(p.v_pages) + offset + (head - p.k.heads) * p.page_head_stride;
}

constexpr int R_THREADS = 256;
constexpr int R_TURNS = 512;      // cosines and sines a block holds: tokens per block x pairs
constexpr int R_MAX_TOKENS = 64;  // per block
constexpr int R_AHEAD = 2;        // units a thread has in flight

// Whole 16-byte vectors on both sides of every pair. A unit is the two vectors that hold the halves of VECTOR pairs (half
// layout) or one vector of whole pairs (interleaved), or one vector that is copied; the pairs of a unit are in one thread,
// so out may be x itself. A block's first loads are issued before its angles are formed.
//
// 16384 tokens x 40 heads x 128 bf16 (336 MB, 51.3 us at the copy rate): see the table of measured times.
template <typename T, bool INTERLEAVED>
__global__ void __launch_bounds__(R_THREADS) rotary_vector_kernel(const RotaryParams p, const RotaryLayout l) {
  constexpr int VECTOR = 16 / (int)sizeof(T);
  __shared__ __align__(16) float cosines[R_TURNS], sines[R_TURNS];
  __shared__ int64_t places[R_MAX_TOKENS];
  const int64_t token0 = (int64_t)blockIdx.x * l.tokens;
  const int tokens = (int)(p.tokens - token0 < l.tokens ? p.tokens - token0 : l.tokens);
  const int all_heads = p.q.heads + p.k.heads + p.v.heads, head0 = blockIdx.y * l.heads;
  const int heads = all_heads - head0 < l.heads ? all_heads - head0 : l.heads;
  const int total = tokens * l.heads * l.units, turned = INTERLEAVED ? 0 : p.pairs / VECTOR;

  struct Unit {
    int token, head, unit;
    uint4 a, b;
  } units[R_AHEAD];
  auto find = [&](Unit& u, int flat) {
    const int row = small_divide(flat, l.units, l.units_mul);
    u.unit = flat - row * l.units;
    u.token = small_divide(row, l.heads, l.heads_mul);
    u.head = row - u.token * l.heads;
    if (flat >= total || u.head >= heads) u.token = -1;
  };
  auto load = [&](Unit& u) {
    if (u.token < 0) return;
    const T* src = head_source<T>(p, token0 + u.token, head0 + u.head);
    if (!INTERLEAVED && u.unit < turned) {
      u.a = *reinterpret_cast<const uint4*>(src + u.unit * VECTOR);
      u.b = *reinterpret_cast<const uint4*>(src + p.pairs + u.unit * VECTOR);
    } else {
      u.a = *reinterpret_cast<const uint4*>(src + (INTERLEAVED ? u.unit : u.unit + turned) * VECTOR);
    }
  };
  auto store = [&](Unit& u) {
    if (u.token < 0) return;
    bool rotated;
    T* dst = head_target<T>(p, token0 + u.token, head0 + u.head, places[u.token], rotated);
    if (dst == nullptr) return;
    T* a = reinterpret_cast<T*>(&u.a);
    if (INTERLEAVED) {
      if (rotated && u.unit * VECTOR < 2 * p.pairs) {
        const float* c = cosines + u.token * p.pairs + u.unit * (VECTOR / 2);
        const float* s = sines + u.token * p.pairs + u.unit * (VECTOR / 2);
#pragma unroll
        for (int i = 0; i < VECTOR / 2; ++i) {
          const float x = to_float(a[2 * i]), y = to_float(a[2 * i + 1]);
          a[2 * i] = from_float<T>(fmaf(x, c[i], -y * s[i]));
          a[2 * i + 1] = from_float<T>(fmaf(y, c[i], x * s[i]));
        }
      }
      *reinterpret_cast<uint4*>(dst + u.unit * VECTOR) = u.a;
    } else if (u.unit < turned) {
      T* b = reinterpret_cast<T*>(&u.b);
      if (rotated) {
        const float4* c4 = reinterpret_cast<const float4*>(cosines + u.token * p.pairs + u.unit * VECTOR);
        const float4* s4 = reinterpret_cast<const float4*>(sines + u.token * p.pairs + u.unit * VECTOR);
#pragma unroll
        for (int i = 0; i < VECTOR / 4; ++i) {
          const float4 cv = c4[i], sv = s4[i];
          const float c[4] = {cv.x, cv.y, cv.z, cv.w}, s[4] = {sv.x, sv.y, sv.z, sv.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float x = to_float(a[4 * i + j]), y = to_float(b[4 * i + j]);
            a[4 * i + j] = from_float<T>(fmaf(x, c[j], -y * s[j]));
            b[4 * i + j] = from_float<T>(fmaf(y, c[j], x * s[j]));
          }
        }
      }
      *reinterpret_cast<uint4*>(dst + u.unit * VECTOR) = u.a;
      *reinterpret_cast<uint4*>(dst + p.pairs + u.unit * VECTOR) = u.b;
    } else {
      *reinterpret_cast<uint4*>(dst + (u.unit + turned) * VECTOR) = u.a;
    }
  };

#pragma unroll
  for (int i = 0; i < R_AHEAD; ++i) {
    find(units[i], threadIdx.x + i * R_THREADS);
    load(units[i]);
  }
  for (int i = threadIdx.x; i < tokens * p.pairs; i += R_THREADS) {
    const int t = i / p.pairs;
    const float2 cs = turn(p, position_of(p, token0 + t), i - t * p.pairs);
    cosines[i] = cs.x;
    sines[i] = cs.y;
  }
  if ((int)threadIdx.x < tokens) places[threadIdx.x] = p.k.heads > 0 ? page_offset(p, token0 + threadIdx.x) : -1;
  __syncthreads();
  for (int base = 0; base < total; base += R_AHEAD * R_THREADS) {
    if (base > 0) {
#pragma unroll
      for (int i = 0; i < R_AHEAD; ++i) {
        find(units[i], base + threadIdx.x + i * R_THREADS);
        load(units[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < R_AHEAD; ++i) store(units[i]);
  }
}

// Any number of pairs, any alignment: rows of heads are staged in shared memory, by 16-byte vectors where the rows allow it
// (WIDE), and each thread writes what it staged with the partners read from there. A pass holds whole rows and reads all of
// them before it writes any.
constexpr int R_MAX_DIM = 1024;

template <typename T, bool INTERLEAVED, bool WIDE>
__global__ void __launch_bounds__(R_THREADS) rotary_staged_kernel(const RotaryParams p, const RotaryLayout l) {
  constexpr int VECTOR = WIDE ? 16 / (int)sizeof(T) : 1, EACH = WIDE ? R_AHEAD : 8, CAPACITY = EACH * R_THREADS;
  __shared__ float2 turns[R_TURNS];
  __shared__ __align__(16) T staged[CAPACITY * VECTOR];
  __shared__ int64_t places[R_MAX_TOKENS];
  const int64_t token0 = (int64_t)blockIdx.x * l.tokens;
  const int tokens = (int)(p.tokens - token0 < l.tokens ? p.tokens - token0 : l.tokens);
  const int all_heads = p.q.heads + p.k.heads + p.v.heads, head0 = blockIdx.y * l.heads;
  const int heads = all_heads - head0 < l.heads ? all_heads - head0 : l.heads;
  const int rows = tokens * l.heads, rows_of_pass = CAPACITY / l.units;   // a unit is one vector here
  for (int i = threadIdx.x; i < tokens * p.pairs; i += R_THREADS) {
    const int t = i / p.pairs;
    turns[i] = turn(p, position_of(p, token0 + t), i - t * p.pairs);
  }
  if ((int)threadIdx.x < tokens) places[threadIdx.x] = p.k.heads > 0 ? page_offset(p, token0 + threadIdx.x) : -1;
  __syncthreads();
  for (int first = 0; first < rows; first += rows_of_pass) {
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int flat = threadIdx.x + i * R_THREADS, row = small_divide(flat, l.units, l.units_mul), unit = flat - row * l.units;
      const int token = small_divide(first + row, l.heads, l.heads_mul), head = first + row - token * l.heads;
      if (row >= rows_of_pass || first + row >= rows || head >= heads) continue;
      const T* src = head_source<T>(p, token0 + token, head0 + head) + unit * VECTOR;
      if (WIDE)
        *reinterpret_cast<uint4*>(staged + flat * VECTOR) = *reinterpret_cast<const uint4*>(src);
      else
        staged[flat] = *src;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int flat = threadIdx.x + i * R_THREADS, row = small_divide(flat, l.units, l.units_mul), unit = flat - row * l.units;
      const int token = small_divide(first + row, l.heads, l.heads_mul), head = first + row - token * l.heads;
      if (row >= rows_of_pass || first + row >= rows || head >= heads) continue;
      bool rotated;
      T* dst = head_target<T>(p, token0 + token, head0 + head, places[token], rotated);
      if (dst == nullptr) continue;
      const T* line = staged + row * l.units * VECTOR;
      const float2* line_turns = turns + token * p.pairs;
      __align__(16) T out[VECTOR];
#pragma unroll
      for (int e = 0; e < VECTOR; ++e) {
        const int d = unit * VECTOR + e;
        out[e] = line[d];
        if (rotated && d < 2 * p.pairs) {
          const bool is_first = INTERLEAVED ? d % 2 == 0 : d < p.pairs;
          const int pair = INTERLEAVED ? d / 2 : (is_first ? d : d - p.pairs), partner = INTERLEAVED ? d ^ 1 : (is_first ? d + p.pairs : pair);
          const float x = to_float(out[e]), y = to_float(line[partner]);
          const float2 cs = line_turns[pair];
          out[e] = from_float<T>(is_first ? fmaf(x, cs.x, -y * cs.y) : fmaf(x, cs.x, y * cs.y));
        }
      }
      if (WIDE)
        *reinterpret_cast<uint4*>(dst + unit * VECTOR) = *reinterpret_cast<const uint4*>(out);
      else
        dst[unit] = out[0];
    }
    __syncthreads();
  }
}

// Tokens and heads per block. Many tokens: as many per block as share the work of R_TURNS angles and still leave several
// blocks per SM. Few: one, its heads cut so that the card is not left to a handful of blocks.
static RotaryLayout rotary_layout(const RotaryParams& p, int units, int per_pass, dim3& grid) {
  RotaryLayout l = {};
  const int64_t heads = p.q.heads + p.k.heads + p.v.heads, target = 4 * (int64_t)sm_count();
  int64_t tokens = p.pairs > 0 ? R_TURNS / p.pairs : R_MAX_TOKENS;
  tokens = tokens < 1 ? 1 : (tokens > R_MAX_TOKENS ? R_MAX_TOKENS : tokens);
  if (tokens > p.tokens / target) tokens = p.tokens / target < 1 ? 1 : p.tokens / target;
  int64_t cut = heads;
  const int64_t fill = (per_pass + units - 1) / units, wanted = p.tokens < target ? target / p.tokens : 1;   // heads of one pass; blocks per token
  if (wanted > 1) cut = (heads + wanted - 1) / wanted;
  if (cut < fill) cut = fill;
  if (cut > heads) cut = heads;
  const int64_t most = 32768 / units;   // units <= 1024: a block's numbers of units and rows stay below 2^16, their products with a divisor below 2^32
  if (cut > most) cut = most;
  if (tokens * cut > most) tokens = most / cut;
  l.tokens = (int)tokens;
  l.heads = (int)cut;
  l.units = units;
  l.units_mul = (uint32_t)(((1ULL << 32) + units - 1) / units);
  l.heads_mul = (uint32_t)(((1ULL << 32) + cut - 1) / cut);
  grid = dim3((unsigned)((p.tokens + tokens - 1) / tokens), (unsigned)((heads + cut - 1) / cut));
  return l;
}

template <typename T>
static int rotary_launch_t(const RotaryParams& p, int interleaved, cudaStream_t s) {
  constexpr int VECTOR = 16 / (int)sizeof(T);
  auto wide = [](const HeadStream& h, const void* base) {
    return h.heads == 0 || (aligned_to(base, 16) && h.token_stride % VECTOR == 0 && h.head_stride % VECTOR == 0);
  };
  const HeadStream q_target = {p.q_out, p.q_out_token_stride, p.q_out_head_stride, p.q.heads};
  const HeadStream pages = {p.k_pages, p.page_stride, p.page_head_stride, p.k.heads};
  const bool vectors = p.dim % VECTOR == 0 && wide(p.q, p.q.src) && wide(p.k, p.k.src) && wide(p.v, p.v.src) && wide(q_target, p.q_out) &&
                       wide(pages, p.k_pages) && wide(pages, p.v_pages);
  const bool whole = vectors && (interleaved ? 2 * p.pairs : p.pairs) % VECTOR == 0;
  dim3 grid;
  if (whole) {
    const int units = interleaved ? p.dim / VECTOR : (p.dim - p.pairs) / VECTOR;
    const RotaryLayout l = rotary_layout(p, units, R_AHEAD * R_THREADS, grid);
    DTN_REQUIRE(grid.y < 65536, DTN_ERR_UNSUPPORTED, "rotary: too many heads for one launch");
    if (interleaved)
      rotary_vector_kernel<T, true><<<grid, R_THREADS, 0, s>>>(p, l);
    else
      rotary_vector_kernel<T, false><<<grid, R_THREADS, 0, s>>>(p, l);
  } else if (vectors) {
    const RotaryLayout l = rotary_layout(p, p.dim / VECTOR, R_AHEAD * R_THREADS, grid);
    DTN_REQUIRE(grid.y < 65536, DTN_ERR_UNSUPPORTED, "rotary: too many heads for one launch");
    if (interleaved)
      rotary_staged_kernel<T, true, true><<<grid, R_THREADS, 0, s>>>(p, l);
    else
      rotary_staged_kernel<T, false, true><<<grid, R_THREADS, 0, s>>>(p, l);
  } else {
    const RotaryLayout l = rotary_layout(p, p.dim, 8 * R_THREADS, grid);
    DTN_REQUIRE(grid.y < 65536, DTN_ERR_UNSUPPORTED, "rotary: too many heads for one launch");
    if (interleaved)
      rotary_staged_kernel<T, true, false><<<grid, R_THREADS, 0, s>>>(p, l);
    else
      rotary_staged_kernel<T, false, false><<<grid, R_THREADS, 0, s>>>(p, l);
  }
  DTN_LAUNCH_CHECK("rotary kernel");
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
