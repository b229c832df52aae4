// Rotary positions, and the same rotation fused with the write of keys and values into the pages of a cache.
//
// Pair i of a head (elements (i, i + r/2) in the half layout, (2i, 2i + 1) interleaved) is turned by the angle p * w_i:
//   (a, b) -> amplitude * (a cos - b sin, b cos + a sin),
// the other elements are copied. The transpose of that map, which the backward pass applies to the gradient, is the same
// with the sine's sign turned.
//
// The angle is p * w_i / 2 pi turns in 64 bits, reduced to a fraction of a turn there (at position 10^6 a 32-bit angle would
// already be off by 0.03 radians) and only then rounded to 32 bits: sincospif of that fraction is off by about 1e-7. That
// rounding and a 32-bit sine and cosine are a choice: f16 and bf16 results round to 2^-11 and 2^-8 anyway, and FP32 ones are off by
// 2.8e-8 in the mean where a 64-bit sine and cosine give 2.4e-8 (4095 x 20 x 96); 2^-21 of a pair's magnitudes bounds it. One
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
__device__ __forceinline__ float2 turn(const RotaryParams& p, double position, int pair) {
  const double turns = position * p.frequencies[pair] * 0.15915494309189533577;   // 1 / (2 pi)
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

constexpr int R_MAX_DIM = 1024;
constexpr int R_THREADS = 256;
constexpr int R_FILL = 8192;   // threads per SM wanted of a launch: 54 us at 16384 x 40 x 128, 59 with 4096, 62 with 16384

// V elements in one access.
template <int BYTES> struct Access;
template <> struct Access<16> { using type = uint4; };
template <> struct Access<8> { using type = uint2; };
template <> struct Access<4> { using type = uint32_t; };
template <> struct Access<2> { using type = uint16_t; };

// A thread keeps one unit of one token: it forms the angles of its pairs once, in registers, and walks over a range of heads
// of one stream with them, so the 64-bit work is done once per token and pair and slice of heads. A unit is the two accesses of
// V elements that hold the halves of V pairs (TWO), or one access of whole pairs (interleaved), or one access that is copied;
// neighbouring threads have neighbouring units, so the accesses of a warp are whole lines whatever V is. The pairs of a unit
// are in one thread and the loads of a head precede its stores, so out may be x itself. The loads of the first heads are
// issued before the angles are formed and before a key or value's page is looked up.
//
// Bound by memory. V is the widest that divides the head, its strides and addresses and, in the half layout, the number of
// pairs: 16 bytes in practice. 16384 tokens x 40 heads x 128 bf16 (336 MB): 54 us, 0.95 of the copy rate; 4095 x 20 x 96 FP32
// interleaved (63 MB): 12 us, 0.80; append of 16000 tokens, 32 + 8 + 8 heads (393 MB): 61.5 us, 0.98, and of 8000 in FP32 64 us,
// 0.94; one token: 2 us. (A
// form with the angles in shared memory and a unit per thread and head took 61, 15.7 and 112 us: its index arithmetic.)
template <typename T, bool TWO, int V>
__global__ void __launch_bounds__(R_THREADS) rotary_kernel(const RotaryParams p, const int interleaved, const int units, const int tokens_per_block,
                                                           const int heads_per_thread, const int q_slices, const int k_slices) {
  using Word = typename Access<V * (int)sizeof(T)>::type;
  constexpr int WORDS = TWO ? 2 : 1, PAIRS = TWO ? V : V / 2, AHEAD = 4;
  const int width = units < R_THREADS ? units : R_THREADS, local = threadIdx.x / width, unit = threadIdx.x - local * width + blockIdx.z * R_THREADS;
  const int64_t token = (int64_t)blockIdx.x * tokens_per_block + local;
  if (local >= tokens_per_block || token >= p.tokens || unit >= units) return;
  int slice = blockIdx.y;
  const bool query = slice < q_slices, key = !query && slice < q_slices + k_slices;
  slice -= query ? 0 : (key ? q_slices : q_slices + k_slices);
  const HeadStream& from = query ? p.q : (key ? p.k : p.v);
  const int head0 = slice * heads_per_thread, heads = from.heads - head0 < heads_per_thread ? from.heads - head0 : heads_per_thread;
  // the unit's first column, how far its pairs' other halves are and how many of its pairs are turned
  const int turned = TWO ? p.pairs / V : 0;
  const bool two = TWO && unit < turned;
  const int other = interleaved ? 1 : p.pairs;   // TWO and interleaved only with V = 1: elements that cannot be moved in pairs
  const int column = !TWO ? unit * V : (two ? (interleaved ? 2 * unit : unit * V) : (unit + turned) * V);
  const int left = TWO ? (two ? PAIRS : 0) : p.pairs - unit * PAIRS, turning = query || key ? left : 0;
  const T* src = static_cast<const T*>(from.src) + token * from.token_stride + head0 * from.head_stride + column;

  Word x[AHEAD][WORDS];
  auto load = [&](int h) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (h + i < heads) {
        x[i][0] = *reinterpret_cast<const Word*>(src + (h + i) * from.head_stride);
        if (TWO && two) x[i][WORDS - 1] = *reinterpret_cast<const Word*>(src + (h + i) * from.head_stride + other);
      }
  };
  load(0);
  float c[PAIRS], s[PAIRS];
  if (turning > 0) {
    const double position = (double)position_of(p, token);
#pragma unroll
    for (int i = 0; i < PAIRS; ++i)
      if (i < turning) {
        const float2 cs = turn(p, position, unit * PAIRS + i);
        c[i] = cs.x;
        s[i] = cs.y;
      }
  }
  T* dst;
  int64_t head_stride;
  if (query) {
    dst = static_cast<T*>(p.q_out) + token * p.q_out_token_stride + head0 * p.q_out_head_stride + column;
    head_stride = p.q_out_head_stride;
  } else {
    const int64_t offset = page_offset(p, token);
    if (offset < 0) return;
    dst = static_cast<T*>(key ? p.k_pages : p.v_pages) + offset + head0 * p.page_head_stride + column;
    head_stride = p.page_head_stride;
  }
  for (int h = 0; h < heads; h += AHEAD) {
    if (h > 0) load(h);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      if (h + i >= heads) break;
      T* a = reinterpret_cast<T*>(&x[i][0]);
      T* b = reinterpret_cast<T*>(&x[i][WORDS - 1]);
#pragma unroll
      for (int j = 0; j < PAIRS; ++j)
        if (j < turning) {
          T& first = TWO ? a[j] : a[2 * j];
          T& second = TWO ? b[j] : a[2 * j + 1];
          const float u = to_float(first), v = to_float(second);
          first = from_float<T>(fmaf(u, c[j], -v * s[j]));
          second = from_float<T>(fmaf(v, c[j], u * s[j]));
        }
      *reinterpret_cast<Word*>(dst + (h + i) * head_stride) = x[i][0];
      if (TWO && two) *reinterpret_cast<Word*>(dst + (h + i) * head_stride + other) = x[i][WORDS - 1];
    }
  }
}

// The heads are cut into slices of one stream until the card has `fill` threads per SM (a thread per head for a handful of
// tokens), each of at least the heads that a thread has in flight while the tokens alone give the card a block per SM.
static int64_t rotary_heads_per_thread(const RotaryParams& p, int units, int ahead, int64_t fill) {
  const int64_t heads = p.q.heads + p.k.heads + p.v.heads, threads = p.tokens * units, slices = fill * sm_count() / threads + 1;
  int64_t each = (heads + slices - 1) / slices;
  if (each > ahead || threads >= (int64_t)R_THREADS * sm_count()) each = (each + ahead - 1) / ahead * ahead;
  return each;
}

template <typename T, bool TWO, int V>
static int rotary_launch_v(const RotaryParams& p, int interleaved, cudaStream_t s) {
  const int units = (TWO ? p.dim - p.pairs : p.dim) / V, width = units < R_THREADS ? units : R_THREADS, tokens = R_THREADS / width;
  const int64_t each = rotary_heads_per_thread(p, units, 4, R_FILL);
  const int64_t q_slices = (p.q.heads + each - 1) / each, k_slices = (p.k.heads + each - 1) / each;
  DTN_REQUIRE(q_slices + 2 * k_slices < 65536, DTN_ERR_UNSUPPORTED, "rotary: too many heads for one launch");
  const dim3 grid((unsigned)((p.tokens + tokens - 1) / tokens), (unsigned)(q_slices + 2 * k_slices), (unsigned)((units + R_THREADS - 1) / R_THREADS));
  rotary_kernel<T, TWO, V><<<grid, tokens * width, 0, s>>>(p, interleaved, units, tokens, (int)each, (int)q_slices, (int)k_slices);
  DTN_LAUNCH_CHECK("rotary_kernel");
  return DTN_OK;
}

// Half layout, heads of whole 16-byte vectors, pairs that are not: a thread keeps one vector of one token and takes the other
// halves of its elements' pairs from shared memory, where every thread of the head puts its vector: two vectors, out of
// which OFF = pairs % V elements are shifted (a constant, so the shift costs no instruction or one per word). Between two
// barriers all loads of R_SHARED heads precede their stores, and a head's threads are in one block, so out may be x itself.
// 16384 x 40 x 128 bf16 with 37 pairs: 92 us against 161 with one element per access; with 38 pairs 92 against 111 with two;
// with 36 pairs 89 against 96 with four. What it pays over whole vectors is twice the angles, one per element.
constexpr int R_SHARED = 4, R_FILL_SHARED = 4096;

template <typename T, int OFF>
__global__ void __launch_bounds__(R_THREADS) rotary_shared_kernel(const RotaryParams p, const int units, const int tokens_per_block, const int heads_per_thread,
                                                                  const int q_slices, const int k_slices) {
  constexpr int V = 16 / (int)sizeof(T);
  __shared__ __align__(16) T staged[R_SHARED][R_THREADS * V];
  const int local = threadIdx.x / units, unit = threadIdx.x - local * units;
  const int64_t token = (int64_t)blockIdx.x * tokens_per_block + local;
  const bool there = token < p.tokens;
  int slice = blockIdx.y;
  const bool query = slice < q_slices, key = !query && slice < q_slices + k_slices;
  slice -= query ? 0 : (key ? q_slices : q_slices + k_slices);
  const HeadStream& from = query ? p.q : (key ? p.k : p.v);
  const int head0 = slice * heads_per_thread, heads = from.heads - head0 < heads_per_thread ? from.heads - head0 : heads_per_thread;
  const int column = unit * V;
  // elements of the vector that are first halves, and that are turned at all
  const int whole = p.pairs / V, firsts = p.pairs - column, turning = there && (query || key) ? 2 * p.pairs - column : 0;
  const T* src = static_cast<const T*>(from.src) + token * from.token_stride + head0 * from.head_stride + column;

  uint4 x[R_SHARED];
  auto load = [&](int h) {
#pragma unroll
    for (int i = 0; i < R_SHARED; ++i)
      if (there && h + i < heads) x[i] = *reinterpret_cast<const uint4*>(src + (h + i) * from.head_stride);
  };
  load(0);
  float c[V], s[V];
  if (turning > 0) {
    const double position = (double)position_of(p, token);
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e < turning) {
        const float2 cs = turn(p, position, e < firsts ? column + e : column + e - p.pairs);
        c[e] = cs.x;
        s[e] = e < firsts ? -cs.y : cs.y;
      }
  }
  T* dst = nullptr;
  int64_t head_stride = 0;
  if (there && query) {
    dst = static_cast<T*>(p.q_out) + token * p.q_out_token_stride + head0 * p.q_out_head_stride + column;
    head_stride = p.q_out_head_stride;
  } else if (there) {
    const int64_t offset = page_offset(p, token);
    if (offset >= 0) dst = static_cast<T*>(key ? p.k_pages : p.v_pages) + offset + head0 * p.page_head_stride + column;
    head_stride = p.page_head_stride;
  }
  for (int h = 0; h < heads; h += R_SHARED) {
    if (h > 0) load(h);
#pragma unroll
    for (int i = 0; i < R_SHARED; ++i)
      if (there && h + i < heads) *reinterpret_cast<uint4*>(&staged[i][threadIdx.x * V]) = x[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < R_SHARED; ++i) {
      if (h + i >= heads || dst == nullptr) break;
      T* a = reinterpret_cast<T*>(&x[i]);
      if (turning > 0) {
        const uint4* line = reinterpret_cast<const uint4*>(staged[i]) + local * units;
        uint4 up[2], down[2];   // the second halves of first ones, the first halves of second ones
        if (firsts > 0) {
          up[0] = line[unit + whole];
          up[1] = line[unit + whole + 1 < units ? unit + whole + 1 : units - 1];   // past the head: not used
        }
        if (firsts < V) {
          down[0] = line[unit - whole - 1 > 0 ? unit - whole - 1 : 0];             // before the head: not used
          down[1] = line[unit - whole];
        }
        const T* up_at = reinterpret_cast<const T*>(up) + OFF;
        const T* down_at = reinterpret_cast<const T*>(down) + V - OFF;
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (e < turning) a[e] = from_float<T>(fmaf(to_float(a[e]), c[e], to_float(e < firsts ? up_at[e] : down_at[e]) * s[e]));
      }
      *reinterpret_cast<uint4*>(dst + (h + i) * head_stride) = x[i];
    }
    __syncthreads();
  }
}

template <typename T, int OFF>
static int rotary_launch_shared(const RotaryParams& p, cudaStream_t s) {
  const int units = p.dim * (int)sizeof(T) / 16, tokens = R_THREADS / units;
  const int64_t each = rotary_heads_per_thread(p, units, R_SHARED, R_FILL_SHARED);
  const int64_t q_slices = (p.q.heads + each - 1) / each, k_slices = (p.k.heads + each - 1) / each;
  DTN_REQUIRE(q_slices + 2 * k_slices < 65536, DTN_ERR_UNSUPPORTED, "rotary: too many heads for one launch");
  const dim3 grid((unsigned)((p.tokens + tokens - 1) / tokens), (unsigned)(q_slices + 2 * k_slices));
  rotary_shared_kernel<T, OFF><<<grid, tokens * units, 0, s>>>(p, units, tokens, (int)each, (int)q_slices, (int)k_slices);
  DTN_LAUNCH_CHECK("rotary_shared_kernel");
  return DTN_OK;
}

template <typename T>
static int rotary_launch_t(const RotaryParams& p, int interleaved, cudaStream_t s) {
  // elements that every head's address and extent and, in the half layout, the distance within a pair are multiples of
  uint64_t common = (uint64_t)p.dim;
  auto add = [&](const void* base, int64_t token_stride, int64_t head_stride, int heads) {
    if (heads > 0) common |= (reinterpret_cast<uintptr_t>(base) / sizeof(T)) | (uint64_t)token_stride | (uint64_t)head_stride;
  };
  add(p.q.src, p.q.token_stride, p.q.head_stride, p.q.heads);
  add(p.q_out, p.q_out_token_stride, p.q_out_head_stride, p.q.heads);
  add(p.k.src, p.k.token_stride, p.k.head_stride, p.k.heads);
  add(p.v.src, p.v.token_stride, p.v.head_stride, p.v.heads);
  add(p.k_pages, p.page_stride, p.page_head_stride, p.k.heads);
  add(p.v_pages, p.page_stride, p.page_head_stride, p.v.heads);
  constexpr int WHOLE = 16 / (int)sizeof(T);
  if (common % WHOLE == 0) {
    if (interleaved) return rotary_launch_v<T, false, WHOLE>(p, 1, s);
    if (p.pairs % WHOLE == 0) return rotary_launch_v<T, true, WHOLE>(p, 0, s);
    if constexpr (WHOLE == 8) {
      switch (p.pairs % 8) {
        case 1: return rotary_launch_shared<T, 1>(p, s);
        case 2: return rotary_launch_shared<T, 2>(p, s);
        case 3: return rotary_launch_shared<T, 3>(p, s);
        case 5: return rotary_launch_shared<T, 5>(p, s);
        case 6: return rotary_launch_shared<T, 6>(p, s);
        case 7: return rotary_launch_shared<T, 7>(p, s);
        default: return rotary_launch_shared<T, 4>(p, s);
      }
    } else {
      switch (p.pairs % 4) {
        case 1: return rotary_launch_shared<T, 1>(p, s);
        case 2: return rotary_launch_shared<T, 2>(p, s);
        default: return rotary_launch_shared<T, 3>(p, s);
      }
    }
  }
  if (!interleaved) common |= (uint64_t)p.pairs;
  if constexpr (sizeof(T) == 2) {
    if (common % 4 == 0) return interleaved ? rotary_launch_v<T, false, 4>(p, 1, s) : rotary_launch_v<T, true, 4>(p, 0, s);
  }
  if (common % 2 == 0) return interleaved ? rotary_launch_v<T, false, 2>(p, 1, s) : rotary_launch_v<T, true, 2>(p, 0, s);
  return rotary_launch_v<T, true, 1>(p, interleaved, s);
}

static int rotary_launch(const RotaryParams& p, int interleaved, int storage, cudaStream_t s) {
  if (p.tokens == 0 || p.dim == 0 || p.q.heads + p.k.heads + p.v.heads == 0) return DTN_OK;
  if (storage == DTN_STORAGE_F32) return rotary_launch_t<float>(p, interleaved, s);
  if (storage == DTN_STORAGE_F16) return rotary_launch_t<__half>(p, interleaved, s);
  return rotary_launch_t<__nv_bfloat16>(p, interleaved, s);
}

}  // namespace dtn

extern "C" {

int dtn_rotary(const dtn_rotary_args* args, void* stream) {
  using namespace dtn;
  DTN_REQUIRE(args != nullptr, DTN_ERR_INVALID, "rotary: no arguments");
  const dtn_rotary_args& a = *args;
  DTN_REQUIRE(a.tokens >= 0 && a.heads >= 0 && a.dim >= 0 && a.pairs >= 0, DTN_ERR_INVALID, "rotary: negative extent");
  DTN_REQUIRE(paged_storage_known(a.storage), DTN_ERR_INVALID, "rotary: unknown storage %lld", (long long)a.storage);
  DTN_REQUIRE(a.dim <= R_MAX_DIM && a.heads < (1 << 20) && a.tokens < (1LL << 31), DTN_ERR_UNSUPPORTED,
              "rotary: heads of at most %d elements, fewer than 2^31 tokens", R_MAX_DIM);
  DTN_REQUIRE(a.pairs <= a.dim / 2, DTN_ERR_INVALID, "rotary: %lld pairs do not fit a head of %lld", (long long)a.pairs, (long long)a.dim);
  if (a.tokens == 0 || a.heads == 0 || a.dim == 0) return DTN_OK;
  DTN_REQUIRE(a.x && a.out && a.positions && (a.frequencies || a.pairs == 0), DTN_ERR_INVALID, "rotary: null pointer");
  RotaryParams p = {};
  p.q = {a.x, a.x_token_stride, a.x_head_stride, (int)a.heads};
  p.q_out = a.out;
  p.q_out_token_stride = a.out_token_stride;
  p.q_out_head_stride = a.out_head_stride;
  p.positions = a.positions;
  p.positions_64 = a.positions_64 != 0;
  p.frequencies = a.frequencies;
  p.pairs = (int)a.pairs;
  p.dim = (int)a.dim;
  p.amplitude = (float)a.amplitude;
  p.sign = a.transpose ? -1.f : 1.f;
  p.tokens = a.tokens;
  return rotary_launch(p, a.interleaved != 0, (int)a.storage, as_stream(stream));
}

int dtn_paged_append(const dtn_paged_append_args* args, void* stream) {
  using namespace dtn;
  DTN_REQUIRE(args != nullptr, DTN_ERR_INVALID, "paged append: no arguments");
  const dtn_paged_append_args& a = *args;
  DTN_REQUIRE(a.tokens >= 0 && a.kv_heads >= 0 && a.dim >= 0 && a.pairs >= 0 && a.q_heads >= 0 && a.pages >= 0 && a.sequences >= 0 &&
                  a.pages_per_sequence >= 0,
              DTN_ERR_INVALID, "paged append: negative extent");
  DTN_REQUIRE(a.page_size >= 1 && a.page_size < (1LL << 31), DTN_ERR_INVALID, "paged append: page size %lld", (long long)a.page_size);
  DTN_REQUIRE(paged_storage_known(a.storage), DTN_ERR_INVALID, "paged append: unknown storage %lld", (long long)a.storage);
  DTN_REQUIRE(a.dim <= R_MAX_DIM && a.kv_heads < (1 << 20) && a.q_heads < (1 << 20) && a.tokens < (1LL << 31) && a.pages < (1LL << 31) &&
                  a.pages_per_sequence < (1LL << 31),
              DTN_ERR_UNSUPPORTED, "paged append: heads of at most %d elements, fewer than 2^31 tokens and pages", R_MAX_DIM);
  DTN_REQUIRE(a.pairs <= a.dim / 2, DTN_ERR_INVALID, "paged append: %lld pairs do not fit a head of %lld", (long long)a.pairs, (long long)a.dim);
  if (a.tokens == 0 || a.dim == 0 || a.kv_heads + a.q_heads == 0) return DTN_OK;
  DTN_REQUIRE(a.k && a.v && a.rows && a.positions && (a.frequencies || a.pairs == 0), DTN_ERR_INVALID, "paged append: null pointer");
  DTN_REQUIRE((a.k_pages && a.v_pages) || a.pages == 0, DTN_ERR_INVALID, "paged append: null pool");
  DTN_REQUIRE(a.tables || a.sequences == 0 || a.pages_per_sequence == 0, DTN_ERR_INVALID, "paged append: null tables");
  DTN_REQUIRE(a.q_heads == 0 || (a.q && a.q_out), DTN_ERR_INVALID, "paged append: null queries");
  RotaryParams p = {};
  p.q = {a.q, a.q_token_stride, a.q_head_stride, (int)a.q_heads};
  p.k = {a.k, a.k_token_stride, a.k_head_stride, (int)a.kv_heads};
  p.v = {a.v, a.v_token_stride, a.v_head_stride, (int)a.kv_heads};
  p.q_out = a.q_out;
  p.q_out_token_stride = a.q_out_token_stride;
  p.q_out_head_stride = a.q_out_head_stride;
  p.k_pages = a.k_pages;
  p.v_pages = a.v_pages;
  p.page_stride = a.page_stride;
  p.page_head_stride = a.page_head_stride;
  p.tables = a.tables;
  p.table_stride = a.table_stride;
  p.rows = a.rows;
  p.sequences = a.sequences;
  p.pages = a.pages;
  p.capacity = a.pages_per_sequence * a.page_size;
  p.page_size = (int)a.page_size;
  p.positions = a.positions;
  p.positions_64 = a.positions_64 != 0;
  p.frequencies = a.frequencies;
  p.pairs = (int)a.pairs;
  p.dim = (int)a.dim;
  p.amplitude = (float)a.amplitude;
  p.sign = 1.f;
  p.tokens = a.tokens;
  p.status = device_status_word_unless_capturing(as_stream(stream));
  return rotary_launch(p, a.interleaved != 0, (int)a.storage, as_stream(stream));
}

}  // extern "C"
