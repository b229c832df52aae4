// Attention of one new token per sequence over a paged key-value cache.
//
// For each sequence and query head: out = sum_t p_t v_t / sum_t p_t, p_t = 2^(x_t - m), x_t = scale log2(e) q.k_t, with the
// running maximum m, denominator and numerator of one pass over the tokens. The bytes of the keys and values are the floor:
// with g query heads on one kv head the work is 2 g multiply-adds per element read, far below what the card does per byte, so
// everything here serves an even, deep and unbroken stream of loads.
//
//   Shares. A unit is one tile of tokens (CHUNK per team of warps) of one item (sequence, kv head, block of query heads), and
//   PA_ITEM_UNITS more stand at an item's end for what finishing it costs; the units of the whole batch, tile fastest, then
//   head, then sequence, are cut into equal contiguous ranges, one per block of a grid that fills the card once. So the split
//   over a sequence's length follows from the lengths on the device: no host copy of them, one launch, any raggedness, and a
//   captured launch follows lengths that change.
//   Pipeline. Each team keeps a ring of stages in shared memory filled by 16-byte asynchronous copies, ahead of the products
//   and across the ends of sequences; a token's row is looked up through the page table one stage before its copies are
//   issued. Nothing but the stage's own warps waits for a stage. Where a set of tokens lies in one page its rows follow one
//   another and the copies' addresses differ by constants. Three blocks of four warps per SM with two stages each read faster
//   than two with three stages (245 against 254 us below): what is short is not bytes in flight but warps whose chains of
//   dependent instructions overlap.
//   Products, 16-bit storage. mma.sync m16n8k16 with the tokens as the 16 rows and the query heads as the 8 columns:
//   scores = K Q^T, numerators = V^T P^T, so that a group of up to 8 heads wastes nothing and the probabilities turn from
//   result to operand layout with one movmatrix per 8 x 8. At the copy rate 8 heads need 80 TFLOP/s of products; tcgen05
//   would need 64 or 128 rows of heads, or P through shared memory. P is split into terms of the storage type, and a chunk's
//   product starts from zero and is added to the FP32 numerator apart: the tensor core's own accumulator truncates. Three
//   bf16 terms leave 2^-24 of a probability. f16 has too few exponents for that: 2^-24 is its smallest step. So its
//   probabilities are 2^BIAS times larger (the factor is in the sums as well and cancels), which puts the largest at 2^15, and
//   the second of two terms is REST = 2^12 times what the first leaves, with a product of its own that is scaled back when it
//   is added. That leaves 2^-23 of a probability, or 2^-44 of 1 where that is more: half a step of the second term, 2^-25, over
//   2^BIAS and REST; 1 is a token whose score is the maximum that the warp keeps. (Two terms of one scale left 2^-25 of 1: 48
//   tokens, one of them with a zero value and all but 4e-5 of the mass, were off by 1e-3, now by 5e-7. Neither form is
//   slower than the other: the 96 users 246.9 and 246.9 us, groups of 16 99.6 and 100.0, head size 80 70.0 and 70.4.)
//   Products, FP32 storage. Plain fused multiply-adds: four lanes share a token's score, a lane owns dim / 32 columns of V.
//   More than 8 query heads per kv head: HB = 2 or 4 warps share a team's stage, each with its 8 heads; beyond 32 the
//   heads are split into blocks that read the keys again. From 16 heads on the products and the instructions around them, not the bytes, set
//   the time.
//   Join. A block that holds a whole item writes it. Otherwise it leaves (m, sum, numerators) in the workspace and counts
//   itself in; the last to arrive adds the parts in the order of the blocks, so the result does not depend on who was last.
//   It leaves the counter at zero for the next launch.
//
// No form may use local memory: a build in which registers spilled read wrong addresses at head sizes above 128.
//
// Measured (kernel in a graph of 30 calls on three sets of inputs in turn, fraction of the 6540 GB/s of a copy):
//   96 users, 17..8192 tokens, 32 heads on 8, 128, f16, 1.62 GB: 244 us (1.01); 16 users, 1..4096, 137 MB: 30 us (0.69, of
//   which 3 us are the launch and the clearing of the counters); one user of 131071, bf16, 537 MB: 88.4 us (0.93; 37 blocks
//   share each head, joining them costs 3 us, the slowest SM is 8 % behind the mean); 9 users, FP32, 16 heads of 64, 124 MB:
//   28.6 us (0.66); 37 tokens of one user: 6 us. 256 users of 128..256 tokens: 0.70. 64 users of 64..8192 tokens, f16: head 64,
//   32 on 8, 0.90; head 256, 16 on 4, 0.91; head 128 in groups of 16 on 4 0.85, of 32 on 2 0.54, of 40 and 64 on 2 0.33 and 0.32
//   (the keys are read twice), of 128 on one 0.17. 32 users, FP32, 8 kv heads: head 64 in groups of 1, 4 and 8 0.95, 0.91 and
//   0.79; head 128 0.95, 0.88 and 0.69, of 16 0.49.
#include <type_traits>

#include "paged.cuh"

namespace dtn {

constexpr int PA_WARPS = 4;
constexpr int PA_MAX_BLOCKS = 1024;        // counters in the workspace
constexpr int PA_COUNTER_BYTES = PA_MAX_BLOCKS * 4;

// position / divisor as a multiplication, for positions below 2^31 and divisors from 1 to 2^31 - 1: mul = floor(2^(31 + s) / d) + 1
// with 2^s >= d exceeds 2^(31 + s) / d by at most 1, so the product exceeds the quotient by less than 2^31 / 2^(31 + s) <= 1 / d:
// the floor is exact. mul <= 2^32 - 1 needs d > 1; for d = 1 the multiplier is 1 and the shift 0.
struct PaDivider {
  uint32_t mul;
  int shift;
  __host__ __device__ __forceinline__ int operator()(int position) const { return (int)(((uint64_t)(uint32_t)position * mul) >> shift); }
};
static PaDivider pa_divider(int64_t divisor) {
  if (divisor == 1) return {1, 0};
  int bits = 1;
  while ((1LL << bits) < divisor) ++bits;
  return {(uint32_t)((1ULL << (31 + bits)) / (uint64_t)divisor + 1), 31 + bits};
}

struct PagedAttentionParams {
  const void *q, *k_pages, *v_pages;
  void* out;
  const int *tables, *lengths, *rows;   // rows may be null: sequence i uses row i
  int64_t count, sequences, pages, table_stride;
  int64_t q_token_stride, q_head_stride, out_token_stride, out_head_stride;   // elements
  int64_t page_stride, page_head_stride;                                      // bytes
  int64_t window;
  int capacity;                         // tokens that a row of the tables covers
  int heads, kv_heads;                  // items per sequence: kv heads x blocks of query heads
  int blocks;                           // blocks of query heads per kv head
  int q_heads, group, dim, page_size, row_bytes;
  PaDivider pages_of;                   // position / page_size
  float scale_log2e;
  int out_f32;
  int q_pairs, out_quads;               // neighbouring elements of q and out can be moved by two (4 bytes) and by four
  int whole_sets;                       // the tokens of a set lie in one page, one after another
  int min_units;                        // a block takes at least this many units
  int* counters;
  float* parts;
  int* status;
};

// Units for the end of an item: the teams' parts are added, the result written, the next query taken (0, 1, 2, 3 and 5 units on
// the 16 users: 35.3, 32.5, 32.1, 31.5 and 31.5 us; on 64 long ones 3 is still free).
constexpr int PA_ITEM_UNITS = 3;
constexpr int PA_JOIN = 8;                 // parts requested at once where they are joined

// First unit of block c of `workers`, and the block that holds a unit: units * c / workers <= unit.
__host__ __device__ __forceinline__ int64_t pa_share_begin(int64_t units, int64_t workers, int64_t c) { return units * c / workers; }
__host__ __device__ __forceinline__ int64_t pa_share_owner(int64_t units, int64_t workers, int64_t unit) {
  return ((unit + 1) * workers - 1) / units;
}
// Blocks that take part: each has at least min_units units, but for the only one.
__host__ __device__ __forceinline__ int64_t pa_workers(int64_t units, int64_t min_units, int64_t grid) {
  const int64_t most = units / min_units;
  return most < 1 ? 1 : (most < grid ? most : grid);
}

template <typename T, int DP, int HB, int NH>
struct PaConfig {
  static constexpr bool HALF = sizeof(T) == 2;
  static constexpr int SUB = HALF ? 16 : 8;              // tokens of one set of products
  // sets that a team takes in one step: one per member keeps as many tokens in work whatever the group; twice that for small
  // rows, whose chain of dependent instructions would otherwise outlast their bytes
  static constexpr int SETS = DP == 64 ? (HB == 1 ? 2 : 4) : (DP == 256 && HB == 4 ? 2 : HB);
  static constexpr int CHUNK = SUB * SETS;               // tokens per stage
  static constexpr int TEAMS = PA_WARPS / HB;
  static constexpr int ROW = DP * (int)sizeof(T);
  static constexpr int STAGE = 2 * CHUNK * ROW;          // keys, then values: 64 * DP * SETS bytes; at an item's end numerators of HB x 8 heads
  static constexpr int RING = (DP == 256 ? 192 : 64) * 1024;
  static constexpr int STAGES = RING / (TEAMS * STAGE);
  static constexpr int QUERY = HALF ? 0 : HB * NH * DP * 4;
  static constexpr int SMEM = RING + QUERY;
  static constexpr int BLOCKS_PER_SM = DP == 256 ? 1 : (HALF || HB == 1 ? 3 : 2);   // 168 registers and 64 KB for three
  static constexpr int HEADS = 8 * HB;                   // query heads of an item (the first NH of each 8 are looked at)
  static constexpr int PART = HEADS * DP + 2 * HEADS;    // floats: numerators, then maximum and sum of each head
  static_assert(STAGES >= 2 && STAGE >= HEADS * DP * 4, "a ring of two stages, numerators that fit one");
};

__device__ __forceinline__ void pa_copy16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void pa_copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// Two FP32 sums in one instruction.
__device__ __forceinline__ void pa_add2(float& a0, float& a1, float b0, float b1) {
  asm("{ .reg .b64 a, b; mov.b64 a, {%0, %1}; mov.b64 b, {%2, %3}; add.rn.f32x2 a, a, b; mov.b64 {%0, %1}, a; }" : "+f"(a0), "+f"(a1) : "f"(b0), "f"(b1));
}
// a += b * c for two.
__device__ __forceinline__ void pa_fma2(float& a0, float& a1, float b0, float b1, float c) {
  asm("{ .reg .b64 a, b, c; mov.b64 a, {%0, %1}; mov.b64 b, {%2, %3}; mov.b64 c, {%4, %4}; fma.rn.f32x2 a, b, c, a; mov.b64 {%0, %1}, a; }"
      : "+f"(a0), "+f"(a1) : "f"(b0), "f"(b1), "f"(c));
}
__device__ __forceinline__ void pa_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void pa_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void pa_ldmatrix(uint32_t (&r)[4], uint32_t address) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(address) : "memory");
}
__device__ __forceinline__ void pa_ldmatrix_t(uint32_t (&r)[4], uint32_t address) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(address) : "memory");
}
__device__ __forceinline__ uint32_t pa_transpose(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ void pa_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void pa_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void pa_mma_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void pa_mma_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
// Rounds a pair to the storage type (low half first) and leaves what the rounding took off.
__device__ __forceinline__ uint32_t pa_take(float& a, float& b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  const float2 f = __half22float2(h);
  a -= f.x;
  b -= f.y;
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pa_take(float& a, float& b, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  const float2 f = __bfloat1622float2(h);
  a -= f.x;
  b -= f.y;
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Counts a block in; what its threads wrote before the barrier ahead of this is seen by whoever reads after the last arrival.
__device__ __forceinline__ int pa_arrive(int* counter) {
  int before;
  asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
  return before;
}

// What is seen of a sequence: its row of the tables and tokens first + skip .. first + seen. A window's tiles start at a
// multiple of SUB tokens, so that sets of tokens lie in one page where they can; the skip tokens before it are not seen.
struct PaSequence {
  int64_t table;
  int first, skip, seen;
};

template <int SUB>
__device__ __forceinline__ PaSequence pa_sequence(const PagedAttentionParams& p, int64_t i) {
  PaSequence s = {0, 0, 0, 0};
  const int64_t row = p.rows ? (int64_t)p.rows[i] : i;
  if (row < 0) return s;
  if (row >= p.sequences) {
    paged_report(p.status, PAGED_STATUS_ATTENTION);
    return s;
  }
  int length = p.lengths[row];
  if (length > p.capacity) {
    paged_report(p.status, PAGED_STATUS_ATTENTION);
    length = p.capacity;
  }
  if (length <= 0) return s;
  s.table = row * p.table_stride;
  const int begin = p.window > 0 && p.window < length ? length - (int)p.window : 0;
  s.skip = begin % SUB;
  s.first = begin - s.skip;
  s.seen = length - s.first;
  return s;
}

template <int UNIT>
__device__ __forceinline__ int pa_tiles(int seen) { return seen <= 0 ? 0 : (seen - 1) / UNIT + 1; }

// Units of one item of a sequence; none where nothing is seen (its zeros are written apart).
__device__ __forceinline__ int64_t pa_item_units(int tiles) { return tiles > 0 ? (int64_t)tiles + PA_ITEM_UNITS : 0; }

// A place in the order of the units, always a tile.
template <int UNIT, int SUB>
struct PaCursor {
  int sequence;
  int left;                      // units of the share from here on
  int kv_head, block;            // block of query heads
  int tile, tiles;
  PaSequence s;

  __device__ __forceinline__ void enter(const PagedAttentionParams& p) {
    s = pa_sequence<SUB>(p, sequence);
    tiles = pa_tiles<UNIT>(s.seen);
  }
  __device__ __forceinline__ void next_item(const PagedAttentionParams& p) {   // from the first unit behind this item's tiles
    left -= PA_ITEM_UNITS;
    tile = 0;
    if (++block < p.blocks) return;
    block = 0;
    if (++kv_head < p.kv_heads) return;
    kv_head = 0;
    do {
      ++sequence;
      if (sequence >= p.count) return;   // past every share
      enter(p);
    } while (tiles == 0);
  }
  __device__ __forceinline__ void step(const PagedAttentionParams& p) {
    --left;
    if (++tile == tiles) next_item(p);
  }
};

template <typename T, int DP, int HB, int NH>
__global__ void __launch_bounds__(PA_WARPS * 32, PaConfig<T, DP, HB, NH>::BLOCKS_PER_SM) paged_attention_kernel(const PagedAttentionParams p) {
  using C = PaConfig<T, DP, HB, NH>;
  constexpr int CHUNK = C::CHUNK, SETS = C::SETS, TEAMS = C::TEAMS, ROW = C::ROW, STAGES = C::STAGES, UNIT = CHUNK * TEAMS, THREADS = PA_WARPS * 32;
  constexpr int LANES = ROW / 16;                  // 16-byte vectors of a row
  constexpr float NONE = -INFINITY;
  constexpr bool SPLIT = std::is_same_v<T, __half>;   // probabilities in two terms of different scales
  constexpr float BIAS = SPLIT ? 7.f : 0.f;           // probabilities are held 2^BIAS times larger than against the maximum
  constexpr float FEWER = SPLIT ? 0.f : 23.f, FEW = SPLIT ? 1.f : 1.f / 8388608.f;   // and 2^FEWER times smaller in a second pass
  constexpr float GROWTH = 8.f;
  constexpr float REST = 4096.f;                      // half a step of the first term, at most 2^3, stays below f16's largest value
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float s_max[PA_WARPS][8], s_sum[PA_WARPS][8];
  __shared__ __align__(16) float s_p[C::HALF ? 1 : PA_WARPS][C::HALF ? 1 : CHUNK][NH], s_alpha[C::HALF ? 1 : PA_WARPS][8];
  __shared__ int64_t s_scan[PA_WARPS];
  __shared__ int64_t s_start[2];
  __shared__ int64_t s_plan[3];                    // units, workers and the share's end: for the end of an item, not worth registers
  __shared__ int s_last;

  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, team = warp / HB, member = warp % HB;
  const int g = lane / 4, t = lane % 4;

  // -- the share of this block: thread i adds up a contiguous part of the sequences ---------------
  const int64_t per = (p.count + THREADS - 1) / THREADS, mine = tid * per, mine_end = mine + per < p.count ? mine + per : p.count;
  int64_t sum = 0;
  for (int64_t i = mine; i < mine_end; ++i) sum += pa_item_units(pa_tiles<UNIT>(pa_sequence<C::SUB>(p, i).seen));
  int64_t before = sum;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int64_t other = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += other;
  }
  if (lane == 31) s_scan[warp] = before;
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w < PA_WARPS; ++w) {
    if (w < warp) before += s_scan[w];
    total += s_scan[w];
  }
  before -= sum;
  for (int64_t i = blockIdx.x; i < p.count; i += gridDim.x) {   // rows that see nothing
    if (pa_sequence<C::SUB>(p, i).seen > 0) continue;
    for (int j = tid; j < p.q_heads * p.dim; j += THREADS) {
      const int64_t to = i * p.out_token_stride + j / p.dim * p.out_head_stride + j % p.dim;
      if (p.out_f32)
        static_cast<float*>(p.out)[to] = 0.f;
      else
        static_cast<T*>(p.out)[to] = from_float<T>(0.f);
    }
  }
  const int64_t units = total * p.heads;
  const int64_t workers = pa_workers(units, p.min_units, gridDim.x);
  if (units == 0 || blockIdx.x >= workers) return;
  const int64_t begin = pa_share_begin(units, workers, blockIdx.x), end = pa_share_begin(units, workers, blockIdx.x + 1);
  if (begin >= before * p.heads && begin < (before + sum) * p.heads) {
    int64_t at = before * p.heads;
    for (int64_t i = mine; i < mine_end; ++i) {
      const int64_t here = pa_item_units(pa_tiles<UNIT>(pa_sequence<C::SUB>(p, i).seen)) * p.heads;
      if (begin < at + here) {
        s_start[0] = i;
        s_start[1] = begin - at;
        break;
      }
      at += here;
    }
  }
  if (tid == 0) s_plan[0] = units, s_plan[1] = workers, s_plan[2] = end;
  __syncthreads();
  PaCursor<UNIT, C::SUB> now, ahead;
  now.left = (int)(end - begin);
  now.sequence = (int)s_start[0];
  now.enter(p);
  {
    const int item = (int)(s_start[1] / pa_item_units(now.tiles));
    now.kv_head = item / p.blocks;
    now.block = item % p.blocks;
    now.tile = (int)(s_start[1] % pa_item_units(now.tiles));
    if (now.tile >= now.tiles) {   // the share begins behind an item's tiles
      now.left += now.tile - now.tiles;
      now.next_item(p);
    }
  }
  ahead = now;

  // -- copies -------------------------------------------------------------------------------------
  uint8_t* ring = smem + team * STAGES * C::STAGE;
  const uint32_t ring_address = smem_u32(ring);
  constexpr int ROWS = CHUNK / HB;                 // of a stage, copied by this warp: rows member * ROWS + 0, 1, ...
  int64_t offset = -1;             // of row lane % ROWS of them in the stage that is copied next; -1: not seen, -2: no such page

  auto look_up = [&]() {
    const int token = (ahead.tile * TEAMS + team) * CHUNK + member * ROWS + lane % ROWS;
    offset = -1;
    if (token < ahead.s.seen && token >= ahead.s.skip) {
      const int position = ahead.s.first + token;
      const int index = p.pages_of(position);
      const int page = p.tables[ahead.s.table + index];
      offset = -2;
      if (page >= 0 && page < p.pages)
        offset = page * p.page_stride + ahead.kv_head * p.page_head_stride + (int64_t)(position - index * p.page_size) * p.row_bytes;
    }
  };
  // Lane l copies vector l % LANES of rows l / LANES, + 32 / LANES, ...: their swizzled places differ by constants.
  const int lane_row = LANES <= 32 ? lane / LANES : 0, lane_column = LANES <= 32 ? lane % LANES : lane;
  const uint8_t *k_pages = static_cast<const uint8_t*>(p.k_pages), *v_pages = static_cast<const uint8_t*>(p.v_pages);
  const uint32_t lane_place = (member * ROWS + lane_row) * ROW +
                              (C::HALF ? lane_column ^ ((member * ROWS + lane_row) & 7) : lane_column ^ (((member * ROWS + lane_row) & 1) << 2)) * 16;
  auto copy = [&](int slot) {
    const uint32_t seen_rows = __ballot_sync(0xffffffffu, offset >= 0);
    const uint32_t stage = ring_address + slot * C::STAGE;
    if (seen_rows == 0xffffffffu && p.whole_sets) {   // one page holds the rows of a set one after another: constant distances
      constexpr int TOGETHER = ROWS < C::SUB ? ROWS : C::SUB, STEP = LANES <= 32 ? 32 / LANES : 1;   // rows between two copies of a lane
      if (p.row_bytes == ROW) {
#pragma unroll
        for (int set = 0; set < ROWS / TOGETHER; ++set) {
          const int64_t at = __shfl_sync(0xffffffffu, offset, set * TOGETHER) + (lane_row * ROW + lane_column * 16);
          const uint8_t *k_at = k_pages + at, *v_at = v_pages + at;
#pragma unroll
          for (int j = 0; j < TOGETHER * LANES / 32; ++j) {
            const int row = LANES <= 32 ? j * STEP : j / 2, half = LANES <= 32 ? 0 : j % 2 * 512;   // a row of 64 vectors takes two copies
            const uint32_t to = ((stage + lane_place) ^ (C::HALF ? (row & 7) << 4 : (row & 1) << 6)) + (set * TOGETHER + row) * ROW + half;
            pa_copy16(to, k_at + row * ROW + half);
            pa_copy16(to + CHUNK * ROW, v_at + row * ROW + half);
          }
        }
      } else {   // narrower rows: zeros in the columns past the head
#pragma unroll
        for (int set = 0; set < ROWS / TOGETHER; ++set) {
          const int64_t at = __shfl_sync(0xffffffffu, offset, set * TOGETHER) + lane_row * p.row_bytes;
#pragma unroll
          for (int j = 0; j < TOGETHER * LANES / 32; ++j) {
            const int row = LANES <= 32 ? j * STEP : j / 2, half = LANES <= 32 ? 0 : j % 2 * 512;
            const uint32_t to = ((stage + lane_place) ^ (C::HALF ? (row & 7) << 4 : (row & 1) << 6)) + (set * TOGETHER + row) * ROW + half;
            const int bytes = lane_column * 16 + half < p.row_bytes ? 16 : 0;
            const int64_t from = bytes ? at + row * p.row_bytes + half + lane_column * 16 : 0;   // copies of nothing name the pool's start
            pa_copy16(to, k_pages + from, bytes);
            pa_copy16(to + CHUNK * ROW, v_pages + from, bytes);
          }
        }
      }
      return;
    }
    const bool bad = __any_sync(0xffffffffu, offset == -2);
    if (bad && lane == 0) paged_report(p.status, PAGED_STATUS_ATTENTION);
    if (!bad && seen_rows == 0 && HB == 1) return;   // nothing of this stage is looked at
#pragma unroll
    for (int j = 0; j < ROWS * LANES / 32; ++j) {
      const int v = lane + 32 * j, own = v / LANES, row = member * ROWS + own, column = v % LANES;
      const int64_t at = __shfl_sync(0xffffffffu, offset, own);
      const int swizzled = C::HALF ? column ^ (row & 7) : column ^ ((row & 1) << 2);
      const uint32_t to = stage + row * ROW + swizzled * 16;
      const bool there = at >= 0 && column * 16 < p.row_bytes;   // else zeros: neither what is not seen nor the columns past a head count
      const int64_t from = there ? at + column * 16 : 0;
      if (at == -2)   // keys of a page that does not exist are NaN, and so is all that sees them
        *reinterpret_cast<uint4*>(ring + (to - ring_address)) = make_uint4(0x7fffffffu, 0x7fffffffu, 0x7fffffffu, 0x7fffffffu);
      else
        pa_copy16(to, k_pages + from, there ? 16 : 0);
      pa_copy16(to + CHUNK * ROW, v_pages + from, there ? 16 : 0);
    }
  };
  auto team_barrier = [&]() {
    if (HB == 1)
      __syncwarp();
    else
      asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(32 * HB) : "memory");
  };

  // -- queries ------------------------------------------------------------------------------------
  constexpr int STEPS_K = DP / 16;
  uint32_t query[C::HALF ? STEPS_K : 1][2], query_next[C::HALF && DP == 64 ? STEPS_K : 1][2];
  float* s_query = reinterpret_cast<float*>(smem + C::RING);
  auto head_of = [&](int block, int h) { return block * C::HEADS + h; };   // within the group
  auto load_query = [&](uint32_t (&to)[C::HALF ? STEPS_K : 1][2], int sequence, int kv_head, int block) {
    // 16-bit storage: columns 2t.. and 2t + 8.. of head g, per 16
    const int h = head_of(block, member * 8 + g);
    const bool there = h < p.group;
    const T* q = static_cast<const T*>(p.q) + sequence * p.q_token_stride + ((int64_t)kv_head * p.group + (there ? h : 0)) * p.q_head_stride + 2 * t;
    if (p.q_pairs && p.dim == DP) {
#pragma unroll
      for (int i = 0; i < 2 * STEPS_K; ++i) to[i / 2][i % 2] = there ? *reinterpret_cast<const uint32_t*>(q + i * 8) : 0u;
    } else {
#pragma unroll
      for (int i = 0; i < 2 * STEPS_K; ++i) {
        uint32_t v = 0;
        if (there && i * 8 + 2 * t < p.dim) {   // dim is even
          if (p.q_pairs)
            v = *reinterpret_cast<const uint32_t*>(q + i * 8);
          else
            v = *reinterpret_cast<const uint16_t*>(q + i * 8) | (uint32_t) * reinterpret_cast<const uint16_t*>(q + i * 8 + 1) << 16;
        }
        to[i / 2][i % 2] = v;
      }
    }
  };
  if constexpr (C::HALF && DP == 64)
    if (now.left > 0) load_query(query_next, now.sequence, now.kv_head, now.block);

  // -- the pass over the tokens -------------------------------------------------------------------
  constexpr int COLUMNS = DP / 32;                 // FP32 storage: columns of V per lane
  float top[2] = {NONE, NONE}, total_p[2] = {0.f, 0.f};   // of heads 2t, 2t + 1
  constexpr int A = C::HALF ? DP / 16 : NH, B = C::HALF ? 4 : COLUMNS;
  float acc[A][B];                                 // numerators: 16 columns of V by 2 heads, or NH heads by COLUMNS
  float growth = GROWTH;                           // how far scores may pass the maximum before it moves
  bool fresh = true, again = false;
  int start = 0;                                   // the item's first tile here
  int slot = 0, filling = STAGES - 1;              // the oldest stage; copies still to be issued before the first stage is read

  if (ahead.left > 0) look_up();
  while (now.left > 0) {
    pa_wait<STAGES - 2>();
    team_barrier();   // the oldest stage is there, and the one before it has been read by all
    if (ahead.left > 0) {
      copy(filling > 0 ? STAGES - 1 - filling : (slot == 0 ? STAGES - 1 : slot - 1));
      ahead.step(p);
      if (ahead.left > 0) look_up();
    }
    pa_commit();
    if (filling > 0) {
      --filling;
      continue;
    }

    if (fresh) {
      fresh = false;
      start = now.tile;
#pragma unroll
      for (int i = 0; i < 2; ++i) top[i] = NONE, total_p[i] = 0.f;
#pragma unroll
      for (int i = 0; i < A; ++i)
#pragma unroll
        for (int j = 0; j < B; ++j) acc[i][j] = 0.f;
      if constexpr (C::HALF && DP > 64) {
        load_query(query, now.sequence, now.kv_head, now.block);   // registers for one item's query only
      } else if constexpr (C::HALF) {
#pragma unroll
        for (int ks = 0; ks < STEPS_K; ++ks) query[ks][0] = query_next[ks][0], query[ks][1] = query_next[ks][1];
        PaCursor<UNIT, C::SUB> next = now;   // the next item's, a whole item ahead
        next.left -= now.tiles - now.tile;
        next.next_item(p);
        if (next.left > 0) load_query(query_next, next.sequence, next.kv_head, next.block);
      } else {
        __syncthreads();
        for (int i = tid; i < HB * NH * DP; i += THREADS) {
          const int h = head_of(now.block, i / DP / NH * 8 + i / DP % NH), d = i % DP;
          s_query[i] = h < p.group && d < p.dim ? static_cast<const float*>(p.q)[now.sequence * p.q_token_stride +
                                                      ((int64_t)now.kv_head * p.group + h) * p.q_head_stride + d] : 0.f;
        }
        __syncthreads();
      }
    }

    const int base = (now.tile * TEAMS + team) * CHUNK, seen = now.s.seen;
    if (base < seen) {
      const uint32_t stage = ring_address + slot * C::STAGE;
      constexpr int EIGHTS = CHUNK / 8;            // tokens g + 8 n of the chunk
      float x[EIGHTS][2];                          // scores, then probabilities, of heads 2t and 2t + 1
      if constexpr (C::HALF) {
        const uint32_t k_place = stage + lane % 16 * ROW + ((lane / 16) ^ (lane % 8)) * 16;   // stages are multiples of 128 bytes
#pragma unroll
        for (int set = 0; set < SETS; ++set) {
          float s[4] = {0.f, 0.f, 0.f, 0.f}, s2[4] = {0.f, 0.f, 0.f, 0.f};   // two chains of products
#pragma unroll
          for (int ks = 0; ks < STEPS_K; ++ks) {
            if (ks == STEPS_K * 3 / 4 && p.dim <= DP * 3 / 4) break;   // the last quarter is zeros
            uint32_t a[4];
            pa_ldmatrix(a, (k_place ^ (ks % 4 * 32)) + ks / 4 * 128 + set * 16 * ROW);
            pa_mma(ks % 2 ? s2 : s, a, query[ks][0], query[ks][1], T());
          }
          x[2 * set][0] = s[0] + s2[0], x[2 * set][1] = s[1] + s2[1];
          x[2 * set + 1][0] = s[2] + s2[2], x[2 * set + 1][1] = s[3] + s2[3];
        }
      } else {
        const float* query_rows = s_query + member * NH * DP;
        float s[SETS][8] = {};
#pragma unroll
        for (int j = 0; j < DP / 16; ++j) {
          const int column = t + 4 * j;
          float4 k[SETS];
#pragma unroll
          for (int set = 0; set < SETS; ++set)
            k[set] = *reinterpret_cast<const float4*>(ring + slot * C::STAGE + (set * 8 + g) * ROW + ((column ^ ((g & 1) << 2)) * 16));
#pragma unroll
          for (int h = 0; h < NH; ++h) {
            const float4 q = *reinterpret_cast<const float4*>(query_rows + h * DP + column * 4);
#pragma unroll
            for (int set = 0; set < SETS; ++set)
              s[set][h] = fmaf(k[set].x, q.x, fmaf(k[set].y, q.y, fmaf(k[set].z, q.z, fmaf(k[set].w, q.w, s[set][h]))));
          }
        }
        // four lanes hold parts of a token's scores; lane t ends with heads 2t and 2t + 1 (those past NH: zeros)
#pragma unroll
        for (int set = 0; set < SETS; ++set) {
          float r[4];
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            const float kept = t & 2 ? s[set][h + 4] : s[set][h], sent = t & 2 ? s[set][h] : s[set][h + 4];
            r[h] = h < NH ? kept + __shfl_xor_sync(0xffffffffu, sent, 2) : 0.f;
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float kept = t & 1 ? r[h + 2] : r[h], sent = t & 1 ? r[h] : r[h + 2];
            x[set][h] = h < NH ? kept + __shfl_xor_sync(0xffffffffu, sent, 1) : 0.f;
          }
        }
      }
#pragma unroll
      for (int n = 0; n < EIGHTS; ++n) x[n][0] *= p.scale_log2e, x[n][1] *= p.scale_log2e;
      if (base + CHUNK > seen || base < now.s.skip) {
#pragma unroll
        for (int n = 0; n < EIGHTS; ++n)
          if (base + g + 8 * n >= seen || base + g + 8 * n < now.s.skip) x[n][0] = x[n][1] = NONE;
      }
      // The maximum moves only when a score passes it by more than GROWTH: until then probabilities reach 2^GROWTH, which
      // FP32 sums do not mind and f16 terms have room for (2^(GROWTH + BIAS) = 2^15), and nothing is exchanged or rescaled.
      bool higher = false;
#pragma unroll
      for (int n = 0; n < EIGHTS; ++n) higher |= x[n][0] > top[0] + growth || x[n][1] > top[1] + growth;
      if (__any_sync(0xffffffffu, higher)) {
        float alpha[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float high = top[i];
#pragma unroll
          for (int n = 0; n < EIGHTS; ++n) high = fmaxf(high, x[n][i]);
#pragma unroll
          for (int o = 4; o < 32; o *= 2) high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
          alpha[i] = ex2_approx_ftz(top[i] - (high == NONE ? 0.f : high));
          top[i] = high;
          total_p[i] *= alpha[i];
        }
        if constexpr (C::HALF) {
#pragma unroll
          for (int mt = 0; mt < DP / 16; ++mt)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[mt][j] *= alpha[j % 2];
        } else {
          if (g == 0) s_alpha[warp][2 * t] = alpha[0], s_alpha[warp][2 * t + 1] = alpha[1];
          __syncwarp();
#pragma unroll
          for (int h = 0; h < NH; ++h) {
            const float a = s_alpha[warp][h];
#pragma unroll
            for (int j = 0; j < COLUMNS; ++j) acc[h][j] *= a;
          }
          __syncwarp();
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float around = top[i] == NONE ? 0.f : top[i] - BIAS;   // every score -inf so far: the exponentials are zeros, not NaN
#pragma unroll
        for (int n = 0; n < EIGHTS; ++n) {
          x[n][i] = ex2_approx_ftz(x[n][i] - around);
          total_p[i] += x[n][i];
        }
      }
      if (!SPLIT && again) {
#pragma unroll
        for (int n = 0; n < EIGHTS; ++n) x[n][0] *= FEW, x[n][1] *= FEW;
      }
      if constexpr (C::HALF) {
        if (!again) {
          constexpr int TERMS = SPLIT ? 2 : 3;
          uint32_t b[SETS][TERMS][2];
#pragma unroll
          for (int set = 0; set < SETS; ++set)
#pragma unroll
            for (int n = 0; n < TERMS; ++n)
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                float &p0 = x[2 * set + half][0], &p1 = x[2 * set + half][1];
                if (SPLIT && n == 1) p0 *= REST, p1 *= REST;
                b[set][n][half] = pa_transpose(pa_take(p0, p1, T()));
              }
          const uint32_t v_place = stage + CHUNK * ROW + (lane % 8 + lane / 16 * 8) * ROW + ((lane / 8 % 2) ^ (lane % 8)) * 16;
          auto load_values = [&](uint32_t(&a)[4], int mt, int set) { pa_ldmatrix_t(a, (v_place ^ (mt % 4 * 32)) + mt / 4 * 128 + set * 16 * ROW); };
          // Registers for one product only: the small terms' is scaled back and goes on as the large ones', which reads the values again.
          constexpr bool TWICE = SPLIT && DP == 256 && SETS > 1;
#pragma unroll
          for (int mt = 0; mt < DP / 16; ++mt) {
            if (mt == DP / 16 * 3 / 4 && p.dim <= DP * 3 / 4) break;
            float y[4];
            if constexpr (TWICE) {
#pragma unroll
              for (int set = 0; set < SETS; ++set) {
                uint32_t a[4];
                load_values(a, mt, set);
                if (set == 0)
                  pa_mma_first(y, a, b[set][1][0], b[set][1][1], T());
                else
                  pa_mma(y, a, b[set][1][0], b[set][1][1], T());
              }
#pragma unroll
              for (int j = 0; j < 4; ++j) y[j] *= 1.f / REST;
            }
            float rest[4];
#pragma unroll
            for (int set = 0; set < SETS; ++set) {
              uint32_t a[4];
              load_values(a, mt, set);
              if constexpr (SPLIT) {
                if (set == 0 && !TWICE) {
                  pa_mma_first(rest, a, b[set][1][0], b[set][1][1], T());
                  pa_mma_first(y, a, b[set][0][0], b[set][0][1], T());
                } else {
                  if (!TWICE) pa_mma(rest, a, b[set][1][0], b[set][1][1], T());
                  pa_mma(y, a, b[set][0][0], b[set][0][1], T());
                }
              } else {
#pragma unroll
                for (int n = TERMS - 1; n >= 0; --n) {   // small terms first
                  if (set == 0 && n == TERMS - 1)
                    pa_mma_first(y, a, b[set][n][0], b[set][n][1], T());
                  else
                    pa_mma(y, a, b[set][n][0], b[set][n][1], T());
                }
              }
            }
            if constexpr (SPLIT && !TWICE) {
              pa_fma2(acc[mt][0], acc[mt][1], rest[0], rest[1], 1.f / REST);
              pa_fma2(acc[mt][2], acc[mt][3], rest[2], rest[3], 1.f / REST);
            }
            pa_add2(acc[mt][0], acc[mt][1], y[0], y[1]);
            pa_add2(acc[mt][2], acc[mt][3], y[2], y[3]);
          }
        } else {
#pragma unroll
          for (int n = 0; n < EIGHTS; ++n) {
#pragma unroll 1
            for (int token = 0; token < 8; ++token) {
              const float p0 = __shfl_sync(0xffffffffu, x[n][0], token * 4 + t), p1 = __shfl_sync(0xffffffffu, x[n][1], token * 4 + t);
              const uint8_t* values = ring + slot * C::STAGE + CHUNK * ROW + (8 * n + token) * ROW + g * 2;
#pragma unroll
              for (int mt = 0; mt < DP / 16; ++mt)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                  const float v = to_float(*reinterpret_cast<const T*>(values + ((2 * mt + j) ^ token) * 16));
                  acc[mt][2 * j] = fmaf(p0, v, acc[mt][2 * j]);
                  acc[mt][2 * j + 1] = fmaf(p1, v, acc[mt][2 * j + 1]);
                }
            }
          }
        }
      } else {
#pragma unroll
        for (int n = 0; n < EIGHTS; ++n) {
          if (2 * t < NH) s_p[warp][8 * n + g][2 * t] = x[n][0];
          if (2 * t + 1 < NH) s_p[warp][8 * n + g][2 * t + 1] = x[n][1];
        }
        __syncwarp();
#pragma unroll
        for (int token = 0; token < CHUNK; ++token) {
          const uint8_t* values = ring + slot * C::STAGE + CHUNK * ROW + token * ROW;
          float v[COLUMNS];
          if constexpr (COLUMNS == 2) {
            *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(values + (((lane / 2) ^ ((token & 1) << 2)) * 16) + (lane % 2) * 8);
          } else {
#pragma unroll
            for (int j = 0; j < COLUMNS / 4; ++j)
              *reinterpret_cast<float4*>(v + 4 * j) = *reinterpret_cast<const float4*>(values + (((lane + 32 * j) ^ ((token & 1) << 2)) * 16));
          }
#pragma unroll
          for (int h = 0; h < NH; ++h) {
            const float pr = s_p[warp][token][h];
#pragma unroll
            for (int j = 0; j < COLUMNS; ++j) acc[h][j] = fmaf(pr, v[j], acc[h][j]);
          }
        }
        __syncwarp();
      }
    }

    // -- the end of an item, or of this block's part of it ----------------------------------------
    const bool to_end = now.tile + 1 == now.tiles;
    if (to_end || now.left == 1) {
      // the teams' parts meet in shared memory: maxima and sums by warp, numerators in the stage that was just read (its
      // refill is a step away). Columns are swizzled by the head so that neither side meets bank conflicts
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int o = 4; o < 32; o *= 2) total_p[i] += __shfl_xor_sync(0xffffffffu, total_p[i], o);
        if (g == 0) {
          s_max[warp][2 * t + i] = again ? top[i] + FEWER : top[i];   // a part is relative to 2^(this - BIAS)
          s_sum[warp][2 * t + i] = again ? total_p[i] * FEW : total_p[i];
        }
      }
      team_barrier();   // every member has read the stage
      float* numerators = reinterpret_cast<float*>(ring + slot * C::STAGE) + member * 8 * DP;
      if constexpr (C::HALF) {
#pragma unroll
        for (int mt = 0; mt < DP / 16; ++mt)
#pragma unroll
          for (int j = 0; j < 4; ++j) numerators[(2 * t + j % 2) * DP + ((mt * 16 + g + 8 * (j / 2)) ^ (t << 3))] = acc[mt][j];
      } else {
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
          for (int j = 0; j < COLUMNS; ++j) {
            const int d = COLUMNS == 2 ? 2 * lane + j : (j / 4) * 128 + 4 * lane + j % 4;
            numerators[h * DP + (d ^ ((h / 2) << 3))] = acc[h][j];
          }
      }
      {
        // Everybody's part is there behind this barrier. Where a numerator is not finite the block goes over its tiles of the item
        // once more. 16-bit storage takes whole probabilities then: an infinite value times one term of a probability, negative
        // or zero, is not what it is times the probability. And where values can be so large that their sum, but not their mean,
        // passes FP32 (bf16 and FP32), the probabilities are 2^-23 at most: 2^23 tokens of the largest value can be added.
        float probe = 0.f;
        if (!again) {
#pragma unroll
          for (int i = 0; i < A; ++i)
#pragma unroll
            for (int j = 0; j < B; ++j) probe = fmaf(acc[i][j], 0.f, probe);
        }
        if (__syncthreads_or(probe != 0.f)) {
          pa_wait<0>();
          __syncthreads();   // no stage is read or written any more
          now.left += now.tile - start;
          now.tile = start;
          ahead = now;
          look_up();
          if constexpr (C::HALF && DP == 64) load_query(query_next, now.sequence, now.kv_head, now.block);
          again = fresh = true;
          if (!SPLIT) growth = 0.f;
          slot = 0;
          filling = STAGES - 1;
          continue;
        }
        again = false;
        growth = GROWTH;
      }
      const bool whole = start == 0 && to_end;
      float* part = p.parts + ((int64_t)blockIdx.x * 2 + (start == 0 ? 1 : 0)) * C::PART;
      auto write = [&](int h, int d, float4 y) {   // h within the group, d a multiple of four
        const int64_t to = now.sequence * p.out_token_stride + ((int64_t)now.kv_head * p.group + h) * p.out_head_stride + d;
        if (p.out_f32) {
          float* out = static_cast<float*>(p.out) + to;
          if (p.out_quads)
            *reinterpret_cast<float4*>(out) = y;
          else
            out[0] = y.x, out[1] = y.y, out[2] = y.z, out[3] = y.w;
        } else {
          T* out = static_cast<T*>(p.out) + to;
          alignas(8) const T rounded[4] = {from_float<T>(y.x), from_float<T>(y.y), from_float<T>(y.z), from_float<T>(y.w)};
          if (p.out_quads && C::HALF)
            *reinterpret_cast<uint2*>(out) = *reinterpret_cast<const uint2*>(rounded);
          else
            out[0] = rounded[0], out[1] = rounded[1], out[2] = rounded[2], out[3] = rounded[3];
        }
      };
#pragma unroll 1
      for (int i = tid; i < C::HEADS * DP / 4; i += THREADS) {
        const int slot_head = i / (DP / 4), d = i % (DP / 4) * 4, h = head_of(now.block, slot_head);
        if (h >= p.group || d >= p.dim) continue;
        float high = NONE;
#pragma unroll
        for (int m = 0; m < TEAMS; ++m) high = fmaxf(high, s_max[m * HB + slot_head / 8][slot_head % 8]);
        const float around = high == NONE ? 0.f : high;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
        float weight_sum = 0.f;
#pragma unroll
        for (int m = 0; m < TEAMS; ++m) {
          const int w = m * HB + slot_head / 8;
          const float weight = ex2_approx_ftz(s_max[w][slot_head % 8] - around) * (1.f / TEAMS);   // finite parts have a finite sum
          const float* from = reinterpret_cast<const float*>(smem + (m * STAGES + slot) * C::STAGE);
          const float4 x = *reinterpret_cast<const float4*>(from + slot_head * DP + (d ^ (((slot_head % 8) / 2) << 3)));
          y.x = fmaf(weight, x.x, y.x), y.y = fmaf(weight, x.y, y.y), y.z = fmaf(weight, x.z, y.z), y.w = fmaf(weight, x.w, y.w);
          weight_sum = fmaf(weight, s_sum[w][slot_head % 8], weight_sum);
        }
        if (whole) {
          const float share = 1.f / weight_sum;
          write(h, d, make_float4(y.x * share, y.y * share, y.z * share, y.w * share));
        } else {
          __stcg(reinterpret_cast<float4*>(part + slot_head * DP + d), y);
          if (d == 0) __stcg(reinterpret_cast<float2*>(part + C::HEADS * DP + 2 * slot_head), make_float2(high, weight_sum));
        }
      }
      if (!whole) {
        const int64_t item = s_plan[2] - now.left - now.tile;   // the item's first unit
        const int64_t first = pa_share_owner(s_plan[0], s_plan[1], item), last = pa_share_owner(s_plan[0], s_plan[1], item + now.tiles - 1);
        __syncthreads();
        if (tid == 0) s_last = pa_arrive(p.counters + first) == (int)(last - first);
        __syncthreads();
        if (s_last) {
          if (tid == 0) p.counters[first] = 0;
          // The parts, added in the order of the blocks: the first block's second part, then every other's first, which lie at
          // one distance; PA_JOIN of them requested at once.
          const int count = (int)(last - first);
          constexpr float SHARED = 1.f / PA_MAX_BLOCKS;   // finite parts have a finite sum
          const float* parts = p.parts + (first * 2 + 1) * C::PART;
#pragma unroll 1
          for (int i = tid; i < C::HEADS * DP / 4; i += THREADS) {
            const int slot_head = i / (DP / 4), d = i % (DP / 4) * 4, h = head_of(now.block, slot_head);
            if (h >= p.group || d >= p.dim) continue;
            const float* number = parts + slot_head * DP + d;
            const float* state = parts + C::HEADS * DP + 2 * slot_head;   // maximum and sum
            float4 y = __ldcg(reinterpret_cast<const float4*>(number));
            const float2 started = __ldcg(reinterpret_cast<const float2*>(state));
            float high = started.x, sum_p = started.y * SHARED;
            y.x *= SHARED, y.y *= SHARED, y.z *= SHARED, y.w *= SHARED;
            number += C::PART, state += C::PART;
#pragma unroll 1
            for (int n = 0; n < count; n += PA_JOIN, number += 2 * PA_JOIN * C::PART, state += 2 * PA_JOIN * C::PART) {
              float4 x[PA_JOIN];
              float2 part[PA_JOIN];
              float up = high;
#pragma unroll
              for (int j = 0; j < PA_JOIN; ++j) {
                part[j] = make_float2(NONE, 0.f);
                x[j] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (n + j < count) {
                  part[j] = __ldcg(reinterpret_cast<const float2*>(state + 2 * j * C::PART));
                  x[j] = __ldcg(reinterpret_cast<const float4*>(number + 2 * j * C::PART));
                }
              }
#pragma unroll
              for (int j = 0; j < PA_JOIN; ++j) up = fmaxf(up, part[j].x);
              const float around = up == NONE ? 0.f : up, before_weight = ex2_approx_ftz(high - around);
              high = up;
              y.x *= before_weight, y.y *= before_weight, y.z *= before_weight, y.w *= before_weight, sum_p *= before_weight;
#pragma unroll
              for (int j = 0; j < PA_JOIN; ++j) {
                const float weight = ex2_approx_ftz(part[j].x - around) * SHARED;
                y.x = fmaf(weight, x[j].x, y.x), y.y = fmaf(weight, x[j].y, y.y), y.z = fmaf(weight, x[j].z, y.z), y.w = fmaf(weight, x[j].w, y.w);
                sum_p = fmaf(weight, part[j].y, sum_p);
              }
            }
            const float share = 1.f / sum_p;
            write(h, d, make_float4(y.x * share, y.y * share, y.z * share, y.w * share));
          }
        }
      }
      __syncthreads();   // the stage and the maxima are free again
      fresh = true;
    }
    now.step(p);
    slot = slot + 1 == STAGES ? 0 : slot + 1;
  }
}


static size_t pa_workspace_bytes() {
  // two parts per block of the form with the most: 32 heads of 128, three blocks per SM
  using Most = PaConfig<__half, 128, 4, 8>;
  static_assert(Most::BLOCKS_PER_SM * Most::PART >= PaConfig<__half, 256, 4, 8>::PART && Most::BLOCKS_PER_SM >= PaConfig<float, 128, 4, 8>::BLOCKS_PER_SM, "largest");
  return PA_COUNTER_BYTES + (size_t)sm_count() * Most::BLOCKS_PER_SM * 2 * Most::PART * sizeof(float);
}

template <typename T, int DP, int HB, int NH>
static int paged_attention_launch_t(PagedAttentionParams& p, cudaStream_t s) {
  using C = PaConfig<T, DP, HB, NH>;
  static thread_local int attr_dev = -1;
  int dev = 0;
  DTN_CUDA_CHECK(cudaGetDevice(&dev));
  if (attr_dev != dev) {
    DTN_CUDA_CHECK(cudaFuncSetAttribute(paged_attention_kernel<T, DP, HB, NH>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    attr_dev = dev;
  }
  p.blocks = (p.group + C::HEADS - 1) / C::HEADS;
  p.heads = p.kv_heads * p.blocks;
  p.whole_sets = p.page_size % C::SUB == 0;
  // Two blocks per SM are enough to read, and where few items are shared by many blocks the fewer parts to join count more:
  // 8 items of head size 128 in 16 bits 88.6 us against 91.4 with three (131071 tokens each) and 32.7 against 33.7 (32768); 24
  // items 70.1 against 68.9, 32 items 44.9 against 43.8. Other forms, 256 to 65536 tokens: up to 1024 tokens equal; 8 items of
  // 16384 tokens, in us against three blocks: f16 128 21.5 / 23.3, 64 15.1 / 16.0, groups of 16 32.2 / 35.9, of 32 49.9 / 56.7,
  // FP32 64 21.5 / 22.3, 128 35.6 / 37.6; of 65536 within 2 % (f16 64 in groups of 16: 41.1 / 39.1). 16 items go either way: f16
  // 128 14.1 / 14.7 at 4096 tokens and 89.7 / 87.3 at 65536, f16 64 53.2 / 51.4 and FP32 128 in groups of 8 228 / 212 there.
  const int64_t per_sm = C::BLOCKS_PER_SM > 2 && p.count <= 16 && p.count * p.heads <= 16 ? 2 : C::BLOCKS_PER_SM;
  int64_t grid = (int64_t)sm_count() * per_sm;
  if (grid > PA_MAX_BLOCKS) grid = PA_MAX_BLOCKS;
  const int64_t unit = C::CHUNK * C::TEAMS, most_tiles = p.capacity > unit ? (p.capacity + unit - 1) / unit : 1;
  DTN_REQUIRE((double)p.count * p.heads * (double)(most_tiles + PA_ITEM_UNITS) < 2147483648.0 * (double)grid, DTN_ERR_UNSUPPORTED,
              "paged attention: the tables cover too many tokens for one launch");
  if (p.count < grid && p.heads < grid && most_tiles < grid && p.count * p.heads * most_tiles < grid) grid = p.count * p.heads * most_tiles;
  paged_attention_kernel<T, DP, HB, NH><<<(unsigned)grid, PA_WARPS * 32, C::SMEM, s>>>(p);
  DTN_LAUNCH_CHECK("paged_attention_kernel");
  return DTN_OK;
}

template <typename T, int DP>
static int paged_attention_launch_d(PagedAttentionParams& p, cudaStream_t s) {
  // FP32 multiply-adds are paid per head: a form for a head or four of the eight that the products of 16-bit storage have anyway
  if constexpr (sizeof(T) == 4) {
    if (p.group == 1) return paged_attention_launch_t<T, DP, 1, 1>(p, s);
    if (p.group <= 4) return paged_attention_launch_t<T, DP, 1, 4>(p, s);
  }
  if (p.group <= 8) return paged_attention_launch_t<T, DP, 1, 8>(p, s);
  if (p.group <= 16) return paged_attention_launch_t<T, DP, 2, 8>(p, s);
  return paged_attention_launch_t<T, DP, 4, 8>(p, s);
}

template <typename T>
static int paged_attention_launch(PagedAttentionParams& p, cudaStream_t s) {
  if (p.dim <= 64) return paged_attention_launch_d<T, 64>(p, s);
  if (p.dim <= 128) return paged_attention_launch_d<T, 128>(p, s);
  return paged_attention_launch_d<T, 256>(p, s);
}

}  // namespace dtn

extern "C" {

int dtn_paged_attention_workspace_bytes(size_t* bytes_out) {
  DTN_REQUIRE(bytes_out != nullptr, DTN_ERR_INVALID, "paged attention: bytes_out is null");
  *bytes_out = dtn::pa_workspace_bytes();
  return DTN_OK;
}

int dtn_paged_attention_plan(const int64_t* tiles, int64_t count, int64_t heads, int64_t min_units, int64_t grid, int64_t* begin_out,
                             int64_t* first_out, int64_t* last_out, int64_t* workers_out) {
  using namespace dtn;
  DTN_REQUIRE(tiles && count > 0 && heads > 0 && min_units > 0 && grid > 0, DTN_ERR_INVALID, "paged attention plan: bad extent");
  int64_t units = 0;
  for (int64_t i = 0; i < count; ++i) {
    DTN_REQUIRE(tiles[i] >= 0, DTN_ERR_INVALID, "paged attention plan: negative tiles");
    units += tiles[i] > 0 ? (tiles[i] + PA_ITEM_UNITS) * heads : 0;
  }
  const int64_t workers = units > 0 ? pa_workers(units, min_units, grid) : 0;
  if (workers_out) *workers_out = workers;
  if (begin_out)
    for (int64_t c = 0; c <= workers; ++c) begin_out[c] = workers > 0 ? pa_share_begin(units, workers, c) : 0;
  int64_t at = 0;
  for (int64_t i = 0; i < count * heads; ++i) {
    const int64_t here = tiles[i / heads];
    if (first_out) first_out[i] = here > 0 ? pa_share_owner(units, workers, at) : -1;
    if (last_out) last_out[i] = here > 0 ? pa_share_owner(units, workers, at + here - 1) : -1;
    at += here > 0 ? here + PA_ITEM_UNITS : 0;
  }
  return DTN_OK;
}

int dtn_paged_attention_pages(const int* positions, int64_t count, int64_t page_size, int* pages_out) {
  using namespace dtn;
  DTN_REQUIRE(count >= 0 && (count == 0 || (positions && pages_out)), DTN_ERR_INVALID, "paged attention pages: null pointer or negative count");
  DTN_REQUIRE(page_size >= 1 && page_size < (1LL << 31), DTN_ERR_INVALID, "paged attention pages: page size %lld", (long long)page_size);
  const PaDivider pages_of = pa_divider(page_size);
  for (int64_t i = 0; i < count; ++i) {
    DTN_REQUIRE(positions[i] >= 0, DTN_ERR_INVALID, "paged attention pages: negative position");
    pages_out[i] = pages_of(positions[i]);
  }
  return DTN_OK;
}

int dtn_paged_attention(const dtn_paged_attention_args* args, void* stream) {
  using namespace dtn;
  DTN_REQUIRE(args != nullptr, DTN_ERR_INVALID, "paged attention: no arguments");
  const dtn_paged_attention_args& a = *args;
  DTN_REQUIRE(a.count >= 0 && a.q_heads >= 0 && a.kv_heads >= 0 && a.dim >= 0 && a.pages >= 0 && a.sequences >= 0 && a.pages_per_sequence >= 0 && a.window >= 0,
              DTN_ERR_INVALID, "paged attention: negative extent");
  DTN_REQUIRE(a.page_size >= 1 && a.page_size < (1LL << 31), DTN_ERR_INVALID, "paged attention: page size %lld", (long long)a.page_size);
  DTN_REQUIRE(paged_storage_known(a.storage), DTN_ERR_INVALID, "paged attention: unknown storage %lld", (long long)a.storage);
  if (a.count == 0 || a.q_heads == 0 || a.dim == 0) return DTN_OK;
  DTN_REQUIRE(a.kv_heads > 0 && a.q_heads % a.kv_heads == 0, DTN_ERR_INVALID, "paged attention: query heads must be a multiple of kv heads");
  DTN_REQUIRE(a.dim <= 256, DTN_ERR_UNSUPPORTED, "paged attention: heads of at most 256 elements");
  const int64_t element = paged_storage_bytes(a.storage);
  DTN_REQUIRE(a.dim * element % 16 == 0 && a.page_stride * element % 16 == 0 && a.page_head_stride * element % 16 == 0 && aligned_to(a.k_pages, 16) &&
                  aligned_to(a.v_pages, 16),
              DTN_ERR_INVALID, "paged attention: the heads of the pools must start on 16-byte boundaries and have a multiple of 16 bytes");
  DTN_REQUIRE(a.q && a.out && (a.lengths || a.sequences == 0) && (a.rows || a.count <= a.sequences), DTN_ERR_INVALID, "paged attention: null pointer");
  DTN_REQUIRE((a.k_pages && a.v_pages) || a.pages == 0, DTN_ERR_INVALID, "paged attention: null pool");
  DTN_REQUIRE(a.sequences == 0 || a.tables || a.pages_per_sequence == 0, DTN_ERR_INVALID, "paged attention: null tables");
  DTN_REQUIRE(a.pages < (1LL << 31) && a.count < (1LL << 31) && a.q_heads < (1LL << 20) && a.pages_per_sequence < (1LL << 31), DTN_ERR_UNSUPPORTED,
              "paged attention: too many rows or pages for one launch");
  DTN_REQUIRE(a.workspace && a.workspace_bytes >= (int64_t)pa_workspace_bytes(), DTN_ERR_WORKSPACE,
              "paged attention: %lld bytes of workspace, %zu needed", (long long)a.workspace_bytes, pa_workspace_bytes());
  DTN_REQUIRE(aligned_to(a.workspace, 16), DTN_ERR_WORKSPACE, "paged attention: the workspace must be 16-byte aligned");
  cudaStream_t s = as_stream(stream);
  const int64_t capacity = a.pages_per_sequence * a.page_size, most = (1LL << 31) - (1 << 16);
  PagedAttentionParams p = {};
  p.q = a.q;
  // an empty pool is never read, but copies of no bytes name an aligned address
  const void* nothing = reinterpret_cast<const void*>(reinterpret_cast<uintptr_t>(a.q) & ~(uintptr_t)15);
  p.k_pages = a.pages ? a.k_pages : nothing;
  p.v_pages = a.pages ? a.v_pages : nothing;
  p.out = a.out;
  p.tables = a.tables;
  p.lengths = a.lengths;
  p.rows = a.rows;
  p.count = a.count;
  p.sequences = a.sequences;
  p.pages = a.pages;
  p.table_stride = a.table_stride;
  p.capacity = (int)(capacity < most ? capacity : most);
  p.q_token_stride = a.q_token_stride;
  p.q_head_stride = a.q_head_stride;
  p.out_token_stride = a.out_token_stride;
  p.out_head_stride = a.out_head_stride;
  p.page_stride = a.page_stride * element;
  p.page_head_stride = a.page_head_stride * element;
  p.kv_heads = (int)a.kv_heads;
  p.q_heads = (int)a.q_heads;
  p.group = (int)(a.q_heads / a.kv_heads);
  p.dim = (int)a.dim;
  p.page_size = (int)a.page_size;
  p.row_bytes = (int)(a.dim * element);
  p.window = a.window;
  p.scale_log2e = (float)(a.scale * 1.4426950408889634);
  p.out_f32 = a.out_f32 != 0;
  p.q_pairs = element == 2 && aligned_to(a.q, 4) && a.q_token_stride % 2 == 0 && a.q_head_stride % 2 == 0;
  const int64_t out_element = a.out_f32 ? 4 : element;
  p.out_quads = aligned_to(a.out, 4 * out_element) && a.out_token_stride % 4 == 0 && a.out_head_stride % 4 == 0;
  p.min_units = 1 + PA_ITEM_UNITS;
  p.pages_of = pa_divider(a.page_size);
  p.counters = static_cast<int*>(a.workspace);
  p.parts = reinterpret_cast<float*>(static_cast<char*>(a.workspace) + PA_COUNTER_BYTES);
  p.status = device_status_word_unless_capturing(s);
  if (a.storage == DTN_STORAGE_F32) return paged_attention_launch<float>(p, s);
  if (a.storage == DTN_STORAGE_F16) return paged_attention_launch<__half>(p, s);
  return paged_attention_launch<__nv_bfloat16>(p, s);
}

}  // extern "C"
