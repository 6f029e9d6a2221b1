// Attention of a drafted step (a tree or a chain of new tokens for each sequence) over the pages of a cache
// (tmh_paged_tree_attention).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "tmh_attend.h"
#include "tmh_internal.h"
#include "tmh_launch.h"
#include "tmh_tree_plan.h"

namespace tmh {
namespace {

struct TreeArgs {
  const void* q;
  const void* k;
  const void* v;
  const int32_t* table;
  const int32_t* lengths;
  const int32_t* starts;
  const uint64_t* mask;  // nullptr: chains
  void* y;
  float* part;    // [2 workers][columns of a tile][head_dim], then their (maximum, sum) pairs
  float2* stats;
  uint32_t part_bytes, stats_bytes;
  uint32_t* meet;  // [workers] parts of the item that begins in a worker, kept so far; zero between calls
  int64_t ldq, ldy, max_pages, rows, most;  // most: max_pages * page_size
  PageShape cache;
  int64_t head_stride;
  int window, words, B, group, kv_heads, head_dim;
  uint32_t workers;
  FastDiv by_group;
  float scale;  // of the scores in base-2 logarithms: scale * log2(e)
  float unit;   // base-2 logarithms to one of the parts' maxima: 1, or, of tiles that keep maxima as the products have them, |scale|
};

template <int UT, int M>
__device__ __forceinline__ Draft draft_at(const TreeArgs& p, int b) {
  return draft_of(p.starts[b], p.starts[b + 1], p.rows, p.lengths[b], p.most, p.window, UT, p.group, M);
}
template <int UT, int M>
__device__ __forceinline__ uint32_t work_at(const TreeArgs& p, int b) {
  return work_of(draft_at<UT, M>(p, b));
}

// All work of one kv head, by one wavefront.
template <int UT, int M>
__device__ __forceinline__ uint32_t all_work(const TreeArgs& p) {
  uint32_t n = 0;
  for (int i = threadIdx.x & 63; i < p.B; i += 64) n += work_at<UT, M>(p, i);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) n += __shfl_xor(n, o);
  return __builtin_amdgcn_readfirstlane(n);  // (known to be the same in all lanes, as what follows from it then is)
}

// The sequence whose work holds `target`, and the work before it.
template <int UT, int M>
__device__ __forceinline__ int find_draft(const TreeArgs& p, uint32_t target, uint32_t& before) {
  const int lane = threadIdx.x & 63;
  uint32_t base = 0;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    const uint32_t mine = b0 + lane < p.B ? work_at<UT, M>(p, b0 + lane) : 0;
    const uint32_t sum = scan64(mine);
    const uint64_t past = __ballot(base + sum > target);
    if (past) {
      const int at = __builtin_ctzll(past);
      before = base + __builtin_amdgcn_readlane(sum - mine, at);
      return b0 + at;
    }
    base += __builtin_amdgcn_readlane(sum, 63);
  }
  before = base;
  return p.B;  // (target is not below the total)
}

// Where `at` lies in a sequence whose work begins at `before`: the item (one kv head and tile of columns) and where it begins.
struct Place {
  uint32_t item, first;
};
__device__ __forceinline__ Place place_in(const Draft& d, uint32_t before, uint32_t at) {
  const uint32_t each = static_cast<uint32_t>(d.units) + kItem, item = (at - before) / each;
  return {item, before + item * each};
}

// Parts of items that several workers shared. Each worker leaves its part in memory (stores that pass the XCD's own L2), then counts
// itself; the one that finds all others counted joins the parts, in their order, whoever it is. Items of more than MOST parts, which
// would keep one workgroup too long, are left to a second kernel (join_most: half a MiB of parts of 128 dimensions). In us so, all by the second
// kernel, and all in the kernel: 32 x 4 over 4000 bf16 62, 65, 62; 8 x 32 42, 51, 59; 2 x 100 over 20000 f16 68, 76, 96. Narrow tiles of 256
// dimensions keep that number of parts, of a MiB then: 1 x 2 over 6000, 8 heads of one kv head, f16 33.0, with half as many 36.5; 4 x 4 over 8000, 16 of
// 4, bf16 52.9 and 56.2.
constexpr int kThrough = 16;                // sc1 of a buffer access: past the XCD's L2, to where all XCDs meet
constexpr uint32_t kNowhere = 0xFFFFFFF0u;  // an offset past every buffer's range here
constexpr uint32_t join_most(int columns, int blocks) { return 1024u / (columns * blocks); }

__device__ __forceinline__ void put_part(const TreeArgs& p, uint32_t quad, float4_t v) {
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(uint4_t, v), buffer_rsrc(p.part, p.part_bytes), quad * 16, 0, kThrough);
}
__device__ __forceinline__ void put_stats(const TreeArgs& p, uint32_t at, float top, float total) {
  __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(uint2_t, make_float2(top, total)), buffer_rsrc(p.stats, p.stats_bytes), at * 8, 0, kThrough);
}
__device__ __forceinline__ void put_value(const TreeArgs& p, uint32_t at, float v) {  // (of a part, counted in values)
  __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, v), buffer_rsrc(p.part, p.part_bytes), at * 4, 0, kThrough);
}
template <int AUX>
__device__ __forceinline__ float4_t get_part(const TreeArgs& p, uint32_t quad, bool there) {
  return __builtin_bit_cast(float4_t, __builtin_amdgcn_raw_buffer_load_b128(buffer_rsrc(p.part, p.part_bytes), there ? quad * 16 : kNowhere, 0, AUX));
}
template <int AUX>
__device__ __forceinline__ float2 get_stats(const TreeArgs& p, uint32_t at, bool there) {
  return __builtin_bit_cast(float2, __builtin_amdgcn_raw_buffer_load_b64(buffer_rsrc(p.stats, p.stats_bytes), there ? at * 8 : kNowhere, 0, AUX));
}

// Whether this worker is the last of an item's to have left its part. (As k_paged_attention counts: this thread's stores have arrived,
// then everybody's, then the count.)
__device__ __forceinline__ bool last_of(const TreeArgs& p, const TreeParts& parts) {
  __shared__ uint32_t others;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    others = __hip_atomic_fetch_add(p.meet + parts.from, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (others == parts.count - 1) __hip_atomic_store(p.meet + parts.from, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  return others == parts.count - 1;
}

// The sum of parts k = first, first + step, ..: QUADS quads of a lane each, at quads quad_at(place of the part, i), with the statistics
// at stats_at(place of the part); four parts on their way at once. AUX: kThrough where other
// workgroups of the same kernel have written them.
template <int AUX, int QUADS, typename QuadAt, typename StatsAt>
__device__ __forceinline__ void join_parts(const TreeArgs& p, const TreeParts& parts, uint32_t first, uint32_t step, float4_t (&acc)[QUADS], float& top,
                                           float& total, QuadAt quad_at, StatsAt stats_at) {
  constexpr int BATCH = 4;
  top = kNone;
  total = 0.f;
#pragma unroll
  for (int i = 0; i < QUADS; ++i) acc[i] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
  for (uint32_t k0 = first; k0 < parts.count; k0 += BATCH * step) {
    float2 st[BATCH];
    float4_t o[BATCH][QUADS];
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {  // (what a batch has too many lies past the buffers' ranges: zeros)
      const uint32_t k = k0 + b * step, place = place_of_part(parts.from + k, k == 0);
      const bool there = k < parts.count;
      st[b] = get_stats<AUX>(p, stats_at(place), there);
#pragma unroll
      for (int i = 0; i < QUADS; ++i) o[b][i] = get_part<AUX>(p, quad_at(place, i), there);
    }
    float next = top;
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      if (k0 + b * step >= parts.count) st[b].x = kNone;
      next = fmaxf(next, st[b].x);
    }
    const float keep = top == next ? 1.f : __builtin_amdgcn_exp2f((top - next) * p.unit);
    top = next;
    total *= keep;
#pragma unroll
    for (int i = 0; i < QUADS; ++i) acc[i] *= keep;
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      const float f = st[b].x == top ? 1.f : __builtin_amdgcn_exp2f((st[b].x - top) * p.unit);
      total += f * st[b].y;
#pragma unroll
      for (int i = 0; i < QUADS; ++i) acc[i] += f * o[b][i];
    }
  }
}

// The item of more than MOST parts, if there is one, whose first part is one of the workers MOST index .. MOST index + MOST - 1's: it
// is what the next such run of workers begins with.
struct Joined {
  Draft d;
  TreeParts parts;
  int kv_head, tile;
};
template <int UT, int M, uint32_t MOST>
__device__ __forceinline__ bool find_joined(const TreeArgs& p, uint32_t index, Joined& j) {
  const uint32_t all = all_work<UT, M>(p) * p.kv_heads, per = units_per_worker(all, p.workers);
  const uint32_t cut = MOST * (index + 1) * per;
  if (per == 0 || cut >= all) return false;
  uint32_t before;
  const int b = find_draft<UT, M>(p, cut / p.kv_heads, before);
  if (b >= p.B) return false;
  j.d = draft_at<UT, M>(p, b);
  const Place place = place_in(j.d, before * p.kv_heads, cut);
  if (place.item >= static_cast<uint32_t>(j.d.tiles * p.kv_heads)) return false;
  j.parts = tree_parts(place.first, static_cast<uint32_t>(j.d.units), per);
  j.kv_head = static_cast<int>(place.item) / j.d.tiles;
  j.tile = static_cast<int>(place.item) % j.d.tiles;
  return j.parts.count > MOST && j.parts.from / MOST == index && j.parts.from + j.parts.count <= p.workers;
}

template <int DT>
__device__ __forceinline__ void store_answer(const TreeArgs& p, int64_t row, int head, int dim, float4_t o) {
  const int64_t out = row * p.ldy + static_cast<int64_t>(head) * p.head_dim + dim;
  if constexpr (DT == DT_F32)
    *reinterpret_cast<float4_t*>(static_cast<float*>(p.y) + out) = o;
  else
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.y) + out) = make_uint2(pack2<DT>(o[0], o[1]), pack2<DT>(o[2], o[3]));
}

// Two probabilities as the sums of two 16-bit parts each, the first cut off, the second rounded (f16: cut off, at 2^-21 of the
// probability). Unlike split2's, the second part may be 0 beside a first that is not, and an infinity in V becomes a NaN.
template <int DT>
__device__ __forceinline__ uint2 cut2(float a, float b) {
  if constexpr (DT == DT_F16) {
    const auto h = __builtin_amdgcn_cvt_pkrtz(a, b);
    const auto r = __builtin_amdgcn_cvt_pkrtz(a - static_cast<float>(h[0]), b - static_cast<float>(h[1]));
    return make_uint2(__builtin_bit_cast(uint32_t, h), __builtin_bit_cast(uint32_t, r));
  } else {
    const uint32_t hi = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, a), 0x07060302u);
    return make_uint2(hi, pack2<DT>(a - __builtin_bit_cast(float, hi << 16), b - __builtin_bit_cast(float, hi & 0xFFFF0000u)));
  }
}

// An infinity or a NaN in V leaves a NaN in every column of its products that does not see it (0 times an infinity), and an infinity may in
// one that sees it with little weight, of which a 16-bit part is 0. Such columns are done again, by each_alone: those whose sums have a NaN
// while the sum of their weights, in which V has no part, has none. (Where it has one, as for a NaN in the query, the answer is NaN
// whatever V holds.) mark: the bits `first` and up of `words`, in LDS, for the GROUP columns of a wavefront in which a lane says so.
template <int GROUP>
__device__ __forceinline__ void mark(uint32_t* words, int first, bool flag) {
  uint64_t b = __ballot(flag);
#pragma unroll
  for (int o = 32; o >= GROUP; o /= 2) b |= b >> o;
  const uint32_t some = static_cast<uint32_t>(b & ((uint64_t{1} << GROUP) - 1));
  if (some && (threadIdx.x & 63) == 0) atomicOr(&words[first / 32], some << (first % 32));
}

// The marked columns of an item's [first, first + columns) over its tokens [from, to), in f32, of the tokens that each sees alone, eight columns
// at a time: a thread takes a token for their scores, then a dimension for their sums. put(column of these, dimension, sum,
// weights' sum) and total(column of these, maximum, weights' sum) take the answers; the maxima are of products times `scale`, each worth
// p.unit base-2 logarithms. Weights are multiplied by `factor`, as the other columns' are. It is slow (4 x 512 over 4096 bf16 with one NaN in
// each kv head's V of one sequence 9.6 ms, 0.16 without): for columns that need it only. `room`: kAloneRoom(THREADS, head_dim) bytes of LDS;
// `marked` lies in LDS too.
constexpr int kAlone = 8;
constexpr int kAloneRoom(int threads, int dim) { return threads * (12 + 4 * kAlone) + (dim + threads / 64 + 3) * 4 * kAlone; }
template <int DT, int THREADS, typename Put, typename Total>
__device__ __forceinline__ void each_alone(const Draft& d, const int32_t* table, int kv_head, int first, int columns, int from,
                                           int to, float scale, float factor, const uint32_t* marked, void* room, Put put, Total total) {
  constexpr int EACH = 256 / THREADS > 0 ? 256 / THREADS : 1;  // dimensions a thread may have
  constexpr int BATCH = 8;                                      // loads of V on their way at once
  // The kernel's arguments (its only one is a TreeArgs) once more, and the thread, as nothing that the compiler knows: what follows from
  // them it would compute ahead of all work and keep in registers (3 x 13 over 1000 f32 13.3 us, so 11.8).
  const auto* args = (const __attribute__((address_space(4))) void*)__builtin_amdgcn_kernarg_segment_ptr();
  int tid = threadIdx.x;
  asm volatile("" : "+s"(args), "+v"(tid));
  TreeArgs p;
  __builtin_memcpy(&p, (const void*)args, sizeof(p));
  const int dim = p.head_dim, wave = tid >> 6;
  int64_t* rows = static_cast<int64_t*>(room);  // of a turn's tokens, negative where there is none
  auto weights = reinterpret_cast<float(*)[kAlone]>(rows + THREADS);
  float* q = &weights[THREADS][0];  // [dim][kAlone]
  auto meet = reinterpret_cast<float(*)[kAlone]>(q + dim * kAlone);                           // [THREADS / 64]
  uint32_t* seen = reinterpret_cast<uint32_t*>(&meet[THREADS / 64][0]);  // by which of the columns, of a turn's tokens
  // The columns (-1: none), their nodes, and the first token that the window leaves them.
  int *column = reinterpret_cast<int*>(seen + THREADS), *node = column + kAlone, *begin = node + kAlone;
  const int64_t head_at = static_cast<int64_t>(kv_head) * p.head_stride;
  int next_column = 0;
#pragma unroll 1
  while (true) {
    if (tid < kAlone) {
      int c = next_column;
      for (int left = tid; c < columns; ++c)
        if ((marked[c / 32] >> (c % 32) & 1u) && left-- == 0) break;
      const int n = static_cast<int>(p.by_group.div(static_cast<uint32_t>(first + min(c, columns - 1))));
      column[tid] = c < columns ? c : -1;
      node[tid] = n;
      begin[tid] = 0;
      if (p.window > 0) {
        if (p.mask) begin[tid] = tree_begin(p.mask + static_cast<int64_t>(d.row + n) * p.words, p.words, d.prefix, d.nodes, p.window);
        else begin[tid] = chain_begin(n, d.prefix, p.window);
      }
    }
    __syncthreads();
    if (column[0] < 0) break;
    next_column = column[kAlone - 1] < 0 ? columns : column[kAlone - 1] + 1;
    for (int i = tid; i < dim * kAlone; i += THREADS) {
      const int k = i % kAlone;
      const int head = kv_head * p.group + first + max(column[k], 0) - node[k] * p.group;
      q[i] = column[k] < 0 ? 0.f : load_as_f32<DT>(p.q, (d.row + node[k]) * p.ldq + static_cast<int64_t>(head) * dim + i / kAlone);
    }
    float top[kAlone], sum[kAlone], o[kAlone][EACH];  // sum: of this thread's tokens, o: dimensions tid + x THREADS
#pragma unroll
    for (int k = 0; k < kAlone; ++k) {
      top[k] = kNone;
      sum[k] = 0.f;
#pragma unroll
      for (int x = 0; x < EACH; ++x) o[k][x] = 0.f;
    }
    __syncthreads();
#pragma unroll 1
    for (int t0 = from; t0 < to; t0 += THREADS) {
      const int token = t0 + tid, some = min(THREADS, to - t0);
      const int64_t row = token < to ? token_offset(p.cache, table, static_cast<uint32_t>(token)) : -1;
      float t[kAlone] = {};
      if (row >= 0) {
#pragma unroll 2
        for (int i = 0; i < dim; i += 8) {
          float y[8];
          load8<DT, true>(p.k, row + head_at + i, 8, y);
#pragma unroll
          for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int k = 0; k < kAlone; ++k) t[k] = fmaf(q[(i + j) * kAlone + k], y[j], t[k]);
        }
      }
      uint32_t by = 0;
#pragma unroll
      for (int k = 0; k < kAlone; ++k) {
        bool sees = column[k] >= 0 && row >= 0 && token >= begin[k];
        if (sees && token >= d.prefix) {
          const uint64_t* mask = p.mask ? p.mask + static_cast<int64_t>(d.row + node[k]) * p.words : nullptr;
          sees = (mask ? tree_bits(mask, p.words, token - d.prefix) : chain_bits(node[k], token - d.prefix)) & 1u;
        }
        by |= sees ? 1u << k : 0u;
        t[k] = sees ? t[k] * scale : kNone;
        float most = t[k];
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) most = fmaxf(most, __shfl_xor(most, x));
        if ((tid & 63) == 0) meet[wave][k] = most;
      }
      __syncthreads();
      rows[tid] = row;
      seen[tid] = by;
#pragma unroll
      for (int k = 0; k < kAlone; ++k) {
        float next = top[k];
#pragma unroll
        for (int w = 0; w < THREADS / 64; ++w) next = fmaxf(next, meet[w][k]);
        const float keep = next == top[k] ? 1.f : __builtin_amdgcn_exp2f((top[k] - next) * p.unit);
        top[k] = next;
        const float w = by >> k & 1u ? __builtin_amdgcn_exp2f((t[k] - (next == kNone ? 0.f : next)) * p.unit) * factor : 0.f;
        weights[tid][k] = w;
        sum[k] = fmaf(sum[k], keep, w);
#pragma unroll
        for (int x = 0; x < EACH; ++x) o[k][x] *= keep;
      }
      __syncthreads();
      if (64 * wave < dim) {
#pragma unroll 1
        for (int i = 0; i < some; i += BATCH) {  // (tokens past `some` are seen by none; the cache's first row is in their place, not used)
          float v[EACH][BATCH];
          bool special = false;
#pragma unroll
          for (int j = 0; j < BATCH; ++j)
#pragma unroll
            for (int x = 0; x < EACH; ++x) {
              v[x][j] = load_as_f32<DT>(p.v, max(rows[i + j], int64_t{0}) + head_at + min(tid + x * THREADS, dim - 1));
              special |= !(fabsf(v[x][j]) < __builtin_inff());
            }
          if (__ballot(special)) {
#pragma unroll
            for (int j = 0; j < BATCH; ++j)
#pragma unroll
              for (int x = 0; x < EACH; ++x) {
                if (fabsf(v[x][j]) < __builtin_inff()) continue;
#pragma unroll
                for (int k = 0; k < kAlone; ++k)
                  if (seen[i + j] >> k & 1u) o[k][x] = fmaf(weights[i + j][k], v[x][j], o[k][x]);
                v[x][j] = 0.f;
              }
          }
#pragma unroll
          for (int j = 0; j < BATCH; ++j)
#pragma unroll
            for (int k = 0; k < kAlone; ++k)
#pragma unroll
              for (int x = 0; x < EACH; ++x) o[k][x] = fmaf(weights[i + j][k], v[x][j], o[k][x]);
        }
      }
      __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < kAlone; ++k) {
#pragma unroll
      for (int x = 1; x < 64; x <<= 1) sum[k] += __shfl_xor(sum[k], x);
      if ((tid & 63) == 0) meet[wave][k] = sum[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kAlone; ++k) {
      if (column[k] < 0) continue;
      sum[k] = meet[0][k];
#pragma unroll
      for (int w = 1; w < THREADS / 64; ++w) sum[k] += meet[w][k];
#pragma unroll
      for (int x = 0; x < EACH; ++x)
        if (tid + x * THREADS < dim) put(column[k], tid + x * THREADS, o[k][x], sum[k]);
      if (tid == 0) total(column[k], top[k], sum[k]);
    }
    __syncthreads();  // the columns have been read
  }
  __syncthreads();  // that there are no more, too
}

// Four dimensions of one column of an item whose parts are rows.
template <int AUX, int DT, int M>
__device__ __forceinline__ void join_item(const TreeArgs& p, const Draft& d, const TreeParts& parts, int kv_head, int tile, int c, int quad, int quads) {
  float4_t o[1];
  float top, total;
  join_parts<AUX, 1>(p, parts, 0, 1, o, top, total, [&](uint32_t place, int) { return (place * M + c) * quads + quad; }, [&](uint32_t place) { return place * M + c; });
  const int of_all = tile * M + c, n = static_cast<int>(p.by_group.div(static_cast<uint32_t>(of_all)));
  store_answer<DT>(p, d.row + n, kv_head * p.group + of_all - n * p.group, 4 * quad,
                   total == 0.f ? float4_t{0.f, 0.f, 0.f, 0.f} : o[0] * (1.f / total));
}

// A tile of M = 16 CB columns (a column: one query head of one node) over a run of units of its sequence's tokens, four
// wavefronts each taking the tiles of TILE tokens of a unit in turn, as attention of one token does (k_paged_attention):
// S^T = K Q^T and O^T = V^T P^T with a token's row as it lies in memory, probabilities staying in the lanes that
// computed them, in two 16-bit parts. K's and V's 16 bytes a lane are used for CB products each, so that a tree's
// rows read the cache once together.
// What a column sees of the step's own tokens is 32 bits a tile; what it does not see has a weight of 0, and where
// an infinity or NaN is there (found by the NaN that it leaves) a column is done again (mark).
// Bound by memory where tokens are many, else by the ways in and out: 32 x 4 nodes over 4000 bf16 (4 kv heads of 4 heads of 128,
// 262 MB of K and V) 62 us, 4.2 TB/s; one of 8 nodes over 700 f16 11.7.
template <int DT, int NB, int CB>  // NB: blocks of 16 E dimensions
__global__ __launch_bounds__(256, NB == 1 && CB <= 2 ? 2 : 1) void k_tree_attention(TreeArgs p) {
  constexpr bool F32 = DT == DT_F32;
  constexpr int SIZE = F32 ? 4 : 2, E = 16 / SIZE, TILE = F32 ? 16 : 32, UT = 4 * TILE, M = 16 * CB;
  constexpr int NH = TILE / 16;           // 16-token halves of a tile
  constexpr int NC = 4 * NB;              // chunks of 4 E dimensions of a row
  constexpr int VT = F32 ? 4 : 8;         // tokens a lane reads of V
  constexpr uint32_t WHOLE = TILE == 32 ? 0xFFFFFFFFu : 0xFFFFu;  // all tokens of a tile
  constexpr float FACTOR = DT == DT_F16 ? 0x1p15f : 0x1p-32f;
  constexpr int ROW = 16 * E * NB + 4;    // floats of a column's answer in LDS (+ 4: off a bank's multiple)
  __shared__ __align__(16) float lds_o[4][16][ROW];
  __shared__ float lds_m[4][16], lds_l[4][16];
  __shared__ uint32_t marks[2];
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t worker = blockIdx.x;
  const int quads = p.head_dim / 4;
  // Zeros for the rows of sequences without tokens.
  for (int b = static_cast<int>(worker); b < p.B; b += static_cast<int>(p.workers)) {
    const Draft d = draft_at<UT, M>(p, b);
    if (d.units != 0) continue;
    const int64_t of_row = static_cast<int64_t>(p.group) * p.kv_heads * quads;
    for (int64_t i = threadIdx.x; i < d.nodes * of_row; i += 256)
      store_answer<DT>(p, d.row + i / of_row, 0, 4 * static_cast<int>(i % of_row), float4_t{0.f, 0.f, 0.f, 0.f});
  }
  const uint32_t all = all_work<UT, M>(p) * p.kv_heads, per = units_per_worker(all, p.workers);
  uint32_t at = worker * per;
  if (per == 0 || at >= all) return;
  const uint32_t stop = min(at + per, all);
  uint32_t before;
  int b = find_draft<UT, M>(p, at / p.kv_heads, before);
  if (b >= p.B) return;
  Draft d = draft_at<UT, M>(p, b);
  before *= p.kv_heads;  // the first unit of the sequence's first item
  const int chunks_of_row = (p.head_dim + 4 * E - 1) / (4 * E);
  const bool ragged = p.head_dim % (4 * E) != 0;
  while (at < stop) {
    while (at - before >= work_of(d) * p.kv_heads) {
      before += work_of(d) * p.kv_heads;
      if (++b >= p.B) return;
      d = draft_at<UT, M>(p, b);
    }
    const Place place = place_in(d, before, at);
    const Share share = share_of(place.first, static_cast<uint32_t>(d.units), at, stop);
    const uint32_t from = share.from, to = share.to;
    at = place.first + kItem + static_cast<uint32_t>(d.units);
    if (from >= to) continue;
    const int kv_head = static_cast<int>(place.item) / d.tiles, tile = static_cast<int>(place.item) % d.tiles;
    const int columns = min(M, d.nodes * p.group - tile * M);
    const char* kb = static_cast<const char*>(p.k) + static_cast<int64_t>(kv_head) * p.head_stride * SIZE;
    const char* vb = static_cast<const char*>(p.v) + static_cast<int64_t>(kv_head) * p.head_stride * SIZE;
    const int32_t* table = p.table + static_cast<int64_t>(b) * p.max_pages;

    uint4_t qf[CB][NC];
    int node[CB], begin[CB];  // of this lane's columns; begin: the first token that the window leaves
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
      const int c = 16 * cb + col, of_all = tile * M + min(c, columns - 1);
      node[cb] = static_cast<int>(p.by_group.div(static_cast<uint32_t>(of_all)));
      const int head = kv_head * p.group + of_all - node[cb] * p.group;
      begin[cb] = 0;
      if (p.window > 0) {
        if (p.mask) begin[cb] = tree_begin(p.mask + static_cast<int64_t>(d.row + node[cb]) * p.words, p.words, d.prefix, d.nodes, p.window);
        else begin[cb] = chain_begin(node[cb], d.prefix, p.window);
      }
#pragma unroll
      for (int x = 0; x < NC; ++x) {
        qf[cb][x] = uint4_t{0u, 0u, 0u, 0u};
        const int dim = 4 * E * x + E * g;
        if (dim < p.head_dim)
          qf[cb][x] = *reinterpret_cast<const uint4_t*>(static_cast<const char*>(p.q) +
                                                        ((d.row + node[cb]) * p.ldq + static_cast<int64_t>(head) * p.head_dim + dim) * SIZE);
      }
    }
    float m[CB], l[CB];  // of column 16 cb + col, l over this lane's tokens only
    float4_t acc[CB][NB][E];
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
      m[cb] = kNone;
      l[cb] = 0.f;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int e = 0; e < E; ++e) acc[cb][nb][e] = float4_t{0.f, 0.f, 0.f, 0.f};
    }

    // Lane i looks token i % TILE of a unit's tile up, a unit ahead: its row's offset in bytes, -1 where there is none.
    auto first_of = [&](uint32_t u) { return (d.unit + static_cast<int>(u)) * UT + wave * TILE; };
    auto look = [&](uint32_t u) -> int64_t {
      const int token = first_of(u) + lane % TILE;
      if (u >= to || token >= d.end) return -1;
      return token_offset(p.cache, table, static_cast<uint32_t>(token)) * SIZE;  // (a page that is none: negative)
    };
    uint4_t kf[NH][NC], vf[VT][NB];
    auto load_k = [&](int64_t offset) {
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        const char* row = kb + __shfl(offset, 16 * h + col);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const int dim = 4 * E * c + E * g;
          if (c < chunks_of_row) kf[h][c] = *reinterpret_cast<const uint4_t*>(row + (dim < p.head_dim ? dim * SIZE : 0));
        }
      }
    };
    auto load_v = [&](int64_t offset) {
#pragma unroll
      for (int j = 0; j < VT; ++j) {
        const char* row = vb + __shfl(offset, 16 * (j / 4) + 4 * g + j % 4);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          const int dim = 16 * E * nb + E * col;
          vf[j][nb] = *reinterpret_cast<const uint4_t*>(row + (dim < p.head_dim ? dim * SIZE : 0));
        }
      }
    };
    // S^T of a tile from kf.
    float4_t s[CB][NH];
    auto scores = [&] {
      if (ragged) {
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
          for (int c = 0; c < NC; ++c)
            if (4 * E * c + E * g >= p.head_dim) kf[h][c] = uint4_t{0u, 0u, 0u, 0u};
      }
#pragma unroll
      for (int cb = 0; cb < CB; ++cb)
#pragma unroll
        for (int h = 0; h < NH; ++h) s[cb][h] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        if (c >= chunks_of_row) continue;
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
          for (int cb = 0; cb < CB; ++cb) {
            if constexpr (F32) {
#pragma unroll
              for (int x = 0; x < 4; ++x)
                s[cb][h] = __builtin_amdgcn_mfma_f32_16x16x4f32(as_float(kf[h][c][x]), as_float(qf[cb][c][x]), s[cb][h], 0, 0, 0);
            } else {
              s[cb][h] = mfma16<DT>(kf[h][c], qf[cb][c], s[cb][h]);
            }
          }
      }
    };
    // What each of the lane's columns sees of the tile that begins at token `first`, `valid` of whose tokens there are: false
    // where all see all of it. Rows of V that are not there become zeros.
    uint32_t sees[CB];
    auto look_at = [&](int first, uint32_t valid) {
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) sees[cb] = valid;
      if (valid == WHOLE && first + TILE <= d.prefix && p.window == 0) return false;
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) {
        if (first + TILE > d.prefix) {
          if (p.mask) sees[cb] &= tree_bits(p.mask + static_cast<int64_t>(d.row + node[cb]) * p.words, p.words, first - d.prefix);
          else sees[cb] &= chain_bits(node[cb], first - d.prefix);
        }
        if (p.window > 0) sees[cb] &= from_bits(begin[cb], first);
      }
      if (valid != WHOLE) {
#pragma unroll
        for (int j = 0; j < VT; ++j)
          if (!(valid >> (16 * (j / 4) + 4 * g + j % 4) & 1u))
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) vf[j][nb] = uint4_t{0u, 0u, 0u, 0u};
      }
      return true;
    };
    float pr[F32 ? CB : 1][4];        // the probabilities, or
    uint4_t parts[F32 ? 1 : CB][2];   // their two parts
    auto softmax = [&](bool masked) {
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) {
        float t[NH][4], top = kNone;
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            t[h][i] = s[cb][h][i] * p.scale;
            if (masked && !(sees[cb] >> (16 * h + 4 * g + i) & 1u)) t[h][i] = kNone;
            top = fmaxf(top, t[h][i]);
          }
        top = column_max(top);
        if (__ballot(top > m[cb])) {
          const float next = fmaxf(m[cb], top);
          const float keep = next == m[cb] ? 1.f : __builtin_amdgcn_exp2f(m[cb] - next);  // (m -inf: 0)
          m[cb] = next;
          l[cb] *= keep;
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int e = 0; e < E; ++e) acc[cb][nb][e] *= keep;
        }
        const float ref = m[cb] == kNone ? 0.f : m[cb];
#pragma unroll
        for (int h = 0; h < NH; ++h) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            t[h][i] = __builtin_amdgcn_exp2f(t[h][i] - ref) * FACTOR;
            l[cb] += t[h][i];
            if constexpr (F32) pr[cb][i] = t[h][i];
          }
          if constexpr (!F32) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const uint2 two = split2<DT>(t[h][2 * x], t[h][2 * x + 1]);
              parts[cb][0][2 * h + x] = two.x;
              parts[cb][1][2 * h + x] = two.y;
            }
          }
        }
      }
    };
    // Of V's dimension E (4 g + i) + e (of block nb) the lane's tokens.
    auto operand = [&](int nb, int e) {
      uint4_t vt;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        if constexpr (F32) vt[x] = vf[x][nb][e];
        else vt[x] = __builtin_amdgcn_perm(vf[2 * x + 1][nb][e >> 1], vf[2 * x][nb][e >> 1], e & 1 ? 0x07060302u : 0x05040100u);
      }
      return vt;
    };
    auto product = [&](int cb, uint4_t v, float4_t c) {
      if constexpr (F32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(as_float(v[i]), pr[cb][i], c, 0, 0, 0);
        return c;
      } else {
        return mfma16<DT>(v, parts[cb][1], mfma16<DT>(v, parts[cb][0], c));
      }
    };

    int64_t found = look(from), coming = look(from + 1);
    load_k(found < 0 ? 0 : found);
    load_v(found < 0 ? 0 : found);
    for (uint32_t u = from; u < to; ++u) {
      const uint32_t valid = static_cast<uint32_t>(__ballot(found >= 0)) & WHOLE;  // (TILE 16: the four copies agree)
      const int64_t next_row = coming < 0 ? 0 : coming;
      const bool more = u + 1 < to;
      found = coming;
      coming = look(u + 2);
      scores();
      if (more) load_k(next_row);
      softmax(look_at(first_of(u), valid));
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const uint4_t vt = operand(nb, e);
#pragma unroll
          for (int cb = 0; cb < CB; ++cb) acc[cb][nb][e] = product(cb, vt, acc[cb][nb][e]);
        }
      if (more) load_v(next_row);
    }

    const bool whole = from == 0 && to == static_cast<uint32_t>(d.units);
    const uint32_t slot = place_of_part(worker, from == 0);
    const TreeParts all_parts = tree_parts(place.first, static_cast<uint32_t>(d.units), per);
    auto join_here = [&] {
      if (whole || all_parts.count > join_most(M, 1) || !last_of(p, all_parts)) return;
      for (int i = threadIdx.x; i < columns * quads; i += 256) {
        const int c = i / quads, quad = i - c * quads;
        join_item<kThrough, DT, M>(p, d, all_parts, kv_head, tile, c, quad, quads);
      }
    };
    bool bad[CB], any = false;  // (mark)
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
      bad[cb] = false;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x = acc[cb][nb][e][i];
            bad[cb] |= x != x;
          }
      any |= bad[cb];
    }
    uint32_t alone = 0;  // columns to do again
    if (__builtin_expect(__syncthreads_or(any), 0)) {
      if (threadIdx.x < 2) marks[threadIdx.x] = 0;
      __syncthreads();
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) {
        mark<16>(&marks[0], 16 * cb, bad[cb]);
        mark<16>(&marks[1], 16 * cb, l[cb] != l[cb]);
      }
      __syncthreads();
      alone = marks[0] & ~marks[1];
    }
    // The wavefronts' parts of the item meet in LDS, sixteen columns at a time.
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
      const float sum = column_sum(l[cb]);
      if (g == 0) {
        lds_m[wave][col] = m[cb];
        lds_l[wave][col] = sum;
      }
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < E; e += 4)
            *reinterpret_cast<float4_t*>(&lds_o[wave][col][16 * E * nb + E * (4 * g + i) + e]) =
                float4_t{acc[cb][nb][e][i], acc[cb][nb][e + 1][i], acc[cb][nb][e + 2][i], acc[cb][nb][e + 3][i]};
      __syncthreads();
      const int some = min(16, columns - 16 * cb);
      for (int i = threadIdx.x; i < some * quads; i += 256) {
        const int c = i / quads, dim = (i - c * quads) * 4;
        if (alone >> (16 * cb + c) & 1u) continue;
        float top = lds_m[0][c], total = 0.f;
#pragma unroll
        for (int w = 1; w < 4; ++w) top = fmaxf(top, lds_m[w][c]);
        float4_t o{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float f = lds_m[w][c] == top ? 1.f : __builtin_amdgcn_exp2f(lds_m[w][c] - top);
          total += f * lds_l[w][c];
          o += f * *reinterpret_cast<const float4_t*>(&lds_o[w][c][dim]);
        }
        if (whole) {
          const int of_all = tile * M + 16 * cb + c, n = static_cast<int>(p.by_group.div(static_cast<uint32_t>(of_all)));
          const float each = total == 0.f ? 0.f : 1.f / total;
          float4_t y = o * each;
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = total == 0.f ? 0.f : y[e];  // (0 * an infinity is none)
          store_answer<DT>(p, d.row + n, kv_head * p.group + of_all - n * p.group, dim, y);
        } else {
          const uint32_t row = slot * M + 16 * cb + c;
          put_part(p, row * quads + dim / 4, o);
          if (dim == 0) put_stats(p, row, top, total);
        }
      }
      __syncthreads();
    }
    if (__builtin_expect(alone, 0)) {
      if (threadIdx.x == 0) marks[0] = alone;
      __syncthreads();
      static_assert(kAloneRoom(256, 16 * E * NB) <= sizeof(lds_o), "");
      each_alone<DT, 256>(
          d, table, kv_head, tile * M, columns, (d.unit + static_cast<int>(from)) * UT, min(d.end, (d.unit + static_cast<int>(to)) * UT),
          p.scale, FACTOR, marks, lds_o,
          [&](int c, int dim, float o, float sum) {
            const int of_all = tile * M + c, n = static_cast<int>(p.by_group.div(static_cast<uint32_t>(of_all)));
            if (whole) store_as<DT>(p.y, (d.row + n) * p.ldy + static_cast<int64_t>(kv_head * p.group + of_all - n * p.group) * p.head_dim + dim, sum == 0.f ? 0.f : o * (1.f / sum));
            else put_value(p, (slot * M + c) * p.head_dim + dim, o);
          },
          [&](int c, float top, float sum) {
            if (!whole) put_stats(p, slot * M + c, top, sum);
          });
    }
    join_here();
  }
}

// Items of many parts (find_joined): workgroup (i, index) sees to columns 16 i .. 16 i + 15.
template <int DT, int M>
__global__ __launch_bounds__(256) void k_tree_join(TreeArgs p) {
  constexpr int UT = DT == DT_F32 ? 64 : 128;
  Joined j;
  if (!find_joined<UT, M, join_most(M, 1)>(p, blockIdx.y, j)) return;
  const int first_column = 16 * blockIdx.x, some = min(16, min(M, j.d.nodes * p.group - j.tile * M) - first_column), quads = p.head_dim / 4;
  for (int i = threadIdx.x; i < some * quads; i += 256) {
    const int c = i / quads;
    join_item<0, DT, M>(p, j.d, j.parts, j.kv_head, j.tile, first_column + c, i - c * quads, quads);
  }
}

// Sixteen bytes a lane from memory into LDS at lds + 16 * lane, past the registers. `lds` must be wavefront-uniform. In assembly,
// as the compiler would wait for it ahead of every transposed read of LDS, whatever that reads; a wait for all loads and a
// barrier stand between it and the reads that it is for.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // (m0 is nobody's for longer than an instruction, so that naming it is remarked on)
__device__ __forceinline__ void to_lds16(const char* from, uint8_t* lds) {
#if defined(__HIP_DEVICE_COMPILE__)
  const uint32_t at = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t*)lds)));
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(at) : "m0");
#endif
}
#pragma clang diagnostic pop

// Of four rows of sixteen 16-bit values, each row by four lanes of eight bytes, to each of sixteen lanes one column.
__device__ __forceinline__ uint2_t columns_of(const uint8_t* lds) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef short short4_t __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(uint2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)(lds)));
#else
  return uint2_t{0u, 0u};
#endif
}

template <int DT>
__device__ __forceinline__ float16_t mfma32(uint4_t a, uint4_t b, float16_t c) {
  typedef typename Lane16<DT>::vec vec;
  if constexpr (DT == DT_F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(vec, a), __builtin_bit_cast(vec, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(vec, a), __builtin_bit_cast(vec, b), c, 0, 0, 0);
}

// v's upper and lower half's values in both halves.
__device__ __forceinline__ void both_halves(float v, float& low, float& high) {
  const auto p = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
  const uint32_t a = p[0], b = p[1];
  low = __builtin_bit_cast(float, a);
  high = __builtin_bit_cast(float, b);
}

// A lane's answers of one column, dimensions dim + 8 q + {0 .. 3} in acc[q].
template <int DT>
__device__ __forceinline__ void answer_column(const TreeArgs& p, const Draft& d, int kv_head, int column, int dim, const float4_t (&acc)[4], float total) {
  const int n = static_cast<int>(p.by_group.div(static_cast<uint32_t>(column)));
  const float each = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    float4_t y = acc[q] * each;
#pragma unroll
    for (int x = 0; x < 4; ++x) y[x] = total == 0.f ? 0.f : y[x];  // (0 * an infinity is none)
    if (dim + 8 * q < p.head_dim) store_answer<DT>(p, d.row + n, kv_head * p.group + column - n * p.group, dim + 8 * q, y);
  }
}
__device__ __forceinline__ void quads_of(const float16_t& v, float4_t (&q)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) q[i] = float4_t{v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]};
}

// 32 dimensions (block db) of 32 columns (wc) of an item whose parts lie lane by lane.
template <int AUX, int DB, int WC>
__device__ __forceinline__ void join_block(const TreeArgs& p, const TreeParts& parts, int wc, int db, int lane, uint32_t first, uint32_t step, float4_t (&o)[4],
                                           float& top, float& total) {
  join_parts<AUX, 4>(p, parts, first, step, o, top, total, [&](uint32_t place, int i) { return ((place * WC + wc) * (4 * DB) + 4 * db + i) * 64 + lane; },
                [&](uint32_t place) { return place * (32 * WC) + 32 * wc + (lane & 31); });
}

// What tokens that are none bring to LDS.
__device__ const uint4_t kZeros[32] = {};

// Tiles of M = 32 WC columns of 16-bit types: WC WT wavefronts, a group of 32 columns each, WT of them sharing a unit's tokens, read K and V
// from LDS, where all of them bring the next unit meanwhile (two stages of 32 KiB). A step is 32 tokens: S^T = K Q^T, whose
// lanes then hold sixteen tokens' scores of one column, in the order in which O^T = V^T P^T takes them: no score leaves its
// lane, and V's columns are read from LDS transposed. Rows lie in LDS as in memory, their pieces of 16 bytes moved within the row,
// K's by the row's number so that the rows that are read together lie on different banks, V's by four pieces a row of four.
// Scores' maxima are kept as they come from the products, in the parts too: a probability is 2^((s - m) a + F) with the scale's
// magnitude a (its sign goes to the queries), at most 2^(F + LAG) whatever size the scores have. It is computed as s a + (F - m a), one
// instruction, up to maxima of FAR, where the roundings move weights by 2^-18 at most (from 2^27 on they would leave the 16-bit
// parts' range); past that a branch subtracts the maximum from the scores first (always so, 4 x 512 over 4096 took 168 us for 164).
// Probabilities go in two 16-bit parts (cut2; one part would make 4 x 512 over
// 4096 13% faster, and show in the answer). Maxima are followed where they grow by more than LAG only, as a rule never after a
// column's first unit (0 instead, one of 64 over 131072 f16: 310 us with 32 heads and so, 297 with 4).
// Bound by the products: 8192 more tokens of 4 x 512 bf16 rows cost 395 us, 1.04 PFLOP/s in all, where a large library product
// comes to 1.20; without any exponentials it is 7% less, without reads of K from LDS no less. Beside that the ways in and out,
// 35 us of the 154 of 4 x 512 over 4096.
template <int DT, int NB, int WC, int WT>
__global__ __launch_bounds__(64 * WC * WT, NB == 1 ? 2 : 1) void k_tree_shared(TreeArgs p) {
  constexpr int THREADS = 64 * WC * WT, UT = 64 / NB, TW = UT / WT, M = 32 * WC;  // TW: a wavefront's tokens of a unit
  constexpr int W = TW / 32, NC = 8 * NB, DB = 4 * NB, PITCH = 256 * NB, STAGE = 2 * UT * PITCH;
  constexpr int RI = 4 / NB, RW = TW / WC;  // rows that an instruction brings, and a wavefront
  constexpr int PLACES = W + 2;             // of a unit's work where loads of the next are asked for
  constexpr uint32_t kNone16 = ~0u;
  constexpr float LAG = DT == DT_F16 ? 4.f : 8.f, F = DT == DT_F16 ? 15.f - LAG : -32.f - LAG, FAR = 64.f;
  static_assert(TW % 32 == 0 && RW % 16 == 0, "");
  __shared__ __align__(16) uint8_t lds[2][STAGE];
  __shared__ float2 lds_ml[WT][M];
  __shared__ uint32_t marks[2 * WC];
  const int lane = threadIdx.x & 63, col = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wc = wave % WC, wt = wave / WC;
  const uint32_t worker = blockIdx.x;
  const int quads = p.head_dim / 4;
  for (int b = static_cast<int>(worker); b < p.B; b += static_cast<int>(p.workers)) {
    const Draft d = draft_at<UT, M>(p, b);
    if (d.units != 0) continue;
    const int64_t of_row = static_cast<int64_t>(p.group) * p.kv_heads * quads;
    for (int64_t i = threadIdx.x; i < d.nodes * of_row; i += THREADS)
      store_answer<DT>(p, d.row + i / of_row, 0, 4 * static_cast<int>(i % of_row), float4_t{0.f, 0.f, 0.f, 0.f});
  }
  const uint32_t all = all_work<UT, M>(p) * p.kv_heads, per = units_per_worker(all, p.workers);
  uint32_t at = worker * per;
  if (per == 0 || at >= all) return;
  const uint32_t stop = min(at + per, all);
  uint32_t before;
  int b = find_draft<UT, M>(p, at / p.kv_heads, before);
  if (b >= p.B) return;
  Draft d = draft_at<UT, M>(p, b);
  before *= p.kv_heads;
  auto clear = [&](int stages) {  // pieces of a row past head_dim are brought by nobody: zeros for all units
    if (p.head_dim == 128 * NB) return;
    for (int i = threadIdx.x; i < stages * STAGE / 16; i += THREADS) reinterpret_cast<uint4_t*>(&lds[0][0])[i] = uint4_t{0u, 0u, 0u, 0u};
    __syncthreads();
  };
  clear(2);
  const float a = p.unit;
  const uint32_t sign = p.scale < 0.f ? 0x80008000u : 0u;
  const uint32_t page16 = static_cast<uint32_t>(p.cache.page_stride / 8), token16 = static_cast<uint32_t>(p.cache.token_stride / 8);
  bool used = false;  // stage 0, by an item's sums
  while (at < stop) {
    while (at - before >= work_of(d) * p.kv_heads) {
      before += work_of(d) * p.kv_heads;
      if (++b >= p.B) return;
      d = draft_at<UT, M>(p, b);
    }
    const Place place = place_in(d, before, at);
    const Share share = share_of(place.first, static_cast<uint32_t>(d.units), at, stop);
    const uint32_t from = share.from, to = share.to;
    at = place.first + kItem + static_cast<uint32_t>(d.units);
    if (from >= to) continue;
    const int kv_head = static_cast<int>(place.item) / d.tiles, tile = static_cast<int>(place.item) % d.tiles;
    const int columns = min(M, d.nodes * p.group - tile * M);
    const char* kb = static_cast<const char*>(p.k) + static_cast<int64_t>(kv_head) * p.head_stride * 2;
    const char* vb = static_cast<const char*>(p.v) + static_cast<int64_t>(kv_head) * p.head_stride * 2;
    const int32_t* table = p.table + static_cast<int64_t>(b) * p.max_pages;
    // Tokens that all columns see, and those that any sees (of chains: up to the tile's first and last nodes).
    const int first_node = static_cast<int>(p.by_group.div(static_cast<uint32_t>(tile * M)));
    const int last_node = static_cast<int>(p.by_group.div(static_cast<uint32_t>(tile * M + columns - 1)));
    const int open = p.mask ? d.prefix : d.prefix + first_node + 1, end = p.mask ? d.end : min(d.end, d.prefix + last_node + 1);
    const uint32_t needed = end > d.unit * UT ? static_cast<uint32_t>((end + UT - 1) / UT - d.unit) : 0, upto = min(to, needed);

    const int of_all = tile * M + min(32 * wc + col, columns - 1);  // this lane's column
    const int node = static_cast<int>(p.by_group.div(static_cast<uint32_t>(of_all)));
    const uint64_t* mask = p.mask ? p.mask + static_cast<int64_t>(d.row + node) * p.words : nullptr;
    const uint64_t word = mask ? mask[0] : 0;  // (all of it, mostly)
    int begin = 0;
    if (p.window > 0) begin = mask ? tree_begin(mask, p.words, d.prefix, d.nodes, p.window) : chain_begin(node, d.prefix, p.window);
    uint4_t qf[NC];
    float m = kNone, l = 0.f;  // of this lane's column, l over this lane's tokens only
    bool far = false;          // a column's maximum is past FAR
    float16_t acc[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[db][i] = 0.f;

    // Lane i looks token i % TW of its wavefront's part of a unit up, in two steps: the page's number is loaded a unit before it is
    // looked at, which would wait for the rows that are on their way by then. A row's offset in 16 bytes, kNone16 where there is none.
    auto first_of = [&](uint32_t u) { return (d.unit + static_cast<int>(u)) * UT + wt * TW; };
    auto page_of = [&](uint32_t u) { return table[p.cache.by_page.div(static_cast<uint32_t>(min(first_of(u) + lane % TW, d.end - 1)))]; };
    auto offset_of = [&](uint32_t u, int32_t id) {
      const int token = first_of(u) + lane % TW;
      const uint32_t in_page = static_cast<uint32_t>(token) - p.cache.by_page.div(static_cast<uint32_t>(token)) * p.cache.by_page.d;
      const uint32_t at_row = static_cast<uint32_t>(id) * page16 + in_page * token16;
      return token < d.end && id >= 0 && id < p.cache.pages ? at_row : kNone16;
    };
    // Brings a unit's rows: a wavefront its share of its part's, PIECES instructions, of which those of `place` of all `places`. Rows
    // that are none bring zeros; where the head is narrower than the unit's rows, lanes past it bring nothing.
    constexpr int J = RW / RI;
    const int slot16 = lane % (16 * NB), in_instruction = lane / (16 * NB);
    const char* k_lane[J];
    const char* v_lane[RI < 4 ? 4 / RI : 1];
#pragma unroll
    for (int j = 0; j < J; ++j) k_lane[j] = kb + 16 * (slot16 ^ ((RI * j + in_instruction) & 15));
#pragma unroll
    for (int j = 0; j < (RI < 4 ? 4 / RI : 1); ++j) v_lane[j] = vb + 16 * (slot16 ^ (((RI * j + in_instruction) & 3) << 2));
    uint32_t rows[J];  // of the unit that is brought: the lane's row of each instruction
    bool plain = true;  // all of its tokens are there, in rows of the full width
    auto rows_of = [&](uint32_t offset) {
#pragma unroll
      for (int j = 0; j < J; ++j) rows[j] = __shfl(offset, RW * wc + RI * j + in_instruction);
      plain = p.head_dim == 128 * NB && __ballot(offset == kNone16) == 0;
    };
    auto bring = [&](int stage, int place, int places) {
#pragma unroll
      for (int j = 0; j < J; ++j) {
        if (j * places / J != place) continue;
        uint8_t* to = &lds[stage][(wt * TW + RW * wc + RI * j) * PITCH];
        const uint64_t row = static_cast<uint64_t>(rows[j]) << 4;
        if (plain) {
          to_lds16(k_lane[j] + row, to);
          to_lds16(v_lane[j % (4 / RI)] + row, to + UT * PITCH);
        } else {
          const char* none = reinterpret_cast<const char*>(kZeros);
          const int k_piece = slot16 ^ ((RI * j + in_instruction) & 15), v_piece = slot16 ^ (((RI * j + in_instruction) & 3) << 2);
          if (8 * k_piece < p.head_dim) to_lds16(rows[j] == kNone16 ? none : k_lane[j] + row, to);
          if (8 * v_piece < p.head_dim) to_lds16(rows[j] == kNone16 ? none : v_lane[j % (4 / RI)] + row, to + UT * PITCH);
        }
      }
    };
    // All of a workgroup's rows have come, and no wavefront reads the unit before any more.
    auto meet = [&] {
      __builtin_amdgcn_s_waitcnt(0);
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    };
    // The TW tokens from `first` on, `valid` of which there are. Meanwhile between() is called PLACES times: a wavefront that
    // asked for all its share of the next unit at once would wait for the queue of such loads.
    auto step = [&](int stage, int first, uint64_t valid, auto between) {
      float16_t s[W];
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const uint8_t* k_row = &lds[stage][(wt * TW + 32 * w + col) * PITCH];
#pragma unroll
        for (int i = 0; i < 16; ++i) s[w][i] = 0.f;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          // (Asked of LDS ahead of all products: the compiler would wait for each by itself.)
          uint4_t kf[8];
#pragma unroll
          for (int c = 0; c < 8; ++c) kf[c] = *reinterpret_cast<const uint4_t*>(k_row + 16 * ((16 * nb + 2 * c + h) ^ (col & 15)));
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int c = 0; c < 8; ++c) s[w] = mfma32<DT>(kf[c], qf[8 * nb + c], s[w]);
        }
        between(w);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (valid != (TW == 64 ? ~uint64_t{0} : 0xFFFFFFFFu) || first + TW > open || p.window > 0) {
        asm volatile("");  // (a branch: as selects it would be paid for in every unit)
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const int from = first + 32 * w;
          uint32_t some = static_cast<uint32_t>(valid >> 32 * w);
          if (from + 32 > d.prefix) {
            if (!p.mask) some &= chain_bits(node, from - d.prefix);
            else some &= p.words == 1 ? tree_bits(&word, 1, from - d.prefix) : tree_bits(mask, p.words, from - d.prefix);
          }
          if (p.window > 0) some &= from_bits(begin, from);
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (!(some >> (8 * (i / 4) + 4 * h + i % 4) & 1u)) s[w][i] = kNone;
        }
      }
      float low, high, top = kNone;
#pragma unroll
      for (int w = 0; w < W; ++w)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, s[w][i]);
      both_halves(top, low, high);
      top = fmaxf(low, high);
      if (__ballot((top - m) * a > LAG)) {  // (m -infinity: infinity; or NaN where top is so too, or infinite as m is)
        const float next = fmaxf(m, top);
        const float keep = next == m ? 1.f : m == kNone ? 0.f : __builtin_amdgcn_exp2f((m - next) * a);
        m = next;
        l *= keep;
#pragma unroll
        for (int db = 0; db < DB; ++db) acc[db] *= keep;
        far = __ballot(m != kNone && fabsf(m * a) > FAR) != 0;
      }
      const float ref = m == kNone ? 0.f : m;
      float c = F - ref * a;
      if (far) {
        asm volatile("");
        c = F;
#pragma unroll
        for (int w = 0; w < W; ++w)
#pragma unroll
          for (int i = 0; i < 16; ++i) s[w][i] -= ref;
      }
      // Half a step's products: of tokens 16 x + 4 h + {0 .. 3, 8 .. 11} V's dimension 32 db + lane % 32.
#pragma unroll
      for (int x = 0; x < 2 * W; ++x) {
        uint4_t vf[DB], parts[2];
        const int in_block = lane & 15, token = 16 * x + 4 * h + in_block / 4;
        const uint8_t* row = &lds[stage][(UT + wt * TW + token) * PITCH];
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          const int at = 16 * ((4 * db + 2 * (col >> 4) + (in_block & 3) / 2) ^ ((token & 3) << 2)) + 8 * (in_block & 1);
          const uint2_t one = columns_of(row + at), two = columns_of(row + 8 * PITCH + at);
          vf[db] = uint4_t{one.x, one.y, two.x, two.y};
        }
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const float p0 = __builtin_amdgcn_exp2f(fmaf(s[x / 2][8 * (x % 2) + 2 * y], a, c));
          const float p1 = __builtin_amdgcn_exp2f(fmaf(s[x / 2][8 * (x % 2) + 2 * y + 1], a, c));
          l += p0 + p1;
          const uint2 part = cut2<DT>(p0, p1);
          parts[0][y] = part.x;
          parts[1][y] = part.y;
        }
        if (x < 2) between(W + x);
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int db = 0; db < DB; ++db) acc[db] = mfma32<DT>(vf[db], parts[y], acc[db]);
      }
    };

    uint32_t found = kNone16;
    int32_t coming = 0;
    __syncthreads();  // the item before has left LDS
    if (WT > 1 && used) clear(1);  // (its sums: as 16-bit values NaN among them, for which it would all be done again)
    used = true;
    // The queries come by whole rows through the second stage, each wavefront's own columns (by 16 bytes of many rows at a time they
    // took 5 us, with the first rows of K and V they come in passing).
    if (from < upto) {
      const int64_t q_row = (d.row + node) * p.ldq + static_cast<int64_t>(kv_head * p.group + of_all - node * p.group) * p.head_dim;
#pragma unroll
      for (int j = 0; j < 32 / RI; ++j) {
        const int row = RI * j + in_instruction, piece = slot16 ^ (row & 15);
        const char* q = static_cast<const char*>(p.q) + __shfl(q_row, row) * 2 + 16 * piece;
        if (8 * piece < p.head_dim) to_lds16(q, &lds[1][(32 * wave + RI * j) * PITCH]);
      }
      found = offset_of(from, page_of(from));
      coming = page_of(from + 1);
      rows_of(found);
      bring(0, 0, 1);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      qf[c] = *reinterpret_cast<const uint4_t*>(&lds[1][(32 * wave + col) * PITCH + 16 * ((2 * c + h) ^ (col & 15))]);
      if (16 * c + 8 * h >= p.head_dim || p.scale == 0.f) qf[c] = uint4_t{0u, 0u, 0u, 0u};
      qf[c] ^= sign;
    }
    int stage = 0;
    for (uint32_t u = from; u < upto; ++u, stage ^= 1) {
      const uint64_t valid = TW == 64 ? __ballot(found != kNone16) : __ballot(found != kNone16) & 0xFFFFFFFFu;
      meet();
      const bool more = u + 1 < upto;
      if (more) {
        found = offset_of(u + 1, coming);
        coming = page_of(u + 2);
        rows_of(found);
      }
      step(stage, first_of(u), valid, [&](int place) {
        if (more) bring(stage ^ 1, place, PLACES);
      });
    }

    const bool whole = from == 0 && to == static_cast<uint32_t>(d.units);
    const uint32_t slot = place_of_part(worker, from == 0);
    const TreeParts parts = tree_parts(place.first, static_cast<uint32_t>(d.units), per);
    auto join_here = [&] {
      if (whole || parts.count > join_most(M, NB) || !last_of(p, parts)) return;
      for (int i = wave; i < WC * DB; i += WC * WT)
        if (32 * (i / DB) < columns && 32 * (i % DB) < p.head_dim) {
          float4_t o[4];
          float top, total;
          join_block<kThrough, DB, WC>(p, parts, i / DB, i % DB, lane, 0, 1, o, top, total);
          if (32 * (i / DB) + col < columns) answer_column<DT>(p, d, kv_head, tile * M + 32 * (i / DB) + col, 32 * (i % DB) + 4 * h, o, total);
        }
    };
    bool bad = false;  // (mark)
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float x = acc[db][i];
        bad |= x != x;
      }
    bool alone = false, mine = false;  // columns to do again, this lane's among them
    if (__builtin_expect(__syncthreads_or(bad), 0)) {
      if (threadIdx.x < 2 * WC) marks[threadIdx.x] = 0;
      __syncthreads();
      mark<32>(marks, 32 * wc, bad);
      mark<32>(marks + WC, 32 * wc, l != l);
      __syncthreads();
#pragma unroll
      for (int w = 0; w < WC; ++w) alone |= (marks[w] & ~marks[WC + w]) != 0;
      mine = (marks[wc] & ~marks[WC + wc]) >> col & 1u;
    }
    // The wavefronts that share a tile's tokens meet in LDS, lane by lane; the first of them answers.
    {
      float low, high;
      both_halves(l, low, high);
      l = low + high;
    }
    float4_t* sums = reinterpret_cast<float4_t*>(&lds[0][0]);
    auto place_of_sum = [&](int part, int i) { return ((part * WC + wc) * (4 * DB) + i) * 64 + lane; };
    lds_ml[wt][32 * wc + col] = make_float2(m, l);
    if (wt > 0) {
#pragma unroll
      for (int i = 0; i < 4 * DB; ++i)
        sums[place_of_sum(wt - 1, i)] = float4_t{acc[i / 4][i % 4 * 4], acc[i / 4][i % 4 * 4 + 1], acc[i / 4][i % 4 * 4 + 2], acc[i / 4][i % 4 * 4 + 3]};
    }
    __syncthreads();
    if (wt == 0 && 32 * wc < columns) {
      float top = m;
#pragma unroll
      for (int w = 1; w < WT; ++w) top = fmaxf(top, lds_ml[w][32 * wc + col].x);
      auto weight = [&](float x) { return x == top ? 1.f : x == kNone ? 0.f : __builtin_amdgcn_exp2f((x - top) * a); };
      const float f0 = weight(m);
      float total = f0 * l;
#pragma unroll
      for (int db = 0; db < DB; ++db) acc[db] *= f0;
#pragma unroll
      for (int w = 1; w < WT; ++w) {
        const float2 ml = lds_ml[w][32 * wc + col];
        const float f = weight(ml.x);
        total += f * ml.y;
#pragma unroll
        for (int i = 0; i < 4 * DB; ++i) {
          const float4_t o = sums[place_of_sum(w - 1, i)];
#pragma unroll
          for (int x = 0; x < 4; ++x) acc[i / 4][i % 4 * 4 + x] += f * o[x];
        }
      }
      if (whole) {
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          float4_t four[4];
          quads_of(acc[db], four);
          if (32 * wc + col < columns && !mine) answer_column<DT>(p, d, kv_head, tile * M + 32 * wc + col, 32 * db + 4 * h, four, total);
        }
      } else if (!mine) {
#pragma unroll
        for (int i = 0; i < 4 * DB; ++i)
          put_part(p, ((slot * WC + wc) * (4 * DB) + i) * 64 + lane, float4_t{acc[i / 4][i % 4 * 4], acc[i / 4][i % 4 * 4 + 1], acc[i / 4][i % 4 * 4 + 2], acc[i / 4][i % 4 * 4 + 3]});
        if (h == 0) put_stats(p, slot * M + 32 * wc + col, top, total);
      }
    }
    if (__builtin_expect(alone, 0)) {
      __syncthreads();  // the wavefronts' sums have been read
      if (threadIdx.x < WC) marks[threadIdx.x] &= ~marks[WC + threadIdx.x];
      __syncthreads();
      static_assert(kAloneRoom(THREADS, 128 * NB) <= sizeof(lds), "");
      each_alone<DT, THREADS>(
          d, table, kv_head, tile * M, columns, (d.unit + static_cast<int>(from)) * UT, min(d.end, (d.unit + static_cast<int>(to)) * UT),
          p.scale == 0.f ? 0.f : copysignf(1.f, p.scale), __builtin_ldexpf(1.f, static_cast<int>(F)), marks, lds,
          [&](int c, int dim, float o, float sum) {
            const int of_all = tile * M + c, n = static_cast<int>(p.by_group.div(static_cast<uint32_t>(of_all)));
            if (whole) store_as<DT>(p.y, (d.row + n) * p.ldy + static_cast<int64_t>(kv_head * p.group + of_all - n * p.group) * p.head_dim + dim, sum == 0.f ? 0.f : o * (1.f / sum));
            else put_value(p, (((slot * WC + c / 32) * (4 * DB) + dim / 8) * 64 + dim / 4 % 2 * 32 + c % 32) * 4 + dim % 4, o);
          },
          [&](int c, float top, float sum) {
            if (!whole) put_stats(p, slot * M + c, top, sum);
          });
      clear(2);
    }
    join_here();
  }
}

// Items of many parts (find_joined): workgroup (wc, db, index) sees to 32 dimensions of 32 columns, its wavefronts to every fourth part.
// (The index last: workgroups go to the XCDs in turn, and items of one length begin in workers that many apart. By index first all of the
// work was one XCD's, 21 us for 8 items of 64 parts.)
template <int DT, int NB, int WC>
__global__ __launch_bounds__(256) void k_tree_shared_join(TreeArgs p) {
  constexpr int UT = 64 / NB, M = 32 * WC;
  __shared__ __align__(16) float4_t sums[3][4][64];
  __shared__ float2 stats[3][64];
  Joined j;
  if (!find_joined<UT, M, join_most(M, NB)>(p, blockIdx.z, j)) return;
  const int wc = blockIdx.x, db = blockIdx.y, columns = min(M, j.d.nodes * p.group - j.tile * M);
  if (32 * wc >= columns || 32 * db >= p.head_dim) return;
  const int lane = threadIdx.x & 63, col = lane & 31, h = lane >> 5;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  float4_t acc[4];
  float top, total;
  join_block<0, 4 * NB, WC>(p, j.parts, wc, db, lane, wave, 4, acc, top, total);
  if (wave) {
    stats[wave - 1][lane] = make_float2(top, total);
#pragma unroll
    for (int q = 0; q < 4; ++q) sums[wave - 1][q][lane] = acc[q];
  }
  __syncthreads();
  if (wave) return;
  float most = top;
#pragma unroll
  for (int w = 0; w < 3; ++w) most = fmaxf(most, stats[w][lane].x);
  const float keep = top == most ? 1.f : __builtin_amdgcn_exp2f((top - most) * p.unit);
  total *= keep;
#pragma unroll
  for (int q = 0; q < 4; ++q) acc[q] *= keep;
#pragma unroll
  for (int w = 0; w < 3; ++w) {
    const float2 st = stats[w][lane];
    const float f = st.x == most ? 1.f : __builtin_amdgcn_exp2f((st.x - most) * p.unit);
    total += f * st.y;
#pragma unroll
    for (int q = 0; q < 4; ++q) acc[q] += f * sums[w][q][lane];
  }
  if (32 * wc + col < columns) answer_column<DT>(p, j.d, j.kv_head, j.tile * M + 32 * wc + col, 32 * db + 4 * h, acc, total);
}

// (`units`: of an item, as far as the host knows. Without items of many parts there is nothing for the second kernel to do.)
template <int DT, int NB, int CB>
void launch_tree(const TreeArgs& p, int64_t units, hipStream_t s) {
  constexpr uint32_t MOST = join_most(16 * CB, 1);
  k_tree_attention<DT, NB, CB><<<p.workers, 256, 0, s>>>(p);
  if (p.workers > MOST && units > MOST) k_tree_join<DT, 16 * CB><<<dim3(CB, p.workers / MOST), 256, 0, s>>>(p);
}
template <int DT, int NB, int WC, int WT>
void launch_shared(const TreeArgs& p, int64_t units, hipStream_t s) {
  constexpr uint32_t MOST = join_most(32 * WC, NB);
  k_tree_shared<DT, NB, WC, WT><<<p.workers, 64 * WC * WT, 0, s>>>(p);
  if (p.workers > MOST && units > MOST) k_tree_shared_join<DT, NB, WC><<<dim3(WC, 4 * NB, p.workers / MOST), 256, 0, s>>>(p);
}

// How columns go to workgroups, by the columns that a sequence has in the mean and the tokens that the table or the window leaves it
// (all the host knows).
struct TreeForm {
  bool shared;
  int columns, unit;  // columns of a tile, tokens of a unit
};
constexpr int kPerCu = 2;  // workgroups a CU
// `near`: rows' offsets fit 32 bits, counted in 16 bytes.
// Wide tiles read K and V less often, narrow ones give every workgroup work where there is little. What little is, by the work of a
// worker in narrow tiles, is from measurements, us in tiles of 16 columns, 64 and 128 (16-bit types, 128 dimensions, sequences x
// nodes over tokens):
//   up to 10 units of 16 columns: 4 x 32 over 500 with 8 kv heads of 4 heads 21, 24, 37; 16 x 30 over 64 to 128 13, 19, 17;
//     4 x 30 over 2000 26, 35, 31; 9 x 40 over 1 to 900 26, 28, 42; past it 8 x 32 over 4000 59, 47, 43;
//   up to 16 units of 64 columns, of sequences of up to 1024 tokens (where more of a worker's time goes to the ways in and out): 512
//     over 512 41, 31, 37; two of them 74, 31, 44; 8 x 64 over 1000 86, 44, 55; past it 8 of 512 327, 109, 82;
//   others: 128 over 4096 60, 48, 44; 8 x 64 over 4000 94, 65, 69.
//   of 256 dimensions, in tiles of 16 and 64: 4 x 32 over 500 48 and 53, 16 x 30 over 64 to 128 29 and 39, 4 x 30 over 2000 61 and 45.
// Columns that fill no second tile of 16 stay in one (32 x 4 over 4000 with 4 heads a kv head 62, 80, 90; 6 nodes 94, 78, 87); up to
// 64 go to tiles of 64 (16 nodes 90, 52, 60; 20 nodes 105, 66, 65). In f32, tiles of 16 and 32: 4 x 8 over 2000 35 and 41, 64 over
// 1000 35 and 38; 8 x 32 over 1000 76 and 65, 32 x 8 over 4000 259 and 196.
TreeForm tree_form(int64_t B, int64_t columns, int64_t tokens, int kv_heads, int64_t workers, bool f32, int head_dim, bool near) {
  auto work = [&](int64_t tile, int64_t unit) {  // of a worker
    return 1.0 * B * kv_heads * ((columns + tile - 1) / tile) * ((tokens + unit - 1) / unit + kItem) / workers;
  };
  if (f32) return {false, head_dim <= 128 && columns > 16 && work(16, 64) > 5 ? 32 : 16, 64};
  if (columns <= 16 || !near || (work(16, 128) <= 10 && (head_dim <= 128 || tokens <= 1024))) return {false, 16, 128};
  if (head_dim > 128) return {true, 64, 32};
  return {true, columns <= 64 || (tokens <= 1024 && work(64, 64) <= 16) ? 64 : 128, 64};
}

}  // namespace
}  // namespace tmh

using namespace tmh;

extern "C" {

int tmh_paged_tree_attention(tmh_ctx* ctx, const void* d_q, int64_t ldq, int64_t T, int heads, const tmh_paged_cache* cache,
                             const int32_t* d_page_table, int64_t B, int64_t max_pages, const int32_t* d_lengths,
                             const int32_t* d_starts, const int64_t* d_mask, int64_t mask_words, float scale,
                             int64_t window, void* d_y, int64_t ldy, void* stream) {
  TMH_TRY(check_cache(ctx, cache));
  if (heads < 1 || heads % cache->kv_heads != 0)
    return fail(ctx, TMH_ERR_INVALID, "%d query heads are no multiple of %d kv heads", heads, cache->kv_heads);
  if (heads > (1 << 20)) return fail(ctx, TMH_ERR_UNSUPPORTED, "attention takes up to 2^20 query heads, got %d", heads);
  if (B < 0 || B > 65535) return fail(ctx, TMH_ERR_INVALID, "attention takes 0 to 65535 sequences, got %lld", (long long)B);
  if (T < 0 || T >= (int64_t{1} << 31)) return fail(ctx, TMH_ERR_INVALID, "attention cannot take %lld rows", (long long)T);
  if (max_pages < 0 || window < 0) return fail(ctx, TMH_ERR_INVALID, "max_pages and window must not be negative");
  if (mask_words < 0 || mask_words > (1 << 20) || (d_mask && mask_words < 1))
    return fail(ctx, TMH_ERR_INVALID, "a tree's mask has 1 to 2^20 words a row, got %lld", (long long)mask_words);
  if (std::isnan(scale)) return fail(ctx, TMH_ERR_INVALID, "the scale is NaN");
  const int64_t width = static_cast<int64_t>(heads) * cache->head_dim;
  if (ldq < width || ldy < width)
    return fail(ctx, TMH_ERR_INVALID, "the leading dimensions of q and y must be at least %lld", (long long)width);
  // (A workgroup counts up to two units past its last, and tokens in 32 bits.)
  if (max_pages > ((int64_t{1} << 31) - 1024) / cache->page_size)
    return fail(ctx, TMH_ERR_UNSUPPORTED, "attention of several tokens needs max_pages * page_size of up to 2^31 - 1024");
  TMH_TRY(use_device(ctx));
  if (B == 0 || T == 0) return TMH_OK;
  if (!d_q || !d_y || !d_lengths || !d_starts || (max_pages && !d_page_table))
    return fail(ctx, TMH_ERR_INVALID, "tmh_paged_tree_attention: NULL pointer");
  const int64_t e = 16 / dtype_size(cache->dtype);
  if (reinterpret_cast<uintptr_t>(d_q) % 16 != 0 || reinterpret_cast<uintptr_t>(d_y) % 16 != 0 || ldq % e != 0 || ldy % e != 0)
    return fail(ctx, TMH_ERR_UNSUPPORTED, "attention's q and y must be aligned to 16 bytes, their leading dimensions too");
  const int group = heads / cache->kv_heads;
  if (T * group >= (int64_t{1} << 31)) return fail(ctx, TMH_ERR_UNSUPPORTED, "attention over too many rows at once");
  const bool f32 = cache->dtype == TMH_F32;
  const unsigned __int128 last_row = static_cast<unsigned __int128>(cache->pages - 1) * cache->page_stride +
                                     static_cast<unsigned __int128>(cache->page_size - 1) * cache->token_stride;
  const bool near = last_row / 8 < (uint64_t{1} << 32) - 1;
  const int64_t most = max_pages * cache->page_size, nodes = (T + B - 1) / B, workers = kPerCu * ctx->num_cus;
  const int64_t tokens = window > 0 && window < most ? std::min(most, window + nodes) : most;
  const TreeForm form = tree_form(B, (T * group + B - 1) / B, tokens, cache->kv_heads, workers, f32, cache->head_dim, near);
  const int64_t unit = form.unit;
  const int64_t items = (T * group / form.columns + B) * cache->kv_heads;
  const int64_t units = (most + unit - 1) / unit;  // of an item
  if (units + kItem >= (int64_t{1} << 31) / items)
    return fail(ctx, TMH_ERR_UNSUPPORTED, "attention over too many rows and tokens at once");
  TreeArgs p;
  p.q = d_q;
  p.k = cache->k;
  p.v = cache->v;
  p.table = d_page_table;
  p.lengths = d_lengths;
  p.starts = d_starts;
  p.mask = reinterpret_cast<const uint64_t*>(d_mask);
  p.y = d_y;
  p.ldq = ldq;
  p.ldy = ldy;
  p.max_pages = max_pages;
  p.rows = T;
  p.most = most;
  p.cache = PageShape{cache->pages, cache->page_stride, cache->token_stride, FastDiv(static_cast<uint32_t>(cache->page_size))};
  p.head_stride = cache->head_stride;
  p.window = static_cast<int>(std::min<int64_t>(window, (int64_t{1} << 31) - 1));
  p.words = static_cast<int>(mask_words);
  p.B = static_cast<int>(B);
  p.group = group;
  p.kv_heads = cache->kv_heads;
  p.head_dim = cache->head_dim;
  p.by_group = FastDiv(static_cast<uint32_t>(group));
  p.scale = scale * 1.44269504088896340736f;
  // (A scale of 0: queries of zeros, so that -infinity times the unit stays what it is.)
  p.unit = !form.shared || p.scale == 0.f ? 1.f : std::fabs(p.scale);
  p.workers = static_cast<uint32_t>(std::max<int64_t>(1, std::min<int64_t>(workers, units * items)));
  hipStream_t s = pick_stream(ctx, stream);
  const size_t rows = 2 * static_cast<size_t>(workers) * form.columns;
  const int width_of_part = form.shared ? (cache->head_dim <= 128 ? 128 : 256) : cache->head_dim;
  void* ws = workspace(ctx, rows * (width_of_part * 4 + sizeof(float2)), s);
  if (!ws) return fail(ctx, TMH_ERR_UNSUPPORTED, "attention's workspace cannot grow here: run one call before the capture");
  p.part = static_cast<float*>(ws);
  p.stats = reinterpret_cast<float2*>(p.part + rows * width_of_part);
  p.part_bytes = static_cast<uint32_t>(rows * width_of_part * 4);
  p.stats_bytes = static_cast<uint32_t>(rows * sizeof(float2));
  p.meet = ctx->meet;
  auto launch = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if constexpr (DT == DT_F32) {
      if (cache->head_dim <= 64) form.columns == 16 ? launch_tree<DT, 1, 1>(p, units, s) : launch_tree<DT, 1, 2>(p, units, s);
      else if (cache->head_dim <= 128) form.columns == 16 ? launch_tree<DT, 2, 1>(p, units, s) : launch_tree<DT, 2, 2>(p, units, s);
      else launch_tree<DT, 4, 1>(p, units, s);
    } else if (cache->head_dim <= 128) {
      if (!form.shared) launch_tree<DT, 1, 1>(p, units, s);
      else form.columns == 64 ? launch_shared<DT, 1, 2, 2>(p, units, s) : launch_shared<DT, 1, 4, 1>(p, units, s);
    } else {
      if (!form.shared) launch_tree<DT, 2, 1>(p, units, s);
      else launch_shared<DT, 2, 2, 1>(p, units, s);
    }
  };
  if (cache->dtype == TMH_F32) launch(std::integral_constant<int, DT_F32>{});
  else if (cache->dtype == TMH_F16) launch(std::integral_constant<int, DT_F16>{});
  else launch(std::integral_constant<int, DT_BF16>{});
  return check_launch(ctx, "k_tree_attention");
}

}  // extern "C"
