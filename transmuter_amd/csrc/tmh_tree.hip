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
  int64_t ldq, ldy, max_pages, rows, most;  // most: max_pages * page_size
  PageShape cache;
  int64_t head_stride;
  int window, words, B, group, kv_heads, head_dim;
  uint32_t workers;
  FastDiv by_group;
  float scale;  // of the scores in base-2 logarithms: scale * log2(e)
};

template <int UT, int M>
__device__ __forceinline__ Draft draft_at(const TreeArgs& p, int b) {
  return draft_of(p.starts[b], p.starts[b + 1], p.rows, p.lengths[b], p.most, p.window, UT, p.group, M);
}
template <int UT, int M>
__device__ __forceinline__ uint32_t work_at(const TreeArgs& p, int b) {  // units of one kv head's tiles
  const Draft d = draft_at<UT, M>(p, b);
  return static_cast<uint32_t>(d.units) * static_cast<uint32_t>(d.tiles);
}

// All units of one kv head, by one wavefront.
template <int UT, int M>
__device__ __forceinline__ uint32_t all_work(const TreeArgs& p) {
  uint32_t n = 0;
  for (int i = threadIdx.x & 63; i < p.B; i += 64) n += work_at<UT, M>(p, i);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) n += __shfl_xor(n, o);
  return __builtin_amdgcn_readfirstlane(n);  // (known to be the same in all lanes, as what follows from it then is)
}

// The sequence whose units hold `target` (below the total), and the units before it.
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
  return p.B;  // (not reached: target is below the total)
}

// Where unit `at` lies: its sequence, the item (one kv head and tile of columns) and the item's first unit. An item beyond
// the sequence's (which only rows that are counted twice, by starts that fall, can give) ends a worker.
struct Place {
  uint32_t item, first;
};
__device__ __forceinline__ Place place_in(const Draft& d, uint32_t before, uint32_t at) {
  const uint32_t units = static_cast<uint32_t>(d.units), item = (at - before) / units;
  return {item, before + item * units};
}

template <int DT>
__device__ __forceinline__ void store_answer(const TreeArgs& p, int64_t row, int head, int dim, float4_t o) {
  const int64_t out = row * p.ldy + static_cast<int64_t>(head) * p.head_dim + dim;
  if constexpr (DT == DT_F32)
    *reinterpret_cast<float4_t*>(static_cast<float*>(p.y) + out) = o;
  else
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.y) + out) = make_uint2(pack2<DT>(o[0], o[1]), pack2<DT>(o[2], o[3]));
}

// A lane's answers of one column, dimension 128 nb + 8 (4 g + i) + e in element i of acc[nb][e].
template <int DT, int NB>
__device__ __forceinline__ void answer_columns(const TreeArgs& p, const Draft& d, int kv_head, int column, int g, const float4_t (&acc)[NB][8],
                                               float total) {
  const int n = static_cast<int>(p.by_group.div(static_cast<uint32_t>(column)));
  const float each = total == 0.f ? 0.f : 1.f / total;
  uint16_t* y = static_cast<uint16_t*>(p.y) + (d.row + n) * p.ldy + static_cast<int64_t>(kv_head * p.group + column - n * p.group) * p.head_dim;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int dim = 128 * nb + 8 * (4 * g + i);
      if (dim >= p.head_dim) continue;
      uint4_t out;
#pragma unroll
      for (int x = 0; x < 4; ++x)  // (0 * an infinity is none)
        out[x] = total == 0.f ? 0u : pack2<DT>(acc[nb][2 * x][i] * each, acc[nb][2 * x + 1][i] * each);
      *reinterpret_cast<uint4_t*>(y + dim) = out;
    }
}

// Whether 16 bytes hold an infinity or a NaN.
template <int DT>
__device__ __forceinline__ bool not_finite(uint4_t x) {
  constexpr uint32_t e = DT == DT_F32 ? 0x7F800000u : DT == DT_F16 ? 0x7C00u : 0x7F80u;
  bool any = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = x[i];
    if constexpr (DT == DT_F32) any |= (w & e) == e;
    else any |= (w & e) == e || (w >> 16 & e) == e;
  }
  return any;
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

// Columns [first, first + columns) of an item over its tokens [from, to), one after another, each product in f32 of what a column
// sees alone: the workgroups' way where a column does not see a token that holds an infinity or a NaN, which a weight of 0 would
// leave in a matrix product. put(column of these, dimension, sum) and total(column of these, maximum, sum) take the answers; the
// maxima are of scores in base-2 logarithms. `room` is THREADS floats of LDS.
template <int DT, int THREADS, typename Put, typename Total>
__device__ __forceinline__ void each_alone(const TreeArgs& p, const Draft& d, const int32_t* table, int kv_head, int first, int columns, int from,
                                           int to, float* room, Put put, Total total) {
  constexpr float FACTOR = DT == DT_F16 ? 0x1p15f : 0x1p-32f;
  const int tid = threadIdx.x, dim = p.head_dim, groups = THREADS / dim, mine = tid / dim;
  const int64_t head_at = static_cast<int64_t>(kv_head) * p.head_stride;
#pragma unroll 1
  for (int c = 0; c < columns; ++c) {
    const int of_all = first + c, node = static_cast<int>(p.by_group.div(static_cast<uint32_t>(of_all)));
    const uint64_t* mask = p.mask ? p.mask + static_cast<int64_t>(d.row + node) * p.words : nullptr;
    int begin = 0;
    if (p.window > 0) begin = mask ? tree_begin(mask, p.words, d.prefix, d.nodes, p.window) : chain_begin(node, d.prefix, p.window);
    const int64_t q = (d.row + node) * p.ldq + static_cast<int64_t>(kv_head * p.group + of_all - node * p.group) * dim;
    float top = kNone, sum = 0.f, o = 0.f;  // o: dimension tid % dim, tokens of this group of threads
#pragma unroll 1
    for (int t0 = from; t0 < to; t0 += THREADS) {
      const int token = t0 + tid, some = min(THREADS, to - t0);
      float t = kNone;
      if (token < to && token >= begin) {
        const int64_t row = token_offset(p.cache, table, static_cast<uint32_t>(token));
        const bool seen = row >= 0 && (token < d.prefix || ((mask ? tree_bits(mask, p.words, token - d.prefix) : chain_bits(node, token - d.prefix)) & 1u));
        if (seen) {
          float dot = 0.f;
#pragma unroll 1
          for (int i = 0; i < dim; ++i) dot = fmaf(load_as_f32<DT>(p.q, q + i), load_as_f32<DT>(p.k, row + head_at + i), dot);
          t = dot * p.scale;
        }
      }
      __syncthreads();
      room[tid] = t;
      __syncthreads();
      float next = top;
#pragma unroll 1
      for (int i = 0; i < some; ++i) next = fmaxf(next, room[i]);
      const float keep = next == top ? 1.f : __builtin_amdgcn_exp2f(top - next), ref = next == kNone ? 0.f : next;
      top = next;
      sum *= keep;
      o *= keep;
#pragma unroll 1
      for (int i = 0; i < some; ++i) {
        const float score = room[i];
        if (score == kNone) continue;
        const float w = __builtin_amdgcn_exp2f(score - ref) * FACTOR;
        sum += w;
        if (mine < groups && i % groups == mine) {
          const int64_t row = token_offset(p.cache, table, static_cast<uint32_t>(t0 + i));
          o = fmaf(w, load_as_f32<DT>(p.v, row + head_at + tid - mine * dim), o);
        }
      }
    }
    __syncthreads();
    room[tid] = o;
    __syncthreads();
    if (tid < dim) {
      for (int i = 1; i < groups; ++i) o += room[i * dim + tid];
      put(c, tid, o, sum);
    }
    if (tid == 0) total(c, top, sum);
  }
  __syncthreads();
}

// A tile of M = 16 CB columns (a column: one query head of one node) over a run of units of its sequence's tokens, four
// wavefronts each taking the tiles of TILE tokens of a unit in turn, as attention of one token does (k_paged_attention):
// S^T = K Q^T and O^T = V^T P^T with a token's row as it lies in memory, probabilities staying in the lanes that
// computed them, in two 16-bit parts. K's and V's 16 bytes a lane are used for CB products each, so that a tree's
// rows read the cache once together.
// What a column sees of the step's own tokens is 32 bits a tile; what it does not see has a weight of 0, and where
// an infinity or NaN is there (found by looking at V where the columns differ) the item is done again, by each_alone.
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
  const uint32_t stop = min(at + per, all), run = at;
  uint32_t before;
  int b = find_draft<UT, M>(p, at / p.kv_heads, before);
  if (b >= p.B) return;
  Draft d = draft_at<UT, M>(p, b);
  before *= p.kv_heads;  // the first unit of the sequence's first item
  const int chunks_of_row = (p.head_dim + 4 * E - 1) / (4 * E);
  const bool ragged = p.head_dim % (4 * E) != 0;
  while (at < stop) {
    while (at - before >= static_cast<uint32_t>(d.units) * d.tiles * p.kv_heads) {
      before += static_cast<uint32_t>(d.units) * d.tiles * p.kv_heads;
      if (++b >= p.B) return;
      d = draft_at<UT, M>(p, b);
    }
    const Place place = place_in(d, before, at);
    const uint32_t from = at - place.first, to = min(stop - place.first, static_cast<uint32_t>(d.units));
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
    // Whether a column does not see a token of the tile that holds an infinity or a NaN, which a weight of 0 would not hide.
    auto hides = [&](uint32_t valid) {
      bool mixed = false, any = false;
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) mixed |= sees[cb] != valid;
      if (!__ballot(mixed)) return false;
#pragma unroll
      for (int j = 0; j < VT; ++j)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) any |= not_finite<DT>(vf[j][nb]);
      return __ballot(any) != 0;
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
    bool alone = false;  // a column does not see an infinity or a NaN
    for (uint32_t u = from; u < to; ++u) {
      const uint32_t valid = static_cast<uint32_t>(__ballot(found >= 0)) & WHOLE;  // (TILE 16: the four copies agree)
      const int64_t next_row = coming < 0 ? 0 : coming;
      const bool more = u + 1 < to;
      found = coming;
      coming = look(u + 2);
      scores();
      if (more) load_k(next_row);
      const bool masked = look_at(first_of(u), valid);
      if (masked) alone |= hides(valid);
      softmax(masked);
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
    const uint32_t slot = part_place(worker, at == run);
    at = place.first + to;
    if (__syncthreads_or(alone)) {
      each_alone<DT, 256>(
          p, d, table, kv_head, tile * M, columns, (d.unit + static_cast<int>(from)) * UT, min(d.end, (d.unit + static_cast<int>(to)) * UT),
          &lds_o[0][0][0],
          [&](int c, int dim, float o, float sum) {
            const int of_all = tile * M + c, n = static_cast<int>(p.by_group.div(static_cast<uint32_t>(of_all)));
            if (whole) store_as<DT>(p.y, (d.row + n) * p.ldy + static_cast<int64_t>(kv_head * p.group + of_all - n * p.group) * p.head_dim + dim, sum == 0.f ? 0.f : o * (1.f / sum));
            else p.part[(static_cast<int64_t>(slot) * M + c) * p.head_dim + dim] = o;
          },
          [&](int c, float top, float sum) {
            if (!whole) p.stats[static_cast<int64_t>(slot) * M + c] = make_float2(top, sum);
          });
      continue;
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
          const int64_t row = static_cast<int64_t>(slot) * M + 16 * cb + c;
          *reinterpret_cast<float4_t*>(p.part + row * p.head_dim + dim) = o;
          if (dim == 0) p.stats[row] = make_float2(top, total);
        }
      }
      __syncthreads();
    }
  }
}

// The parts of an item that several workers shared: workgroup (w, i) sees to 16 columns of the item that begins in worker w
// and goes on in the next.
template <int DT, int M>
__global__ __launch_bounds__(256) void k_tree_join(TreeArgs p) {
  constexpr int UT = DT == DT_F32 ? 64 : 128;
  const uint32_t all = all_work<UT, M>(p) * p.kv_heads, per = units_per_worker(all, p.workers);
  const uint32_t cut = (blockIdx.x + 1) * per;  // the first unit of the next worker
  if (per == 0 || cut >= all) return;
  uint32_t before;
  const int b = find_draft<UT, M>(p, cut / p.kv_heads, before);
  if (b >= p.B) return;
  const Draft d = draft_at<UT, M>(p, b);
  const Place place = place_in(d, before * p.kv_heads, cut);
  if (place.item >= static_cast<uint32_t>(d.tiles * p.kv_heads) || place.first >= cut) return;
  const Parts parts = parts_of(place.first, static_cast<uint32_t>(d.units), per);
  if (parts.from != blockIdx.x || parts.from + parts.count > p.workers) return;
  const int kv_head = static_cast<int>(place.item) / d.tiles, tile = static_cast<int>(place.item) % d.tiles;
  const int first_column = 16 * blockIdx.y, some = min(16, min(M, d.nodes * p.group - tile * M) - first_column);
  const int quads = p.head_dim / 4;
  for (int i = threadIdx.x; i < some * quads; i += 256) {
    const int c = first_column + i / quads, dim = (i % quads) * 4;
    auto row_of = [&](uint32_t k) { return static_cast<int64_t>(place_of(parts, k)) * M + c; };
    float top = kNone, total = 0.f;
    for (uint32_t k = 0; k < parts.count; ++k) top = fmaxf(top, p.stats[row_of(k)].x);
    float4_t o{0.f, 0.f, 0.f, 0.f};
    for (uint32_t k = 0; k < parts.count; ++k) {
      const float2 st = p.stats[row_of(k)];
      const float f = st.x == top ? 1.f : __builtin_amdgcn_exp2f(st.x - top);
      total += f * st.y;
      o += f * *reinterpret_cast<const float4_t*>(p.part + row_of(k) * p.head_dim + dim);
    }
    const int of_all = tile * M + c, n = static_cast<int>(p.by_group.div(static_cast<uint32_t>(of_all)));
    store_answer<DT>(p, d.row + n, kv_head * p.group + of_all - n * p.group, dim,
                     total == 0.f ? float4_t{0.f, 0.f, 0.f, 0.f} : o * (1.f / total));
  }
}

// Sixteen bytes a lane from memory into LDS at lds + 16 * lane, past the registers. `lds` must be wavefront-uniform.
__device__ __forceinline__ void to_lds16(const char* from, uint8_t* lds) {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from, (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
#endif
}

// The same for tiles of many columns, M = 64 C, whose products a wavefront's own columns do not keep waiting for memory: eight
// wavefronts, four groups of 16 C columns for each half of a unit's tokens, read K and V from LDS, where all of them bring the
// next unit meanwhile (a stage is 64 KiB, two of them fit a CU). Rows lie in LDS as in memory, K's pieces of 16 bytes moved within
// their row so that the sixteen rows a product reads at once lie on different banks.
// Scores' maxima are kept as they come from the products: a probability is 2^(s a - m a + F) with the scale's magnitude a (its
// sign goes to the queries), one fused multiply-add ahead of the exponential. What m a is rounded by is in all of a column's
// weights and drops out.
template <int DT, int NB, int C>
__global__ __launch_bounds__(512, 2) void k_tree_shared(TreeArgs p) {
  constexpr int TW = 64 / NB, UT = 2 * TW, M = 64 * C;  // a wavefront's tokens of a unit
  constexpr int W = TW / 32, NC = 4 * NB, PITCH = 256 * NB;
  constexpr int STAGE = 2 * UT * PITCH;
  constexpr int RI = 4 / NB, RW = TW / 4;  // rows that an instruction brings, and a wavefront
  constexpr float F = DT == DT_F16 ? 15.f : -32.f;
  __shared__ __align__(16) uint8_t lds[2][STAGE];
  __shared__ float lds_m[4][16 * C], lds_l[4][16 * C];
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wc = wave & 3, wt = wave >> 2;
  const uint32_t worker = blockIdx.x;
  const int quads = p.head_dim / 4;
  for (int b = static_cast<int>(worker); b < p.B; b += static_cast<int>(p.workers)) {
    const Draft d = draft_at<UT, M>(p, b);
    if (d.units != 0) continue;
    const int64_t of_row = static_cast<int64_t>(p.group) * p.kv_heads * quads;
    for (int64_t i = threadIdx.x; i < d.nodes * of_row; i += 512)
      store_answer<DT>(p, d.row + i / of_row, 0, 4 * static_cast<int>(i % of_row), float4_t{0.f, 0.f, 0.f, 0.f});
  }
  const uint32_t all = all_work<UT, M>(p) * p.kv_heads, per = units_per_worker(all, p.workers);
  uint32_t at = worker * per;
  if (per == 0 || at >= all) return;
  const uint32_t stop = min(at + per, all), run = at;
  uint32_t before;
  int b = find_draft<UT, M>(p, at / p.kv_heads, before);
  if (b >= p.B) return;
  Draft d = draft_at<UT, M>(p, b);
  before *= p.kv_heads;
  // Pieces of a row past head_dim are brought by nobody: zeros for all units.
  if (p.head_dim < 128 * NB) {
    for (int i = threadIdx.x; i < 2 * STAGE / 16; i += 512) reinterpret_cast<uint4_t*>(&lds[0][0])[i] = uint4_t{0u, 0u, 0u, 0u};
    __syncthreads();
  }
  // (A scale of 0: queries of zeros, so that -infinity times it stays what it is.)
  const float a = p.scale == 0.f ? 1.f : fabsf(p.scale);
  const uint32_t sign = p.scale < 0.f ? 0x80008000u : 0u;
  while (at < stop) {
    while (at - before >= static_cast<uint32_t>(d.units) * d.tiles * p.kv_heads) {
      before += static_cast<uint32_t>(d.units) * d.tiles * p.kv_heads;
      if (++b >= p.B) return;
      d = draft_at<UT, M>(p, b);
    }
    const Place place = place_in(d, before, at);
    const uint32_t from = at - place.first, to = min(stop - place.first, static_cast<uint32_t>(d.units));
    const int kv_head = static_cast<int>(place.item) / d.tiles, tile = static_cast<int>(place.item) % d.tiles;
    const int columns = min(M, d.nodes * p.group - tile * M);
    const char* kb = static_cast<const char*>(p.k) + static_cast<int64_t>(kv_head) * p.head_stride * 2;
    const char* vb = static_cast<const char*>(p.v) + static_cast<int64_t>(kv_head) * p.head_stride * 2;
    const int32_t* table = p.table + static_cast<int64_t>(b) * p.max_pages;

    uint4_t qf[C][NC];
    int node[C], begin[C];
    uint64_t word[C];  // of masks of one word
#pragma unroll
    for (int cb = 0; cb < C; ++cb) {
      const int of_all = tile * M + min(16 * (C * wc + cb) + col, columns - 1);
      node[cb] = static_cast<int>(p.by_group.div(static_cast<uint32_t>(of_all)));
      const int head = kv_head * p.group + of_all - node[cb] * p.group;
      begin[cb] = 0;
      const uint64_t* mask = p.mask + static_cast<int64_t>(d.row + node[cb]) * p.words;
      word[cb] = p.mask ? mask[0] : 0;
      if (p.window > 0) begin[cb] = p.mask ? tree_begin(mask, p.words, d.prefix, d.nodes, p.window) : chain_begin(node[cb], d.prefix, p.window);
#pragma unroll
      for (int x = 0; x < NC; ++x) {
        const int dim = 32 * x + 8 * g;
        qf[cb][x] = uint4_t{0u, 0u, 0u, 0u};
        if (dim < p.head_dim && p.scale != 0.f)
          qf[cb][x] = *reinterpret_cast<const uint4_t*>(static_cast<const char*>(p.q) +
                                                        ((d.row + node[cb]) * p.ldq + static_cast<int64_t>(head) * p.head_dim + dim) * 2);
        qf[cb][x] ^= sign;
      }
    }
    float m[C], l[C];  // of column 16 (C wc + cb) + col, l over this lane's tokens only
    float4_t acc[C][NB][8];
#pragma unroll
    for (int cb = 0; cb < C; ++cb) {
      m[cb] = kNone;
      l[cb] = 0.f;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[cb][nb][e] = float4_t{0.f, 0.f, 0.f, 0.f};
    }

    // Lane i looks token i % TW of its wavefront's half of a unit up, in two steps: the page's number is loaded a unit before it is
    // looked at, which would wait for the rows that are on their way by then. A row's offset in bytes, -1 where there is none.
    auto first_of = [&](uint32_t u) { return (d.unit + static_cast<int>(u)) * UT + wt * TW; };
    auto page_of = [&](uint32_t u) { return table[p.cache.by_page.div(static_cast<uint32_t>(min(first_of(u) + lane % TW, d.end - 1)))]; };
    auto offset_of = [&](uint32_t u, int32_t id) -> int64_t {
      const int token = first_of(u) + lane % TW;
      if (u >= to || token >= d.end || id < 0 || id >= p.cache.pages) return -1;
      const uint32_t place = static_cast<uint32_t>(token) - p.cache.by_page.div(static_cast<uint32_t>(token)) * p.cache.by_page.d;
      return (id * p.cache.page_stride + place * p.cache.token_stride) * 2;
    };
    // Brings a unit's rows: a wavefront a quarter of its half's (rows that are masked: row 0 of page 0, not used).
    auto bring = [&](int64_t offset, int stage) {
      const int64_t row = offset < 0 ? 0 : offset;
      int64_t from_row[RW / RI];
#pragma unroll
      for (int j = 0; j < RW / RI; ++j) from_row[j] = __shfl(row, RW * wc + RI * j + lane / (16 * NB));
      auto each = [&](auto whole) {
#pragma unroll
        for (int j = 0; j < RW / RI; ++j) {
          const int mine = RW * wc + RI * j + lane / (16 * NB), slot = lane % (16 * NB);  // row of the half, piece of the row
          uint8_t* to_k = &lds[stage][(wt * TW + RW * wc + RI * j) * PITCH];
          const int piece = slot ^ frag_swizzle<16>(mine);
          if (whole || 8 * piece < p.head_dim) to_lds16(kb + from_row[j] + 16 * piece, to_k);
          if (whole || 8 * slot < p.head_dim) to_lds16(vb + from_row[j] + 16 * slot, to_k + UT * PITCH);
        }
      };
      if (p.head_dim == 128 * NB) each(std::true_type{});
      else each(std::false_type{});
    };
    // All of a workgroup's rows have come, and no wavefront reads the unit before any more.
    auto meet = [&] {
      __builtin_amdgcn_s_waitcnt(0);
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    };

    // What each of the lane's columns sees of the 32 tokens from `first` on, `valid` of which there are.
    auto sees = [&](int cb, int first, uint32_t valid) {
      if (first + 32 > d.prefix) {
        if (!p.mask) valid &= chain_bits(node[cb], first - d.prefix);
        else if (p.words == 1) valid &= tree_bits(&word[cb], 1, first - d.prefix);
        else valid &= tree_bits(p.mask + static_cast<int64_t>(d.row + node[cb]) * p.words, p.words, first - d.prefix);
      }
      if (p.window > 0) valid &= from_bits(begin[cb], first);
      return valid;
    };
    // 16 bytes of V of each of a lane's tokens 32 w + 16 (j / 4) + 4 g + j % 4 of the half.
    auto values_of = [&](int stage, int w, int nb, uint4_t (&vf)[8]) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        vf[j] = *reinterpret_cast<const uint4_t*>(&lds[stage][(UT + wt * TW + 32 * w + 16 * (j / 4) + 4 * g + j % 4) * PITCH + 256 * nb + 16 * col]);
    };
    // A step of 32 tokens. Its rows are asked of LDS at once, ahead of all products (the compiler would wait for each by itself).
    auto step = [&](int stage, int w, int first, uint32_t valid) {
      uint4_t kf[2][NC], vf[8];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint8_t* row = &lds[stage][(wt * TW + 32 * w + 16 * h + col) * PITCH];
#pragma unroll
        for (int c = 0; c < NC; ++c) kf[h][c] = *reinterpret_cast<const uint4_t*>(row + 16 * ((4 * c + g) ^ frag_swizzle<16>(col)));
      }
      values_of(stage, w, 0, vf);
      __builtin_amdgcn_sched_barrier(0);
      float4_t s[C][2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int cb = 0; cb < C; ++cb) s[cb][h] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int cb = 0; cb < C; ++cb) s[cb][h] = mfma16<DT>(kf[h][c], qf[cb][c], s[cb][h]);
      }
      const bool masked = valid != ~0u || first + 32 > d.prefix || p.window > 0;
      if (masked) {
        asm volatile("");  // (a branch: as selects it would be paid for in every step)
#pragma unroll
        for (int cb = 0; cb < C; ++cb) {
          const uint32_t some = sees(cb, first, valid);
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (!(some >> (16 * h + 4 * g + i) & 1u)) s[cb][h][i] = kNone;
        }
      }
      uint4_t parts[C][2];  // the probabilities' two parts
#pragma unroll
      for (int cb = 0; cb < C; ++cb) {
        float top = kNone;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) top = fmaxf(top, s[cb][h][i]);
        top = column_max(top);
        if (__ballot(top > m[cb])) {
          const float next = fmaxf(m[cb], top);
          const float keep = next == m[cb] ? 1.f : m[cb] == kNone ? 0.f : __builtin_amdgcn_exp2f((m[cb] - next) * a);
          m[cb] = next;
          l[cb] *= keep;
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[cb][nb][e] *= keep;
        }
        const float c = F - (m[cb] == kNone ? 0.f : m[cb] * a);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const float p0 = __builtin_amdgcn_exp2f(fmaf(s[cb][h][2 * x], a, c)), p1 = __builtin_amdgcn_exp2f(fmaf(s[cb][h][2 * x + 1], a, c));
            l[cb] += p0 + p1;
            const uint2 part = cut2<DT>(p0, p1);
            parts[cb][0][2 * h + x] = part.x;
            parts[cb][1][2 * h + x] = part.y;
          }
      }
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        if (nb) values_of(stage, w, nb, vf);
        if (masked) {
          asm volatile("");  // (as above)
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (!(valid >> (16 * (j / 4) + 4 * g + j % 4) & 1u)) vf[j] = uint4_t{0u, 0u, 0u, 0u};
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          uint4_t vt;  // of V's dimension 8 (4 g + i) + e (of block nb) the lane's tokens
#pragma unroll
          for (int x = 0; x < 4; ++x)
            vt[x] = __builtin_amdgcn_perm(vf[2 * x + 1][e >> 1], vf[2 * x][e >> 1], e & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
          for (int cb = 0; cb < C; ++cb) {
            acc[cb][nb][e] = mfma16<DT>(vt, parts[cb][0], acc[cb][nb][e]);
            acc[cb][nb][e] = mfma16<DT>(vt, parts[cb][1], acc[cb][nb][e]);
          }
        }
      }
    };

    int64_t found = offset_of(from, page_of(from));
    int32_t coming = page_of(from + 1);
    __syncthreads();  // the item before has left LDS
    bring(found, 0);
    int stage = 0;
    for (uint32_t u = from; u < to; ++u, stage ^= 1) {
      const uint64_t valid = TW == 64 ? __ballot(found >= 0) : __ballot(found >= 0) & 0xFFFFFFFFu;
      meet();
      found = offset_of(u + 1, coming);
      coming = page_of(u + 2);
      if (u + 1 < to) bring(found, stage ^ 1);
#pragma unroll 1
      for (int w = 0; w < W; ++w) step(stage, w, first_of(u) + 32 * w, static_cast<uint32_t>(valid >> 32 * w));
    }
    // An infinity or a NaN in V leaves a NaN in every column of its products, whether the column sees it or not (0 times an
    // infinity): such an item is done again.
    bool alone = false;
#pragma unroll
    for (int cb = 0; cb < C; ++cb)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x = acc[cb][nb][e][i];
            alone |= x != x;
          }

    const bool whole = from == 0 && to == static_cast<uint32_t>(d.units);
    const int64_t slot = part_place(worker, at == run);
    at = place.first + to;
    if (__syncthreads_or(alone)) {
      each_alone<DT, 512>(
          p, d, table, kv_head, tile * M, columns, (d.unit + static_cast<int>(from)) * UT, min(d.end, (d.unit + static_cast<int>(to)) * UT),
          reinterpret_cast<float*>(&lds[0][0]),
          [&](int c, int dim, float o, float sum) {
            const int of_all = tile * M + c, n = static_cast<int>(p.by_group.div(static_cast<uint32_t>(of_all)));
            if (whole) store_as<DT>(p.y, (d.row + n) * p.ldy + static_cast<int64_t>(kv_head * p.group + of_all - n * p.group) * p.head_dim + dim, sum == 0.f ? 0.f : o * (1.f / sum));
            else p.part[(((slot * 4 * C + c / 16) * (NB * 8) + dim / 128 * 8 + dim % 8) * 64 + dim % 128 / 32 * 16 + c % 16) * 4 + dim % 32 / 8] = o;
          },
          [&](int c, float top, float sum) {
            if (!whole) p.stats[slot * M + c] = make_float2(top, sum);
          });
      if (p.head_dim < 128 * NB) {  // (what it used of LDS may have been pieces of zeros)
        for (int i = threadIdx.x; i < 2 * STAGE / 16; i += 512) reinterpret_cast<uint4_t*>(&lds[0][0])[i] = uint4_t{0u, 0u, 0u, 0u};
        __syncthreads();
      }
      continue;
    }

    // The halves' parts meet in LDS, lane by lane; the first half's wavefronts answer.
    float4_t* mine = reinterpret_cast<float4_t*>(&lds[0][0]) + wc * (C * NB * 8) * 64 + lane;
#pragma unroll
    for (int cb = 0; cb < C; ++cb) l[cb] = column_sum(l[cb]);
    if (wt == 1) {
#pragma unroll
      for (int cb = 0; cb < C; ++cb) {
        if (g == 0) {
          lds_m[wc][16 * cb + col] = m[cb];
          lds_l[wc][16 * cb + col] = l[cb];
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < 8; ++e) mine[((cb * NB + nb) * 8 + e) * 64] = acc[cb][nb][e];
      }
    }
    __syncthreads();
    if (wt == 0) {
#pragma unroll
      for (int cb = 0; cb < C; ++cb) {
        const int c = 16 * (C * wc + cb) + col;
        const float other = lds_m[wc][16 * cb + col], top = fmaxf(m[cb], other);
        const float f0 = m[cb] == top ? 1.f : m[cb] == kNone ? 0.f : __builtin_amdgcn_exp2f((m[cb] - top) * a);
        const float f1 = other == top ? 1.f : other == kNone ? 0.f : __builtin_amdgcn_exp2f((other - top) * a);
        const float total = f0 * l[cb] + f1 * lds_l[wc][16 * cb + col];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[cb][nb][e] = f0 * acc[cb][nb][e] + f1 * mine[((cb * NB + nb) * 8 + e) * 64];
        if (16 * (C * wc + cb) >= columns) continue;
        if (whole) {
          if (c < columns) answer_columns<DT, NB>(p, d, kv_head, tile * M + c, g, acc[cb], total);
        } else {
          float4_t* part = reinterpret_cast<float4_t*>(p.part) + ((slot * 4 + wc) * (C * NB * 8) + cb * NB * 8) * 64 + lane;
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int e = 0; e < 8; ++e) part[(nb * 8 + e) * 64] = acc[cb][nb][e];
          if (g == 0) p.stats[slot * M + c] = make_float2(top == kNone ? kNone : top * a, total);
        }
      }
    }
  }
}

// The parts of an item that several workers shared: workgroup (w, i) sees to 16 columns of the item that begins in worker w
// and goes on in the next, its four wavefronts to every fourth part.
template <int DT, int NB, int C>
__global__ __launch_bounds__(256) void k_tree_shared_join(TreeArgs p) {
  constexpr int UT = 128 / NB, M = 64 * C;
  const uint32_t all = all_work<UT, M>(p) * p.kv_heads, per = units_per_worker(all, p.workers);
  const uint32_t cut = (blockIdx.x + 1) * per;  // the first unit of the next worker
  if (per == 0 || cut >= all) return;
  uint32_t before;
  const int b = find_draft<UT, M>(p, cut / p.kv_heads, before);
  if (b >= p.B) return;
  const Draft d = draft_at<UT, M>(p, b);
  const Place place = place_in(d, before * p.kv_heads, cut);
  if (place.item >= static_cast<uint32_t>(d.tiles * p.kv_heads) || place.first >= cut) return;
  const Parts parts = parts_of(place.first, static_cast<uint32_t>(d.units), per);
  if (parts.from != blockIdx.x || parts.from + parts.count > p.workers) return;
  const int kv_head = static_cast<int>(place.item) / d.tiles, tile = static_cast<int>(place.item) % d.tiles;
  const int block = blockIdx.y;  // 16 columns
  const int columns = min(M, d.nodes * p.group - tile * M);
  if (16 * block >= columns) return;
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  float top = kNone, total = 0.f;
  float4_t acc[NB][8];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[nb][e] = float4_t{0.f, 0.f, 0.f, 0.f};
  auto join = [&](float other, float sum, auto from) {
    const float next = fmaxf(top, other);
    const float f0 = top == next ? 1.f : __builtin_amdgcn_exp2f(top - next), f1 = other == next ? 1.f : __builtin_amdgcn_exp2f(other - next);
    top = next;
    total = f0 * total + f1 * sum;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[nb][e] = f0 * acc[nb][e] + f1 * from(nb * 8 + e);
  };
#pragma unroll 2
  for (uint32_t k = wave; k < parts.count; k += 4) {
    const int64_t slot = place_of(parts, k);
    const float2 st = p.stats[slot * M + 16 * block + col];
    const float4_t* part = reinterpret_cast<const float4_t*>(p.part) + (slot * 4 * C + block) * (NB * 8) * 64 + lane;
    join(st.x, st.y, [&](int i) { return part[i * 64]; });
  }
  __shared__ __align__(16) float4_t sums[3][NB * 8][64];
  __shared__ float2 stats[3][64];
  if (wave) {
    stats[wave - 1][lane] = make_float2(top, total);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int e = 0; e < 8; ++e) sums[wave - 1][nb * 8 + e][lane] = acc[nb][e];
  }
  __syncthreads();
  if (wave) return;
  for (int w = 0; w < 3; ++w) join(stats[w][lane].x, stats[w][lane].y, [&](int i) { return sums[w][i][lane]; });
  if (16 * block + col < columns) answer_columns<DT, NB>(p, d, kv_head, tile * M + 16 * block + col, g, acc, total);
}

template <int DT, int NB, int CB>
void launch_tree(const TreeArgs& p, hipStream_t s) {
  k_tree_attention<DT, NB, CB><<<p.workers, 256, 0, s>>>(p);
  if (p.workers > 1) k_tree_join<DT, 16 * CB><<<dim3(p.workers - 1, CB), 256, 0, s>>>(p);
}
template <int DT, int NB, int C>
void launch_shared(const TreeArgs& p, hipStream_t s) {
  k_tree_shared<DT, NB, C><<<p.workers, 512, 0, s>>>(p);
  if (p.workers > 1) k_tree_shared_join<DT, NB, C><<<dim3(p.workers - 1, 4 * C), 256, 0, s>>>(p);
}

// How columns go to workgroups, by the columns that a sequence has in the mean (all the host knows).
struct TreeForm {
  bool shared;
  int columns, unit, per_cu;  // columns of a tile, tokens of a unit, workgroups a CU
};
TreeForm tree_form(int64_t columns, bool f32, int head_dim) {
  if (f32) return {false, head_dim <= 128 && columns > 16 ? 32 : 16, 64, 2};
  if (columns <= 16) return {false, 16, 128, 2};
  return {true, columns <= 64 || head_dim > 128 ? 64 : 128, head_dim <= 128 ? 128 : 64, 1};
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
  if (max_pages >= (int64_t{1} << 31) / cache->page_size)
    return fail(ctx, TMH_ERR_UNSUPPORTED, "attention needs max_pages * page_size below 2^31");
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
  const TreeForm form = tree_form((T * group + B - 1) / B, f32, cache->head_dim);
  const int64_t unit = form.unit;
  const int64_t most = max_pages * cache->page_size;
  const int64_t items = (T * group / form.columns + B) * cache->kv_heads;
  if ((most + unit - 1) / unit >= (int64_t{1} << 31) / items)
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
  p.workers = static_cast<uint32_t>(std::max<int64_t>(1, std::min<int64_t>(form.per_cu * ctx->num_cus, (most + unit - 1) / unit * items)));
  hipStream_t s = pick_stream(ctx, stream);
  const size_t rows = 2 * static_cast<size_t>(form.per_cu * ctx->num_cus) * form.columns;
  const int width_of_part = form.shared ? (cache->head_dim <= 128 ? 128 : 256) : cache->head_dim;
  void* ws = workspace(ctx, rows * (width_of_part * 4 + sizeof(float2)), s);
  if (!ws) return fail(ctx, TMH_ERR_UNSUPPORTED, "attention's workspace cannot grow here: run one call before the capture");
  p.part = static_cast<float*>(ws);
  p.stats = reinterpret_cast<float2*>(p.part + rows * width_of_part);
  auto launch = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if constexpr (DT == DT_F32) {
      if (cache->head_dim <= 64) form.columns == 16 ? launch_tree<DT, 1, 1>(p, s) : launch_tree<DT, 1, 2>(p, s);
      else if (cache->head_dim <= 128) form.columns == 16 ? launch_tree<DT, 2, 1>(p, s) : launch_tree<DT, 2, 2>(p, s);
      else launch_tree<DT, 4, 1>(p, s);
    } else if (cache->head_dim <= 128) {
      if (!form.shared) launch_tree<DT, 1, 1>(p, s);
      else form.columns == 64 ? launch_shared<DT, 1, 1>(p, s) : launch_shared<DT, 1, 2>(p, s);
    } else {
      if (!form.shared) launch_tree<DT, 2, 1>(p, s);
      else launch_shared<DT, 2, 1>(p, s);
    }
  };
  if (cache->dtype == TMH_F32) launch(std::integral_constant<int, DT_F32>{});
  else if (cache->dtype == TMH_F16) launch(std::integral_constant<int, DT_F16>{});
  else launch(std::integral_constant<int, DT_BF16>{});
  return check_launch(ctx, "k_tree_attention");
}

}  // extern "C"
