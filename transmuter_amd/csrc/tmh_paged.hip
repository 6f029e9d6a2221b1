// A paged cache of keys and values: rotary positions and the new tokens into their slots
// (tmh_paged_append), and attention of one new token a sequence over its pages (tmh_paged_attention).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "tmh_f8.h"
#include "tmh_internal.h"

namespace tmh {
namespace {

// ------------------------------------------------------------------ append

struct AppendArgs {
  const void* q;
  const void* k;
  const void* v;
  const int64_t* positions;
  const void* cos;
  const void* sin;
  const int64_t* slots;
  void* q_out;
  void* k_cache;
  void* v_cache;
  int64_t ldq, ldk, ldv, ldqo, max_positions;
  int64_t page_stride, token_stride, head_stride;
  int64_t num_slots;
  int table_dtype, rotary, interleaved, heads, kv_heads;
  // A token's pieces: of each query and key head (`turned` of them pairs of eight dimensions half a rotary row
  // apart), then of each value head.
  uint32_t pieces, value_pieces;
  int turned, head_dim;
  FastDiv by_pieces, by_head, by_value, by_page;
};

// Eight entries of a rotary table row.
__device__ __forceinline__ void load_table(const void* p, int dtype, int64_t at, bool vec, float (&v)[8]) {
  if (vec && dtype == DT_F32) load8<DT_F32, true>(p, at, 8, v);
  else if (vec && dtype == DT_F16) load8<DT_F16, true>(p, at, 8, v);
  else if (vec) load8<DT_BF16, true>(p, at, 8, v);
  else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = load_float_rt(p, dtype, at + i);
  }
}

// A thread answers eight dimensions of one head of one token, and with VEC of those that turn by halves their
// partners too. VEC: rows and partners lie on 16 bytes. Bound by memory: 4096 bf16 tokens of 32 and 4 heads of 128
// 16.8 us, 5.1 TB/s (20.0 with each half read by two threads).
template <int DT, bool VEC>
__global__ __launch_bounds__(256) void k_paged_append(AppendArgs p, int64_t first, uint32_t count, bool table_vec, bool pairs_vec) {
  // Every line of the arguments at once: one that is first looked at further on would cost its way then (1000 f16 tokens
  // 6.8 us without this, 6.2 with it).
  asm volatile("" ::"s"(p.q), "s"(p.k_cache), "s"(p.num_slots), "s"(p.by_page.d), "s"(count));
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i >= count) return;
  const uint32_t tl = p.by_pieces.div(i);
  const int64_t t = first + tl;
  const uint32_t piece = i - tl * p.pieces;
  const bool is_v = piece >= p.pieces - p.value_pieces;
  const uint32_t local = is_v ? piece - (p.pieces - p.value_pieces) : piece;
  const FastDiv by = is_v ? p.by_value : p.by_head;
  const int head = static_cast<int>(by.div(local)), at = static_cast<int>(local - head * by.d), head_dim = p.head_dim;
  const bool is_q = !is_v && head < p.heads, is_k = !is_v && !is_q, pair = !is_v && at < p.turned;
  const int dim = 8 * (is_v || pair ? at : at + p.turned);
  int64_t slot = 0;
  if (!is_q) {
    slot = p.slots[t];
    if (slot < 0 || slot >= p.num_slots) return;
  }
  const void* src = is_q ? p.q : is_k ? p.k : p.v;
  const int h = is_k ? head - p.heads : head;
  const int64_t row = (is_q ? p.ldq : is_k ? p.ldk : p.ldv) * t + static_cast<int64_t>(h) * head_dim;
  auto put = [&](int at, const float (&x)[8]) {
    if (is_q) {
      store8<DT, VEC>(p.q_out, t * p.ldqo + static_cast<int64_t>(h) * head_dim + at, 8, x);
    } else {
      const uint32_t page = p.by_page.div(static_cast<uint32_t>(slot));
      const uint32_t place = static_cast<uint32_t>(slot) - page * p.by_page.d;
      store8<DT, true>(is_k ? p.k_cache : p.v_cache,
                       page * p.page_stride + place * p.token_stride + h * p.head_stride + at, 8, x);
    }
  };
  float v[8];
  load8<DT, VEC>(src, row + dim, 8, v);
  if ((is_q || is_k) && dim < p.rotary) {
    const int64_t position = min(max(p.positions[t], int64_t{0}), p.max_positions - 1);
    const int half = p.rotary / 2;
    const int64_t table = position * half;
    if (p.interleaved) {
      float c[4], s[4];
      if (pairs_vec) {
        const float4_t cv = *reinterpret_cast<const float4_t*>(static_cast<const float*>(p.cos) + table + dim / 2);
        const float4_t sv = *reinterpret_cast<const float4_t*>(static_cast<const float*>(p.sin) + table + dim / 2);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          c[j] = cv[j];
          s[j] = sv[j];
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bool in = dim + 2 * j < p.rotary;
          c[j] = in ? load_float_rt(p.cos, p.table_dtype, table + dim / 2 + j) : 1.f;
          s[j] = in ? load_float_rt(p.sin, p.table_dtype, table + dim / 2 + j) : 0.f;
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (!pairs_vec && dim + 2 * j >= p.rotary) continue;
        const float a = v[2 * j], b = v[2 * j + 1];
        v[2 * j] = a * c[j] - b * s[j];
        v[2 * j + 1] = fmaf(a, s[j], b * c[j]);
      }
    } else if (VEC) {  // a pair
      float o[8], c[8], s[8];
      load8<DT, VEC>(src, row + dim + half, 8, o);
      load_table(p.cos, p.table_dtype, table + dim, table_vec, c);
      load_table(p.sin, p.table_dtype, table + dim, table_vec, s);
      float high[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        high[j] = fmaf(v[j], s[j], o[j] * c[j]);
        v[j] = v[j] * c[j] - o[j] * s[j];
      }
      put(dim + half, high);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int d = dim + j;
        if (d >= p.rotary) continue;
        const bool low = d < half;
        const int at = low ? d : d - half;
        const float o = load_as_f32<DT>(src, row + (low ? d + half : d - half));
        const float c = load_float_rt(p.cos, p.table_dtype, table + at);
        const float s = load_float_rt(p.sin, p.table_dtype, table + at);
        v[j] = low ? v[j] * c - o * s : fmaf(o, s, v[j] * c);
      }
    }
  }
  put(dim, v);
}

template <int DT>
void launch_append(const AppendArgs& p, int64_t T, bool vec, bool table_vec, bool pairs_vec, hipStream_t s) {
  const int64_t most = ((int64_t{1} << 31) - 256) / p.pieces;  // tokens a launch, within the divisions' range
  for (int64_t first = 0; first < T; first += most) {
    const uint32_t count = static_cast<uint32_t>(std::min(most, T - first) * p.pieces);
    const unsigned grid = (count + 255) / 256;
    if (vec) k_paged_append<DT, true><<<grid, 256, 0, s>>>(p, first, count, table_vec, pairs_vec);
    else k_paged_append<DT, false><<<grid, 256, 0, s>>>(p, first, count, table_vec, pairs_vec);
  }
}

// ------------------------------------------------------------------ attention

constexpr float kNone = -__builtin_inff();
constexpr uint32_t kNowhere = 1u << 31;  // an offset past every buffer's range here
constexpr int kThrough = 16;  // sc1 of a buffer access: past the XCD's L2, to where all XCDs meet
typedef uint32_t uint2_t __attribute__((ext_vector_type(2)));

struct AttendArgs {
  const void* q;
  const void* k;
  const void* v;
  const int32_t* table;
  const int32_t* lengths;
  void* y;
  float* part;    // [2 workers][heads of an item][head_dim], then their (maximum, sum) pairs
  float2* stats;
  uint32_t part_bytes, stats_bytes;
  uint32_t* meet;  // [workers] parts of the item that begins in a worker, kept so far; zero between calls
  int64_t ldq, ldy, max_pages;
  PageShape cache;
  int64_t head_stride;
  int64_t window, most;  // most: max_pages * page_size
  int B, group, kv_heads, chunks, head_dim;
  uint32_t workers;
  FastDiv by_units, by_items;  // EACH: units of an item, items of a sequence
  float scale;  // of the scores in base-2 logarithms: scale * log2(e)
};

template <int UT>
__device__ __forceinline__ Span span_at(const AttendArgs& p, int b) {
  return span_of(p.lengths[b], p.most, p.window, UT);
}

// The units of the sequences before b (all of them for b = B), by one wavefront. (The host has checked that all
// items' units are below 2^31.)
template <int UT>
__device__ __forceinline__ uint32_t units_before(const AttendArgs& p, int b) {
  uint32_t n = 0;
  for (int i = threadIdx.x & 63; i < b; i += 64) n += static_cast<uint32_t>(span_at<UT>(p, i).units);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) n += __shfl_xor(n, o);
  return n;
}

__device__ __forceinline__ uint32_t scan64(uint32_t v) {  // the sum over the lanes up to this one
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t up = __shfl_up(v, o);
    if ((threadIdx.x & 63) >= o) v += up;
  }
  return v;
}

// The sequence whose units hold `target` (below the total), and the units before it.
template <int UT>
__device__ __forceinline__ int find_sequence(const AttendArgs& p, uint32_t target, uint32_t& before) {
  const int lane = threadIdx.x & 63;
  uint32_t base = 0;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    const uint32_t mine = b0 + lane < p.B ? static_cast<uint32_t>(span_at<UT>(p, b0 + lane).units) : 0;
    const uint32_t sum = scan64(mine);
    const uint64_t past = __ballot(base + sum > target);
    if (past) {
      const int at = __builtin_ctzll(past);
      before = base + __shfl(sum - mine, at);
      return b0 + at;
    }
    base += __shfl(sum, 63);
  }
  before = base;
  return p.B - 1;  // (not reached: target is below the total)
}

// (By value: __builtin_bit_cast of a vector's element, an lvalue, reads element 0.)
__device__ __forceinline__ float as_float(uint32_t v) { return __builtin_bit_cast(float, v); }

template <int DT>
struct Lane16 {  // 16 bytes of a lane as MFMA operands
  typedef _Float16 vec __attribute__((ext_vector_type(8)));
};
template <>
struct Lane16<DT_BF16> {
  typedef __bf16 vec __attribute__((ext_vector_type(8)));
};

template <int DT>
__device__ __forceinline__ float4_t mfma16(uint4_t a, uint4_t b, float4_t c) {
  typedef typename Lane16<DT>::vec vec;
  if constexpr (DT == DT_F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(vec, a), __builtin_bit_cast(vec, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(vec, a), __builtin_bit_cast(vec, b), c, 0, 0, 0);
}

// Two probabilities as the sums of two 16-bit parts each: cut off, and the rest, rounded. What is cut is a little less
// than the probability, so that the rest is not 0 beside a first part that is not, and an infinity in V stays what
// it is in both products (f16: of probabilities of 2^-23, 2^-38 of the largest, and more; others give NaN with it).
// A probability of 0 gives zeros: a token without weight has no part in the answer, whatever its value.
template <int DT>
__device__ __forceinline__ uint2 split2(float a, float b) {
  constexpr float less = 1.f - 0x1p-20f;
  if constexpr (DT == DT_F16) {
    const auto h = __builtin_amdgcn_cvt_pkrtz(fmaf(a, less, -0x1p-24f), fmaf(b, less, -0x1p-24f));
    return make_uint2(__builtin_bit_cast(uint32_t, h), pack2<DT>(a - static_cast<float>(h[0]), b - static_cast<float>(h[1])));
  } else {
    const uint32_t hi = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, b * less), __builtin_bit_cast(uint32_t, a * less), 0x07060302u);
    return make_uint2(hi, pack2<DT>(a - __builtin_bit_cast(float, hi << 16), b - __builtin_bit_cast(float, hi & 0xFFFF0000u)));
  }
}

// The maximum (sum) over the four lanes of one column of an MFMA tile, in all of them.
__device__ __forceinline__ float column_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float column_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// One workgroup's share of the units. Four wavefronts take the tiles of a unit (TILE tokens each), with
// running maxima, sums and answers of their own, which meet in LDS where an item ends or the share does.
//
// A tile: S^T = K Q^T on MFMA, a lane's operand rows being 16 bytes of a token's row as it lies in memory (both
// operands take the dimensions in the same order, any order). A lane then holds four (two times four, TILE 32)
// tokens' scores of one head, column l & 15, which are the operand that O^T = V^T P^T wants in the order
// token(g, j) = 16 (j / 4) + 4 g + j % 4 of its lane row g = l / 16: no score leaves its lane. V's rows come
// as they lie in memory too, 16 bytes of token(g, j) a lane (a load reads four whole rows of 128 dimensions),
// and pairs of tokens are put side by side with one v_perm_b32 per two values. The answer's dimension
// E (4 g + i) + e (of a block of 16 E, E values to 16 bytes) lies in element i of product e: a lane's answers of one i
// are 16 consecutive bytes.
// f32: the same with v_mfma_f32_16x16x4_f32, whose operands are single values.
//
// Probabilities are split into two 16-bit parts, each multiplied: the sum keeps 16 bits (bf16) or 21 (f16, and
// multiples of 2^-39 of the largest) of each (one part would round each to 8 or 11, as far off as the answer's own type).
// f16 parts are taken of 2^15 times the probability, so that small ones of long rows do not fall below f16's
// range; f32 and bf16 ones of 2^-32 times it, so that sums of up to 2^31 values near the type's largest stay
// finite. The factor is in the running sum too and drops out.
//
// Bound by memory where there are many tokens: 4 x 131072 f16 181 us, 5.7 TB/s; 32 x 1..8000 bf16 57.2 us, 4.6 TB/s,
// of which about 12 us are the way in (lengths, page table, first rows) and out; one sequence of 700 tokens 7.5 us,
// all of it such ways. Runs of units of equal number to each of two workgroups a CU (their registers' limit) even
// ragged lengths out; three a CU would spill.
//
// What happens to items that several workers share:
//  JOIN  they meet here. Each leaves its part in memory (stores that pass the XCD's own L2), then counts itself; the one that
//        finds all others counted joins the parts in their order, whoever it is, so the answer does not depend on who comes
//        last.
//  PARTS k_paged_join joins them.
//  WHOLE there are none: a workgroup (WHOLE8: of eight wavefronts) takes an item, and looks at its own sequence's length only.
//  EACH  JOIN with a worker to each unit that the table has room for, where no window moves them: a worker knows its
//        tokens without the lengths, so that it looks their pages up meanwhile. Those past the length leave.
template <int DT, int NB, int HOW>  // NB: blocks of 16 E dimensions
__global__ __launch_bounds__(HOW == WHOLE8 ? 512 : 256, NB == 1 || (DT == DT_F32 && NB == 2) ? 2 : 1) void k_paged_attention(AttendArgs p) {
  // Every line of the arguments at once: one that is first looked at further on would cost its way then (us: one token of
  // f16 4.7 without this, 4.5 with it; of f32 and 256 dimensions 8.9 and 8.3).
  asm volatile("" ::"s"(p.q), "s"(p.part_bytes), "s"(p.window), "s"(p.scale));
  constexpr bool F32 = DT == DT_F32, ALONE = HOW == WHOLE || HOW == WHOLE8, MEET = HOW == JOIN || HOW == EACH;
  constexpr int WAVES = HOW == WHOLE8 ? 8 : 4, THREADS = 64 * WAVES;
  constexpr int SIZE = F32 ? 4 : 2, E = 16 / SIZE, TILE = F32 ? 16 : 32, UT = WAVES * TILE;
  constexpr int NH = TILE / 16;           // 16-token halves of a tile
  constexpr int NC = 4 * NB;              // chunks of 4 E dimensions of a row
  constexpr int VT = F32 ? 4 : 8;         // tokens a lane reads of V
  constexpr float FACTOR = DT == DT_F16 ? 0x1p15f : 0x1p-32f;
  constexpr int ROW = 16 * E * NB + 4;    // floats of a head's answer in LDS (+ 4: off a bank's multiple)
  __shared__ __align__(16) float lds_o[WAVES][kHeads][ROW];
  __shared__ float lds_m[WAVES][kHeads], lds_l[WAVES][kHeads];
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t items = static_cast<uint32_t>(p.kv_heads * p.chunks);
  const uint32_t worker = blockIdx.x;
  [[maybe_unused]] const auto parts_rsrc = buffer_rsrc(p.part, p.part_bytes), stats_rsrc = buffer_rsrc(p.stats, p.stats_bytes);
  auto store = [&](int b, int head, int dim, float4_t o) {
    const int64_t out = b * p.ldy + static_cast<int64_t>(head) * p.head_dim + dim;
    if constexpr (F32)
      *reinterpret_cast<float4_t*>(static_cast<float*>(p.y) + out) = o;
    else
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.y) + out) = make_uint2(pack2<DT>(o[0], o[1]), pack2<DT>(o[2], o[3]));
  };
  if constexpr (HOW == JOIN) {  // zeros for the sequences without tokens
    const int quads = p.group * p.kv_heads * p.head_dim / 4;
    for (int b = static_cast<int>(worker); b < p.B; b += static_cast<int>(p.workers))
      if (span_at<UT>(p, b).units == 0)
        for (int i = threadIdx.x; i < quads; i += 256) store(b, 0, 4 * i, float4_t{0.f, 0.f, 0.f, 0.f});
  }
  uint32_t per = 0, at, stop, before = 0;
  int b;
  [[maybe_unused]] uint32_t each_item = 0, each_unit = 0;
  [[maybe_unused]] int32_t length = 0;
  if constexpr (HOW == EACH) {
    const uint32_t of_all = p.by_units.div(worker);
    each_unit = worker - of_all * p.by_units.d;
    b = static_cast<int>(p.by_items.div(of_all));
    each_item = of_all - b * items;
    int of_lane = b;  // (by a vector load, like the table's below: both are then waited for at once)
    asm volatile("" : "+v"(of_lane));
    length = p.lengths[of_lane];
    per = 1;
    at = worker;
    stop = worker + 1;
  } else if constexpr (ALONE) {
    b = static_cast<int>(worker / items);
    const uint32_t units = static_cast<uint32_t>(span_at<UT>(p, b).units), item = worker - b * items;
    at = item * units;
    stop = at + units;
    if (units == 0) {
      const int kv_head = static_cast<int>(item) / p.chunks, chunk = static_cast<int>(item) % p.chunks;
      const int quads = min(kHeads, p.group - chunk * kHeads) * p.head_dim / 4;
      for (int i = threadIdx.x; i < quads; i += THREADS) store(b, kv_head * p.group + chunk * kHeads, 4 * i, float4_t{0.f, 0.f, 0.f, 0.f});
      return;
    }
  } else {
    // Up to 64 sequences: one look at their lengths tells the total and where this worker's units are.
    uint32_t mine = 0, upto = 0, all;
    if (p.B <= 64) {
      mine = lane < p.B ? static_cast<uint32_t>(span_at<UT>(p, lane).units) : 0;
      upto = scan64(mine);
      all = __shfl(upto, 63) * items;
    } else {
      all = units_before<UT>(p, p.B) * items;
    }
    per = units_per_worker(all, p.workers);
    at = worker * per;
    if (per == 0 || at >= all) return;
    stop = min(at + per, all);
    if (p.B <= 64) {
      b = __builtin_ctzll(__ballot(upto > at / items));
      before = __shfl(upto - mine, b);
    } else {
      b = find_sequence<UT>(p, at / items, before);
    }
  }
  [[maybe_unused]] const uint32_t run = at;
  Span sp{};
  if constexpr (HOW != EACH) sp = span_at<UT>(p, b);
  uint32_t first = before * items;  // the first unit of the sequence's first item
  const int chunks_of_row = (p.head_dim + 4 * E - 1) / (4 * E);
  const bool ragged = p.head_dim % (4 * E) != 0;
  while (at < stop) {
    uint32_t item = each_item, item_first = at - each_unit, from = each_unit, to = each_unit + 1;
    if constexpr (HOW != EACH) {
      while (at >= first + static_cast<uint32_t>(sp.units) * items) {
        first += static_cast<uint32_t>(sp.units) * items;
        sp = span_at<UT>(p, ++b);
      }
      item = (at - first) / static_cast<uint32_t>(sp.units);
      item_first = first + item * sp.units;
      from = at - item_first;
      to = min(stop - item_first, static_cast<uint32_t>(sp.units));
    }
    const int kv_head = static_cast<int>(item) / p.chunks, chunk = static_cast<int>(item) % p.chunks;
    const int heads = min(kHeads, p.group - chunk * kHeads);
    const int head0 = kv_head * p.group + chunk * kHeads;
    const char* kb = static_cast<const char*>(p.k) + static_cast<int64_t>(kv_head) * p.head_stride * SIZE;
    const char* vb = static_cast<const char*>(p.v) + static_cast<int64_t>(kv_head) * p.head_stride * SIZE;
    const int32_t* table = p.table + static_cast<int64_t>(b) * p.max_pages;

    uint4_t qf[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      qf[c] = uint4_t{0u, 0u, 0u, 0u};
      const int dim = 4 * E * c + E * g;
      if (col < heads && dim < p.head_dim)
        qf[c] = *reinterpret_cast<const uint4_t*>(static_cast<const char*>(p.q) +
                                                  (b * p.ldq + static_cast<int64_t>(head0 + col) * p.head_dim + dim) * SIZE);
    }
    float m = kNone, l = 0.f;  // of column col, l over this lane's tokens only
    float4_t acc[NB][E];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int e = 0; e < E; ++e) acc[nb][e] = float4_t{0.f, 0.f, 0.f, 0.f};

    // Lane i looks token i % TILE of a unit's tile up, a unit ahead: its row's offset in bytes, -1 where it is masked.
    auto look = [&](uint32_t u) -> int64_t {
      const int token = (sp.unit + static_cast<int>(u)) * UT + wave * TILE + lane % TILE;
      if (HOW == EACH ? token >= p.most : (u >= to || token < sp.begin || token >= sp.end)) return -1;
      return token_offset(p.cache, table, static_cast<uint32_t>(token)) * SIZE;  // (a page that is none: negative)
    };
    // The loads are a unit ahead of the products, without more registers: K's next rows follow when the scores have
    // read these, V's when the answers have. Rows that are masked are row 0 of page 0, not used.
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
    int64_t found = look(from), coming = HOW == EACH ? -1 : look(from + 1);
    if constexpr (HOW == EACH) {
      sp = span_of(__builtin_amdgcn_readfirstlane(length), p.most, 0, UT);
      if (from >= static_cast<uint32_t>(sp.units)) {
        if (from == 0)
          for (int i = threadIdx.x; i < heads * (p.head_dim / 4); i += THREADS) store(b, head0, 4 * i, float4_t{0.f, 0.f, 0.f, 0.f});
        return;
      }
      if (static_cast<int>(from) * UT + wave * TILE + lane % TILE >= sp.end) found = -1;
    }
    load_k(found < 0 ? 0 : found);
    load_v(found < 0 ? 0 : found);
    for (uint32_t u = from; u < to; ++u) {
      const uint32_t valid = static_cast<uint32_t>(__ballot(found >= 0));  // (TILE 16: the four copies agree)
      const int64_t next_row = coming < 0 ? 0 : coming;
      const bool more = u + 1 < to;
      found = coming;
      if constexpr (HOW != EACH) coming = look(u + 2);
      const bool full = TILE == 32 ? valid == 0xFFFFFFFFu : (valid & 0xFFFFu) == 0xFFFFu;
      if (ragged) {
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
          for (int c = 0; c < NC; ++c)
            if (4 * E * c + E * g >= p.head_dim) kf[h][c] = uint4_t{0u, 0u, 0u, 0u};
      }
      float4_t s[NH];
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        s[h] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          if (c >= chunks_of_row) continue;
          if constexpr (F32) {
#pragma unroll
            for (int x = 0; x < 4; ++x)
              s[h] = __builtin_amdgcn_mfma_f32_16x16x4f32(as_float(kf[h][c][x]),
                                                          as_float(qf[c][x]), s[h], 0, 0, 0);
          } else {
            s[h] = mfma16<DT>(kf[h][c], qf[c], s[h]);
          }
        }
      }
      if (more) load_k(next_row);
      float t[NH][4], top = kNone;
#pragma unroll
      for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          t[h][i] = s[h][i] * p.scale;
          if (!full && !(valid >> (16 * h + 4 * g + i) & 1u)) t[h][i] = kNone;
          top = fmaxf(top, t[h][i]);
        }
      top = column_max(top);
      if (!full) {
#pragma unroll
        for (int j = 0; j < VT; ++j)
          if (!(valid >> (16 * (j / 4) + 4 * g + j % 4) & 1u))
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) vf[j][nb] = uint4_t{0u, 0u, 0u, 0u};
      }
      if (__ballot(top > m)) {
        const float next = fmaxf(m, top);
        const float keep = next == m ? 1.f : __builtin_amdgcn_exp2f(m - next);  // (m -inf: 0)
        m = next;
        l *= keep;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < E; ++e) acc[nb][e] *= keep;
      }
      // (The factor by a product, which is exact; its exponent in the argument would round that at its size: f32 1.4e-6 of
      // the answer in the 2-norm over 1000 tokens, 1.0e-6 so.)
      const float ref = m == kNone ? 0.f : m;
      float pr[NH][4];
#pragma unroll
      for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          pr[h][i] = __builtin_amdgcn_exp2f(t[h][i] - ref) * FACTOR;
          l += pr[h][i];
        }
      if constexpr (F32) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int e = 0; e < E; ++e)
              acc[nb][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(as_float(vf[i][nb][e]), pr[0][i],
                                                                acc[nb][e], 0, 0, 0);
      } else {
        uint4_t hi, lo;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const uint2 parts = split2<DT>(pr[x >> 1][2 * (x & 1)], pr[x >> 1][2 * (x & 1) + 1]);
          hi[x] = parts.x;
          lo[x] = parts.y;
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < E; ++e) {
            uint4_t vt;
#pragma unroll
            for (int x = 0; x < 4; ++x)
              vt[x] = __builtin_amdgcn_perm(vf[2 * x + 1][nb][e >> 1], vf[2 * x][nb][e >> 1],
                                            e & 1 ? 0x07060302u : 0x05040100u);
            acc[nb][e] = mfma16<DT>(vt, hi, acc[nb][e]);
            acc[nb][e] = mfma16<DT>(vt, lo, acc[nb][e]);
          }
      }
      if (more) load_v(next_row);
    }

    // The wavefronts' parts of the item meet in LDS.
    l = column_sum(l);
    if (g == 0) {
      lds_m[wave][col] = m;
      lds_l[wave][col] = l;
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < E; e += 4)
          *reinterpret_cast<float4_t*>(&lds_o[wave][col][16 * E * nb + E * (4 * g + i) + e]) =
              float4_t{acc[nb][e][i], acc[nb][e + 1][i], acc[nb][e + 2][i], acc[nb][e + 3][i]};
    __syncthreads();
    const bool whole = ALONE || (from == 0 && to == static_cast<uint32_t>(sp.units));
    [[maybe_unused]] const uint32_t slot = part_place(worker, at == run);
    const int part_heads = min(kHeads, p.group), quads = p.head_dim / 4;
    auto joined = [&](int hd, int dim, float& top, float& total) {
      top = lds_m[0][hd];
#pragma unroll
      for (int w = 1; w < WAVES; ++w) top = fmaxf(top, lds_m[w][hd]);
      total = 0.f;
      float4_t o{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        const float f = lds_m[w][hd] == top ? 1.f : __builtin_amdgcn_exp2f(lds_m[w][hd] - top);
        total += f * lds_l[w][hd];
        o += f * *reinterpret_cast<const float4_t*>(&lds_o[w][hd][dim]);
      }
      return o;
    };
    for (int i = threadIdx.x; i < heads * quads; i += THREADS) {
      const int hd = i / quads, dim = (i - hd * quads) * 4;
      float top, total;
      const float4_t o = joined(hd, dim, top, total);
      const int64_t row = static_cast<int64_t>(slot) * part_heads + hd;
      if (whole) {
        const float each = total == 0.f ? 0.f : 1.f / total;
        float4_t y = o * each;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = total == 0.f ? 0.f : y[e];  // (0 * an infinity is none)
        store(b, head0 + hd, dim, y);
      } else if constexpr (MEET) {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(uint4_t, o), parts_rsrc, static_cast<uint32_t>(row * p.head_dim + dim) * 4, 0, kThrough);
        if (dim == 0)
          __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(uint2_t, make_float2(top, total)), stats_rsrc, static_cast<uint32_t>(row) * 8, 0, kThrough);
      } else {
        *reinterpret_cast<float4_t*>(p.part + row * p.head_dim + dim) = o;
        if (dim == 0) p.stats[row] = make_float2(top, total);
      }
    }
    at = item_first + to;
    if constexpr (MEET) {
      if (!whole) {
        const Parts parts = parts_of(item_first, static_cast<uint32_t>(sp.units), per);
        // The parts are stored and loaded past the XCDs' L2 caches, so that the order is all that is left to see to:
        // this thread's stores have arrived, then everybody's, then the count. (Fences of that scope would also write
        // the L2 back and empty it: 32 x 8000 tokens took 163 us with them, 58 without.)
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        __shared__ uint32_t others;
        if (threadIdx.x == 0) {
          others = __hip_atomic_fetch_add(p.meet + parts.from, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          if (others == parts.count - 1) __hip_atomic_store(p.meet + parts.from, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (others == parts.count - 1) {
          // A thread takes four dimensions of one head and every so many parts, a batch of parts' loads at a time (as many
          // as the registers hold, or four where that is all), with a running maximum; the threads of the same dimensions
          // then meet in LDS. What a batch has too many lies past the buffers' ranges: nothing is fetched for it.
          const int all_quads = heads * quads, groups = max(256 / all_quads, 1), mine_group = static_cast<int>(threadIdx.x) / all_quads;
          float4_t* sums = reinterpret_cast<float4_t*>(&lds_o[0][0][0]);
          float2* tops = reinterpret_cast<float2*>(sums + 256);
          for (int i0 = 0; i0 < all_quads; i0 += 256) {
            const int i = groups > 1 ? static_cast<int>(threadIdx.x) - mine_group * all_quads : i0 + static_cast<int>(threadIdx.x);
            const int hd = i / quads, dim = (i - hd * quads) * 4;
            float top = kNone, total = 0.f;
            float4_t o{0.f, 0.f, 0.f, 0.f};
            auto batches = [&](auto batch) {
              constexpr int BATCH = decltype(batch)::value;
              for (uint32_t k0 = mine_group; k0 < parts.count; k0 += BATCH * groups) {
                float2 st[BATCH];
                float4_t po[BATCH];
#pragma unroll
                for (int k = 0; k < BATCH; ++k) {
                  const bool there = k0 + k * groups < parts.count;
                  const uint32_t row = place_of(parts, k0 + k * groups) * part_heads + hd;
                  st[k] = __builtin_bit_cast(float2, __builtin_amdgcn_raw_buffer_load_b64(stats_rsrc, there ? row * 8 : kNowhere, 0, kThrough));
                  po[k] = __builtin_bit_cast(float4_t, __builtin_amdgcn_raw_buffer_load_b128(parts_rsrc, there ? (row * p.head_dim + dim) * 4 : kNowhere, 0, kThrough));
                }
                float next = top;
#pragma unroll
                for (int k = 0; k < BATCH; ++k) {
                  if (k0 + k * groups >= parts.count) st[k].x = kNone;
                  next = fmaxf(next, st[k].x);
                }
                const float keep = top == next ? 1.f : __builtin_amdgcn_exp2f(top - next);
                total *= keep;
                o *= keep;
                top = next;
#pragma unroll
                for (int k = 0; k < BATCH; ++k) {
                  const float f = st[k].x == top ? 1.f : __builtin_amdgcn_exp2f(st[k].x - top);
                  total += f * st[k].y;
                  o += f * po[k];
                }
              }
            };
            if (mine_group < groups && i < all_quads) {
              if (parts.count <= 4u * groups) batches(std::integral_constant<int, 4>{});
              else batches(std::integral_constant<int, F32 && NB == 2 ? 8 : 12>{});
            }
            if (groups > 1) {
              sums[threadIdx.x] = o;
              tops[threadIdx.x] = make_float2(top, total);
              __syncthreads();
              if (mine_group == 0) {
                float most = top;
                for (int k = 1; k < groups; ++k) most = fmaxf(most, tops[k * all_quads + i].x);
                const float keep = top == most ? 1.f : __builtin_amdgcn_exp2f(top - most);
                total *= keep;
                o *= keep;
                for (int k = 1; k < groups; ++k) {
                  const float2 t = tops[k * all_quads + i];
                  const float f = t.x == most ? 1.f : __builtin_amdgcn_exp2f(t.x - most);
                  total += f * t.y;
                  o += f * sums[k * all_quads + i];
                }
              }
            }
            if (mine_group == 0 && i < all_quads) store(b, head0 + hd, dim, total == 0.f ? float4_t{0.f, 0.f, 0.f, 0.f} : o * (1.f / total));
          }
        }
      }
    }
    __syncthreads();
  }
}

// The parts of an item that several workers shared (one workgroup a query head), and zeros for sequences
// without tokens. Which workers those are follows from the lengths, as in the kernel above.
template <int DT>
__global__ __launch_bounds__(256) void k_paged_join(AttendArgs p) {
  constexpr int UT = DT == DT_F32 ? 64 : 128;
  const int b = blockIdx.y;
  const int head = blockIdx.x, kv_head = head / p.group, in_group = head - kv_head * p.group;
  const int chunk = in_group / kHeads, hd = in_group - chunk * kHeads;
  const Span sp = span_at<UT>(p, b);
  const int quads = p.head_dim / 4;  // at most 64
  auto store = [&](int dim, float4_t o) {
    const int64_t out = b * p.ldy + static_cast<int64_t>(head) * p.head_dim + dim;
    if constexpr (DT == DT_F32)
      *reinterpret_cast<float4_t*>(static_cast<float*>(p.y) + out) = o;
    else
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.y) + out) = make_uint2(pack2<DT>(o[0], o[1]), pack2<DT>(o[2], o[3]));
  };
  if (sp.units == 0) {
    if (static_cast<int>(threadIdx.x) < quads) store(4 * threadIdx.x, float4_t{0.f, 0.f, 0.f, 0.f});
    return;
  }
  const uint32_t items = static_cast<uint32_t>(p.kv_heads * p.chunks);
  const uint32_t all = units_before<UT>(p, p.B) * items;
  const uint32_t first = units_before<UT>(p, b) * items + static_cast<uint32_t>(kv_head * p.chunks + chunk) * sp.units;
  const Parts parts = parts_of(first, static_cast<uint32_t>(sp.units), units_per_worker(all, p.workers));
  if (parts.count == 1) return;
  auto row_of = [&](uint32_t i) { return static_cast<int64_t>(place_of(parts, i)) * min(kHeads, p.group) + hd; };
  __shared__ float red[4];
  __shared__ __align__(16) float4_t sums[256];
  __shared__ float totals[256];
  float top = kNone;
  for (uint32_t i = threadIdx.x; i < parts.count; i += 256) top = fmaxf(top, p.stats[row_of(i)].x);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
  __syncthreads();
  top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  // 256 / quads threads to a group of four dimensions, each every so many parts.
  const int groups = 256 / quads, mine = threadIdx.x / quads, dim = (threadIdx.x - mine * quads) * 4;
  float total = 0.f;
  float4_t o{0.f, 0.f, 0.f, 0.f};
  if (mine < groups) {
    for (uint32_t i = mine; i < parts.count; i += groups) {
      const int64_t row = row_of(i);
      const float2 st = p.stats[row];
      const float f = st.x == top ? 1.f : __builtin_amdgcn_exp2f(st.x - top);
      total += f * st.y;
      o += f * *reinterpret_cast<const float4_t*>(p.part + row * p.head_dim + dim);
    }
  }
  sums[threadIdx.x] = o;
  totals[threadIdx.x] = total;
  __syncthreads();
  if (static_cast<int>(threadIdx.x) >= quads) return;
  for (int i = 1; i < groups; ++i) {
    total += totals[i * quads + threadIdx.x];
    o += sums[i * quads + threadIdx.x];
  }
  store(dim, total == 0.f ? float4_t{0.f, 0.f, 0.f, 0.f} : o * (1.f / total));
}

int check_cache(tmh_ctx* ctx, const tmh_paged_cache* c) {
  if (!c) return fail(ctx, TMH_ERR_INVALID, "the paged cache is NULL");
  if (!is_float_dtype(c->dtype))
    return fail(ctx, TMH_ERR_INVALID, "a paged cache holds f32, f16 or bf16 values, got %s", dtype_name(c->dtype));
  if (c->kv_heads < 1 || c->page_size < 1 || c->pages < 1)
    return fail(ctx, TMH_ERR_INVALID, "a paged cache needs kv_heads, page_size and pages of at least 1, got %d, %d, %lld",
                c->kv_heads, c->page_size, (long long)c->pages);
  if (c->head_dim < 8 || c->head_dim > 256 || c->head_dim % 8 != 0)
    return fail(ctx, TMH_ERR_UNSUPPORTED, "a paged cache's head_dim must be a multiple of 8 up to 256, got %d", c->head_dim);
  if (c->pages >= (int64_t{1} << 31) / c->page_size + ((int64_t{1} << 31) % c->page_size != 0))
    return fail(ctx, TMH_ERR_UNSUPPORTED, "a paged cache needs pages * page_size below 2^31");
  if (!c->k || !c->v) return fail(ctx, TMH_ERR_INVALID, "a paged cache's k and v must not be NULL");
  const int64_t e = 16 / dtype_size(c->dtype);
  if (reinterpret_cast<uintptr_t>(c->k) % 16 != 0 || reinterpret_cast<uintptr_t>(c->v) % 16 != 0 || c->page_stride % e != 0 ||
      c->token_stride % e != 0 || c->head_stride % e != 0)
    return fail(ctx, TMH_ERR_UNSUPPORTED, "a paged cache's k, v and strides must be multiples of 16 bytes");
  if (c->page_stride < 0 || c->token_stride < 0 || c->head_stride < 0)
    return fail(ctx, TMH_ERR_INVALID, "a paged cache's strides must not be negative");
  return TMH_OK;
}

template <int DT, int HOW>
void launch_attention(const AttendArgs& p, int heads, hipStream_t s) {
  constexpr int per_block = DT == DT_F32 ? 64 : 128;
  const int nb = (p.head_dim + per_block - 1) / per_block;
  constexpr int threads = HOW == WHOLE8 ? 512 : 256;
  constexpr int most = HOW != WHOLE8 ? (DT == DT_F32 ? 4 : 2) : (DT == DT_F32 ? 2 : 1);  // (eight wavefronts' registers)
  if (nb == 1) k_paged_attention<DT, 1, HOW><<<p.workers, threads, 0, s>>>(p);
  if constexpr (most >= 2)
    if (nb == 2) k_paged_attention<DT, 2, HOW><<<p.workers, threads, 0, s>>>(p);
  if constexpr (most >= 4)
    if (nb > 2) k_paged_attention<DT, 4, HOW><<<p.workers, threads, 0, s>>>(p);
  if constexpr (HOW == PARTS) k_paged_join<DT><<<dim3(static_cast<unsigned>(heads), static_cast<unsigned>(p.B)), 256, 0, s>>>(p);
}

}  // namespace
}  // namespace tmh

using namespace tmh;

extern "C" {

int tmh_paged_append(tmh_ctx* ctx, const void* d_q, int64_t ldq, const void* d_k, int64_t ldk, const void* d_v,
                     int64_t ldv, int64_t T, int heads, const int64_t* d_positions, const void* d_cos,
                     const void* d_sin, int table_dtype, int64_t max_positions, int rotary_dim, int interleaved,
                     const int64_t* d_slots, const tmh_paged_cache* cache, void* d_q_out, int64_t ldqo, void* stream) {
  TMH_TRY(check_cache(ctx, cache));
  const int dim = cache->head_dim;
  if (T < 0 || heads < 0 || T >= (int64_t{1} << 31) || static_cast<int64_t>(heads) + 2 * static_cast<int64_t>(cache->kv_heads) > (1 << 20))
    return fail(ctx, TMH_ERR_INVALID, "cannot append %lld tokens of %d query heads", (long long)T, heads);
  if (rotary_dim < 0 || rotary_dim > dim || rotary_dim % 2 != 0)
    return fail(ctx, TMH_ERR_INVALID, "rotary_dim must be even and from 0 to head_dim=%d, got %d", dim, rotary_dim);
  if (rotary_dim && !is_float_dtype(table_dtype))
    return fail(ctx, TMH_ERR_INVALID, "rotary tables must be f32, f16 or bf16, got %s", dtype_name(table_dtype));
  if (rotary_dim && max_positions < 1) return fail(ctx, TMH_ERR_INVALID, "rotary tables hold no positions");
  const int64_t kv_width = static_cast<int64_t>(cache->kv_heads) * dim, q_width = static_cast<int64_t>(heads) * dim;
  if (ldk < kv_width || ldv < kv_width || (heads && (ldq < q_width || ldqo < q_width)))
    return fail(ctx, TMH_ERR_INVALID, "the leading dimensions of q, k and v must be at least their heads' widths");
  TMH_TRY(use_device(ctx));
  if (T == 0) return TMH_OK;
  if (!d_k || !d_v || !d_slots || (heads && (!d_q || !d_q_out)) || (rotary_dim && (!d_positions || !d_cos || !d_sin)))
    return fail(ctx, TMH_ERR_INVALID, "tmh_paged_append: NULL pointer");
  if (heads && rotary_dim && d_q_out == d_q) return fail(ctx, TMH_ERR_INVALID, "rotated queries need a place of their own");
  AppendArgs p;
  p.q = d_q;
  p.k = d_k;
  p.v = d_v;
  p.positions = d_positions;
  p.cos = d_cos;
  p.sin = d_sin;
  p.slots = d_slots;
  p.q_out = d_q_out;
  p.k_cache = cache->k;
  p.v_cache = cache->v;
  p.ldq = ldq;
  p.ldk = ldk;
  p.ldv = ldv;
  p.ldqo = ldqo;
  p.max_positions = max_positions;
  p.page_stride = cache->page_stride;
  p.token_stride = cache->token_stride;
  p.head_stride = cache->head_stride;
  p.num_slots = cache->pages * cache->page_size;
  p.table_dtype = table_dtype;
  p.rotary = rotary_dim;
  p.interleaved = interleaved;
  p.heads = heads;
  p.kv_heads = cache->kv_heads;
  p.by_page = FastDiv(static_cast<uint32_t>(cache->page_size));
  const int64_t e = 16 / dtype_size(cache->dtype);
  auto on16 = [](const void* x) { return reinterpret_cast<uintptr_t>(x) % 16 == 0; };
  const bool vec = on16(d_k) && on16(d_v) && ldk % e == 0 && ldv % e == 0 &&
                   (!heads || (on16(d_q) && on16(d_q_out) && ldq % e == 0 && ldqo % e == 0)) &&
                   (interleaved ? true : rotary_dim % 16 == 0);
  p.head_dim = dim;
  p.turned = vec && !interleaved ? rotary_dim / 16 : 0;
  const uint32_t of_head = static_cast<uint32_t>(dim / 8 - p.turned);
  p.value_pieces = static_cast<uint32_t>(cache->kv_heads * (dim / 8));
  p.pieces = static_cast<uint32_t>(heads + cache->kv_heads) * of_head + p.value_pieces;
  p.by_pieces = FastDiv(p.pieces);
  p.by_head = FastDiv(of_head);
  p.by_value = FastDiv(static_cast<uint32_t>(dim / 8));
  const bool table_vec = on16(d_cos) && on16(d_sin) && rotary_dim % 16 == 0;
  const bool pairs_vec = table_dtype == TMH_F32 && on16(d_cos) && on16(d_sin) && rotary_dim % 8 == 0;  // four pairs an access
  hipStream_t s = pick_stream(ctx, stream);
  if (cache->dtype == TMH_F32) launch_append<DT_F32>(p, T, vec, table_vec, pairs_vec, s);
  else if (cache->dtype == TMH_F16) launch_append<DT_F16>(p, T, vec, table_vec, pairs_vec, s);
  else launch_append<DT_BF16>(p, T, vec, table_vec, pairs_vec, s);
  return check_launch(ctx, "k_paged_append");
}

int tmh_paged_attention(tmh_ctx* ctx, const void* d_q, int64_t ldq, int64_t B, int heads, const tmh_paged_cache* cache,
                        const int32_t* d_page_table, int64_t max_pages, const int32_t* d_lengths, float scale,
                        int64_t window, void* d_y, int64_t ldy, void* stream) {
  TMH_TRY(check_cache(ctx, cache));
  if (heads < 1 || heads % cache->kv_heads != 0)
    return fail(ctx, TMH_ERR_INVALID, "%d query heads are no multiple of %d kv heads", heads, cache->kv_heads);
  if (heads > (1 << 20)) return fail(ctx, TMH_ERR_UNSUPPORTED, "attention takes up to 2^20 query heads, got %d", heads);
  if (B < 0 || B > 65535) return fail(ctx, TMH_ERR_INVALID, "attention takes 0 to 65535 sequences, got %lld", (long long)B);
  if (max_pages < 0 || window < 0) return fail(ctx, TMH_ERR_INVALID, "max_pages and window must not be negative");
  if (std::isnan(scale)) return fail(ctx, TMH_ERR_INVALID, "the scale is NaN");
  const int64_t width = static_cast<int64_t>(heads) * cache->head_dim;
  if (ldq < width || ldy < width)
    return fail(ctx, TMH_ERR_INVALID, "the leading dimensions of q and y must be at least %lld", (long long)width);
  if (max_pages >= (int64_t{1} << 31) / cache->page_size)
    return fail(ctx, TMH_ERR_UNSUPPORTED, "attention needs max_pages * page_size below 2^31");
  TMH_TRY(use_device(ctx));
  if (B == 0) return TMH_OK;
  if (!d_q || !d_y || !d_lengths || (max_pages && !d_page_table)) return fail(ctx, TMH_ERR_INVALID, "tmh_paged_attention: NULL pointer");
  const int64_t e = 16 / dtype_size(cache->dtype);
  if (reinterpret_cast<uintptr_t>(d_q) % 16 != 0 || reinterpret_cast<uintptr_t>(d_y) % 16 != 0 || ldq % e != 0 || ldy % e != 0)
    return fail(ctx, TMH_ERR_UNSUPPORTED, "attention's q and y must be aligned to 16 bytes, their leading dimensions too");
  const int group = heads / cache->kv_heads, chunks = (group + kHeads - 1) / kHeads;
  const int64_t unit = cache->dtype == TMH_F32 ? 64 : 128;
  const int64_t units = (max_pages * cache->page_size + unit - 1) / unit * B * cache->kv_heads * chunks;
  if (units >= (int64_t{1} << 31)) return fail(ctx, TMH_ERR_UNSUPPORTED, "attention over too many tokens at once");
  AttendArgs p;
  p.q = d_q;
  p.k = cache->k;
  p.v = cache->v;
  p.table = d_page_table;
  p.lengths = d_lengths;
  p.y = d_y;
  p.ldq = ldq;
  p.ldy = ldy;
  p.max_pages = max_pages;
  p.cache = PageShape{cache->pages, cache->page_stride, cache->token_stride, FastDiv(static_cast<uint32_t>(cache->page_size))};
  p.head_stride = cache->head_stride;
  p.window = window;
  p.most = max_pages * cache->page_size;
  p.B = static_cast<int>(B);
  p.group = group;
  p.kv_heads = cache->kv_heads;
  p.chunks = chunks;
  p.head_dim = cache->head_dim;
  p.scale = scale * 1.44269504088896340736f;
  const AttentionPlan plan = attention_plan(B, cache->kv_heads, group, cache->head_dim, p.most, window, cache->dtype == TMH_F32, ctx->num_cus);
  p.workers = plan.workers;
  hipStream_t s = pick_stream(ctx, stream);
  const size_t rows = 2 * static_cast<size_t>(2 * ctx->num_cus) * std::min(kHeads, group);
  void* ws = workspace(ctx, rows * (cache->head_dim * 4 + sizeof(float2)), s);
  if (!ws) return fail(ctx, TMH_ERR_UNSUPPORTED, "attention's workspace cannot grow here: run one call before the capture");
  p.meet = ctx->meet;
  p.part = static_cast<float*>(ws);
  p.stats = reinterpret_cast<float2*>(p.part + rows * cache->head_dim);
  p.part_bytes = static_cast<uint32_t>(rows * cache->head_dim * 4);
  p.stats_bytes = static_cast<uint32_t>(rows * sizeof(float2));
  if (plan.way == EACH) {
    p.by_units = FastDiv(plan.units);
    p.by_items = FastDiv(static_cast<uint32_t>(cache->kv_heads * chunks));
  }
  auto launch = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    switch (plan.way) {
      case WHOLE: launch_attention<DT, WHOLE>(p, heads, s); break;
      case WHOLE8: launch_attention<DT, WHOLE8>(p, heads, s); break;
      case EACH: launch_attention<DT, EACH>(p, heads, s); break;
      case JOIN: launch_attention<DT, JOIN>(p, heads, s); break;
      case PARTS: launch_attention<DT, PARTS>(p, heads, s); break;
    }
  };
  if (cache->dtype == TMH_F32) launch(std::integral_constant<int, DT_F32>{});
  else if (cache->dtype == TMH_F16) launch(std::integral_constant<int, DT_F16>{});
  else launch(std::integral_constant<int, DT_BF16>{});
  return check_launch(ctx, "k_paged_attention");
}

}  // extern "C"
