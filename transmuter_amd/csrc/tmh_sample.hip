// Tokens drawn from rows of logits by temperature, top-k, top-p, min-p and given random numbers (tmh_sample).
//
// A row's weights are whole numbers (units of 2^-44 of the largest), so that sums of them do not depend on an order. Three kernels,
// each with `slices` workgroups a row, the last of which to finish does what needs the whole row:
//  k_sample_top   the largest logit.
//  k_sample_sum   rows that keep all tokens, or those of min-p: the weights of every chunk of tokens, and the draw. Rows by top-k: how
//                 many tokens lie in each bin (a sixteenth of a factor of two in weight), and down to which bin the k largest reach.
//                 Others, by top-p alone: the weights of each bin, and the bin in which they reach top-p of the whole.
//  k_sample_draw  rows by top-k: the tokens down to that bin go to a list. By top-p alone: those of that bin do, and the weights above
//                 it to chunks. The list, sorted out in LDS, gives the least logit kept and the last of its equals that is; then the draw.
// Rows of at most kShort tokens are a list from the start: k_sample_short, one kernel and a workgroup a row.
// Bound by latency (what one kernel leaves the next, a row's last workgroup alone) and by the weights' exponentials in 64 bits; in us
// k_sample_top, k_sample_sum, k_sample_draw: 1 x 151936 f32 by top-k and top-p 4, 12, 10; 64 x 151936 bf16 by top-p 10, 21, 36;
// 500 x 32003 f16 of all kinds 14, 36, 42; 256 x 151936 f32 by min-p 34, 36: 4.6 and 4.3 TB/s.
// A list that does not fit (thousands of tokens of almost the same logit) leaves its row to the last workgroup, which goes over all
// of it a few times.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "tmh_device.h"
#include "tmh_internal.h"
#include "tmh_launch.h"

namespace tmh {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kUnit = 44;
constexpr int kPerOctave = 16, kWeightBins = kPerOctave * kUnit + 4;  // (a few more than have weights: bins are found in f32)
constexpr int kList = 4096;        // tokens of a row's list
constexpr int kShort = 8192;       // tokens of a row that one workgroup takes
constexpr int kDigits = 2048;      // of a selection's turn
constexpr int kMostRows = 512;     // of a launch: each has a counter

enum Mode : int { GREEDY, ALL, TOP_K, TOP_P };

struct SampleArgs {
  const void* x;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  const float* u;
  int64_t* tokens;
  int64_t ld;
  int vocabulary, slices, chunks;  // chunks: of a row
  // The workspace: of each row and slice the largest logit and its place, the bins and the list with its count; of each row the chunks'
  // weights and what k_sample_sum tells k_sample_draw.
  uint64_t* best;    // [rows][slices]
  uint64_t* bins;    // [rows][slices][kWeightBins]
  uint64_t* list;    // [rows][slices][kList]
  uint32_t* counts;  // [rows][slices]
  uint64_t* sums;    // [rows][chunks]
  uint64_t* told;    // [rows][4]: border bin, weight above it, weight of all
  uint32_t* meet;    // [rows] slices that have finished; zero between launches
};

// Logits as numbers that order as they do, NaN with -infinity, the lowest.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (!(x > -__builtin_inff())) x = -__builtin_inff();
  if (x == 0.f) x = 0.f;  // (-0 as 0)
  const uint32_t b = __builtin_bit_cast(uint32_t, x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __builtin_bit_cast(float, key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}
constexpr uint32_t kLowestKey = 0x007FFFFFu;  // of -infinity

// 2^(j / 128) in units of 2^-44 of 1, j < 128, in LDS: e^y with y = j ln 2 / 128 up to 0.7, whose series ends with y^15 / 15! (the next
// term is below 2^-53).
constexpr int kSteps = 128;
__device__ __forceinline__ const double* powers() {
  __shared__ double table[kSteps];
  if (threadIdx.x < kSteps) {
    const double y = threadIdx.x * (0.69314718055994530942 / kSteps);
    double term = 0x1p44, sum = 0x1p44;
#pragma unroll
    for (int i = 1; i <= 15; ++i) {
      term *= y * (1.0 / i);
      sum += term;
    }
    table[threadIdx.x] = sum;
  }
  __syncthreads();
  return table;
}

// What a row's WG knows of its row.
struct Row {
  Mode mode;
  int k;
  float top;          // the largest logit
  uint32_t top_key, top_index;
  double c;           // 128 log2(e) / temperature
  const double* table;  // of powers()
  float per_bin;      // bins a logit
  double top_p, least;  // least: the smallest weight that min-p keeps, in units
  float low;          // logits below it are certainly left out by min-p, or weigh nothing
  float u;
  // exp((x - top) / temperature) in units of 2^-44, not rounded; 0 where it is less than one. It is 2^(t / 128): the whole part n of t gives
  // a power of two and a place of the table, the rest z, up to a half, 2^(z / 128) by its series up to z^4 (the next term is 2^-49).
  __device__ __forceinline__ double units(float x) const {
    constexpr double kRound = 0x1.8p52;  // (added, its low bits are the whole part)
    if (top == __builtin_inff()) return x == top ? 0x1p44 : 0.0;
    const double t = (static_cast<double>(x) - static_cast<double>(top)) * c;
    if (!(t >= -kUnit * kSteps)) return 0.0;
    const double whole = t + kRound, z = t - (whole - kRound);
    const int n = static_cast<int>(__builtin_bit_cast(uint64_t, whole));
    constexpr double l = 0.69314718055994530942 / kSteps;
    double s = fma(z, l * l * l * l / 24.0, l * l * l / 6.0);
    s = fma(s, z, l * l / 2.0);
    s = fma(s, z, l);
    s = fma(s, z, 1.0) * table[n & (kSteps - 1)];
    return __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, s) + (static_cast<uint64_t>(static_cast<uint32_t>(n >> 7) << 20) << 32));
  }
  // A whole number of units: added to 2^52, the low bits.
  static __device__ __forceinline__ uint64_t rounded(double units) { return __builtin_bit_cast(uint64_t, units + 0x1p52) & ((uint64_t{1} << 52) - 1); }
  __device__ __forceinline__ uint64_t weight(float x) const { return rounded(units(x)); }
  // The same, 0 where min-p leaves the token out.
  __device__ __forceinline__ uint64_t kept_weight(float x) const {
    const double w = units(x);
    return w >= least ? rounded(w) : 0;
  }
  // The bin of a logit: of the largest 0, kWeightBins and more where it has no weight. Not falling as logits fall.
  __device__ __forceinline__ int bin(float x) const {
    const float b = fminf((top - x) * per_bin, static_cast<float>(kWeightBins));  // (of NaN the other)
    return x == top ? 0 : static_cast<int>(b);
  }
};

// The sum over the lanes up to this one: within rows of 16 lanes, then the rows' last lanes to the rows behind (DPP moves; a lane that
// a move does not reach adds 0).
template <int CONTROL, int ROWS>
__device__ __forceinline__ uint64_t moved(uint64_t v) {
  const uint32_t low = __builtin_amdgcn_update_dpp(0, static_cast<int>(v), CONTROL, ROWS, 0xF, false);
  const uint32_t high = __builtin_amdgcn_update_dpp(0, static_cast<int>(v >> 32), CONTROL, ROWS, 0xF, false);
  return static_cast<uint64_t>(high) << 32 | low;
}
__device__ __forceinline__ uint64_t wave_scan(uint64_t v) {
  v += moved<0x111, 0xF>(v);
  v += moved<0x112, 0xF>(v);
  v += moved<0x114, 0xF>(v);
  v += moved<0x118, 0xF>(v);
  v += moved<0x142, 0xA>(v);
  return v + moved<0x143, 0xC>(v);
}
__device__ __forceinline__ uint64_t of_lane(uint64_t v, int i) {
  return static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v >> 32), i))) << 32 |
         static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), i));
}
__device__ __forceinline__ uint64_t wave_sum(uint64_t v) { return of_lane(wave_scan(v), 63); }
__device__ __forceinline__ uint64_t wave_max(uint64_t v) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) v = max(v, static_cast<uint64_t>(__shfl_xor(v, o)));
  return v;
}
__device__ __forceinline__ void put64(uint64_t* p, uint64_t v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ uint64_t get64(const uint64_t* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// A row in chunks of 64 E tokens, a wavefront's 16 bytes a lane; chunk 0 begins with the 16 bytes that the row's first token lies in.
template <int DT>
struct Chunks {
  static constexpr int E = DT == DT_F32 ? 4 : 8, SIZE = DT == DT_F32 ? 4 : 2;
  const char* row;  // chunk 0
  int before, n;    // places of chunk 0 ahead of the row, tokens
  __device__ Chunks(const SampleArgs& p, int64_t r) : n(p.vocabulary) {
    const char* first = static_cast<const char*>(p.x) + r * p.ld * SIZE;
    before = static_cast<int>(reinterpret_cast<uintptr_t>(first) % 16) / SIZE;
    row = first - before * SIZE;
  }
  // The lane's first token of chunk q (its E tokens may begin before 0 or end past n).
  __device__ __forceinline__ int token(int q) const { return (q * 64 + static_cast<int>(threadIdx.x & 63)) * E - before; }
  __device__ __forceinline__ uint4_t raw(int q) const {
    const int t = token(q);
    if (t >= 0 && t + E <= n) return *reinterpret_cast<const uint4_t*>(row + static_cast<int64_t>(t + before) * SIZE);
    uint4_t v = uint4_t{0u, 0u, 0u, 0u};  // (16 bytes that are not all the row's: one token after another)
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (t + e >= 0 && t + e < n) {
        const char* at = row + static_cast<int64_t>(t + e + before) * SIZE;
        if constexpr (DT == DT_F32) v[e] = *reinterpret_cast<const uint32_t*>(at);
        else v[e / 2] |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(at)) << 16 * (e % 2);
      }
    return v;
  }
  // Its E logits, -infinity in the place of tokens that there are not.
  __device__ __forceinline__ void logits(int q, uint4_t v, float (&x)[E]) const {
    const int t = token(q);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if constexpr (DT == DT_F32) {
        const uint32_t w = v[e];
        x[e] = __builtin_bit_cast(float, w);
      } else {
        const uint32_t w = v[e / 2] >> 16 * (e % 2);
        x[e] = DT == DT_F16 ? f16_bits_to_f32(static_cast<uint16_t>(w)) : __builtin_bit_cast(float, w << 16);
      }
      if (t + e < 0 || t + e >= n) x[e] = -__builtin_inff();
    }
  }
};

// Calls each(q, logits) for the chunks [from, to), a wavefront taking every kWaves-th, with AHEAD loads on their way; the first of them
// are loaded where it is made.
template <int DT, int AHEAD = 4>
struct OverChunks {
  const Chunks<DT>& row;
  int from, to;
  uint4_t v[AHEAD];
  __device__ __forceinline__ void load(int q0) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (q0 + i * kWaves < to) v[i] = row.raw(q0 + i * kWaves);
  }
  __device__ __forceinline__ OverChunks(const Chunks<DT>& r, int first, int end) : row(r), from(first + static_cast<int>(threadIdx.x >> 6)), to(end) {
    load(from);
  }
  template <typename Each>
  __device__ __forceinline__ void operator()(Each each) {
    for (int q0 = from; q0 < to; q0 += AHEAD * kWaves) {
      if (q0 != from) load(q0);
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int q = q0 + i * kWaves;
        if (q >= to) break;
        float x[Chunks<DT>::E];
        row.logits(q, v[i], x);
        each(q, x);
      }
    }
  }
};

struct Slice {
  int64_t row;
  int at, from, to;  // which, its chunks
};
__device__ __forceinline__ Slice slice_of(const SampleArgs& p) {
  Slice s;
  s.row = blockIdx.x / p.slices;
  s.at = static_cast<int>(blockIdx.x - s.row * p.slices);
  s.from = static_cast<int>(static_cast<int64_t>(p.chunks) * s.at / p.slices);
  s.to = static_cast<int>(static_cast<int64_t>(p.chunks) * (s.at + 1) / p.slices);
  return s;
}

// Whether this workgroup is the last of its row's. What the others have stored (past their XCD's L2, put64) it may load (get64).
__device__ __forceinline__ bool last_of_row(const SampleArgs& p, int64_t row) {
  __shared__ uint32_t others;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    others = p.slices == 1 ? 0 : __hip_atomic_fetch_add(p.meet + row, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (p.slices > 1 && others == static_cast<uint32_t>(p.slices) - 1) __hip_atomic_store(p.meet + row, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  return others == static_cast<uint32_t>(p.slices) - 1;
}

template <typename Join>
__device__ __forceinline__ uint64_t block_join(uint64_t v, Join join) {  // (of all threads; v is its wavefront's)
  __shared__ uint64_t red[kWaves];
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  uint64_t all = red[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) all = join(all, red[w]);
  return all;
}
__device__ __forceinline__ uint64_t block_sum(uint64_t v) {
  return block_join(wave_sum(v), [](uint64_t a, uint64_t b) { return a + b; });
}

// The sum over the threads before this one, and over all.
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t& all) {
  __shared__ uint64_t parts[kWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint64_t upto = wave_scan(v);
  __syncthreads();
  if (lane == 63) parts[wave] = upto;
  __syncthreads();
  uint64_t before = upto - v;
  all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) before += parts[w];
    all += parts[w];
  }
  return before;
}

template <int DT>
__global__ __launch_bounds__(kThreads) void k_sample_top(SampleArgs p) {
  const Slice s = slice_of(p);
  const Chunks<DT> row(p, s.row);
  uint32_t top = 0, at = 0;  // (a thread's tokens come in their order: the first of equals stays)
  OverChunks<DT>(row, s.from, s.to)([&](int q, const float (&x)[Chunks<DT>::E]) {
    const int t = row.token(q);
#pragma unroll
    for (int e = 0; e < Chunks<DT>::E; ++e) {
      const uint32_t key = key_of(x[e]);
      at = key > top ? t + e : at;
      top = max(top, key);
    }
  });
  uint64_t best = static_cast<uint64_t>(top) << 32 | static_cast<uint32_t>(~at);
  best = block_join(wave_max(best), [](uint64_t a, uint64_t b) { return max(a, b); });
  if (threadIdx.x == 0) p.best[s.row * p.slices + s.at] = best;
}

// A row's choices; in GREEDY rows the token is known (the largest; -1 where no logit is above -infinity).
__device__ __forceinline__ Row row_of(const SampleArgs& p, int64_t r, uint64_t best) {
  Row row;
  row.table = powers();
  row.top_key = static_cast<uint32_t>(best >> 32);
  row.top_index = static_cast<uint32_t>(~best);
  row.top = value_of(row.top_key);
  const float temperature = p.temperature ? p.temperature[r] : 1.f;
  row.c = kSteps * 1.4426950408889634074 / static_cast<double>(temperature);
  row.per_bin = static_cast<float>(row.c * (1.0 * kPerOctave / kSteps));
  row.k = p.top_k ? p.top_k[r] : 0;
  row.top_p = p.top_p ? p.top_p[r] : 1.0;
  const float min_p = p.min_p ? p.min_p[r] : 0.f;
  row.least = min_p > 0.f ? fmin(static_cast<double>(min_p), 1.0) * 0x1p44 : 0.0;
  row.u = p.u[r];
  // (A factor of two below: more than f32's roundings are.)
  const float octaves = 1.f + (min_p > 0.f ? fminf(-log2f(fminf(min_p, 1.f)), kUnit) : kUnit);
  row.low = row.top == __builtin_inff() ? row.top : static_cast<float>(row.top - octaves * kSteps / row.c);
  row.mode = !(temperature > 0.f) || row.top_key == kLowestKey ? GREEDY : row.k > 0 && row.k < p.vocabulary ? TOP_K : row.top_p < 1.0 ? TOP_P : ALL;
  return row;
}

__device__ __forceinline__ Row row_of(const SampleArgs& p, int64_t r) {
  uint64_t best = 0;
  for (int i = threadIdx.x & 63; i < p.slices; i += 64) best = max(best, p.best[r * p.slices + i]);
  return row_of(p, r, wave_max(best));
}

// The draw: the first token, by index, up to which the weights sum to more than u of their whole. sums: of each chunk, in LDS.
// weight(logit, token): a token's, 0 where it is not kept.
template <int DT, typename Weight>
__device__ __forceinline__ void draw(const SampleArgs& p, const Row& r, const Chunks<DT>& row, int64_t at_row, const uint64_t* sums, Weight weight) {
  constexpr int E = Chunks<DT>::E;
  __shared__ uint64_t found_before;
  __shared__ int found;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // Each thread some chunks in a row.
  const int each = (p.chunks + kThreads - 1) / kThreads, first = tid * each;
  uint64_t mine = 0;
  for (int i = 0; i < each; ++i)
    if (first + i < p.chunks) mine += sums[first + i];
  if (tid == 0) found = -1;
  uint64_t total;
  uint64_t before = block_scan(mine, total);
  const double target = static_cast<double>(r.u) * static_cast<double>(total);
  // (Where no sum is above the target, as for u >= 1, the last token of any weight is taken. A NaN is above nothing.)
  auto past = [&](uint64_t sum) { return static_cast<double>(sum) > target || sum == total; };
  if (mine && past(before + mine) && !(before && past(before))) {
    for (int i = 0; i < each && first + i < p.chunks; ++i) {
      const uint64_t w = sums[first + i];
      if (w && past(before + w)) {
        found = first + i;
        found_before = before;
        break;
      }
      before += w;
    }
  }
  __syncthreads();
  if (wave != 0 || found < 0) return;
  const int q = found, t = row.token(q);
  float x[E];
  row.logits(q, row.raw(q), x);
  uint64_t w[E], sum = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    w[e] = x[e] > -__builtin_inff() ? weight(x[e], t + e) : 0;
    sum += w[e];
  }
  uint64_t so_far = wave_scan(sum) - sum + found_before;
  int token = -1;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    so_far += w[e];
    if (token < 0 && w[e] && past(so_far)) token = t + e;
  }
  const uint64_t any = __ballot(token >= 0);
  if (any && lane == __builtin_ctzll(any)) p.tokens[at_row] = token;
}

// The key at which the sum of measures over items of falling keys reaches `need` (reached(sum)), and the sum above it, by 11 bits of the
// keys a turn, of those in which they differ. items(each) calls each(key, measure) for the thread's items.
template <typename Items, typename Reached>
__device__ __forceinline__ uint32_t select(uint64_t* bins, Items items, Reached reached, uint64_t& above) {
  static_assert(kDigits == 2 * kThreads, "");
  __shared__ uint32_t found_digit;
  __shared__ uint64_t found_sum;
  const uint32_t tid = threadIdx.x;
  uint32_t low = ~0u, high = 0;
  items([&](uint32_t key, uint64_t) {
    low = min(low, key);
    high = max(high, key);
  });
  // (Both ends' largest in one number: the low half holds the complement of the lowest.)
  auto both = [](uint64_t a, uint64_t b) {
    const uint32_t x = max(static_cast<uint32_t>(a >> 32), static_cast<uint32_t>(b >> 32)), y = max(static_cast<uint32_t>(a), static_cast<uint32_t>(b));
    return static_cast<uint64_t>(x) << 32 | y;
  };
  uint64_t ends = static_cast<uint64_t>(high) << 32 | static_cast<uint32_t>(~low);
  ends = both(ends, moved<0x111, 0xF>(ends));
  ends = both(ends, moved<0x112, 0xF>(ends));
  ends = both(ends, moved<0x114, 0xF>(ends));
  ends = both(ends, moved<0x118, 0xF>(ends));
  ends = both(ends, moved<0x142, 0xA>(ends));
  ends = both(ends, moved<0x143, 0xC>(ends));
  ends = block_join(of_lane(ends, 63), both);
  low = ~static_cast<uint32_t>(ends);
  high = static_cast<uint32_t>(ends >> 32);
  above = 0;
  int shift = high > low ? max(32 - __builtin_clz(high - low) - 11, 0) : 0;
  uint32_t base = low, span = high - low;  // the keys that are left are base .. base + span
#pragma unroll 1
  while (true) {
    bins[2 * tid] = 0;
    bins[2 * tid + 1] = 0;
    if (tid == 0) found_digit = ~0u;
    __syncthreads();
    items([&](uint32_t key, uint64_t measure) {
      if (key >= base && key - base <= span)
        atomicAdd(reinterpret_cast<unsigned long long*>(&bins[(key - base) >> shift]), static_cast<unsigned long long>(measure));
    });
    __syncthreads();
    // Each thread two digits, from the highest down.
    const uint32_t digit = kDigits - 1 - 2 * tid;
    const uint64_t first = bins[digit], second = bins[digit - 1], lowest = bins[0];
    uint64_t all;
    const uint64_t before = block_scan(first + second, all) + above;
    // The first to reach it.
    if ((first + second) && reached(before + first + second) && !(before != above && reached(before))) {
      const bool upper = first && reached(before + first);
      found_digit = upper ? digit : digit - 1;
      found_sum = upper ? before : before + first;
    }
    __syncthreads();
    const uint32_t found = found_digit;
    above = found == ~0u ? above + all - lowest : found_sum;  // (the lowest that there is, should the sums not reach it)
    base += (found == ~0u ? 0 : found) << shift;
    if (shift == 0) return base;
    span = (1u << shift) - 1;
    shift = max(shift - 11, 0);
    __syncthreads();
  }
}

// How many of equal weights `each` it takes, beside `above`, to reach `need`.
__device__ __forceinline__ uint64_t equals_needed(double need, uint64_t above, uint64_t each) {
  if (!each || static_cast<double>(above + each) >= need) return 1;
  uint64_t n = static_cast<uint64_t>((need - static_cast<double>(above)) / static_cast<double>(each));
  if (n) --n;  // (the quotient is rounded: counted up from just below)
  while (static_cast<double>(above + n * each) < need) ++n;
  return n;
}

// What top-k and top-p keep: keys above `key`, and of its equals the tokens up to `last`. items(each) calls each(key, token) for the
// thread's items, the tokens that may be the border's; those above all of them weigh `above`. `whole`: the weight that top-p is of, or
// 0: that of what top-k keeps.
struct Edge {
  uint32_t key, last;
  __device__ __forceinline__ bool keeps(uint32_t k, uint32_t token) const { return k > key || (k == key && token <= last); }
};
template <int DT, typename Items>
__device__ __forceinline__ Edge edge_of(const Row& r, uint64_t* bins, Items items, uint64_t above, uint64_t whole) {
  // (The low bits of 16-bit types' keys are all alike, 0 or, of numbers below 0, 1.)
  constexpr int QUIET = DT == DT_F32 ? 0 : DT == DT_F16 ? 13 : 16;
  auto key_again = [](uint32_t k) { return k << QUIET | (k >> (31 - QUIET) ? 0 : (1u << QUIET) - 1); };
  uint32_t edge = 0;
  uint64_t ties = ~uint64_t{0};
  if (r.mode == TOP_K) {
    uint64_t more;
    edge = key_again(select(bins, [&](auto each) { items([&](uint32_t key, uint32_t) { each(key >> QUIET, uint64_t{1}); }); },
                            [&](uint64_t sum) { return sum >= static_cast<uint64_t>(r.k); }, more));
    ties = static_cast<uint64_t>(r.k) - more;
  }
  if (r.top_p < 1.0) {
    uint64_t at_edge = ties;
    if (!whole) {
      // Of tokens at the edge only `ties` count.
      uint64_t sum = 0, equal = 0;
      items([&](uint32_t key, uint32_t) {
        if (key > edge) sum += r.weight(value_of(key));
        equal += key == edge;
      });
      whole = block_sum(sum);
      at_edge = min(block_sum(equal), ties);
      whole += at_edge * r.weight(value_of(edge));
    }
    const double need = fmax(r.top_p * static_cast<double>(whole), 1.0);  // (one token at least)
    const uint32_t by_k = edge;
    uint64_t more;
    edge = key_again(select(bins, [&](auto each) { items([&](uint32_t key, uint32_t) { if (key >= by_k) each(key >> QUIET, r.weight(value_of(key))); }); },
                            [&](uint64_t sum) { return static_cast<double>(above + sum) >= need; }, more));
    ties = equals_needed(need, above + more, r.weight(value_of(edge)));
    if (edge == by_k) ties = min(ties, at_edge);
  }
  uint64_t equal = 0;
  items([&](uint32_t key, uint32_t) { equal += key == edge; });
  if (block_sum(equal) <= ties) return {edge, ~0u};
  uint64_t more;
  return {edge, ~select(bins, [&](auto each) { items([&](uint32_t key, uint32_t token) { if (key == edge) each(~token, uint64_t{1}); }); },
                        [&](uint64_t sum) { return sum >= ties; }, more)};
}

template <int DT>
__global__ __launch_bounds__(kThreads) void k_sample_sum(SampleArgs p) {
  constexpr int E = Chunks<DT>::E;
  extern __shared__ uint64_t bins[];  // kWeightBins (or, for the draw, the chunks' weights)
  const Slice s = slice_of(p);
  const Chunks<DT> row(p, s.row);
  OverChunks<DT> over(row, s.from, s.to);
  const Row r = row_of(p, s.row);
  const int tid = threadIdx.x, lane = tid & 63;
  if (r.mode == GREEDY) {
    if (s.at == 0 && tid == 0) p.tokens[s.row] = r.top_key == kLowestKey ? -1 : static_cast<int64_t>(r.top_index);
    return;
  }
  uint64_t* sums = p.sums + s.row * p.chunks;
  if (r.mode == ALL) {
    over([&](int q, const float (&x)[E]) {
      uint64_t sum = 0;
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (!(x[e] < r.low)) sum += r.kept_weight(x[e]);
      if (__ballot(sum != 0)) sum = wave_sum(sum);
      if (lane == 0) put64(sums + q, sum);
    });
    if (!last_of_row(p, s.row)) return;
    for (int i = tid; i < p.chunks; i += kThreads) bins[i] = get64(sums + i);
    __syncthreads();
    draw<DT>(p, r, row, s.row, bins, [&](float x, int) { return r.kept_weight(x); });
    return;
  }
  for (int i = tid; i < kWeightBins; i += kThreads) bins[i] = 0;
  __syncthreads();
  over([&](int q, const float (&x)[E]) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int b = r.bin(x[e]);
      if (b >= kWeightBins) continue;
      atomicAdd(reinterpret_cast<unsigned long long*>(&bins[b]), static_cast<unsigned long long>(r.mode == TOP_K ? 1 : r.weight(x[e])));
    }
  });
  __syncthreads();
  uint64_t* all = p.bins + s.row * p.slices * kWeightBins;
  for (int i = tid; i < kWeightBins; i += kThreads) put64(all + s.at * kWeightBins + i, bins[i]);
  if (!last_of_row(p, s.row)) return;
  uint64_t mine = 0;
  if (tid < kWeightBins)
#pragma unroll 8
    for (int i = 0; i < p.slices; ++i) mine += get64(all + i * kWeightBins + tid);
  static_assert(kWeightBins <= kThreads, "");
  // The first bin with which the sum of the bins reaches k tokens, or top-p of the whole.
  __shared__ uint32_t border;
  __shared__ uint64_t above;
  if (tid == 0) {
    border = kWeightBins;
    above = 0;
  }
  uint64_t total;
  const uint64_t before = block_scan(mine, total);
  const double need = fmax(r.top_p * static_cast<double>(total), 1.0);
  auto reached = [&](uint64_t sum) { return r.mode == TOP_K ? sum >= static_cast<uint64_t>(r.k) : static_cast<double>(sum) >= need; };
  if (mine && reached(before + mine) && !(before && reached(before))) {
    border = tid;
    above = before;
  }
  __syncthreads();
  if (tid == 0) {
    p.told[4 * s.row] = border;
    p.told[4 * s.row + 1] = r.mode == TOP_K ? 0 : above;
    p.told[4 * s.row + 2] = r.mode == TOP_K ? 0 : total;
  }
}

// A row by top-k whose list has up to 64 tokens, a lane each, by one wavefront: what comes before a token by logit, and of what is kept
// by index, is summed over the lanes one after another.
__device__ __forceinline__ void draw_few(const SampleArgs& p, const Row& r, int64_t at_row, const uint64_t* list, int n, int lane) {
  const bool there = lane < n;
  const uint64_t mine = there ? list[lane] : 0;
  const uint32_t key = static_cast<uint32_t>(mine >> 32), token = static_cast<uint32_t>(mine);
  uint64_t w = there ? r.weight(value_of(key)) : 0;
  int rank = 0;
  uint64_t before = 0;
  for (int i = 0; i < n; ++i) {
    const uint64_t other = of_lane(mine, i), weight = of_lane(w, i);
    const uint32_t k = static_cast<uint32_t>(other >> 32), t = static_cast<uint32_t>(other);
    const bool ahead = k > key || (k == key && t < token);
    rank += ahead;
    before += ahead ? weight : 0;
  }
  bool kept = there && rank < r.k;
  if (r.top_p < 1.0) {
    const double need = fmax(r.top_p * static_cast<double>(wave_sum(kept ? w : 0)), 1.0);
    kept = kept && static_cast<double>(before) < need;
  }
  w = kept ? r.kept_weight(value_of(key)) : 0;
  const uint64_t total = wave_sum(w);
  before = 0;
  for (int i = 0; i < n; ++i) {
    const uint64_t weight = of_lane(w, i);
    const uint32_t t = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(token), i));
    before += t < token ? weight : 0;
  }
  const double target = static_cast<double>(r.u) * static_cast<double>(total);
  auto past = [&](uint64_t sum) { return static_cast<double>(sum) > target || sum == total; };
  if (w && past(before + w) && !(before && past(before))) p.tokens[at_row] = token;
}

// A row of up to kShort tokens by one workgroup, as the others do the tokens of a list.
template <int DT>
__global__ __launch_bounds__(kThreads) void k_sample_short(SampleArgs p) {
  constexpr int E = Chunks<DT>::E;
  __shared__ uint64_t bins[kDigits];
  extern __shared__ uint64_t sums[];  // of each chunk
  uint32_t* keys = reinterpret_cast<uint32_t*>(sums + p.chunks);
  const int64_t at = blockIdx.x;
  const Chunks<DT> row(p, at);
  const int tid = threadIdx.x, lane = tid & 63;
  const uint32_t n = static_cast<uint32_t>(p.vocabulary);
  uint64_t best = 0;
  OverChunks<DT>(row, 0, p.chunks)([&](int q, const float (&x)[E]) {
    const int t = row.token(q);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (t + e < 0 || t + e >= row.n) continue;
      const uint32_t key = key_of(x[e]);
      keys[t + e] = key;
      best = max(best, static_cast<uint64_t>(key) << 32 | static_cast<uint32_t>(~(t + e)));
    }
  });
  const Row r = row_of(p, at, block_join(wave_max(best), [](uint64_t a, uint64_t b) { return max(a, b); }));
  if (r.mode == GREEDY) {
    if (tid == 0) p.tokens[at] = r.top_key == kLowestKey ? -1 : static_cast<int64_t>(r.top_index);
    return;
  }
  auto items = [&](auto each) {
    for (uint32_t i = tid; i < n; i += kThreads) each(keys[i], i);
  };
  Edge edge{0, ~0u};
  if (r.mode == TOP_P) {  // (of all)
    uint64_t sum = 0;
    items([&](uint32_t key, uint32_t) { sum += r.weight(value_of(key)); });
    edge = edge_of<DT>(r, bins, items, 0, block_sum(sum));
  } else if (r.mode == TOP_K) {
    edge = edge_of<DT>(r, bins, items, 0, 0);
  }
  auto weight = [&](float x, int token) { return edge.keeps(key_of(x), static_cast<uint32_t>(token)) ? r.kept_weight(x) : 0; };
  for (int q = tid >> 6; q < p.chunks; q += kWaves) {
    const int t = row.token(q);
    uint64_t sum = 0;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (t + e >= 0 && t + e < row.n) sum += weight(value_of(keys[t + e]), t + e);
    sum = wave_sum(sum);
    if (lane == 0) sums[q] = sum;
  }
  __syncthreads();
  draw<DT>(p, r, row, at, sums, weight);
}

template <int DT>
__global__ __launch_bounds__(kThreads) void k_sample_draw(SampleArgs p) {
  constexpr int E = Chunks<DT>::E;
  __shared__ uint64_t bins[kDigits];
  __shared__ uint64_t list[kList];  // key << 32 | token
  extern __shared__ uint64_t sums[];  // of each chunk
  __shared__ uint32_t count;
  const Slice s = slice_of(p);
  const Chunks<DT> row(p, s.row);
  OverChunks<DT> over(row, s.from, s.to);
  const Row r = row_of(p, s.row);
  const int tid = threadIdx.x, lane = tid & 63;
  if (r.mode == GREEDY || r.mode == ALL) return;
  const uint32_t border = static_cast<uint32_t>(p.told[4 * s.row]);
  const uint64_t above = p.told[4 * s.row + 1], whole = p.told[4 * s.row + 2];
  uint64_t* all_sums = p.sums + s.row * p.chunks;
  uint64_t* lists = p.list + s.row * p.slices * kList;
  uint32_t* counts = p.counts + s.row * p.slices;
  if (tid == 0) count = 0;
  __syncthreads();
  over([&](int q, const float (&x)[E]) {
    const int t = row.token(q);
    uint64_t sum = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint32_t b = static_cast<uint32_t>(r.bin(x[e]));
      if (b > border || b >= kWeightBins) continue;
      if (b == border || r.mode == TOP_K) {
        const uint32_t at = atomicAdd(&count, 1u);
        if (at < kList) list[at] = static_cast<uint64_t>(key_of(x[e])) << 32 | static_cast<uint32_t>(t + e);
      } else {
        sum += r.kept_weight(x[e]);
      }
    }
    if (r.mode == TOP_P) {
      sum = wave_sum(sum);
      if (lane == 0) put64(all_sums + q, sum);
    }
  });
  __syncthreads();
  if (p.slices > 1) {
    for (uint32_t i = tid; i < min(count, static_cast<uint32_t>(kList)); i += kThreads) put64(lists + s.at * kList + i, list[i]);
    if (tid == 0) __hip_atomic_store(counts + s.at, count, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (!last_of_row(p, s.row)) return;
    // All slices' lists, one behind the other (a slice's that did not fit: neither does the whole).
    const uint32_t some = tid < p.slices ? __hip_atomic_load(counts + tid, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0;
    uint64_t all;
    const uint64_t before = block_scan(some, all);
    uint32_t* begins = reinterpret_cast<uint32_t*>(bins);  // (and ends)
    if (tid < p.slices) {
      begins[2 * tid] = static_cast<uint32_t>(min(before, uint64_t{kList}));
      begins[2 * tid + 1] = static_cast<uint32_t>(min(before + some, uint64_t{kList}));
    }
    if (tid == 0) count = static_cast<uint32_t>(min(all, uint64_t{kList} + 1));
    __syncthreads();
    for (int i = tid >> 6; i < p.slices; i += kWaves)
      for (uint32_t k = begins[2 * i] + lane; k < begins[2 * i + 1]; k += 64) list[k] = get64(lists + i * kList + k - begins[2 * i]);
    __syncthreads();
  }
  const uint32_t n = count;
  const bool fits = n <= kList;
  for (int i = tid; i < p.chunks; i += kThreads) sums[i] = fits && r.mode == TOP_P ? get64(all_sums + i) : 0;
  // The edge, from the list or from the whole row.
  auto from_list = [&](auto each) {
    for (uint32_t i = tid; i < n; i += kThreads) each(static_cast<uint32_t>(list[i] >> 32), static_cast<uint32_t>(list[i]));
  };
  auto from_row = [&](auto each) {
    OverChunks<DT, 1>(row, 0, p.chunks)([&](int q, const float (&x)[E]) {
      const int t = row.token(q);
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (x[e] > -__builtin_inff()) each(key_of(x[e]), static_cast<uint32_t>(t + e));
    });
  };
  const bool cut = border < kWeightBins;  // (without: fewer than k tokens have a weight)
  Edge edge{0, ~0u};
  if (n <= 64 && r.mode == TOP_K) {
    if (tid < 64) draw_few(p, r, s.row, list, static_cast<int>(n), lane);
    return;
  }
  if (cut || r.top_p < 1.0) {
    Row rr = r;
    if (!cut) rr.mode = TOP_P;
    edge = fits ? edge_of<DT>(rr, bins, from_list, r.mode == TOP_P ? above : 0, whole) : edge_of<DT>(rr, bins, from_row, 0, whole);
  }
  __syncthreads();
  auto weight = [&](float x, int token) { return edge.keeps(key_of(x), static_cast<uint32_t>(token)) ? r.kept_weight(x) : 0; };
  if (fits) {
    for (uint32_t i = tid; i < n; i += kThreads) {
      const uint32_t token = static_cast<uint32_t>(list[i]);
      const uint64_t w = weight(value_of(static_cast<uint32_t>(list[i] >> 32)), static_cast<int>(token));
      if (w) atomicAdd(reinterpret_cast<unsigned long long*>(&sums[(token + row.before) / (64 * E)]), static_cast<unsigned long long>(w));
    }
  } else {
    OverChunks<DT, 1>(row, 0, p.chunks)([&](int q, const float (&x)[E]) {
      const int t = row.token(q);
      uint64_t sum = 0;
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (x[e] > -__builtin_inff()) sum += weight(x[e], t + e);
      sum = wave_sum(sum);
      if (lane == 0) sums[q] = sum;
    });
  }
  __syncthreads();
  draw<DT>(p, r, row, s.row, sums, weight);
}

// The workgroups of a row, of `most` at most. One fits a CU (the weights' pass has registers for one), so that they take turns of
// what a slice's tokens take and its ways in and out beside, which cost as much as 24000 tokens. (In us, with the CUs' share of
// workgroups a row rounded down and so: 132 x 139374 f16 by top-p 153 and 117, 300 x 150000 bf16 269 and 227, 160 x 100000 117 and 105,
// by top-k and top-p 69 and 77; 64 x 151936 with 8 a row, in two turns, 81, with 4 68.)
int slices_of(int64_t rows, int64_t vocabulary, int64_t most, int64_t cus) {
  int64_t best = 1, least = INT64_MAX;
  for (int64_t s = 1; s <= std::max<int64_t>(most, 1) && (s == 1 || rows * s <= 4 * cus); ++s) {
    const int64_t cost = (rows * s + cus - 1) / cus * (vocabulary / s + 24000);
    if (cost < least) {
      least = cost;
      best = s;
    }
  }
  return static_cast<int>(best);
}

}  // namespace
}  // namespace tmh

using namespace tmh;

extern "C" {

int tmh_sample(tmh_ctx* ctx, const void* d_logits, int64_t ld, int dtype, int64_t T, int64_t V, const float* d_temperature,
               const int32_t* d_top_k, const float* d_top_p, const float* d_min_p, const float* d_random, int64_t* d_tokens,
               void* stream) {
  if (!is_float_dtype(dtype)) return fail(ctx, TMH_ERR_INVALID, "sampling takes f32, f16 or bf16 logits, got %s", dtype_name(dtype));
  if (T < 0 || T >= (int64_t{1} << 31)) return fail(ctx, TMH_ERR_INVALID, "sampling cannot take %lld rows", (long long)T);
  if (V < 1) return fail(ctx, TMH_ERR_INVALID, "sampling needs a vocabulary, got %lld tokens", (long long)V);
  if (V >= (1 << 20)) return fail(ctx, TMH_ERR_UNSUPPORTED, "sampling takes fewer than 2^20 tokens, got %lld", (long long)V);
  if (ld < V) return fail(ctx, TMH_ERR_INVALID, "the logits' leading dimension must be at least %lld", (long long)V);
  TMH_TRY(use_device(ctx));
  if (T == 0) return TMH_OK;
  if (!d_logits || !d_random || !d_tokens) return fail(ctx, TMH_ERR_INVALID, "tmh_sample: NULL pointer");
  const int64_t size = dtype_size(dtype), chunk = 64 * 16 / size;
  if (reinterpret_cast<uintptr_t>(d_logits) % size != 0) return fail(ctx, TMH_ERR_UNSUPPORTED, "the logits must lie on multiples of their size");
  hipStream_t s = pick_stream(ctx, stream);
  // In us, by one workgroup a row and by the three kernels: 31 x 703 f16 17.7 and 30.4, 174 x 196 f32 13.5 and 22.4; of all kinds 24 x
  // 8192 bf16 22.4 and 29.6, 193 f32 31.4 and 34.9, 500 f16 47.2 and 52.5, 24 x 16384 31.6 and 32.3, 193 44.6 and 41.1, 500 71.4 and
  // 63.4. (One row by top-k and top-p, of 8192, 23.8 and 19.5.)
  const bool is_short = V <= kShort;
  const int64_t most_rows = std::min<int64_t>(kMostRows, 2 * ctx->num_cus);
  const int64_t rows = std::min(T, most_rows);
  SampleArgs p{};
  p.ld = ld;
  p.vocabulary = static_cast<int>(V);
  p.chunks = static_cast<int>((V + 16 / size - 1 + chunk - 1) / chunk);  // (rows that begin inside 16 bytes may take one more)
  p.slices = is_short ? 1 : slices_of(rows, V, p.chunks / kWaves, ctx->num_cus);
  if (!is_short) {
    const size_t of_rows = static_cast<size_t>(rows) * p.slices;
    const size_t bytes = 8 * (of_rows * (1 + kWeightBins + (p.slices > 1 ? kList : 0)) + static_cast<size_t>(rows) * (p.chunks + 4)) + 4 * of_rows;
    void* ws = workspace(ctx, bytes, s);
    if (!ws) return fail(ctx, TMH_ERR_UNSUPPORTED, "sampling's workspace cannot grow here: run one call before the capture");
    p.best = static_cast<uint64_t*>(ws);
    p.bins = p.best + of_rows;
    p.list = p.bins + of_rows * kWeightBins;
    p.sums = p.list + (p.slices > 1 ? of_rows * kList : 0);
    p.told = p.sums + static_cast<size_t>(rows) * p.chunks;
    p.counts = reinterpret_cast<uint32_t*>(p.told + static_cast<size_t>(rows) * 4);
    p.meet = ctx->meet;
  }
  in_launches(T, is_short ? most_a_launch(kThreads, 1, 1) : most_rows, [&](int64_t first, int64_t some) {
    auto from = [&](auto* a) { return a ? a + first : a; };
    p.x = static_cast<const char*>(d_logits) + first * ld * size;
    p.temperature = from(d_temperature);
    p.top_k = from(d_top_k);
    p.top_p = from(d_top_p);
    p.min_p = from(d_min_p);
    p.u = from(d_random);
    p.tokens = d_tokens + first;
    const unsigned grid = static_cast<unsigned>(some * p.slices);
    auto launch = [&](auto dt) {
      constexpr int DT = decltype(dt)::value;
      if (is_short) {
        k_sample_short<DT><<<static_cast<unsigned>(some), kThreads, 8 * p.chunks + 4 * p.vocabulary, s>>>(p);
        return;
      }
      k_sample_top<DT><<<grid, kThreads, 0, s>>>(p);
      k_sample_sum<DT><<<grid, kThreads, 8 * std::max(kWeightBins, p.chunks), s>>>(p);
      if (d_top_k || d_top_p) k_sample_draw<DT><<<grid, kThreads, 8 * p.chunks, s>>>(p);
    };
    if (dtype == TMH_F32) launch(std::integral_constant<int, DT_F32>{});
    else if (dtype == TMH_F16) launch(std::integral_constant<int, DT_F16>{});
    else launch(std::integral_constant<int, DT_BF16>{});
  });
  return check_launch(ctx, "sampling");
}

}  // extern "C"
