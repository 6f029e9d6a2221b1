// Tokens drawn from rows of logits by temperature, top-k, top-p, min-p and given random numbers (tmh_sample).
#include <cmath>
#include <type_traits>

#include "tmh_device.h"
#include "tmh_internal.h"
#include "tmh_launch.h"

namespace tmh {
namespace {

struct SampleArgs {
  const void* x;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  const float* u;
  int64_t* tokens;
  int64_t ld;
  int vocabulary;
};

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kUnit = 44;  // weights are multiples of 2^-44 (of the largest's): sums of up to 2^20 of them in 64 bits
constexpr int kSegment = 512;
constexpr int kMostSegments = (1 << 20) / kSegment;
constexpr int kBins = 2048;

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

// 2^x, x <= 0, in 64 bits: 2^n e^y with y = (x - n) ln 2 of magnitude up to 0.35, whose series ends with y^12 / 12! (the
// next term is 2^-52).
__device__ __forceinline__ double exp2_of(double x) {
  const double n = __builtin_rint(x), y = (x - n) * 0.69314718055994530942;
  double s = 1.0 / 479001600.0;
  s = fma(s, y, 1.0 / 39916800.0);
  s = fma(s, y, 1.0 / 3628800.0);
  s = fma(s, y, 1.0 / 362880.0);
  s = fma(s, y, 1.0 / 40320.0);
  s = fma(s, y, 1.0 / 5040.0);
  s = fma(s, y, 1.0 / 720.0);
  s = fma(s, y, 1.0 / 120.0);
  s = fma(s, y, 1.0 / 24.0);
  s = fma(s, y, 1.0 / 6.0);
  s = fma(s, y, 0.5);
  s = fma(s, y, 1.0);
  s = fma(s, y, 1.0);
  return __builtin_amdgcn_ldexp(s, static_cast<int>(n));
}

struct Weigh {
  float top;  // the row's largest logit
  double c;   // log2(e) / temperature
  double least;
  // exp((x - top) / temperature) in units of 2^-44; 0 where it is less than one, or less than `least`.
  __device__ __forceinline__ uint64_t operator()(float x) const {
    if (top == __builtin_inff()) return x == top ? uint64_t{1} << kUnit : 0;
    const double e = (static_cast<double>(x) - static_cast<double>(top)) * c;
    if (!(e >= -kUnit)) return 0;
    const double w = exp2_of(e);
    return w >= least ? static_cast<uint64_t>(__builtin_rint(w * 0x1p44)) : 0;
  }
};

__device__ __forceinline__ uint64_t wave_sum(uint64_t v) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ __forceinline__ uint64_t wave_max(uint64_t v) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) v = max(v, static_cast<uint64_t>(__shfl_xor(v, o)));
  return v;
}
// The sum over the lanes up to this one.
__device__ __forceinline__ uint64_t wave_scan(uint64_t v) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint64_t up = __shfl_up(v, o);
    if ((threadIdx.x & 63) >= o) v += up;
  }
  return v;
}

// One workgroup a row. Weights are whole numbers, so that their sums do not depend on an order.
template <int DT>
__global__ __launch_bounds__(kThreads) void k_sample(SampleArgs p, int64_t first) {
  __shared__ uint64_t bins[kBins];
  __shared__ uint64_t red[kWaves];
  __shared__ uint64_t seg_sum[kMostSegments];
  __shared__ uint32_t seg_ties[kMostSegments];
  __shared__ uint64_t found[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = p.vocabulary;
  const int64_t row = first + blockIdx.x;
  const int64_t base = row * p.ld;
  auto logit = [&](int i) { return load_as_f32<DT>(p.x, base + i); };
  auto block = [&](uint64_t v, auto join) {  // (all threads)
    __syncthreads();
    if (lane == 0) red[wave] = v;
    __syncthreads();
    uint64_t all = red[0];
    for (int w = 1; w < kWaves; ++w) all = join(all, red[w]);
    return all;
  };
  // The largest logit, and of equal ones the first.
  uint64_t best = 0;
  for (int i = tid; i < n; i += kThreads) best = max(best, static_cast<uint64_t>(key_of(logit(i))) << 32 | static_cast<uint32_t>(~i));
  best = block(wave_max(best), [](uint64_t a, uint64_t b) { return max(a, b); });
  const uint32_t top_key = static_cast<uint32_t>(best >> 32);
  const float temperature = p.temperature ? p.temperature[row] : 1.f;
  if (top_key == key_of(-__builtin_inff())) {  // no token
    if (tid == 0) p.tokens[row] = -1;
    return;
  }
  if (!(temperature > 0.f)) {
    if (tid == 0) p.tokens[row] = static_cast<uint32_t>(~best);
    return;
  }
  Weigh weigh{value_of(top_key), 1.4426950408889634074 / static_cast<double>(temperature), 0.0};

  // Kept are the keys above `edge`, and the first `ties` tokens of that key.
  uint32_t edge = 0;
  uint64_t ties = ~uint64_t{0};
  // The key at which the sum of measure(key) over kept keys, from the largest down, reaches `need`, and the sum above it.
  auto select = [&](auto measure, auto reached, uint64_t& above) {
    uint32_t prefix = 0, mask = 0;
    above = 0;
#pragma unroll 1
    for (int shift : {21, 10, 0}) {
      const uint32_t digits = shift ? 2047u : 1023u;
      __syncthreads();
      for (int i = tid; i < kBins; i += kThreads) bins[i] = 0;
      __syncthreads();
      for (int i = tid; i < n; i += kThreads) {
        const uint32_t key = key_of(logit(i));
        if (key < edge || (key & mask) != prefix) continue;
        atomicAdd(reinterpret_cast<unsigned long long*>(&bins[key >> shift & digits]), static_cast<unsigned long long>(measure(key)));
      }
      __syncthreads();
      if (wave == 0) {  // lane l: bins from digits - 32 l down
        uint64_t mine = 0;
        for (int i = 0; i < 32; ++i)
          if (static_cast<int>(digits) - 32 * lane - i >= 0) mine += bins[digits - 32 * lane - i];
        const uint64_t upto = wave_scan(mine) + above;
        const uint64_t past = __ballot(reached(upto));
        const int at = past ? __builtin_ctzll(past) : digits / 32;  // (always reached by the last)
        if (lane == at) {
          uint64_t sum = upto - mine;
          int i = 0;
          for (; i < 31 && static_cast<int>(digits) - 32 * lane - i > 0; ++i) {
            if (reached(sum + bins[digits - 32 * lane - i])) break;
            sum += bins[digits - 32 * lane - i];
          }
          found[0] = digits - 32 * lane - i;
          found[1] = sum;
        }
      }
      __syncthreads();
      prefix |= static_cast<uint32_t>(found[0]) << shift;
      mask |= digits << shift;
      above = found[1];
    }
    return prefix;
  };
  const int k = p.top_k ? p.top_k[row] : 0;
  if (k > 0 && k < n) {
    uint64_t above;
    edge = select([](uint32_t) { return uint64_t{1}; }, [&](uint64_t sum) { return sum >= static_cast<uint64_t>(k); }, above);
    ties = static_cast<uint64_t>(k) - above;
  }
  const float top_p = p.top_p ? p.top_p[row] : 1.f;
  if (top_p < 1.f) {
    // Of tokens at the edge only `ties` count: they weigh the same, so the rest of theirs is taken off the sum.
    uint64_t sum = 0, at_edge = 0;
    for (int i = tid; i < n; i += kThreads) {
      const float x = logit(i);
      const uint32_t key = key_of(x);
      if (key > edge) sum += weigh(x);
      at_edge += key == edge;
    }
    auto add = [](uint64_t a, uint64_t b) { return a + b; };
    sum = block(wave_sum(sum), add);
    at_edge = min(block(wave_sum(at_edge), add), ties);
    sum += at_edge * weigh(value_of(edge));
    const double need = fmax(static_cast<double>(top_p) * static_cast<double>(sum), 1.0);  // (one token at least)
    uint64_t above;
    const uint32_t last = edge;
    const uint64_t last_ties = at_edge;
    edge = select([&](uint32_t key) { return weigh(value_of(key)); }, [&](uint64_t s) { return static_cast<double>(s) >= need; }, above);
    const uint64_t each = weigh(value_of(edge));
    ties = 1;
    if (each && static_cast<double>(above + each) < need) {
      ties = static_cast<uint64_t>((need - static_cast<double>(above)) / static_cast<double>(each));
      if (ties) --ties;  // (the quotient is rounded: counted up from just below)
      while (static_cast<double>(above + ties * each) < need) ++ties;
    }
    if (edge == last) ties = min(ties, last_ties);
  }
  if (p.min_p && p.min_p[row] > 0.f) weigh.least = fmin(static_cast<double>(p.min_p[row]), 1.0);
  const uint64_t each = weigh(value_of(edge));

  // Sums of segments in the order of the tokens, then the segment where they pass u of the whole.
  const int segments = (n + kSegment - 1) / kSegment;
  __syncthreads();
  for (int s = wave; s < segments; s += kWaves) {
    uint64_t sum = 0;
    uint32_t equal = 0;
    for (int j = 0; j < kSegment / 64; ++j) {
      const int i = s * kSegment + j * 64 + lane;
      if (i >= n) continue;
      const float x = logit(i);
      const uint32_t key = key_of(x);
      if (key > edge) sum += weigh(x);
      equal += key == edge;
    }
    sum = wave_sum(sum);
    equal = static_cast<uint32_t>(wave_sum(equal));
    if (lane == 0) {
      seg_sum[s] = sum;
      seg_ties[s] = equal;
    }
  }
  __syncthreads();
  if (wave != 0) return;
  // (A segment's kept ties: as many of its own as `ties` has left for it.)
  uint64_t total = 0, before_ties = 0;
  for (int s0 = 0; s0 < segments; s0 += 64) {
    const int s = s0 + lane;
    const uint64_t equal = s < segments ? seg_ties[s] : 0, upto = wave_scan(equal) + before_ties;
    const uint64_t start = min(upto - equal, ties), kept = min(upto, ties) - start;
    if (s < segments) seg_sum[s] += kept * each;
    total += wave_sum(s < segments ? seg_sum[s] : 0);
    before_ties = __shfl(upto, 63);
  }
  const float u = p.u[row];
  const double target = static_cast<double>(u) * static_cast<double>(total);
  uint64_t before = 0, ties_before = 0;
  int segment = -1;
  for (int s0 = 0; s0 < segments; s0 += 64) {
    const int s = s0 + lane;
    const uint64_t mine = s < segments ? seg_sum[s] : 0, upto = wave_scan(mine) + before;
    const uint64_t equal = s < segments ? seg_ties[s] : 0, ties_upto = wave_scan(equal) + ties_before;
    // (Where no sum is above the target, as for u >= 1, the last token of any weight is taken.)
    const uint64_t past = __ballot(mine != 0 && (static_cast<double>(upto) > target || upto == total));
    if (past) {
      const int at = __builtin_ctzll(past);
      segment = s0 + at;
      before = __shfl(upto - mine, at);
      ties_before = __shfl(ties_upto - equal, at);
      break;
    }
    before = __shfl(upto, 63);
    ties_before = __shfl(ties_upto, 63);
  }
  if (segment < 0) return;  // (not reached: the largest logit has a weight)
  for (int j = 0; j < kSegment / 64; ++j) {
    const int i = segment * kSegment + j * 64 + lane;
    uint64_t w = 0, equal = 0;
    if (i < n) {
      const float x = logit(i);
      const uint32_t key = key_of(x);
      equal = key == edge;
      if (key > edge) w = weigh(x);
    }
    const uint64_t ties_upto = wave_scan(equal) + ties_before;
    if (equal && ties_upto <= ties) w = each;
    const uint64_t upto = wave_scan(w) + before;
    const uint64_t past = __ballot(w != 0 && (static_cast<double>(upto) > target || upto == total));
    if (past) {
      if (lane == __builtin_ctzll(past)) p.tokens[row] = i;
      return;
    }
    before = __shfl(upto, 63);
    ties_before = __shfl(ties_upto, 63);
  }
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
  SampleArgs p{d_logits, d_temperature, d_top_k, d_top_p, d_min_p, d_random, d_tokens, ld, static_cast<int>(V)};
  hipStream_t s = pick_stream(ctx, stream);
  in_launches(T, most_a_launch(kThreads, 1, 1), [&](int64_t first, int64_t rows) {
    const unsigned grid = static_cast<unsigned>(rows);
    if (dtype == TMH_F32) k_sample<DT_F32><<<grid, kThreads, 0, s>>>(p, first);
    else if (dtype == TMH_F16) k_sample<DT_F16><<<grid, kThreads, 0, s>>>(p, first);
    else k_sample<DT_BF16><<<grid, kThreads, 0, s>>>(p, first);
  });
  return check_launch(ctx, "k_sample");
}

}  // extern "C"
