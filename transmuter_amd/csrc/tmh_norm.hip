// The root-mean-square norm with the residual's addition, and rows in 8 bits (tmh_rms_norm, tmh_quantize_rows). Both
// are bound by memory: each input is read once and each output written once. 4096 x 2048 bf16 with a residual,
// answered in bf16 and 8 bits: 13.0 us, 5.8 TB/s; the gated 2048 x 11008 f16 20.6 us, 5.5 TB/s (a large copy: 4.8).
#include <algorithm>
#include <type_traits>

#include "tmh_f8.h"
#include "tmh_internal.h"
#include "tmh_launch.h"

namespace tmh {
namespace {

struct NormArgs {
  const void* x;
  const void* residual;
  const void* gamma;
  void* sum;
  void* y;
  uint8_t* q;
  float* scales;
  int64_t ldx, ldr, lds, ldy, ldq, rows;
  int cols, gamma_dtype;
  float eps;
  uint32_t count;  // rows of this launch, whose first the pointers are at (`rows`: of the call, the scales' pitch)
};

// Consecutive rows on one XCD (workgroups go to the eight XCDs in turn): their scales of one block lie side by
// side, and lines that one XCD's L2 holds whole are written to memory whole.
__device__ __forceinline__ int64_t xcd_row_group(uint32_t block, uint32_t blocks) {
  const uint32_t per = blocks / 8;
  return block < 8 * per ? (block & 7) * per + (block >> 3) : block;
}

__device__ __forceinline__ void load_gamma(const NormArgs& p, int col, int n, Raw8& raw) {
  if (p.gamma_dtype == DT_F32) load_raw8<DT_F32>(p.gamma, col, n, raw);
  else load_raw8<DT_F16>(p.gamma, col, n, raw);  // (or bf16: 16 bits)
}
__device__ __forceinline__ void gamma_of(const NormArgs& p, const Raw8& raw, float (&g)[8]) {
  if (p.gamma_dtype == DT_F16) floats_of<DT_F16>(raw, g);
  else if (p.gamma_dtype == DT_BF16) floats_of<DT_BF16>(raw, g);
  else floats_of<DT_F32>(raw, g);
}
__device__ __forceinline__ void load_gamma(const NormArgs& p, int col, int n, float (&g)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) g[i] = i * kLaneStep < n ? load_float_rt(p.gamma, p.gamma_dtype, col + i * kLaneStep) : 0.f;
}

// The sum of a value over the threads of a row (a wavefront, or with WIDE a workgroup), in all of them.
template <bool WIDE>
__device__ __forceinline__ float row_total(float v) {
  v = row_sum(v);
  v += __shfl_xor(v, 16);
  v += __shfl_xor(v, 32);
  if constexpr (WIDE) {
    __shared__ float part[16];
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = part[0];
    for (uint32_t i = 1; i < blockDim.x / 64; ++i) v += part[i];
  }
  return v;
}

// r and f with h * f * r = h / sqrt(mean(h^2) + eps) for a row, given a thread's own sum of (f h)^2 for a factor f: 1, but
// for rows that f32 has no room for. Squares of values of 2^64 and more overflow, though their root would not: a row whose
// total is infinite (for all its threads) is summed again with f = 2^-80, which leaves room for 2^30 of the largest
// numbers. Squares below 2^-126 lose bits, and count where the mean and eps are below 2^-96: then f = 2^96, which makes
// squares of the smallest numbers normal ones and 2^30 of 2^96 at most. (Rows of zeros without an eps are 0 / 0.)
struct RowScale {
  float f, r;
};
template <bool WIDE, typename Sum>
__device__ __forceinline__ RowScale row_scale(const NormArgs& p, Sum sum) {
  float total = row_total<WIDE>(sum(1.f));
  const float mean = total / static_cast<float>(p.cols) + p.eps;
  if (total != __builtin_inff() && !(mean < 0x1p-96f)) return {1.f, 1.f / sqrtf(mean)};
  const float f = total == __builtin_inff() ? 0x1p-80f : 0x1p96f;
  if constexpr (WIDE) __syncthreads();  // every thread has read the wavefronts' sums
  total = row_total<WIDE>(sum(f));
  return {f, 1.f / sqrtf(total / static_cast<float>(p.cols) + p.eps * f * f)};
}

template <int DT, bool VEC>
__device__ __forceinline__ void norm_outputs(const NormArgs& p, int64_t row, int col, int n, const float (&h)[8],
                                             const float (&g)[8], float rstd) {
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = h[i] * rstd * g[i];
  if (p.y) store8<DT, VEC, kLaneStep>(p.y, row * p.ldy + col, n, v);
  if (p.q) {
    uint2 q;
    const float scale = f8_block(v, q);
    store8_f8<VEC, kLaneStep>(p.q, row * p.ldq + col, n, q);
    if (n > 0 && (threadIdx.x & 15) == 0) p.scales[static_cast<int64_t>(col / kF8Block) * p.rows + row] = scale;
  }
}

// A row to a wavefront, or with WIDE to a workgroup, each thread with NCH pieces of eight columns in registers, so
// that a row is read once; the sum of squares is f32, taken in a tree. Sixteen lanes hold a block of 128 columns,
// whose largest magnitude they find among themselves. Rows of up to 512 columns go to a wavefront each (no barrier),
// others to as many wavefronts as hold them, with one piece a thread while a workgroup can: 4096 rows of 4096 f16
// with a residual 26.4 us, 30.3 with two pieces and half the threads, 45.0 with a wavefront to a row.
template <int DT, bool WIDE, int NCH, bool VEC>
__global__ __launch_bounds__(WIDE ? 1024 : 256) void k_rms_norm(NormArgs p) {
  const int tpr = WIDE ? static_cast<int>(blockDim.x) : 64;
  const int t = WIDE ? static_cast<int>(threadIdx.x) : static_cast<int>(threadIdx.x) % 64;
  const int64_t group = xcd_row_group(blockIdx.x, gridDim.x);
  const int64_t row = WIDE ? group : group * 4 + threadIdx.x / 64;
  // (A workgroup's own row always exists, but the question brings its arguments ahead of the loads: 512 rows of 32768 bf16
  // 33.5 us, 34.4 without it.)
  if (row >= (WIDE ? p.rows : p.count)) return;
  auto column = [&](int c) { return c * tpr * 8 + (t >> 4) * kF8Block + lane_columns(VEC); };
  float h[NCH][8], g[NCH][8];
  if constexpr (VEC) {  // every load, then what waits for them (4096 x 2048 bf16 13.5 us one after another, 13.0 so)
    Raw8 x[NCH], r[NCH], w[NCH];
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int col = column(c);
      load_raw8<DT>(p.x, row * p.ldx + col, p.cols - col, x[c]);
      if (p.residual) load_raw8<DT>(p.residual, row * p.ldr + col, p.cols - col, r[c]);
      load_gamma(p, col, p.cols - col, w[c]);
    }
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      floats_of<DT>(x[c], h[c]);
      if (p.residual) {
        float more[8];
        floats_of<DT>(r[c], more);
#pragma unroll
        for (int i = 0; i < 8; ++i) h[c][i] += more[i];
      }
      gamma_of(p, w[c], g[c]);
    }
  } else {
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int col = column(c);
      load8<DT, false, kLaneStep>(p.x, row * p.ldx + col, p.cols - col, h[c]);
      load_gamma(p, col, p.cols - col, g[c]);
      if (p.residual) {
        float r[8];
        load8<DT, false, kLaneStep>(p.residual, row * p.ldr + col, p.cols - col, r);
#pragma unroll
        for (int i = 0; i < 8; ++i) h[c][i] += r[i];
      }
    }
  }
  auto squares = [&](float f) {
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) s = fmaf(f * h[c][i], f * h[c][i], s);
    return s;
  };
  if (p.sum) {
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int col = column(c);
      store8<DT, VEC, kLaneStep>(p.sum, row * p.lds + col, p.cols - col, h[c]);
    }
  }
  const RowScale scale = row_scale<WIDE>(p, squares);
  if (scale.f != 1.f) {
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) h[c][i] *= scale.f;
  }
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int col = column(c);
    norm_outputs<DT, VEC>(p, row, col, p.cols - col, h[c], g[c], scale.r);
  }
}

// Rows of more than 32768 columns: the inputs are read twice, the second time from the caches. An
// output may be an input's memory: a row is read whole ahead of the barrier, and its outputs are written by the
// thread that has just read the same elements again.
template <int DT>
__global__ __launch_bounds__(1024) void k_rms_norm_any(NormArgs p) {
  const int64_t row = xcd_row_group(blockIdx.x, gridDim.x);
  const int own = static_cast<int>(threadIdx.x >> 4) * kF8Block + lane_columns(false);
  auto load = [&](int col, float (&h)[8]) {
    load8<DT, false, kLaneStep>(p.x, row * p.ldx + col, p.cols - col, h);
    if (p.residual) {
      float r[8];
      load8<DT, false, kLaneStep>(p.residual, row * p.ldr + col, p.cols - col, r);
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] += r[i];
    }
  };
  const RowScale scale = row_scale<true>(p, [&](float f) {
    float s = 0.f;
    for (int col = own; col < p.cols; col += 8 * static_cast<int>(blockDim.x)) {
      float h[8];
      load(col, h);
#pragma unroll
      for (int i = 0; i < 8; ++i) s = fmaf(f * h[i], f * h[i], s);
    }
    return s;
  });
  // Whole blocks of 16 lanes stay together: lanes past the row hold zeros.
  for (int col = own; col - static_cast<int>(threadIdx.x & 15) < p.cols; col += 8 * static_cast<int>(blockDim.x)) {
    float h[8], g[8];
    load(col, h);
    load_gamma(p, col, p.cols - col, g);
    if (p.sum) store8<DT, false, kLaneStep>(p.sum, row * p.lds + col, p.cols - col, h);
    if (scale.f != 1.f) {
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] *= scale.f;
    }
    norm_outputs<DT, false>(p, row, col, p.cols - col, h, g, scale.r);
  }
}

struct QuantizeArgs {
  const void* x;
  const void* gate;
  uint8_t* q;
  float* scales;
  int64_t ldx, ldg, ldq, rows;
  int cols;
  uint32_t blocks;  // of 128 columns in a row
  FastDiv by_blocks;
};

// g / (1 + e^-g), as (g / 4) / (1/4 + e^-g / 4): the reciprocal, which ends at the smallest normal number, is that of a
// quarter of the sum, and so serves sums up to 2^128, where f32 ends (g of -88.7; the answer is 0 below), not 2^126.
__device__ __forceinline__ float silu(float g) {
  return 0.25f * g * __builtin_amdgcn_rcpf(0.25f + __builtin_amdgcn_exp2f(fmaf(g, -1.44269504088896340736f, -2.f)));
}

// Sixteen lanes to a block of 128 columns, the blocks of the rows one after another. A gated value took 21
// instructions with the divisions' general forms (25.5 us where 20.6 are now: it was bound by them).
template <int DT, bool VEC, bool GATE>
__global__ __launch_bounds__(256) void k_quantize_rows(QuantizeArgs p, int64_t first) {
  const int64_t all = p.rows * p.blocks;
  const uint32_t local = blockIdx.x * 16 + (threadIdx.x >> 4);
  const int64_t block = first * p.blocks + local;
  if (block >= all) return;  // whole rows of lanes
  const uint32_t r = p.by_blocks.div(local);
  const int64_t row = first + r;
  const uint32_t b = local - r * p.blocks;
  const int col = static_cast<int>(b) * kF8Block + lane_columns(VEC), n = p.cols - col;
  float v[8];
  load8<DT, VEC, kLaneStep>(p.x, row * p.ldx + col, n, v);
  if constexpr (GATE) {
    float g[8];
    load8<DT, VEC, kLaneStep>(p.gate, row * p.ldg + col, n, g);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= silu(g[i]);
  }
  uint2 q;
  const float scale = f8_block(v, q);
  store8_f8<VEC, kLaneStep>(p.q, row * p.ldq + col, n, q);
  if ((threadIdx.x & 15) == 0) p.scales[static_cast<int64_t>(b) * p.rows + row] = scale;
}

bool aligned(const void* p, int64_t ld, int dtype, int64_t bytes = 16) {
  return !p || (reinterpret_cast<uintptr_t>(p) % bytes == 0 && ld * (dtype == TMH_F8E4M3 ? 1 : dtype_size(dtype)) % bytes == 0);
}

template <int DT>
void launch_norm(const NormArgs& call, bool vec, hipStream_t s) {
  NormArgs p = call;
  // Whole wavefronts of `pieces` pieces of eight columns a thread.
  auto threads_of = [&](int pieces) { return (p.cols + 512 * pieces - 1) / (512 * pieces) * 64; };
  const bool four = p.cols <= 512;  // rows a workgroup
  const int threads = four ? 256 : p.cols <= 8192 ? threads_of(1) : p.cols <= 16384 ? threads_of(2) : p.cols <= 32768 ? threads_of(4) : 1024;
  in_launches(p.rows, most_a_launch(threads, four ? 4 : 1, 1), [&](int64_t first, int64_t count) {
    auto at = [&](auto* base, int64_t ld, int64_t size) {
      return base ? reinterpret_cast<decltype(base)>(reinterpret_cast<uintptr_t>(base) + first * ld * size) : nullptr;
    };
    constexpr int64_t size = DT == DT_F32 ? 4 : 2;
    p.x = at(call.x, p.ldx, size);
    p.residual = at(call.residual, p.ldr, size);
    p.sum = at(call.sum, p.lds, size);
    p.y = at(call.y, p.ldy, size);
    p.q = at(call.q, p.ldq, 1);
    p.scales = at(call.scales, 1, sizeof(float));
    p.count = static_cast<uint32_t>(count);
    const unsigned grid = static_cast<unsigned>(four ? (count + 3) / 4 : count);
    auto launch = [&](auto v) {
      constexpr bool VEC = decltype(v)::value;
      if (four) k_rms_norm<DT, false, 1, VEC><<<grid, threads, 0, s>>>(p);
      else if (p.cols <= 8192) k_rms_norm<DT, true, 1, VEC><<<grid, threads, 0, s>>>(p);
      else if (p.cols <= 16384) k_rms_norm<DT, true, 2, VEC><<<grid, threads, 0, s>>>(p);
      else if (p.cols <= 32768) k_rms_norm<DT, true, 4, VEC><<<grid, threads, 0, s>>>(p);
      else k_rms_norm_any<DT><<<grid, threads, 0, s>>>(p);
    };
    if (vec) launch(std::true_type{});
    else launch(std::false_type{});
  });
}

template <int DT>
void launch_quantize(const QuantizeArgs& p, bool vec, hipStream_t s) {
  // (Their blocks are within the division's range of 2^31, too.)
  in_launches(p.rows, most_a_launch(256, 16, p.blocks), [&](int64_t first, int64_t rows) {
    const unsigned grid = static_cast<unsigned>((rows * p.blocks + 15) / 16);
    if (p.gate) {
      if (vec) k_quantize_rows<DT, true, true><<<grid, 256, 0, s>>>(p, first);
      else k_quantize_rows<DT, false, true><<<grid, 256, 0, s>>>(p, first);
    } else {
      if (vec) k_quantize_rows<DT, true, false><<<grid, 256, 0, s>>>(p, first);
      else k_quantize_rows<DT, false, false><<<grid, 256, 0, s>>>(p, first);
    }
  });
}

}  // namespace
}  // namespace tmh

using namespace tmh;

extern "C" {

int tmh_rms_norm(tmh_ctx* ctx, const void* d_x, int64_t ldx, const void* d_residual, int64_t ldr, int dtype,
                 int64_t T, int64_t N, const void* d_gamma, int gamma_dtype, float eps, void* d_sum, int64_t lds,
                 void* d_y, int64_t ldy, void* d_q, int64_t ldq, float* d_q_scales, void* stream) {
  if (!is_float_dtype(dtype)) return fail(ctx, TMH_ERR_INVALID, "the norm takes f32, f16 or bf16 rows, got %s", dtype_name(dtype));
  if (!is_float_dtype(gamma_dtype)) return fail(ctx, TMH_ERR_INVALID, "the norm's gamma must be f32, f16 or bf16, got %s", dtype_name(gamma_dtype));
  if (T < 0 || N < 1 || T >= (int64_t{1} << 31) || N > (int64_t{1} << 30))
    return fail(ctx, TMH_ERR_INVALID, "the norm cannot take %lld rows of %lld columns", (long long)T, (long long)N);
  if (!(eps >= 0.f)) return fail(ctx, TMH_ERR_INVALID, "the norm's eps must not be negative or NaN");
  if (!d_y && !d_q) return fail(ctx, TMH_ERR_INVALID, "the norm has no output: y and q are NULL");
  if (!d_q != !d_q_scales) return fail(ctx, TMH_ERR_INVALID, "the norm's q and its scales go together");
  if (ldx < N || (d_residual && ldr < N) || (d_sum && lds < N) || (d_y && ldy < N) || (d_q && ldq < N))
    return fail(ctx, TMH_ERR_INVALID, "the norm's leading dimensions must be at least N=%lld", (long long)N);
  TMH_TRY(use_device(ctx));
  if (T == 0) return TMH_OK;
  if (!d_x || !d_gamma) return fail(ctx, TMH_ERR_INVALID, "tmh_rms_norm: NULL pointer");
  NormArgs p{d_x, d_residual, d_gamma, d_sum, d_y, static_cast<uint8_t*>(d_q), d_q_scales, ldx, ldr, lds, ldy, ldq, T,
             static_cast<int>(N), gamma_dtype, eps, 0};
  const bool vec = N % 8 == 0 && aligned(d_x, ldx, dtype) && aligned(d_residual, ldr, dtype) && aligned(d_sum, lds, dtype) &&
                   aligned(d_y, ldy, dtype) && aligned(d_q, ldq, TMH_F8E4M3, 8) && aligned(d_gamma, 0, gamma_dtype);
  hipStream_t s = pick_stream(ctx, stream);
  if (dtype == TMH_F32) launch_norm<DT_F32>(p, vec, s);
  else if (dtype == TMH_F16) launch_norm<DT_F16>(p, vec, s);
  else launch_norm<DT_BF16>(p, vec, s);
  return check_launch(ctx, "k_rms_norm");
}

int tmh_quantize_rows(tmh_ctx* ctx, const void* d_x, int64_t ldx, const void* d_gate, int64_t ldg, int dtype,
                      int64_t T, int64_t N, void* d_q, int64_t ldq, float* d_q_scales, void* stream) {
  if (!is_float_dtype(dtype)) return fail(ctx, TMH_ERR_INVALID, "rows to quantize must be f32, f16 or bf16, got %s", dtype_name(dtype));
  if (T < 0 || N < 1 || T >= (int64_t{1} << 31) || N > (int64_t{1} << 30))
    return fail(ctx, TMH_ERR_INVALID, "cannot quantize %lld rows of %lld columns", (long long)T, (long long)N);
  if (ldx < N || (d_gate && ldg < N) || ldq < N)
    return fail(ctx, TMH_ERR_INVALID, "the leading dimensions of rows to quantize must be at least N=%lld", (long long)N);
  TMH_TRY(use_device(ctx));
  if (T == 0) return TMH_OK;
  if (!d_x || !d_q || !d_q_scales) return fail(ctx, TMH_ERR_INVALID, "tmh_quantize_rows: NULL pointer");
  const uint32_t blocks = static_cast<uint32_t>((N + kF8Block - 1) / kF8Block);
  QuantizeArgs p{d_x, d_gate, static_cast<uint8_t*>(d_q), d_q_scales, ldx, ldg, ldq, T, static_cast<int>(N), blocks,
                 FastDiv(blocks)};
  const bool vec = N % 8 == 0 && aligned(d_x, ldx, dtype) && aligned(d_gate, ldg, dtype) && aligned(d_q, ldq, TMH_F8E4M3, 8);
  hipStream_t s = pick_stream(ctx, stream);
  if (dtype == TMH_F32) launch_quantize<DT_F32>(p, vec, s);
  else if (dtype == TMH_F16) launch_quantize<DT_F16>(p, vec, s);
  else launch_quantize<DT_BF16>(p, vec, s);
  return check_launch(ctx, "k_quantize_rows");
}

}  // extern "C"
