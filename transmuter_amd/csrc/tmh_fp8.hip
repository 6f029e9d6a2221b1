// The product of 8-bit rows with an 8-bit weight (tmh_matmul_fp8): one matrix product a block of 128 of K, whose
// result is multiplied by the row's and the weight block's scales as it is added to the f32 sums.
//
// For a 16-bit Y a block is one v_mfma_f32_16x16x128_f8f6f4. That unit sums products eight at a time, each cut to a
// multiple of 2^-13 of the power of two at or below the largest of the eight (measured: seven products of 2^-13.2
// beside one of 1 vanish), and these sums in f32: over random factors 1.5e-5 to 5e-5 of Y in the 2-norm, against
// 2e-4 (f16) and 1.7e-3 (bf16) that Y's own rounding leaves. An f32 Y would show it, so its factors are converted
// to f16, which holds every e4m3 value, and multiplied by v_mfma_f32_16x16x32_f16, whose products are exact and
// summed in f32 (8e-8 in the 2-norm), at half the rate or less.
#include <algorithm>
#include <new>

#include "tmh_f8.h"
#include "tmh_internal.h"

// Tiles of 16 rows x 128 of K, 2 KiB each in the order [N / 16][K / 128]: two halves (64 of K each) of 1 KiB,
// lane l = 16 g + r of a wavefront holding row r, k = 64 h + 16 g .. + 15 at offset 16 l of half h. A
// wavefront's 16-byte loads of a tile are its MFMA operand (the order of k within a block is free, as long as
// both factors share it), and read 1 KiB in a row. Rows past N and k past K are zeros.
struct tmh_fp8_weight {
  int device = 0;
  int64_t K = 0, N = 0;
  int64_t kb = 0, tiles = 0;    // blocks of 128 of K, tiles of 16 rows
  uint8_t* d_q = nullptr;       // tiles * kb * 2048 bytes
  float* d_scales = nullptr;    // [ceil(N / 128)][kb]
  size_t device_bytes = 0;
};

namespace tmh {
namespace {

typedef int int8v_t __attribute__((ext_vector_type(8)));

constexpr int kTileBytes = 2048;

// Sixteen bytes of a row's block as MFMA operands: e4m3, or (EXACT) the same values in f16.
template <bool EXACT>
struct Piece {
  uint4_t q;
  __device__ __forceinline__ void set(uint4_t v) { q = v; }
};
template <>
struct Piece<true> {
  half8_t h[2];
  __device__ __forceinline__ void set(uint4_t v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const half2_t lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v[i], 1.f, false);
      const half2_t hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v[i], 1.f, true);
      h[i >> 1][4 * (i & 1)] = lo[0];
      h[i >> 1][4 * (i & 1) + 1] = lo[1];
      h[i >> 1][4 * (i & 1) + 2] = hi[0];
      h[i >> 1][4 * (i & 1) + 3] = hi[1];
    }
  }
};

__device__ __forceinline__ float4_t block_product(const Piece<false> (&w)[2], const Piece<false> (&a)[2]) {
  const int8v_t x = __builtin_shufflevector(__builtin_bit_cast(int4_t, w[0].q), __builtin_bit_cast(int4_t, w[1].q), 0, 1, 2, 3, 4, 5, 6, 7);
  const int8v_t y = __builtin_shufflevector(__builtin_bit_cast(int4_t, a[0].q), __builtin_bit_cast(int4_t, a[1].q), 0, 1, 2, 3, 4, 5, 6, 7);
  const float4_t zero = {0.f, 0.f, 0.f, 0.f};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, zero, 0, 0, 0, 0, 0, 0);  // both e4m3, unscaled
}
__device__ __forceinline__ float4_t block_product(const Piece<true> (&w)[2], const Piece<true> (&a)[2]) {
  float4_t c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[i >> 1].h[i & 1], a[i >> 1].h[i & 1], c, 0, 0, 0);
  return c;
}

// W [N][K] into its tiles: a workgroup's four wavefronts take a tile each.
template <bool VEC>
__global__ __launch_bounds__(256) void k_f8_tile(const uint8_t* __restrict__ w, int64_t N, int64_t K, int64_t kb, int64_t tiles,
                                                 uint8_t* __restrict__ q) {
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (at >= tiles * kb) return;
  const int64_t tile = at / kb, b = at - tile * kb;
  const int lane = threadIdx.x & 63;
  const int64_t n = tile * 16 + (lane & 15);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t k = b * kF8Block + 64 * h + 16 * (lane >> 4);
    uint4_t v{0u, 0u, 0u, 0u};
    if (n < N) {
      if constexpr (VEC) {
        if (k < K) v = *reinterpret_cast<const uint4_t*>(w + n * K + k);
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (k + e < K) v[e >> 2] |= static_cast<uint32_t>(w[n * K + k + e]) << (8 * (e & 3));
      }
    }
    *reinterpret_cast<uint4_t*>(q + at * kTileBytes + h * 1024 + lane * 16) = v;
  }
}

// Rows of K bytes at any address and pitch into rows of Kp bytes, a multiple of 16, zeros past K.
__global__ __launch_bounds__(256) void k_f8_pad_rows(const uint8_t* __restrict__ a, int64_t lda, int64_t M, int64_t K, int64_t Kp,
                                                     uint8_t* __restrict__ out) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t row = i / (Kp / 16), k = (i - row * (Kp / 16)) * 16;
  if (row >= M) return;
  uint4_t v{0u, 0u, 0u, 0u};
#pragma unroll
  for (int e = 0; e < 16; ++e)
    if (k + e < K) v[e >> 2] |= static_cast<uint32_t>(a[row * lda + k + e]) << (8 * (e & 3));
  *reinterpret_cast<uint4_t*>(out + row * Kp + k) = v;
}

struct F8Args {
  const uint8_t* w;
  const float* w_scales;
  const uint8_t* a;
  const float* a_scales;
  const void* bias;
  void* y;
  float* part;  // [splits][M][N] partial sums, or NULL
  int64_t lda, ldy;
  int M, N, K, kb, tiles;
  int bias_dtype, y_dtype;
  int splits, per;  // parts of K (grid z), and blocks of 128 a part
};

// Four consecutive columns n .. n + 3 of row m: rounded to Y (with the bias), or f32 partial sums.
__device__ __forceinline__ void store4(const F8Args& p, int64_t m, int n, float4_t v) {
  if (p.part) {
    float* out = p.part + (static_cast<int64_t>(blockIdx.z) * p.M + m) * p.N + n;
    if (p.N % 4 == 0) {
      *reinterpret_cast<float4_t*>(out) = v;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < p.N) out[e] = v[e];
    }
    return;
  }
  if (p.bias) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < p.N) v[e] += load_float_rt(p.bias, p.bias_dtype, n + e);
  }
  const int64_t at = m * p.ldy + n;
  const bool vec = n + 3 < p.N && (reinterpret_cast<uintptr_t>(p.y) + at * (p.y_dtype == DT_F32 ? 4 : 2)) % (p.y_dtype == DT_F32 ? 16 : 8) == 0;
  if (vec) {
    if (p.y_dtype == DT_F32) *reinterpret_cast<float4_t*>(static_cast<float*>(p.y) + at) = v;
    else if (p.y_dtype == DT_F16)
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.y) + at) = make_uint2(pack2<DT_F16>(v[0], v[1]), pack2<DT_F16>(v[2], v[3]));
    else
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.y) + at) = make_uint2(pack2<DT_BF16>(v[0], v[1]), pack2<DT_BF16>(v[2], v[3]));
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < p.N) store_float_rt(p.y, p.y_dtype, at + e, v[e]);
  }
}

// Few rows: a workgroup of KW wavefronts takes one tile of 16 columns of Y for all (up to 16 MT) rows, the
// wavefronts every KW-th block of K each, and adds their sums in LDS.
template <int MT, int KW, bool EXACT>
__global__ __launch_bounds__(64 * KW) void k_f8_rows(F8Args p) {
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tile = blockIdx.x;
  const uint8_t* w = p.w + (static_cast<int64_t>(tile) * p.kb) * kTileBytes + lane * 16;
  const float* ws = p.w_scales + static_cast<int64_t>(tile / 8) * p.kb;
  float4_t acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = float4_t{0.f, 0.f, 0.f, 0.f};
  const int first = blockIdx.z * p.per, last = min(first + p.per, p.kb);
  for (int b = first + wave; b < last; b += KW) {
    Piece<EXACT> wp[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) wp[h].set(*reinterpret_cast<const uint4_t*>(w + static_cast<int64_t>(b) * kTileBytes + 1024 * h));
    const float sw = ws[b];
    const int k = b * kF8Block + 16 * g;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const int m = 16 * t + r;
      uint4_t a0{0u, 0u, 0u, 0u}, a1{0u, 0u, 0u, 0u};
      float sa = 0.f;
      if (m < p.M) {
        const uint8_t* a = p.a + m * p.lda + k;
        if (k < p.K) a0 = *reinterpret_cast<const uint4_t*>(a);
        if (k + 64 < p.K) a1 = *reinterpret_cast<const uint4_t*>(a + 64);
        sa = p.a_scales[static_cast<int64_t>(b) * p.M + m];
      }
      Piece<EXACT> ap[2];
      ap[0].set(a0);
      ap[1].set(a1);
      acc[t] += block_product(wp, ap) * (sa * sw);
    }
  }
  __shared__ __align__(16) float4_t part[KW > 1 ? KW - 1 : 1][MT][64];
  if (wave > 0) {
#pragma unroll
    for (int t = 0; t < MT; ++t) part[wave - 1][t][lane] = acc[t];
  }
  __syncthreads();
  // Wavefront t adds up and stores row tile t (all of them wavefront 0 where there are fewer wavefronts).
  if (wave > 0) return;
#pragma unroll
  for (int t = 0; t < MT; ++t) {
#pragma unroll
    for (int i = 0; i < KW - 1; ++i) acc[t] += part[i][t][lane];
    const int m = 16 * t + r, n = 16 * tile + 4 * g;
    if (m < p.M && n < p.N) store4(p, m, n, acc[t]);
  }
}

// At most N (below 16) vector-memory operations of this thread outstanding, and no LDS operation.
template <int N>
__device__ __forceinline__ void wait_vm() {
  __builtin_amdgcn_s_waitcnt(N | (7 << 4));
}

// Many rows: BM rows of A times BN of W a workgroup, WM x WN wavefronts of (BM / WM) x (BN / WN) outputs each.
// A step is one block of K: both operands' bytes go global -> LDS (buffer_load ... lds) in the order of the MFMA
// operands, 1 KiB an instruction, a step ahead, and each wavefront reads its fragments back 16 bytes a lane in a
// row, without conflicts. Offsets are scalar along k; what lies past M, N or K is past the buffers' ranges and
// arrives as zeros.
template <int BM, int BN, int WM, int WN, bool EXACT>
__global__ __launch_bounds__(64 * WM * WN) void k_f8_gemm(F8Args p) {
  constexpr int NW = WM * WN, TM = BM / 16 / WM, TN = BN / 16 / WN;
  constexpr int A_TILES = BM / 16, W_TILES = BN / 16;
  constexpr int STAGE = (A_TILES + W_TILES) * kTileBytes;
  constexpr int A_DMA = 2 * A_TILES / NW, W_DMA = 2 * W_TILES / NW;
  static_assert(A_DMA * NW == 2 * A_TILES && W_DMA * NW == 2 * W_TILES, "whole instructions a wavefront");
  extern __shared__ __align__(16) uint8_t lds[];
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;
  // Workgroups go to the eight XCDs in turn: XCD x takes a run of the tiles, in an order that walks groups of four
  // row tiles, rows fastest, so that an XCD's tiles share few rows of A and of W (its own L2).
  uint32_t tile = blockIdx.y * gridDim.x + blockIdx.x;
  const uint32_t tiles = gridDim.x * gridDim.y;
  if (tiles >= 8) {
    const uint32_t per = tiles / 8;
    if (tile < 8 * per) tile = (tile % 8) * per + tile / 8;
  }
  const uint32_t group = tile / (4 * gridDim.x), first_m = 4 * group;
  const uint32_t group_m = min(4u, gridDim.y - first_m), in_group = tile - group * 4 * gridDim.x;
  const int m0 = static_cast<int>(first_m + in_group % group_m) * BM;
  const int n0 = static_cast<int>(in_group / group_m) * BN;
  const int64_t a_bytes = (static_cast<int64_t>(p.M) - m0 - 1) * p.lda + p.K;
  const int64_t w_bytes = (static_cast<int64_t>(p.tiles) - n0 / 16) * p.kb * kTileBytes;
  const auto a_rsrc = buffer_rsrc(p.a + m0 * p.lda, static_cast<uint32_t>(min(a_bytes, int64_t{0x7FFFFFF0})));
  const auto w_rsrc = buffer_rsrc(p.w + static_cast<int64_t>(n0 / 16) * p.kb * kTileBytes,
                                  static_cast<uint32_t>(min(w_bytes, int64_t{0x7FFFFFF0})));
  // Instruction j of this wavefront fills half h of tile t, 2 t + h = A_DMA * wave + j.
  uint32_t a_off[A_DMA], w_off[W_DMA];
#pragma unroll
  for (int j = 0; j < A_DMA; ++j) {
    const int i = A_DMA * wave + j, row = 16 * (i >> 1) + r;
    // A row past M starts past the range by itself; one before the last may not run on into the next.
    a_off[j] = m0 + row < p.M ? static_cast<uint32_t>(row * p.lda) + 64 * (i & 1) + 16 * g : 0x80000000u;
  }
#pragma unroll
  for (int j = 0; j < W_DMA; ++j) {
    const int i = W_DMA * wave + j;
    w_off[j] = n0 / 16 + (i >> 1) < p.tiles ? static_cast<uint32_t>(i >> 1) * p.kb * kTileBytes + (i & 1) * 1024 + lane * 16 : 0x80000000u;
  }
  const int first = blockIdx.z * p.per, last = min(first + p.per, p.kb);
  auto issue = [&](int b) {
    uint8_t* sa = lds + ((b - first) & 1) * STAGE;
    uint8_t* sw = sa + A_TILES * kTileBytes;
    const uint32_t k0 = static_cast<uint32_t>(b) * kF8Block;
    if (b * kF8Block + kF8Block <= p.K) {
#pragma unroll
      for (int j = 0; j < A_DMA; ++j) lds_dma16(a_rsrc, sa + (A_DMA * wave + j) * 1024, a_off[j], k0);
    } else {
#pragma unroll
      for (int j = 0; j < A_DMA; ++j) {
        const int i = A_DMA * wave + j;
        const bool in = static_cast<int>(k0) + 64 * (i & 1) + 16 * g < p.K;
        lds_dma16(a_rsrc, sa + i * 1024, in ? a_off[j] + (a_off[j] < 0x80000000u ? k0 : 0u) : 0x80000000u, 0);
      }
    }
#pragma unroll
    for (int j = 0; j < W_DMA; ++j)
      lds_dma16(w_rsrc, sw + (W_DMA * wave + j) * 1024, w_off[j], static_cast<uint32_t>(b) * kTileBytes);
  };
  auto barrier = [&]() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  float4_t acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = float4_t{0.f, 0.f, 0.f, 0.f};
  const int m_wave = m0 + wm * (BM / WM), n_wave = n0 + wn * (BN / WN);
  // The wavefront's columns lie in one block of 128 rows of W (n0 and BN / WN divide it).
  const float* ws = p.w_scales + static_cast<int64_t>(min(n_wave, p.N - 1) / kF8Block) * p.kb;
  int sa_row[TM];
#pragma unroll
  for (int i = 0; i < TM; ++i) sa_row[i] = min(m_wave + 16 * i + r, p.M - 1);
  if (first < last) issue(first);
  for (int b = first; b < last; ++b) {
    float sa[TM];
#pragma unroll
    for (int i = 0; i < TM; ++i) sa[i] = p.a_scales[static_cast<int64_t>(b) * p.M + sa_row[i]];
    const float sw = ws[b];
    wait_vm<0>();  // this step's stage, and its scales
    barrier();     // everybody's; and everybody has read the stage that the next issue overwrites
    if (b + 1 < last) issue(b + 1);
    const uint8_t* la = lds + ((b - first) & 1) * STAGE + wm * TM * kTileBytes + lane * 16;
    const uint8_t* lw = lds + ((b - first) & 1) * STAGE + (A_TILES + wn * TN) * kTileBytes + lane * 16;
    Piece<EXACT> wf[TN][2];
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) wf[j][h].set(*reinterpret_cast<const uint4_t*>(lw + j * kTileBytes + h * 1024));
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      Piece<EXACT> af[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) af[h].set(*reinterpret_cast<const uint4_t*>(la + i * kTileBytes + h * 1024));
      const float s = sa[i] * sw;
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const float4_t c = block_product(wf[j], af);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(c[e], s, acc[i][j][e]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int m = m_wave + 16 * i + r;
    if (m >= p.M) continue;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int n = n_wave + 16 * j + 4 * g;
      if (n < p.N) store4(p, m, n, acc[i][j]);
    }
  }
}

// Y = the sum of the parts (+ bias), in order.
__global__ __launch_bounds__(256) void k_f8_reduce(F8Args p) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t all = static_cast<int64_t>(p.M) * p.N;
  if (i >= all) return;
  float v = p.part[i];
  for (int s = 1; s < p.splits; ++s) v += p.part[s * all + i];
  const int64_t m = i / p.N;
  const int n = static_cast<int>(i - m * p.N);
  if (p.bias) v += load_float_rt(p.bias, p.bias_dtype, n);
  store_float_rt(p.y, p.y_dtype, m * p.ldy + n, v);
}

template <int BM, int BN, int WM, int WN, bool EXACT>
void launch_gemm(const F8Args& p, hipStream_t s) {
  constexpr int kLds = 2 * (BM + BN) / 16 * kTileBytes;
  static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(&k_f8_gemm<BM, BN, WM, WN, EXACT>),
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
  (void)attr;
  const dim3 grid(static_cast<unsigned>((p.N + BN - 1) / BN), static_cast<unsigned>((p.M + BM - 1) / BM),
                  static_cast<unsigned>(p.splits));
  k_f8_gemm<BM, BN, WM, WN, EXACT><<<grid, 64 * WM * WN, kLds, s>>>(p);
}

}  // namespace
}  // namespace tmh

using namespace tmh;

extern "C" {

int tmh_fp8_weight_prepare(tmh_ctx* ctx, const void* d_b, const float* d_scales, int64_t K, int64_t N, void* stream,
                           tmh_fp8_weight** out) {
  if (!out) return fail(ctx, TMH_ERR_INVALID, "tmh_fp8_weight_prepare: out is NULL");
  *out = nullptr;
  if (K < 1 || N < 1) return fail(ctx, TMH_ERR_INVALID, "an 8-bit weight must have K, N >= 1");
  if (K > (int64_t{1} << 22) || N > (int64_t{1} << 22))
    return fail(ctx, TMH_ERR_UNSUPPORTED, "an 8-bit weight's K and N must be at most 2^22, got %lld, %lld", (long long)K, (long long)N);
  TMH_TRY(use_device(ctx));
  if (!d_b || !d_scales) return fail(ctx, TMH_ERR_INVALID, "tmh_fp8_weight_prepare: NULL pointer");
  const int64_t kb = (K + kF8Block - 1) / kF8Block, tiles = (N + 15) / 16;
  auto* w = new (std::nothrow) tmh_fp8_weight();
  if (!w) return fail(ctx, TMH_ERR_OOM, "tmh_fp8_weight_prepare: out of host memory");
  w->device = ctx->device;
  w->K = K;
  w->N = N;
  w->kb = kb;
  w->tiles = tiles;
  const size_t bytes = static_cast<size_t>(tiles * kb) * kTileBytes;
  const size_t scale_bytes = static_cast<size_t>((N + kF8Block - 1) / kF8Block * kb) * sizeof(float);
  int st = check_hip(ctx, hipMalloc(reinterpret_cast<void**>(&w->d_q), bytes), "hipMalloc");
  if (st == TMH_OK) st = check_hip(ctx, hipMalloc(reinterpret_cast<void**>(&w->d_scales), scale_bytes), "hipMalloc");
  w->device_bytes = bytes + scale_bytes;
  hipStream_t s = pick_stream(ctx, stream);
  if (st == TMH_OK) {
    const unsigned grid = static_cast<unsigned>((tiles * kb + 3) / 4);
    const auto* b = static_cast<const uint8_t*>(d_b);
    if (K % 16 == 0 && reinterpret_cast<uintptr_t>(d_b) % 16 == 0) k_f8_tile<true><<<grid, 256, 0, s>>>(b, N, K, kb, tiles, w->d_q);
    else k_f8_tile<false><<<grid, 256, 0, s>>>(b, N, K, kb, tiles, w->d_q);
    st = check_launch(ctx, "k_f8_tile");
  }
  if (st == TMH_OK)
    st = check_hip(ctx, hipMemcpyAsync(w->d_scales, d_scales, scale_bytes, hipMemcpyDeviceToDevice, s), "hipMemcpyAsync D2D");
  if (st != TMH_OK) {
    tmh_fp8_weight_free(w);
    return st;
  }
  *out = w;
  return TMH_OK;
}

void tmh_fp8_weight_free(tmh_fp8_weight* w) {
  if (!w) return;
  int prev = 0;
  (void)hipGetDevice(&prev);
  (void)hipSetDevice(w->device);
  (void)hipFree(w->d_q);
  (void)hipFree(w->d_scales);
  (void)hipSetDevice(prev);
  delete w;
}

int tmh_fp8_weight_info(const tmh_fp8_weight* w, int64_t* K, int64_t* N, size_t* device_bytes) {
  if (!w) return fail(nullptr, TMH_ERR_INVALID, "tmh_fp8_weight_info: the weight is NULL");
  if (K) *K = w->K;
  if (N) *N = w->N;
  if (device_bytes) *device_bytes = w->device_bytes;
  return TMH_OK;
}

int tmh_matmul_fp8(tmh_ctx* ctx, const tmh_fp8_weight* w, const void* d_a, int64_t M, int64_t lda, const float* d_a_scales,
                   const void* d_bias, int bias_dtype, void* d_y, int y_dtype, int64_t ldy, void* stream) {
  if (!w) return fail(ctx, TMH_ERR_INVALID, "the 8-bit product's weight is NULL");
  if (!is_float_dtype(y_dtype)) return fail(ctx, TMH_ERR_INVALID, "the 8-bit product's y must be f32, f16 or bf16, got %s", dtype_name(y_dtype));
  if (d_bias && !is_float_dtype(bias_dtype))
    return fail(ctx, TMH_ERR_INVALID, "the 8-bit product's bias must be f32, f16 or bf16, got %s", dtype_name(bias_dtype));
  if (M < 0) return fail(ctx, TMH_ERR_INVALID, "M must not be negative");
  if (M > (int64_t{1} << 22) || lda > (int64_t{1} << 22))
    return fail(ctx, TMH_ERR_UNSUPPORTED, "the 8-bit product takes M and lda up to 2^22, got %lld, %lld", (long long)M, (long long)lda);
  if (lda < w->K || ldy < w->N)
    return fail(ctx, TMH_ERR_INVALID, "the 8-bit product needs lda >= K=%lld and ldy >= N=%lld", (long long)w->K, (long long)w->N);
  TMH_TRY(use_device(ctx));
  if (w->device != ctx->device)
    return fail(ctx, TMH_ERR_INVALID, "the 8-bit weight lies on device %d, the context uses %d", w->device, ctx->device);
  if (M == 0) return TMH_OK;
  if (!d_a || !d_a_scales || !d_y) return fail(ctx, TMH_ERR_INVALID, "tmh_matmul_fp8: NULL pointer");
  hipStream_t s = pick_stream(ctx, stream);
  F8Args p;
  p.w = w->d_q;
  p.w_scales = w->d_scales;
  p.a = static_cast<const uint8_t*>(d_a);
  p.a_scales = d_a_scales;
  p.bias = d_bias;
  p.y = d_y;
  p.part = nullptr;
  p.lda = lda;
  p.ldy = ldy;
  p.M = static_cast<int>(M);
  p.N = static_cast<int>(w->N);
  p.K = static_cast<int>(w->K);
  p.kb = static_cast<int>(w->kb);
  p.tiles = static_cast<int>(w->tiles);
  p.bias_dtype = bias_dtype;
  p.y_dtype = y_dtype;
  p.splits = 1;
  p.per = p.kb;
  const bool pad = w->K % 16 != 0 || lda % 16 != 0 || reinterpret_cast<uintptr_t>(d_a) % 16 != 0;
  const int64_t Kp = (w->K + 15) / 16 * 16;
  const size_t pad_bytes = pad ? static_cast<size_t>(M * Kp + 255) / 256 * 256 : 0;
  if (pad_bytes) {
    void* ws = workspace(ctx, pad_bytes, s);
    if (!ws) return fail(ctx, TMH_ERR_UNSUPPORTED, "the 8-bit product's workspace cannot grow here: run one call before the capture");
    k_f8_pad_rows<<<static_cast<unsigned>((M * (Kp / 16) + 255) / 256), 256, 0, s>>>(p.a, lda, M, w->K, Kp, static_cast<uint8_t*>(ws));
    TMH_TRY(check_launch(ctx, "k_f8_pad_rows"));
    p.a = static_cast<const uint8_t*>(ws);
    p.lda = Kp;
    p.K = static_cast<int>(Kp);
  }
  const unsigned tiles = static_cast<unsigned>(p.tiles);
  if (y_dtype == TMH_F32) {
    if (M <= 16) k_f8_rows<1, 8, true><<<tiles, 512, 0, s>>>(p);
    else if (M <= 32) k_f8_rows<2, 8, true><<<tiles, 512, 0, s>>>(p);
    else launch_gemm<128, 128, 2, 2, true>(p, s);
  } else {
    if (M <= 16) k_f8_rows<1, 8, false><<<tiles, 512, 0, s>>>(p);
    else if (M <= 32) k_f8_rows<2, 8, false><<<tiles, 512, 0, s>>>(p);
    else if (M <= 128) launch_gemm<128, 128, 2, 2, false>(p, s);
    else launch_gemm<256, 256, 2, 4, false>(p, s);
  }
  return check_launch(ctx, "k_f8_gemm");
}

}  // extern "C"
