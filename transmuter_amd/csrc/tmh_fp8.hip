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
#include <type_traits>

#include "tmh_f8.h"
#include "tmh_fp8_plan.h"
#include "tmh_internal.h"
#include "tmh_launch.h"

// Tiles of 16 rows x 128 of K, 2 KiB each in the order [N / 16][K / 128]: two halves (64 of K each) of 1 KiB, lane l
// = 16 g + r of a wavefront holding row r (of the pair of tiles' 32, tile_row), k = 64 h + 16 g .. + 15 at offset 16
// l of half h. A wavefront's 16-byte loads of a tile are its MFMA operand (the order of k within a block is free, as
// long as both factors share it), and read 1 KiB in a row. Rows past N and k past K are zeros; tiles come in pairs.
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

// Row r of a tile. Tiles t and t + 1 (t even) share 32 rows of W in turns of four, so that a lane's outputs of the
// pair (rows 4 g .. + 3 of each) are eight consecutive columns of Y.
__host__ __device__ __forceinline__ int64_t tile_row(int64_t tile, int r) {
  return (tile >> 1) * 32 + (r >> 2) * 8 + (tile & 1) * 4 + (r & 3);
}

// W [N][K] into its tiles: a workgroup's four wavefronts take a tile each.
template <bool VEC>
__global__ __launch_bounds__(256) void k_f8_tile(const uint8_t* __restrict__ w, int64_t N, int64_t K, int64_t kb, int64_t tiles,
                                                 uint8_t* __restrict__ q, int64_t first) {
  const int64_t at = first + static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (at >= tiles * kb) return;
  const int64_t tile = at / kb, b = at - tile * kb;
  const int lane = threadIdx.x & 63;
  const int64_t n = tile_row(tile, lane & 15);
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
                                                     uint8_t* __restrict__ out, int64_t first) {
  const int64_t i = first + static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
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

// Four consecutive columns n .. n + 3 of row m, with the bias, rounded to Y.
__device__ __forceinline__ void store4(const F8Args& p, int64_t m, int n, float4_t v) {
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

// 4 bytes per lane from a buffer into LDS at lds + 4 * lane (lds_dma16's form for single values).
__device__ __forceinline__ void lds_dma4(__amdgpu_buffer_rsrc_t rsrc, uint8_t* lds, uint32_t voffset, uint32_t soffset) {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)(lds), 4, voffset, soffset, 0, 0);
#endif
}

// No LDS operation of this thread outstanding (any number of vector-memory ones).
constexpr int kAllLds = 15 | 3 << 14 | 7 << 4;

// At most N (below 64) vector-memory operations of this thread outstanding, and no LDS operation.
template <int N>
__device__ __forceinline__ void wait_vm() {
  __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4 << 14) | (7 << 4));
}

// Few rows: a workgroup of KW wavefronts takes NT tiles of 16 columns of Y for 16 MT rows, the wavefronts every KW-th
// block of K each, and adds their sums in LDS. A wavefront has the next DEPTH - 1 blocks' loads on their way while it
// multiplies one: W's tiles to registers, A's rows to a place of its own in LDS (no barrier), eight lanes to a row's
// line (the fragments' own 16 bytes of 16 rows would be 64 lookups a load, k_f8_gemm). Bound by the weights' bytes
// where they are many (one row 2048 -> 22016: 8.7 us, 5.2 TB/s), by what a CU takes in of A and W and the way there
// where they are few (32 rows 11008 -> 2048 7.1 us, 3.2 TB/s; 13.8 with fragments loaded as they lie, one block at a
// time).
template <int MT, int NT, int KW, int DEPTH, bool EXACT>
__global__ __launch_bounds__(64 * KW) void k_f8_rows(F8Args p) {
  constexpr int STAGE = MT * kTileBytes;
  extern __shared__ __align__(16) uint8_t lds[];  // [KW][DEPTH][STAGE]; then the sums, [KW - 1][MT * NT][64] float4
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int groups = p.tiles / NT, row_group = blockIdx.x / groups, tile = (blockIdx.x - row_group * groups) * NT;
  const uint8_t* w = p.w + (static_cast<int64_t>(tile) * p.kb) * kTileBytes + lane * 16;
  const auto ws_rsrc = buffer_rsrc(p.w_scales + static_cast<int64_t>(tile / 8) * p.kb, static_cast<uint32_t>(p.kb) * 4);
  const int last = p.kb;
  uint8_t* mine = lds + wave * DEPTH * STAGE;
  const int a_row = lane >> 3, a_chunk = (lane & 7) ^ a_row;
  const int m0 = row_group * 16 * MT;
  const auto a_rsrc = buffer_rsrc(p.a + m0 * p.lda, static_cast<uint32_t>(min((static_cast<int64_t>(p.M) - m0 - 1) * p.lda + p.K, int64_t{0x7FFFFFF0})));
  const uint32_t a_off = static_cast<uint32_t>(a_row * p.lda) + 16 * a_chunk, a_rows = static_cast<uint32_t>(8 * p.lda);
  const uint32_t a_at[2] = {static_cast<uint32_t>(r * 128 + 16 * (g ^ (r & 7))), static_cast<uint32_t>(r * 128 + 16 * ((g + 4) ^ (r & 7)))};
  uint4_t wr[DEPTH][NT][2];
  float sw[DEPTH], sa[DEPTH][MT];
  constexpr int LOADS = 2 * NT + 1 + 3 * MT;
  // A block's rows first, then what goes to registers, whose own waits the compiler sees to: so the wait for the rows
  // below holds with all of them and with fewer. (The scales by vector loads like the others, in this order: they are
  // counted.)
  auto load = [&](int b, int buf) {
    const int k0 = b * kF8Block;
#pragma unroll
    for (int q = 0; q < 2 * MT; ++q)
      lds_dma16(a_rsrc, mine + buf * STAGE + q * 1024, k0 + 16 * a_chunk < p.K ? a_off + q * a_rows : 0x80000000u, static_cast<uint32_t>(k0));
    asm volatile("" ::: "memory");
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        wr[buf][j][h] = *reinterpret_cast<const uint4_t*>(w + (static_cast<int64_t>(j) * p.kb + b) * kTileBytes + 1024 * h);
    sw[buf] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(ws_rsrc, 0, static_cast<uint32_t>(b) * 4, 0));
#pragma unroll
    for (int t = 0; t < MT; ++t) sa[buf][t] = p.a_scales[static_cast<int64_t>(b) * p.M + min(m0 + 16 * t + r, p.M - 1)];
    asm volatile("" ::: "memory");
  };
  float4_t acc[MT][NT];
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[t][j] = float4_t{0.f, 0.f, 0.f, 0.f};
  auto block = [&](int b, int buf) {
    const int ahead = b + (DEPTH - 1) * KW;
    if (ahead < last) {
      __builtin_amdgcn_s_waitcnt(kAllLds);  // the block before has been read from the stage that is filled here
      asm volatile("" ::: "memory");
      load(ahead, (buf + DEPTH - 1) % DEPTH);
      wait_vm<(DEPTH - 1) * LOADS>();  // this block's loads: the later ones' are the youngest
    } else if (DEPTH > 2 && ahead - KW < last) {
      wait_vm<LOADS>();
    } else {
      wait_vm<0>();
    }
    asm volatile("" ::: "memory");
    Piece<EXACT> wp[NT][2];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) wp[j][h].set(wr[buf][j][h]);
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      Piece<EXACT> ap[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) ap[h].set(*reinterpret_cast<const uint4_t*>(mine + buf * STAGE + t * kTileBytes + a_at[h]));
      const float s = sa[buf][t] * sw[buf];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const float4_t c = block_product(wp[j], ap);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[t][j][e] = fmaf(c[e], s, acc[t][j][e]);
      }
    }
  };
  int b = wave;
#pragma unroll
  for (int d = 0; d < DEPTH - 1; ++d)
    if (b + d * KW < last) load(b + d * KW, d);
  for (; b < last; b += DEPTH * KW) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d)
      if (b + d * KW < last) block(b + d * KW, d);
  }
  wait_vm<0>();     // nothing is on its way to LDS
  __syncthreads();  // where the sums lie now
  float4_t* part = reinterpret_cast<float4_t*>(lds);
  if (wave > 0) {
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int j = 0; j < NT; ++j) part[((wave - 1) * MT * NT + t * NT + j) * 64 + lane] = acc[t][j];
  }
  __syncthreads();
  // The wavefronts take the tiles of Y in turn: their sums in the wavefronts' order.
  if (wave == 0) {
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int j = 0; j < NT; ++j) part[((KW - 1) * MT * NT + t * NT + j) * 64 + lane] = acc[t][j];
  }
  if constexpr (MT * NT > 1) __syncthreads();
  for (int i = wave; i < MT * NT; i += KW) {
    float4_t sum = part[((KW - 1) * MT * NT + i) * 64 + lane];
#pragma unroll
    for (int k = 0; k < KW - 1; ++k) sum += part[(k * MT * NT + i) * 64 + lane];
    const int m = m0 + 16 * (i / NT) + r, n = static_cast<int>(tile_row(tile + i % NT, 4 * g));
    if (m < p.M && n < p.N) store4(p, m, n, sum);
  }
}

// A wavefront's outputs. A lane holds eight consecutive columns of a row for each pair of tiles, but its
// neighbours other rows: the lanes trade (l = 16 g + r's answers go to lane 4 r + g), so that four lanes
// in a row write a row's 32 columns and a store is 16 lines' work, not 64. Where rows of Y do not lie on 16 bytes they
// go through LDS (`own`, kOwnBytes of the wavefront's), and half a wavefront writes a row's 32 columns one each, or a quarter
// two each where rows lie on pairs (bf16 4000 x 2048 -> 8194: 104 us by ones, 84 by twos).
constexpr int kOwnPitch = 36, kOwnBytes = 16 * kOwnPitch * 4;

template <int DT, bool PART, int TM, int TN>
__device__ __forceinline__ void gemm_outputs(const F8Args& p, const float4_t (&acc)[TM][TN], int m_wave, int n_wave, uint8_t* own) {
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4, to_r = lane >> 2, to_g = lane & 3;
  const int source = 4 * (16 * to_g + to_r);
  auto trade = [&](uint32_t v) { return static_cast<uint32_t>(__builtin_amdgcn_ds_bpermute(source, static_cast<int>(v))); };
  constexpr int SIZE = DT == DT_F32 ? 4 : 2;
  char* base = PART ? reinterpret_cast<char*>(p.part + static_cast<int64_t>(blockIdx.z) * p.M * p.N) : static_cast<char*>(p.y);
  const int64_t ld = PART ? p.N : p.ldy;
  const bool on16 = (reinterpret_cast<uintptr_t>(base) | static_cast<uintptr_t>(ld * SIZE)) % 16 == 0;
  const bool on_pairs = (reinterpret_cast<uintptr_t>(base) | static_cast<uintptr_t>(ld * SIZE)) % (2 * SIZE) == 0;
  if (!on16) __syncthreads();  // every wavefront has read the last of A, and no load of A is on its way
#pragma unroll
  for (int jp = 0; jp < TN / 2; ++jp) {
    const int n_pair = n_wave + 32 * jp, from = n_pair + 8 * g, n = n_pair + 8 * to_g;
    float bias[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) bias[e] = 0.f;
    if (!PART && p.bias) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (from + e < p.N) bias[e] = load_float_rt(p.bias, p.bias_dtype, from + e);
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = acc[i][2 * jp + (e >> 2)][e & 3] + bias[e];
      if (!on16) {
        float* rows = reinterpret_cast<float*>(own);
#pragma unroll
        for (int e = 0; e < 8; e += 4)
          *reinterpret_cast<float4_t*>(rows + r * kOwnPitch + 8 * g + e) = float4_t{v[e], v[e + 1], v[e + 2], v[e + 3]};
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        if (on_pairs) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int row = 4 * k + (lane >> 4), m = m_wave + 16 * i + row, col = n_pair + 2 * (lane & 15);
            const float2 x = *reinterpret_cast<const float2*>(rows + row * kOwnPitch + 2 * (lane & 15));
            if (m >= p.M || col >= p.N) continue;
            char* out = base + (m * ld + col) * SIZE;
            if (col + 1 == p.N) store_as<DT>(base, m * ld + col, x.x);
            else if constexpr (DT == DT_F32) *reinterpret_cast<float2*>(out) = x;
            else *reinterpret_cast<uint32_t*>(out) = pack2<DT>(x.x, x.y);
          }
        } else
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int m = m_wave + 16 * i + 2 * k + (lane >> 5), col = lane & 31;
          const float x = rows[(2 * k + (lane >> 5)) * kOwnPitch + col];
          if (m < p.M && n_pair + col < p.N) store_as<DT>(base, m * ld + n_pair + col, x);
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        continue;
      }
      uint32_t w[2 * SIZE];
#pragma unroll
      for (int e = 0; e < 2 * SIZE; ++e) w[e] = trade(SIZE == 4 ? __builtin_bit_cast(uint32_t, v[e]) : pack2<DT>(v[(2 * e) & 7], v[(2 * e + 1) & 7]));
      const int m = m_wave + 16 * i + to_r;
      if (m >= p.M || n >= p.N) continue;
      char* out = base + (m * ld + n) * SIZE;
      if (n + 8 <= p.N) {
#pragma unroll
        for (int e = 0; e < SIZE / 2; ++e) *reinterpret_cast<uint4_t*>(out + 16 * e) = uint4_t{w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]};
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (n + e >= p.N) continue;
          if constexpr (SIZE == 4) reinterpret_cast<uint32_t*>(out)[e] = w[e];
          else reinterpret_cast<uint16_t*>(out)[e] = static_cast<uint16_t>(w[e >> 1] >> (16 * (e & 1)));
        }
      }
    }
  }
}

// Many rows: BM rows of A times BN of W a workgroup, WM x WN wavefronts of (BM / WM) x (BN / WN) outputs each. A step
// is one block of K. A's bytes go global -> LDS (buffer_load ... lds), 1 KiB an instruction, DA steps ahead, with the
// step's row scales; W's tiles, which are operands as they lie, go to registers DW steps ahead and past LDS, whose
// reads would bound the loop otherwise. What lies past M, N or K is past the buffers' ranges and arrives as zeros.
//
// 4096 x 2048 -> 22016 (f16 Y, 128 x 256): 203 to 210 us, 1.8 PFLOP/s, with operands that come from memory, 167 us with
// those that the last-level cache holds; 8192 x 8192 x 8192 2.4. The matrix unit is busy 54% of the cycles there, at
// a clock that its own power holds at 1.9 GHz. A block's product needs four FMAs of its own beside it: a loop of
// nothing but both reaches 3.5 PFLOP/s (4.0 without them). On the way: 16-byte pieces of 64 rows of A an instruction
// and 8-byte stores 277 us, whole lines 231; two workgroups of 128 x 256 a CU instead of one of 256 x 256 224; the
// loads one by one between the products 210 (all ahead of them 224).
template <int BM, int BN, int WM, int WN, int DW, int DA, bool EXACT, bool TOUCH>
__global__ __launch_bounds__(64 * WM * WN, 2) void k_f8_gemm(F8Args p) {
  constexpr int NW = WM * WN, TM = BM / 16 / WM, TN = BN / 16 / WN;
  constexpr int A_TILES = BM / 16, A_DMA = 2 * A_TILES / NW;
  constexpr int STAGE = A_TILES * kTileBytes;
  static_assert(A_DMA * NW == 2 * A_TILES && BM % 64 == 0 && TN % 2 == 0, "whole instructions a wavefront, pairs of tiles");
  static_assert(NW * kOwnBytes <= (DA + 1) * STAGE, "the outputs' way through LDS");
  constexpr int STAGES = DA + 1;
  static_assert(DA >= DW, "a block's rows are asked for no later than its weights");
  extern __shared__ __align__(16) uint8_t lds[];  // [STAGES][STAGE], then the rows' scales [STAGES][BM]
  float* lds_s = reinterpret_cast<float*>(lds + STAGES * STAGE);
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;
  // Workgroups go to the eight XCDs in turn: XCD x takes a run of the tiles, in an order that walks groups of eight
  // row tiles, rows fastest, so that an XCD's tiles share few rows of A and of W (its own L2).
  const uint32_t cols = static_cast<uint32_t>((p.N + BN - 1) / BN), rows = static_cast<uint32_t>((p.M + BM - 1) / BM), tiles = cols * rows;
  uint32_t tile = blockIdx.x;
  if (tiles >= 8) {
    const uint32_t per = tiles / 8;
    if (tile < 8 * per) tile = (tile % 8) * per + tile / 8;
  }
  const uint32_t group = tile / (8 * cols), first_m = 8 * group;
  const uint32_t group_m = min(8u, rows - first_m), in_group = tile - group * 8 * cols;
  const int m0 = static_cast<int>(first_m + in_group % group_m) * BM;
  const int n0 = static_cast<int>(in_group / group_m) * BN;
  const int64_t a_bytes = (static_cast<int64_t>(p.M) - m0 - 1) * p.lda + p.K;
  const int64_t w_bytes = (static_cast<int64_t>(p.tiles) - n0 / 16) * p.kb * kTileBytes;
  const auto a_rsrc = buffer_rsrc(p.a + m0 * p.lda, static_cast<uint32_t>(min(a_bytes, int64_t{0x7FFFFFF0})));
  const auto w_rsrc = buffer_rsrc(p.w + static_cast<int64_t>(n0 / 16) * p.kb * kTileBytes,
                                  static_cast<uint32_t>(min(w_bytes, int64_t{0x7FFFFFF0})));
  // Instruction j of this wavefront fetches rows 8 i .. 8 i + 7, i = A_DMA * wave + j: eight lanes to a row's 128
  // bytes, one line, which the cache then looks up once (16 bytes of 64 rows each would be 64 lookups). Chunk c (16
  // bytes) of a row lies at place c ^ (row % 8) of its 128 bytes in LDS, so that the fragments' reads below meet no
  // bank twice.
  // (A row past M starts past the range by itself.)
  const int a_row = 8 * A_DMA * wave + (lane >> 3), a_chunk = (lane & 7) ^ (lane >> 3);
  const uint32_t a_off = static_cast<uint32_t>(a_row * p.lda) + 16 * a_chunk, a_rows = static_cast<uint32_t>(8 * p.lda);
  // (Tiles past the last are the last again: their columns are not stored.)
  uint32_t w_off[TN];
#pragma unroll
  for (int j = 0; j < TN; ++j)
    w_off[j] = static_cast<uint32_t>(min(wn * TN + j, p.tiles - 1 - n0 / 16)) * static_cast<uint32_t>(p.kb) * kTileBytes;
  const int first = blockIdx.z * p.per, last = min(first + p.per, p.kb);
  const int n_wave = n0 + wn * (BN / WN), m_wave = m0 + wm * (BM / WM);
  // The wavefront's columns lie in one block of 128 rows of W (n0 and BN / WN divide it).
  const auto ws_rsrc = buffer_rsrc(p.w_scales + static_cast<int64_t>(min(n_wave, p.N - 1) / kF8Block) * p.kb, static_cast<uint32_t>(p.kb) * 4);
  const int s_part = wave % (BM / 64);
  uint4_t wr[DW + 1][TN][2];
  float sw[DW + 1];
  // The loads of a step, one at a time: W's tiles of block b + DW, then A's rows and scales of block b + DA. (No
  // branches, which the compiler would move the products' FMAs behind: past the last block the loads of A have no
  // range and those of W and the scales are the last block's again.)
  constexpr int LOADS_W = 2 * TN + 1, LOADS_A = A_DMA + 1;
  // TOUCH: a look at W's lines four blocks further on, a line a lane, each line by one of the row tiles that walk
  // together, which brings them from memory to the XCD's L2 (the loads of the next block alone would arrive late).
  const bool mine = TOUCH && lane < 16 * TN && (lane >> 3) % group_m == in_group % group_m;
  const uint32_t touch_off = mine ? static_cast<uint32_t>(min(wn * TN + (lane >> 4), p.tiles - 1 - n0 / 16)) * static_cast<uint32_t>(p.kb) * kTileBytes + (lane & 15) * 128
                                  : 0x80000000u;
  auto touch = [&](int b) {
    lds_dma4(w_rsrc, lds + STAGES * (STAGE + BM * 4) + wave * 256, touch_off, static_cast<uint32_t>(min(b, last - 1)) * kTileBytes);
  };
  auto load_w = [&](int q, int at, int buf) {
    const int b = min(at, last - 1);
    if (q < 2 * TN)
      wr[buf][q >> 1][q & 1] = __builtin_bit_cast(uint4_t, __builtin_amdgcn_raw_buffer_load_b128(
          w_rsrc, lane * 16 + 1024 * (q & 1), w_off[q >> 1] + static_cast<uint32_t>(b) * kTileBytes, 0));
    else  // (a vector load like the others: they are counted)
      sw[buf] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(ws_rsrc, 0, static_cast<uint32_t>(b) * 4, 0));
  };
  auto load_a = [&](int q, int b, int slot) {
    if (q < A_DMA) {
      const int k0 = b < last ? b * kF8Block : 0, left = b < last ? p.K - k0 : 0;
      lds_dma16(a_rsrc, lds + slot * STAGE + (A_DMA * wave + q) * 1024, 16 * a_chunk < left ? a_off + q * a_rows : 0x80000000u, static_cast<uint32_t>(k0));
    } else {
      const auto s_rsrc = buffer_rsrc(p.a_scales + static_cast<int64_t>(min(b, last - 1)) * p.M + m0, static_cast<uint32_t>(min(BM, p.M - m0)) * 4);
      // (Where there are more wavefronts than 64 rows each, several load the same scales.)
      lds_dma4(s_rsrc, reinterpret_cast<uint8_t*>(lds_s + slot * BM + s_part * 64), (s_part * 64 + lane) * 4, 0);
    }
  };
  const uint32_t a_at[2] = {static_cast<uint32_t>(r * 128 + 16 * (g ^ (r & 7))), static_cast<uint32_t>(r * 128 + 16 * ((g + 4) ^ (r & 7)))};
  float4_t acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = float4_t{0.f, 0.f, 0.f, 0.f};
  int slot = 0;
  auto barrier = [&]() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  // MORE: with the loads of later blocks. (Without, what it reads has been waited for.)
  auto step = [&](int b, int buf, auto more) {
    constexpr bool MORE = decltype(more)::value;
    if constexpr (MORE) {
      // This step's W, scales and A are there: behind them the steps before have asked for later blocks. The barrier:
      // everybody's are, and everybody has read the stage that is filled next.
      constexpr int A_STEP = LOADS_W + LOADS_A + TOUCH;
      wait_vm<(DW - 1) * A_STEP + (DA > DW ? LOADS_A + TOUCH : TOUCH)>();
      barrier();
    }
    const int free_slot = slot == 0 ? DA : slot - 1;
    auto load = [&](int q) {
      if (!MORE) return;
      if (q < LOADS_W) load_w(q, b + DW, (buf + DW) % (DW + 1));
      else if (q < LOADS_W + LOADS_A) load_a(q - LOADS_W, b + DA, free_slot);
      else touch(b + 4);
    };
    const uint8_t* la = lds + slot * STAGE + wm * TM * kTileBytes;
    const float* ls = lds_s + slot * BM + wm * (BM / WM) + r;
    auto load_af = [&](int i, Piece<EXACT> (&af)[2]) {
#pragma unroll
      for (int h = 0; h < 2; ++h) af[h].set(*reinterpret_cast<const uint4_t*>(la + i * kTileBytes + a_at[h]));
    };
    Piece<EXACT> wf[TN][2];
    constexpr int LOADS = LOADS_W + LOADS_A + TOUCH;
    if constexpr (EXACT) {
      // A's next fragment is read, and a share of the loads issued, while this one is converted and multiplied.
      uint4_t raw[2][2];
      auto read_a = [&](int i) {
#pragma unroll
        for (int h = 0; h < 2; ++h) raw[i & 1][h] = *reinterpret_cast<const uint4_t*>(la + i * kTileBytes + a_at[h]);
      };
      read_a(0);
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) wf[j][h].set(wr[buf][j][h]);
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        if (i + 1 < TM) read_a(i + 1);
#pragma unroll
        for (int q = (i * LOADS + TM - 1) / TM; q < ((i + 1) * LOADS + TM - 1) / TM; ++q) load(q);
        Piece<EXACT> af[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) af[h].set(raw[i & 1][h]);
        const float s = ls[16 * i] * sw[buf];
        float4_t c[TN];
#pragma unroll
        for (int j = 0; j < TN; ++j) c[j] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int j = 0; j < TN; ++j) c[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wf[j][x >> 1].h[x & 1], af[x >> 1].h[x & 1], c[j], 0, 0, 0);
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(c[j][e], s, acc[i][j][e]);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) wf[j][h].set(wr[buf][j][h]);
      // A product's four FMAs come three products later, when it has left the matrix unit, a fragment is read while
      // the one before it is multiplied, and the loads are spread over the step (in a row they would hold
      // the wavefronts up until the address unit has taken them all): in this order, which the compiler would give
      // up to save registers.
      constexpr int LAG = 3, ALL = TM * TN;
      Piece<EXACT> af[2][2];
      constexpr int SR = (LAG + TN - 1) / TN + 1;  // rows whose scales the pending FMAs hold
      float sr[2], s[SR];
      float4_t c[LAG + 1];
      load_af(0, af[0]);
      sr[0] = ls[0];
#pragma unroll
      for (int t = 0; t < ALL + LAG; ++t) {
        const int i = t / TN, j = t % TN;
        if (t < ALL) {
          if (j == 0 && i + 1 < TM) {
            load_af(i + 1, af[(i + 1) & 1]);
            sr[(i + 1) & 1] = ls[16 * (i + 1)];
          }
#pragma unroll
          for (int q = (t * LOADS + ALL - 1) / ALL; q < ((t + 1) * LOADS + ALL - 1) / ALL; ++q) load(q);
          c[t % (LAG + 1)] = block_product(wf[j], af[i & 1]);
          if (j == 0) s[i % SR] = sr[i & 1] * sw[buf];
        }
        if (t >= LAG) {
          const int u = t - LAG;
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[u / TN][u % TN][e] = fmaf(c[u % (LAG + 1)][e], s[u / TN % SR], acc[u / TN][u % TN][e]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    slot = slot == DA ? 0 : slot + 1;
  };
#pragma unroll
  for (int d = 0; d < DA; ++d) {  // what the steps before the first would have asked for, in their order
    if (d >= DA - DW) {
#pragma unroll
      for (int q = 0; q < LOADS_W; ++q) load_w(q, first + d - (DA - DW), d - (DA - DW));
      asm volatile("" ::: "memory");
    }
#pragma unroll
    for (int q = 0; q < LOADS_A; ++q) load_a(q, first + d, d);
    if (TOUCH && d >= DA - DW) touch(first + 2);
    asm volatile("" ::: "memory");
  }
  int b = first;
  for (; b + DW < last; b += DW + 1) {
#pragma unroll
    for (int d = 0; d < DW + 1; ++d) step(b + d, d, std::true_type{});
  }
  // Up to DW steps are left. Their loads have no later ones behind them, so they are all waited for. What was loaded has a
  // reader here on every way out of the loop, so that no load that its waits count can be left out as one that nobody reads.
#pragma unroll
  for (int d = 0; d < DW; ++d) {
    asm volatile("" ::"v"(sw[d]));
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) asm volatile("" ::"v"(wr[d][j][h]));
  }
  wait_vm<0>();
  barrier();
#pragma unroll
  for (int d = 0; d < DW; ++d)
    if (b + d < last) step(b + d, d, std::false_type{});
  if (p.part) gemm_outputs<DT_F32, true, TM, TN>(p, acc, m_wave, n_wave, lds + wave * kOwnBytes);
  else if (EXACT) gemm_outputs<DT_F32, false, TM, TN>(p, acc, m_wave, n_wave, lds + wave * kOwnBytes);
  else if (p.y_dtype == DT_F16) gemm_outputs<DT_F16, false, TM, TN>(p, acc, m_wave, n_wave, lds + wave * kOwnBytes);
  else gemm_outputs<DT_BF16, false, TM, TN>(p, acc, m_wave, n_wave, lds + wave * kOwnBytes);
}

// Y = the sum of the parts (+ bias), in order. A thread takes four columns (their parts lie on 16 bytes where four
// divides N).
__global__ __launch_bounds__(256) void k_f8_reduce(F8Args p, int64_t first) {
  const int64_t i = first + static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int quads = (p.N + 3) / 4;
  const int64_t m = i / quads;
  if (m >= p.M) return;
  const int n = static_cast<int>(i - m * quads) * 4;
  const int64_t all = static_cast<int64_t>(p.M) * p.N;
  const float* part = p.part + m * p.N + n;
  float4_t v{0.f, 0.f, 0.f, 0.f};
  if (p.N % 4 == 0) {
    v = *reinterpret_cast<const float4_t*>(part);
#pragma unroll 4
    for (int s = 1; s < p.splits; ++s) v += *reinterpret_cast<const float4_t*>(part + s * all);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      for (int s = 0; s < p.splits && n + e < p.N; ++s) v[e] += part[s * all + e];
  }
  store4(p, m, n, v);
}

template <int MT, int NT, int KW, int DEPTH, bool EXACT>
void launch_rows(const F8Args& p, hipStream_t s) {
  // The wavefronts' stages of A, and in their place (or past it) their sums.
  constexpr int kLds = KW * MT * std::max(DEPTH * kTileBytes, NT * 1024);
  static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(&k_f8_rows<MT, NT, KW, DEPTH, EXACT>),
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
  (void)attr;
  const unsigned grid = static_cast<unsigned>(p.tiles / NT) * static_cast<unsigned>((p.M + 16 * MT - 1) / (16 * MT));
  k_f8_rows<MT, NT, KW, DEPTH, EXACT><<<grid, 64 * KW, kLds, s>>>(p);
}

template <int BM, int BN, int WM, int WN, int DW, int DA, bool EXACT, bool TOUCH = false>
void launch_gemm(const F8Args& p, hipStream_t s) {
  constexpr int kLds = (DA + 1) * (BM / 16 * kTileBytes + 4 * BM) + (TOUCH ? 256 * WM * WN : 0);
  static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(&k_f8_gemm<BM, BN, WM, WN, DW, DA, EXACT, TOUCH>),
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
  (void)attr;
  const dim3 grid(static_cast<unsigned>((p.N + BN - 1) / BN) * static_cast<unsigned>((p.M + BM - 1) / BM), 1,
                  static_cast<unsigned>(p.splits));
  k_f8_gemm<BM, BN, WM, WN, DW, DA, EXACT, TOUCH><<<grid, 64 * WM * WN, kLds, s>>>(p);
}

template <bool F32>
void launch_plan(const F8Plan& plan, const F8Args& p, hipStream_t s) {
  switch (plan.kernel) {
    case ROWS16: launch_rows<1, 1, 8, 3, F32>(p, s); break;
    case ROWS16_WIDE: launch_rows<1, 2, 8, 2, F32>(p, s); break;
    case ROWS32_WIDE: launch_rows<2, 2, 8, 2, F32>(p, s); break;
    case ROWS64: launch_rows<4, 1, 8, 2, F32>(p, s); break;
    case GEMM_64x64: launch_gemm<64, 64, 2, 2, F32 ? 2 : 3, F32 ? 2 : 3, F32>(p, s); break;
    case GEMM_64x128: launch_gemm<64, 128, 1, 4, 2, 2, F32>(p, s); break;
    case GEMM_128x128: launch_gemm<128, 128, 1, 4, 1, 2, F32>(p, s); break;
    case GEMM_128x256:
      if constexpr (!F32) {
        // Touches pay where W comes from memory and cost where the last-level cache (256 MB) holds it, which a call cannot
        // know: it takes operands of up to 90 MB for held, as those of three calls in turn are. us without touches and
        // with, 38 sizes from 21 to 234 MB: over nine sets of operands in turn 1024 rows 11008 -> 2048 (38 MB) 0.85 of the
        // time with, 512 rows 8192 -> 8192 (80 MB) 0.81, 1024 rows 2048 -> 22016 (92 MB) 0.90, 4096 rows (234 MB) 0.92
        // (1.02 to 0.81 over all); over three, up to 80 MB 1.01 to 1.05, from 84 MB on 0.99 to 0.84, 4096 rows
        // 2048 -> 22016 222.6 and 203.1; over one, held whole, 1.00 to 1.06, 166.8 and 167.5 there.
        const int64_t bytes = static_cast<int64_t>(p.M) * p.K + static_cast<int64_t>(p.tiles) * p.kb * kTileBytes + 2 * static_cast<int64_t>(p.M) * p.N;
        if (bytes > 90'000'000) launch_gemm<128, 256, 1, 4, 1, 2, false, true>(p, s);
        else launch_gemm<128, 256, 1, 4, 1, 2, false>(p, s);
      }
      break;
  }
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
  const int64_t kb = (K + kF8Block - 1) / kF8Block, tiles = (N + 31) / 32 * 2;
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
    const auto* b = static_cast<const uint8_t*>(d_b);
    in_launches(tiles * kb, most_a_launch(256, 4, 1), [&](int64_t first, int64_t count) {
      const unsigned grid = static_cast<unsigned>((count + 3) / 4);
      if (K % 16 == 0 && reinterpret_cast<uintptr_t>(d_b) % 16 == 0) k_f8_tile<true><<<grid, 256, 0, s>>>(b, N, K, kb, tiles, w->d_q, first);
      else k_f8_tile<false><<<grid, 256, 0, s>>>(b, N, K, kb, tiles, w->d_q, first);
    });
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
  const F8Plan plan = plan_of(M, w->N, p.kb, w->tiles, y_dtype == TMH_F32, ctx->num_cus);
  p.per = (p.kb + plan.splits - 1) / plan.splits;
  p.splits = (p.kb + p.per - 1) / p.per;  // (no part is empty)
  const bool pad = w->K % 16 != 0 || lda % 16 != 0 || reinterpret_cast<uintptr_t>(d_a) % 16 != 0;
  const int64_t Kp = (w->K + 15) / 16 * 16;
  const size_t pad_bytes = pad ? static_cast<size_t>(M * Kp + 255) / 256 * 256 : 0;
  const size_t part_bytes = p.splits > 1 ? static_cast<size_t>(p.splits) * M * w->N * sizeof(float) : 0;
  uint8_t* ws = nullptr;
  if (pad_bytes + part_bytes) {
    ws = static_cast<uint8_t*>(workspace(ctx, pad_bytes + part_bytes, s));
    if (!ws) return fail(ctx, TMH_ERR_UNSUPPORTED, "the 8-bit product's workspace cannot grow here: run one call before the capture");
    if (part_bytes) p.part = reinterpret_cast<float*>(ws + pad_bytes);
  }
  if (pad) {
    in_launches(M * (Kp / 16), most_a_launch(256, 256, 1), [&](int64_t first, int64_t count) {
      k_f8_pad_rows<<<static_cast<unsigned>((count + 255) / 256), 256, 0, s>>>(p.a, lda, M, w->K, Kp, ws, first);
    });
    TMH_TRY(check_launch(ctx, "k_f8_pad_rows"));
    p.a = ws;
    p.lda = Kp;
    p.K = static_cast<int>(Kp);
  }
  if (y_dtype == TMH_F32) launch_plan<true>(plan, p, s);
  else launch_plan<false>(plan, p, s);
  if (p.splits > 1) {
    TMH_TRY(check_launch(ctx, "k_f8_gemm"));
    in_launches(M * ((w->N + 3) / 4), most_a_launch(256, 256, 1), [&](int64_t first, int64_t count) {
      k_f8_reduce<<<static_cast<unsigned>((count + 255) / 256), 256, 0, s>>>(p, first);
    });
  }
  return check_launch(ctx, "k_f8_gemm");
}

}  // extern "C"
