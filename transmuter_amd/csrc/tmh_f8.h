// F8E4M3 rows with a scale for each block of 128 columns: what the norm and the quantizer write and
// the 8-bit product reads.
#pragma once

#include "tmh_device.h"
#include "tmh_paged_plan.h"

namespace tmh {

constexpr int kF8Block = 128;
constexpr float kF8Max = 448.f;

// The largest of a value over the 16 lanes of a row of lanes, in all of them: exchanges within pairs, quads,
// halves and the row (DPP moves, no LDS). The values are magnitudes' bit patterns, which order as unsigned
// integers with NaNs above infinity, so a NaN among them stays the largest.
__device__ __forceinline__ uint32_t row_max_bits(uint32_t v) {
  v = max(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0xB1, 0xF, 0xF, true)));   // lane ^ 1
  v = max(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x4E, 0xF, 0xF, true)));   // lane ^ 2
  v = max(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x141, 0xF, 0xF, true)));  // 7 - lane
  v = max(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x140, 0xF, 0xF, true)));  // 15 - lane
  return v;
}

__device__ __forceinline__ float row_sum(float v) {
  auto add = [](float x, int y) { return x + __builtin_bit_cast(float, y); };
  v = add(v, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0xB1, 0xF, 0xF, true));
  v = add(v, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x4E, 0xF, 0xF, true));
  v = add(v, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x141, 0xF, 0xF, true));
  v = add(v, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x140, 0xF, 0xF, true));
  return v;
}

// Eight f32 values of a lane, 16 lanes holding a block: the block's scale (largest magnitude / 448, at least
// the smallest normal number so that its reciprocal is finite, 1 for zeros), and the values divided by it in
// e4m3. The quotients are at most 448 but for the last bits of the two roundings, which e4m3's rounding takes
// back, so they need no clamp (which would turn a NaN into a number).
// The quotient and the reciprocal are estimates with one correction each (the divisions' general forms were a fifth
// of the gated quantizer's instructions, which it is bound by).
__device__ __forceinline__ float f8_block(const float (&v)[8], uint2& q) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __builtin_bit_cast(uint32_t, v[i]) & 0x7FFFFFFFu);
  top = row_max_bits(top);
  const float most = __builtin_bit_cast(float, top);
  float scale = most * (1.f / kF8Max);
  scale = fmaf(fmaf(-scale, kF8Max, most), 1.f / kF8Max, scale);
  if (top == 0) scale = 1.f;
  else if (scale < 1.17549435e-38f) scale = 1.17549435e-38f;  // (false for a NaN)
  float inv = __builtin_amdgcn_rcpf(scale);
  inv = fmaf(fmaf(-scale, inv, 1.f), inv, inv);
  if (top == 0x7F800000u) {  // the corrections of an infinity are NaN
    scale = most;
    inv = 0.f;
  }
  int lo = 0, hi = 0;
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, v[1] * inv, lo, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inv, v[3] * inv, lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4] * inv, v[5] * inv, hi, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6] * inv, v[7] * inv, hi, true);
  q = make_uint2(static_cast<uint32_t>(lo), static_cast<uint32_t>(hi));
  return scale;
}

// Eight elements of type DT: consecutive ones in one or two 16-byte accesses (VEC), or every STEP-th one at a time,
// those below `n` from the first (past which loads give zeros and stores leave memory alone). Where 16 lanes hold a
// block of 128 one element at a time, each takes every sixteenth, so that an access is 16 neighbours (quantizing 4096
// rows of 2050 f16: 16.8 us with eight neighbours to a lane, 11.1 so).
constexpr int kLaneStep = 16;
__device__ __forceinline__ int lane_columns(bool vec) {  // a lane's first column of its block
  return vec ? (threadIdx.x & 15) * 8 : threadIdx.x & 15;
}

// Eight consecutive elements as they lie (16-bit ones in `lo`), apart from what turns them into floats, so that a
// thread's loads can all be on their way before the first is waited for.
struct Raw8 {
  uint4_t lo{0u, 0u, 0u, 0u}, hi{0u, 0u, 0u, 0u};
};
template <int DT>
__device__ __forceinline__ void load_raw8(const void* p, int64_t at, int n, Raw8& raw) {
  if (n <= 0) return;
  const uint4_t* f = reinterpret_cast<const uint4_t*>(static_cast<const char*>(p) + at * (DT == DT_F32 ? 4 : 2));
  raw.lo = f[0];
  if constexpr (DT == DT_F32) raw.hi = f[1];
}
template <int DT>
__device__ __forceinline__ void floats_of(const Raw8& raw, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == DT_F32) {
      const uint32_t a = raw.lo[i], b = raw.hi[i];  // (a bit cast of an element itself would take the first)
      v[i] = __builtin_bit_cast(float, a);
      v[4 + i] = __builtin_bit_cast(float, b);
    } else {
      const uint32_t w = raw.lo[i];
      v[2 * i] = DT == DT_F16 ? f16_bits_to_f32(static_cast<uint16_t>(w)) : __builtin_bit_cast(float, w << 16);
      v[2 * i + 1] = DT == DT_F16 ? f16_bits_to_f32(static_cast<uint16_t>(w >> 16)) : __builtin_bit_cast(float, w & 0xFFFF0000u);
    }
  }
}

template <int DT, bool VEC, int STEP = 1>
__device__ __forceinline__ void load8(const void* p, int64_t at, int n, float (&v)[8]) {
  if constexpr (VEC) {
    Raw8 raw;
    load_raw8<DT>(p, at, n, raw);
    floats_of<DT>(raw, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i * STEP < n ? load_as_f32<DT>(p, at + i * STEP) : 0.f;
  }
}

template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (DT == DT_BF16) return pack_bf16_rne(a, b);
  else return static_cast<uint32_t>(f32_to_f16_bits(a)) | static_cast<uint32_t>(f32_to_f16_bits(b)) << 16;
}

template <int DT, bool VEC, int STEP = 1>
__device__ __forceinline__ void store8(void* p, int64_t at, int n, const float (&v)[8]) {
  if constexpr (VEC) {
    if (n <= 0) return;
    if constexpr (DT == DT_F32) {
      float4_t* f = reinterpret_cast<float4_t*>(static_cast<float*>(p) + at);
      f[0] = float4_t{v[0], v[1], v[2], v[3]};
      f[1] = float4_t{v[4], v[5], v[6], v[7]};
    } else {
      *reinterpret_cast<uint4_t*>(static_cast<uint16_t*>(p) + at) =
          uint4_t{pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3]), pack2<DT>(v[4], v[5]), pack2<DT>(v[6], v[7])};
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i * STEP < n) store_as<DT>(p, at + i * STEP, v[i]);
  }
}

template <bool VEC, int STEP = 1>
__device__ __forceinline__ void store8_f8(uint8_t* p, int64_t at, int n, uint2 q) {
  if constexpr (VEC) {
    if (n > 0) *reinterpret_cast<uint2*>(p + at) = q;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i * STEP < n) p[at + i * STEP] = static_cast<uint8_t>((i < 4 ? q.x >> (8 * i) : q.y >> (8 * (i - 4))) & 0xFFu);
  }
}

}  // namespace tmh
