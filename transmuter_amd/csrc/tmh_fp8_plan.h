// Which kernel multiplies 8-bit rows with an 8-bit weight (tmh_fp8.hip), and in how many parts of K: whole numbers and
// prices only, on the host (whose tests go over them).
#pragma once

#include <algorithm>
#include <cmath>
#include <cstdint>

namespace tmh {

// The kernels of a product, and how many parts K is cut into.
enum : int { ROWS16, ROWS16_WIDE, ROWS32_WIDE, ROWS64, GEMM_64x64, GEMM_64x128, GEMM_128x128, GEMM_128x256 };
struct F8Plan {
  int kernel, splits;
};

// k_f8_gemm: one workgroup's step of 128 of K, in us: alone on its CU (the loads' latency), and with the CU full (the
// matrix and memory units), as measured over K at sizes that fill the chip once and several times. How far ahead the
// loads are (DW, DA) is what the registers leave room for, and three blocks with 64 x 64 against one: us, 512 rows
// 2048 -> 2048 7.1 (9.4 with one), 256 rows 4096 -> 4096 10.5 (15.3); two with 64 x 128: 1024 rows 11008 -> 2048 31.5
// (41.6); one with 128 x 128, whose third workgroup on a CU two would cost: 2048 rows 2048 -> 22016 109 (115 with
// two).
struct F8Shape {
  int kernel, bm, bn;
  float alone[2], full[2];  // for a 16-bit Y, and for an f32 Y
};
constexpr F8Shape kF8Shapes[] = {
    {GEMM_64x64, 64, 64, {0.25f, 0.48f}, {0.25f, 0.34f}},
    {GEMM_64x128, 64, 128, {0.34f, 0.75f}, {0.33f, 0.60f}},
    {GEMM_128x128, 128, 128, {0.60f, 1.40f}, {0.54f, 1.05f}},
    {GEMM_128x256, 128, 256, {0.95f, 0.f}, {0.87f, 0.f}},  // (its f32 form's registers would not fit)
};
// k_f8_rows by row tiles (of 16), column tiles and wavefronts: a CU takes in 88 KB of weights and rows of A a us, a
// wavefront a block of K every 0.33 us at most, and a turn of workgroups costs `turn` us beside (ROWS64 fills a CU's LDS,
// so that its turns do not overlap).
struct F8Rows {
  int kernel, row_tiles, col_tiles, waves;
  double first, turn;
};
constexpr F8Rows kF8Rows[] = {{ROWS16, 1, 1, 8, 2.0, 0.35}, {ROWS16_WIDE, 1, 2, 8, 2.0, 0.35}, {ROWS32_WIDE, 2, 2, 8, 2.0, 0.5},
                              {ROWS64, 4, 1, 8, 1.4, 1.0}};

// The kernel by what it is expected to take; parts of K cost their sums' way to memory and back (4.5 TB/s, 8 TB/s
// while the last-level cache holds them) and the second launch (2.4 us). Measured, us (f16 Y): one row 2048 -> 22016
// 8.5 by ROWS16_WIDE, 8.9 by ROWS16; 2048 -> 2048 3.7 by ROWS16, 3.9 by ROWS16_WIDE; 32 rows 11008 -> 2048 6.5 by
// ROWS16 (twice over W); 64 rows 8.0 by ROWS16_WIDE, 10.0 by ROWS16, 12.1 by ROWS64, 10.3 by 64x64 in 8 parts (a form of 32
// rows and 16 columns, which no size was best with, 7.8 and 8.8); 64 rows 4096 -> 4096 6.1 by ROWS32_WIDE, 7.1 by ROWS64, 9.7 by 64x64 in 4 parts; 64 rows
// 2048 -> 22016 11.1 by 64x64, 21.9 by ROWS64; 128 rows 11008 -> 2048 14.1 by 64x64 in 8 parts, 15.7 in 4, 39.6 in
// one of 64x128; 512 rows 2048 -> 2048 6.9 by 64x64, 11.1 by 128x128; 512 rows 2048 -> 22016 27.0 by 128x128, 28.3 by
// 128x256, 43.9 by 64x64; 4096 rows 11008 -> 2048 81 by 128x256, 87 by 128x128, 119 by a tile of 256 x 256, which no
// size was best with.
inline F8Plan plan_of(int64_t M, int64_t N, int kb, int64_t tiles, bool f32, int num_cus) {
  F8Plan best{GEMM_128x128, 1};
  double least = 1e30;
  auto offer = [&](int kernel, int splits, double us) {
    const double sums = 8.0 * splits * static_cast<double>(M) * static_cast<double>(N);
    if (splits > 1) us += 2.4 + sums / (sums > 128e6 ? 4.5e6 : 8e6);
    if (us < least) {
      least = us;
      best = {kernel, splits};
    }
  };
  auto turns = [&](double groups) { return groups <= 4 ? std::ceil(groups) : groups + 0.4; };
  for (const F8Rows& r : kF8Rows) {
    const int64_t rows = 16 * r.row_tiles;
    const double groups = static_cast<double>(tiles / r.col_tiles * ((M + rows - 1) / rows)) / num_cus;
    const double work = std::max(0.33 * ((kb + r.waves - 1) / r.waves), kb * 2.048 * (r.row_tiles + r.col_tiles) / 88);
    // (An f32 Y: conversions, and twice the answers. 512 rows 2048 -> 2048 17.0 by ROWS64, 11.2 by 64x64.)
    offer(r.kernel, 1, r.first + turns(groups) * (f32 ? r.turn + 0.6 + 1.2 * work : r.turn + work));
  }
  if (M <= 16) return best;
  for (int splits = 1; splits <= 8; splits *= 2) {
    const int per = (kb + splits - 1) / splits;
    if (splits > 1 && per < 4) break;
    for (const F8Shape& f : kF8Shapes) {
      if (f.full[f32] == 0.f) continue;
      const double groups = static_cast<double>((M + f.bm - 1) / f.bm * ((N + f.bn - 1) / f.bn) * splits) / num_cus;
      offer(f.kernel, splits, 2.6 + std::max<double>(f.alone[f32], f.full[f32] * turns(groups)) * per);
    }
  }
  return best;
}

}  // namespace tmh
