// Where the tokens of a paged cache lie and how attention over them is shared out: whole numbers only, the same
// on the host (whose tests go over every case) and on the device.
#pragma once

#include <algorithm>
#include <cstdint>

#include "tmh_launch.h"

#if defined(__HIPCC__)
#define TMH_HD __host__ __device__ __forceinline__
#else
#define TMH_HD inline
#endif

namespace tmh {

// n / d for a fixed d >= 1 and n below 2^31, as a multiplication: with 2^s < d <= 2^(s + 1) and
// mul = ceil(2^(32 + s) / d) (below 2^32), n * mul / 2^(32 + s) exceeds n / d by n e / (d 2^(32 + s)), where
// e = mul d - 2^(32 + s) <= d - 1 < 2^(s + 1): less than 1 / d, so the whole parts are equal.
struct FastDiv {
  uint32_t d = 1, mul = 0, shift = 0;
  FastDiv() = default;
  explicit FastDiv(uint32_t divisor) : d(divisor) {
    if (d == 1) return;
    while ((uint64_t{2} << shift) < d) ++shift;
    mul = static_cast<uint32_t>(((uint64_t{1} << (32 + shift)) + d - 1) / d);
  }
  TMH_HD uint32_t div(uint32_t n) const {
    return d == 1 ? n : static_cast<uint32_t>((static_cast<uint64_t>(n) * mul) >> 32) >> shift;
  }
};

struct PageShape {
  int64_t pages, page_stride, token_stride;
  FastDiv by_page;  // its d: the page size
};

// The offset of token `token` of a sequence with the pages `table` (in elements, of head 0), or -1 where the
// table names no page of the cache. `token` is below the table's pages * page size.
TMH_HD int64_t token_offset(const PageShape& c, const int32_t* table, uint32_t token) {
  const uint32_t page = c.by_page.div(token);
  const int32_t id = table[page];
  if (id < 0 || id >= c.pages) return -1;
  return id * c.page_stride + static_cast<int64_t>(token - page * c.by_page.d) * c.token_stride;
}

// A sequence's tokens [begin, end), and the units (`unit_tokens` tokens each, counted from token 0) that hold
// them: `units` of them from `unit` on. Lengths are clamped to what the table has room for (`most` tokens, below
// 2^31), a window of 0 is none.
struct Span {
  int begin, end, unit, units;
};
TMH_HD Span span_of(int32_t length, int64_t most, int64_t window, int unit_tokens) {
  const int64_t n = length < 0 ? 0 : length < most ? length : most;
  Span s;
  s.end = static_cast<int>(n);
  s.begin = window > 0 && n > window ? static_cast<int>(n - window) : 0;
  s.unit = s.begin / unit_tokens;
  s.units = n > 0 ? static_cast<int>((n + unit_tokens - 1) / unit_tokens) - s.unit : 0;
  return s;
}

// The units of all items (an item: one sequence, kv head and chunk of query heads) lie in order and are cut
// into equal runs of `per` units, one a worker: worker w takes [w per, (w + 1) per). What a worker has of an item that
// it does not have whole is a part, kept in one of the worker's two places: the first of its run in 2 w, else (the
// last of its run, then) 2 w + 1.
TMH_HD uint32_t units_per_worker(uint32_t all, uint32_t workers) { return (all + workers - 1) / workers; }
TMH_HD uint32_t part_place(uint32_t worker, bool first_of_run) { return 2 * worker + (first_of_run ? 0 : 1); }

// The parts of an item of the units [first, first + units): those of the workers `from` .. `from + count - 1`
// (count 1: the worker has it whole, and there is no part).
struct Parts {
  uint32_t from, count;
  bool from_first;  // the item is the first of worker `from`'s run
};
TMH_HD Parts parts_of(uint32_t first, uint32_t units, uint32_t per) {
  Parts p;
  p.from = first / per;
  p.count = (first + units - 1) / per - p.from + 1;
  p.from_first = p.from * per == first;
  return p;
}
// The place of part i: every part but the item's first is the first of its worker's run.
TMH_HD uint32_t place_of(const Parts& p, uint32_t i) { return part_place(p.from + i, i > 0 || p.from_first); }

// What happens to items that several workers share:
//  JOIN  they meet in the kernel: the last worker to finish a part joins an item's parts.
//  PARTS a second kernel joins them.
//  WHOLE there are none: a workgroup (WHOLE8: of eight wavefronts) takes an item.
//  EACH  JOIN with a worker to each unit that the table has room for, where no window moves them.
enum Way : int { JOIN, PARTS, WHOLE, WHOLE8, EACH };

constexpr int kHeads = 16;  // query heads of one kv head that a workgroup answers (the columns of an MFMA tile)
constexpr int64_t kJoinBytes = 72 << 10;

struct AttentionPlan {
  Way way;
  uint32_t workers;  // workgroups
  uint32_t units;    // of an item, as far as the host knows
};

// The way of B sequences whose table has room for `most` tokens each (their lengths are the device's), of kv_heads groups
// of `group` query heads. B * kv_heads * chunks * units is below 2^31.
inline AttentionPlan attention_plan(int64_t B, int64_t kv_heads, int64_t group, int head_dim, int64_t most, int64_t window, bool f32,
                                    int num_cus) {
  const int64_t unit = f32 ? 64 : 128, chunks = (group + kHeads - 1) / kHeads;
  const int64_t all_items = B * kv_heads * chunks, units = (most + unit - 1) / unit * all_items;
  // Two workgroups a compute unit, or one a unit of work where the table has room for fewer.
  const int64_t workers = std::max<int64_t>(1, std::min<int64_t>(2 * num_cus, units));
  // Tokens that a sequence may have, and the units they lie in.
  const int64_t tokens = window > 0 ? std::min(most, window) : most;
  auto units_of = [&](int64_t u) { return (tokens + u - 1) / u + (tokens < most ? 1 : 0); };
  // JOIN where one workgroup has few parts to read (kJoinBytes of equal lengths; of others it may be more). us as JOIN and
  // as PARTS: one sequence of 4096 (64 KiB) 9.5 and 11.6, 32 x 4000 55.1 and 57.0, 64 x 2000 with 64 heads of 4 kv
  // heads 56.6 and 64.0, with 16 heads of one kv head (80 KiB) 20.2 and 20.8; one of 16384 (256 KiB) 20.2 and 19.5, 16 x 4000
  // with 16 heads of one kv head (256 KiB) 21.0 and 16.1, one of 65536 with those (2 MiB) 82 and 35. EACH instead where the table's
  // units are no more than the CUs: one sequence of 700 8.1 us as JOIN, 7.5 so; 8 x 1000 9.4 and 8.6. (With up to
  // two a CU: 4 x 4000 14.2 and 13.2, but tables that are not full leave the workers unevenly on the CUs: 5 x
  // 1..2600 9.3 and 9.8, 9 x 1..900 of 256 dimensions 12.3 and 15.2.)
  const int64_t parts = std::min<int64_t>(units_of(unit), workers / all_items + 2);
  const bool join = parts * std::min<int64_t>(kHeads, group) * head_dim * 4 <= kJoinBytes;
  const bool each = join && tokens == most && units > 0 && units <= num_cus;
  // WHOLE where an item is one unit, which cannot be cut (116 x 1..45, bf16 4 kv heads of 256, 17.1 us as JOIN, 13.4
  // whole; one token of f16 4 kv heads of 128 4.5, as EACH 4.7), or two that EACH cannot take (4 x 200 of 256
  // dimensions 10.8 us, as EACH 9.5). Few items of a few units go WHOLE8, where the registers allow it, if that is one
  // turn of 256 tokens (f32: 128), as a further one costs 2.6 us (3.6), f16 4 kv heads of 128: 8 x 200 6.1 us (7.4 as
  // EACH), but 8 x 500 9.4 (7.8); and with workgroups for half the CUs and more, 32 x 400 10.1 (10.2), 32 x 500 10.4
  // (11.3), 32 x 700 12.8 (16.1 as JOIN), 60 x 1..1000 16.4 (20.0 as JOIN).
  const bool half = all_items >= num_cus / 2;
  const bool eight = head_dim <= 128 && all_items <= num_cus && (units_of(2 * unit) == 1 || (units_of(2 * unit) <= 4 && half));
  // (Of more items than HIP takes workgroups JOIN's share as any others.)
  const bool whole = (units_of(unit) == 1 && all_items <= most_a_launch(256, 1, 1)) ||
                     (!eight && all_items <= num_cus && ((units_of(unit) <= 2 && !each) || (units_of(unit) <= 4 && half)));
  const Way way = whole ? WHOLE : eight ? WHOLE8 : each ? EACH : join ? JOIN : PARTS;
  return {way, static_cast<uint32_t>(whole || eight ? all_items : each ? units : workers), static_cast<uint32_t>(units_of(unit))};
}

}  // namespace tmh
