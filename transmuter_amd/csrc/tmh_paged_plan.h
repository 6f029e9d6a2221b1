// Where the tokens of a paged cache lie and how attention over them is shared out: whole numbers only, the same
// on the host (whose tests go over every case) and on the device.
#pragma once

#include <cstdint>

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

}  // namespace tmh
