// q8_ranges.cuh -- how the attention over the paged 8-bit cache deals its units
// of work to CTAs, and the descriptors by which the pieces of a cut segment are
// joined.  Plain integer arithmetic, for host and device alike.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace fnmoe {

// Equal contiguous ranges of `total` units for the CTAs: CTA i takes
// [begin(i), begin(i + 1)), the first `more` CTAs one unit more than the
// others.  At most a CTA per unit is used, so that no range between two others
// is empty.
struct Ranges {
  long long total, per;
  int used, more;
  __host__ __device__ __forceinline__ Ranges(long long units, int ctas) : total(units) {
    const long long most = units > 1 ? units : 1;
    used = static_cast<int>(ctas < most ? ctas : most);
    per = units <= 0xFFFFFFFFll ? static_cast<uint32_t>(units) / static_cast<uint32_t>(used) : units / used;
    more = static_cast<int>(units - per * used);
  }
  __host__ __device__ __forceinline__ long long begin(int i) const {
    i = i < used ? i : used;
    return per * i + (i < more ? i : more);
  }
  // The CTA whose range holds `unit`.
  __host__ __device__ __forceinline__ int owner(long long unit) const {
    const long long big = (per + 1) * more;
    const long long rest = unit < big ? unit : unit - big, n = unit < big ? per + 1 : per;
    const int q = rest <= 0xFFFFFFFFll && n <= 0xFFFFFFFFll ? static_cast<uint32_t>(rest) / static_cast<uint32_t>(n)
                                                            : static_cast<int>(rest / n);
    return unit < big ? q : more + q;
  }
};

// Where a CTA's range begins.  When that is the first cut inside a segment
// (work of one sequence, kv head and tile that several CTAs share), the join
// finds here all it needs: {sequence, kv head, tile, last CTA of the segment,
// with bit 30 set when the CTA before, the segment's first, began earlier than
// the segment}; otherwise the sequence is -1.
__host__ __device__ __forceinline__ int4 cut_of(const Ranges &ranges, int b, int h, int tile, long long seg_begin,
                                                long long first_unit, long long last_unit, int cta) {
  if (ranges.owner(first_unit) != cta - 1) return make_int4(-1, 0, 0, 0);
  const int late = ranges.begin(cta - 1) < seg_begin ? 1 << 30 : 0;
  return make_int4(b, h, tile, ranges.owner(last_unit) | late);
}
__host__ __device__ __forceinline__ int last_cta(int4 cut) { return cut.w & 0x3FFFFFFF; }

// Whether a descriptor can be followed: the join's indexes then lie inside its
// arrays, whatever the descriptor's memory held.  c0 and h: the segment's first
// CTA and kv head (in a table by segment c0 comes from the descriptor, else h).
__host__ __device__ __forceinline__ bool cut_fits(int4 cut, int c0, int h, int batch, int heads, int ctas) {
  return cut.x >= 0 && cut.x < batch && h >= 0 && h < heads && cut.z >= 0 && cut.w >= 0 && c0 >= 0 &&
         last_cta(cut) > c0 && last_cta(cut) < ctas;
}

}  // namespace fnmoe
