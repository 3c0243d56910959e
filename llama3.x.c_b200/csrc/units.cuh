// A row of fp32 numbers that begins at any element, taken in units of 16 aligned bytes. Its first and last unit may hold
// elements that are not the row's; those are nobody's to read, so such a unit is loaded element by element.
#pragma once

#include <stdint.h>

struct UnitRow {
  const float *data;  // the row's first element
  int n;              // elements
  int off, count;     // elements of the first unit that come before the row; units
};
__host__ __device__ __forceinline__ UnitRow unit_row(const float *data, int n) {
  UnitRow r;
  r.data = data, r.n = n;
  r.off = (int)((reinterpret_cast<uintptr_t>(data) & 15) / 4);
  r.count = (int)(((long long)r.off + n + 3) / 4);
  return r;
}
// Part p of `parts` of its units.
__host__ __device__ __forceinline__ void part_of(const UnitRow &r, int p, int parts, int *first, int *end) {
  *first = (int)((long long)r.count * p / parts);
  *end = (int)((long long)r.count * (p + 1) / parts);
}
// Element i of a unit: its place in the row, or -1 where it is not the row's.
__host__ __device__ __forceinline__ int element_of(const UnitRow &r, int unit, int i) {
  const long long at = 4ll * unit + i - r.off;
  return at >= 0 && at < r.n ? (int)at : -1;
}
// Whether all of a unit of the row is the row's.
__host__ __device__ __forceinline__ bool whole(const UnitRow &r, int unit) {
  return !(unit == 0 && r.off) && !(unit == r.count - 1 && (((unsigned)r.off + (unsigned)r.n) & 3));
}
// The whole units among [first, end), which are the row's: [*from, *to).
__host__ __device__ __forceinline__ void whole_of(const UnitRow &r, int first, int end, int *from, int *to) {
  *from = first, *to = end;
  if (*from < *to && !whole(r, *from))
    ++*from;
  if (*from < *to && !whole(r, *to - 1))
    --*to;
}
// A whole unit's address.
__host__ __device__ __forceinline__ const float *unit_at(const UnitRow &r, int unit) {
  return r.data + (4ll * unit - r.off);
}
