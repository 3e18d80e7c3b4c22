// Work laid end to end and cut into one equal stretch per workgroup: the arithmetic that kf_few_rows.h and kf_flash.hip share.
// Every position is at least 0 and below kNoWork; the host refuses sizes whose work could be more.  Offsets that do not
// ascend can still add up to more than the sizes allow: such sums stay at kNoWork, which stands for no work at all, so an
// item always ends where the sum says, and every stretch that is named from a position is one of those launched.
#pragma once

#include <stdint.h>

namespace kf {

constexpr int kNoWork = 0x7fffffff;

__device__ __forceinline__ int add_work(int a, int b) {
  const uint32_t sum = (uint32_t)a + (uint32_t)b;
  return (int)(sum < (uint32_t)kNoWork ? sum : (uint32_t)kNoWork);
}

struct Stretch {
  int begin, end;
  // Whether it begins in the run of work of length `length` from `at` on.
  __device__ __forceinline__ bool begins_in(int at, int length) const {
    return begin < end && begin >= at && begin - at < length;
  }
};
// Stretch `me` of those of `per` units each; past the work's end they are empty.
__device__ __forceinline__ Stretch stretch_of(int total, int per, int me) {
  const int64_t from = (int64_t)me * per;  // 64 bits: workgroups past the end begin past it
  const int begin = from < total ? (int)from : total;
  return Stretch{begin, begin + (per < total - begin ? per : total - begin)};
}

// The stretch in which an item ends.
__device__ __forceinline__ int last_stretch(int item_at, int cost, int per) { return (item_at + cost - 1) / per; }

}  // namespace kf
