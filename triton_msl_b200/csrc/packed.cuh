// Packed sequences: where sequence b of a batch lies in the token axis.
#pragma once
#include <cstdint>

namespace b2 {
namespace packed {

// Offsets outside [0, T] or descending are clamped to an empty or shorter
// sequence, so that no kernel reads out of range whatever the array holds.
// The pseudo-sequences -1 and B are the tokens before and after the batch's;
// they have no keys and get zeros.
// Where offsets descend, spans of the query axis would overlap: a sequence then
// begins no earlier than the ones before it end (Span::after), so that the spans of
// -1 .. B always cover every token once and the work is bounded by T and B.
struct Span {
  int start, len;
  __device__ __forceinline__ Span after(int end) const {
    const int s = max(start, end);
    return {s, max(start + len - s, 0)};
  }
};
__device__ __forceinline__ Span span_of(const int32_t* cu, int b, int B, int T) {
  int s, e;
  if (b < 0) {
    s = 0;
    e = min(max(cu[0], 0), T);
  } else if (b >= B) {
    s = min(max(cu[B], 0), T);
    e = T;
  } else {
    s = min(max(cu[b], 0), T);
    e = min(max(cu[b + 1], s), T);
  }
  return {s, e - s};
}
__device__ __forceinline__ bool span_bad(const int32_t* cu, int b, int T) {
  return cu[b] < 0 || cu[b + 1] < cu[b] || cu[b + 1] > T;
}

}  // namespace packed
}  // namespace b2
