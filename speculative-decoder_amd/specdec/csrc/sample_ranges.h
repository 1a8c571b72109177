// The ranges that a search over a row of logits cuts its values into.
#pragma once

#include <math.h>

namespace specdec {

constexpr int kSampleBins = 2048;

// kSampleBins ranges of one width over lo .. hi, lo < hi, both finite, from the
// largest value down; what lies below lo is in the last.  A difference of floats
// goes down to 2^-149, where 2048 over it is no fp32 number: differences of narrow
// ranges are taken times 2^100 first.  So `scale` is finite, hi is in range 0 and
// lo, some 2048 (1 - 2^-22) widths off or more, in the last: each cut of lo .. hi
// parts the two, and a search that goes on with the least and the largest value of
// one range ends at one value.
struct SampleRanges {
  float hi, up, scale;
  __device__ __forceinline__ SampleRanges(float lo, float hi_) : hi(hi_) {
    const double width = (double)hi - (double)lo;
    up = width < 0x1p-100 ? 0x1p100f : 1.0f;
    scale = (float)(kSampleBins / (width * (double)up));
  }
  __device__ __forceinline__ int of(float v) const { return (int)fminf((hi - v) * up * scale, kSampleBins - 1.0f); }
};

}  // namespace specdec
