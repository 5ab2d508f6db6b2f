// paged_split.h — the arithmetic of a sequence's splits and of the places of
// partial results, for the kernels and, as plain C++, for the host's tests.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define DRACO_BOTH __host__ __device__ __forceinline__
#else
#define DRACO_BOTH inline
#endif

namespace draco {

// Splits of `kend` keys at `ck` keys each (one at least), and the end of the one
// that begins at `kbeg`.  Neither sum leaves 32 bits however near kend is to the
// largest length and ck to kend.
DRACO_BOTH int split_count(int kend, int ck) { return kend > 0 ? 1 + (kend - 1) / ck : 1; }
DRACO_BOTH int split_end(int kbeg, int kend, int ck) { return kend - kbeg < ck ? kend : kbeg + ck; }

}  // namespace draco
