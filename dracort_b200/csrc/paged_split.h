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

// Places of partial results for the row tiles (R rows each) of the sequences of
// `from` new tokens or more, among n tokens, `group` rows a token: the tile at row
// row0 of the sequence that begins at token `start`.  They are distinct without a
// sum over the sequences: a sequence of m >= from tokens moves the next one's first
// place on by floor(m group / R) + 1 at least, which its tiles need.
DRACO_BOTH int64_t record_place(int start, int row0, int group, int R, int from) {
  return (int64_t)start * group / R + start / from + row0 / R;
}
DRACO_BOTH int64_t record_places(int n, int group, int R, int from) { return (int64_t)n * group / R + n / from; }

}  // namespace draco
