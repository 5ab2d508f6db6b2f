// paged_attn.cuh — what the two paged attention kernels share: the call's
// arguments and the row tiles.
#pragma once

#include "paged.cuh"
#include "paged_split.h"

namespace draco {

constexpr int kPagedCounters = 2048;  // (row tile, kv head) pairs that may be split over CTAs
// workspace: int32 counters [kPagedCounters], status word, padding to this; then partial results
constexpr int kPagedHead = kPagedCounters * 4 + 64;
static_assert(kPagedHead == DRACO_PAGED_WORKSPACE_HEAD && kPagedCounters * 4 == DRACO_PAGED_WORKSPACE_STATUS, "header");

// One call.  The rows of sequence s are its new tokens' query heads of one
// key/value head, ordered (token, head in group); a row tile takes `R`
// consecutive rows.
struct PagedAttnArgs {
  PagedView c;
  const void* q;
  void* out;
  int64_t ldq, ldo;
  const int* q_start;
  const int* kv_len;
  float* recs;   // partial results of splits
  int* counters;
  float scale_log2;  // softmax scale * log2(e)
  int n, n_seqs, heads, group, n_splits;
  int min_new, max_new;  // this kernel takes the sequences with min_new <= new tokens < max_new
  int per_seq;           // row tiles of every sequence, or 0: tiles by the tokens' places
  float want;            // warp MMA: CTAs of a key/value head that run at a time
  int waves;             // ... and how often over at most
};

struct RowTile {
  int s;         // sequence, -1: none
  int start;     // its first token in q
  int new_tok;   // its new tokens
  int row0;      // first row of the tile
  int rows;      // rows of the sequence (new_tok * group)
  int kv;        // its cached keys
};

__device__ __forceinline__ int seq_begin(const PagedAttnArgs& a, int s) {
  return min(max(__ldg(a.q_start + s), 0), a.n);
}

// Tile t of R rows.  With per_seq the sequences own that many tiles each (short
// chunks: a decode step finds its sequence without a search).  Otherwise
// sequence s owns the tiles from floor(start_s * group / R)
// + s on: enough for its rows whatever the other lengths are, so that no
// prefix sum over the sequences is needed, and strictly increasing in s, so
// that a warp finds s with a 32-ary search (one round of loads up to 32
// sequences).  Tiles past a sequence's rows are empty.  All lanes of the warp
// take part.
__device__ __forceinline__ RowTile find_tile(const PagedAttnArgs& a, int t, int R) {
  const int lane = threadIdx.x & 31;
  int lo = 0, cnt = a.n_seqs;
  if (a.per_seq) lo = t / a.per_seq, cnt = 1;
  while (cnt > 1) {
    const int step = (cnt + 31) / 32;
    const int s = lo + lane * step;
    const bool le = s < lo + cnt && (int)((int64_t)seq_begin(a, s) * a.group / R) + s <= t;
    const unsigned m = __ballot_sync(0xffffffffu, le);
    const int k = max(__popc(m), 1) - 1;
    cnt = min(step, cnt - k * step);
    lo += k * step;
  }
  RowTile r;
  r.s = -1;
  r.start = seq_begin(a, lo);
  const int end = max(seq_begin(a, lo + 1), r.start);
  r.new_tok = end - r.start;
  r.rows = r.new_tok * a.group;
  r.row0 = (a.per_seq ? t % a.per_seq : t - (int)((int64_t)r.start * a.group / R) - lo) * R;
  const int64_t cap = (int64_t)a.c.max_pages << a.c.page_shift;
  const int kv = __ldg(a.kv_len + lo);
  r.kv = (int)(kv < 0 ? 0 : kv > cap ? cap : kv);
  if (r.row0 >= 0 && r.row0 < r.rows && r.new_tok >= a.min_new && r.new_tok < a.max_new) r.s = lo;
  return r;
}

// keys that row `row` of the tile's sequence sees (may be <= 0: none)
__device__ __forceinline__ int row_limit(const PagedAttnArgs& a, const RowTile& t, int row) {
  return t.kv - t.new_tok + row / a.group + 1;
}

// Scores past 2^20.  m is the largest c S rounded to fp32, and c S - m in one step
// is that rounding at the largest key: up to 2 at 2^25, where fp16's P overflows,
// and up to 128 at 2^31, where any does.  With c S rounded first the largest gives
// 0, and others at most kPaLazy, but for the rounding of m + kPaLazy: the minimum.
constexpr float kPaLazy = 8.f;     // log2 units by which scores may outgrow m
constexpr float kPaHuge = 1048576.f;
__device__ __forceinline__ bool is_huge(float m) { return fabsf(m) > kPaHuge && m != -INFINITY; }
__device__ __forceinline__ float huge_exponent(float s, float sc, float m) {
  float x = __fsub_rn(__fmul_rn(s, sc), m == -INFINITY ? 0.f : m);  // (NaN for infinite scores)
  asm("min.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(kPaLazy));
  return x;
}

// the tensor-memory kernel (paged_attn_tc.cu)
// New tokens from which a sequence goes there: 65 rows.  Its CTA takes 256 rows at
// a time however few there are.
constexpr int kTcMinRows = 64;
inline int tc_min_tokens(int group) { return kTcMinRows / group + 1; }
struct TcPlan {
  int rt, splits;
  int by_tokens;  // partial results by record_place (else by tile)
  int64_t tiles, units;
  size_t bytes;  // of partial results
};
bool paged_attn_tc_takes(const PagedView& c, int hd, int dtype, int group, int page_size);
TcPlan paged_attn_tc_plan(int n, int n_seqs, int group, int kv_heads, int hd, int max_kv);
int paged_attn_tc_launch(const PagedAttnArgs& a, int hd, const TcPlan& p, int* status, cudaStream_t st, char* msg,
                         size_t ml);

}  // namespace draco
