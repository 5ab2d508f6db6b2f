// verify.cu — verification of drafted tokens (draco_verify_drafts): speculative
// sampling, and with one row per sequence plain sampling.
//
// Row r of a sequence holds the target's logits after the tokens before draft
// r; p = softmax(logits / T).  Draft x_r is taken while u_r q_r(x_r) <
// p_r(x_r), q the drafter's probabilities (1 at x_r without them).  At the
// first one that is not, the next token is drawn from max(p - q, 0); after the
// last row from p itself: the first index whose cumulative weight exceeds
// u times the total.  T = 0: the first index of the largest logit.
//
// Bound by bytes: the logits are read once.  One cluster of 8 or 16 CTAs per
// sequence, the vocabulary cut into one range per CTA, so that one launch does
// everything: row maxima and sums meet in distributed shared memory, every CTA
// walks the same accept decisions, and only the row that is drawn from is read
// again (from L2).  Sums of exponentials that decide an acceptance are fp32; a
// decision whose sides lie within their errors (some 1e-5 of each other) is made
// from fp64 sums of its row.  The cumulative weights of the drawn row are fp64,
// since an index out of 10^5 hangs on differences of one in 10^5 or less.
//
// Measured: 48 sequences of 2-8 rows of 128000 fp32 logits with the drafter's
// probabilities 73 us (2.1 TB/s); for a sequence of five rows 15 us of it read
// the logits, 17 are the two passes of fp64 weights over the row drawn from (the
// sum of p, then of max(p - q, 0)), 5 find the token, 13 go to barriers and
// decisions.  The rest is imbalance: a sequence's rows are all read by its own 8
// CTAs, eight rows as well as two, and the longest sequences end last.  bf16 logits
// 62 us; greedy 37; 48 sequences of one row 27.  One sequence of five rows of 32000
// 11.6 us, greedy 5.7; of one row of 128000 13.
#include <cooperative_groups.h>

#include <cstdio>

#include "internal.h"
#include "paged.cuh"

namespace draco {

namespace cg = cooperative_groups;

constexpr int kVfCtas = 16;  // CTAs of a cluster at most
constexpr int kVfThreads = 384;
constexpr int kVfWarps = kVfThreads / 32;
constexpr int kVfBlocks = 16;
constexpr int kVfRows = 64;  // rows whose statistics are held at a time

struct VerifyArgs {
  const void* logits;
  const float* probs;
  const int* row_start;
  const int* drafts;
  const float* accept_u;
  const float* sample_u;
  int* accepted;
  int* tokens;
  int64_t ld_logits, ld_probs, ld_tokens;
  double inv_t;
  float inv_t_log2;
  float tol;  // relative error of a row's fp32 sum, and of a weight but for its exponent's part
  int n, vocab, max_rows, greedy;
};

// A row's maximum, the sum of exp2((x - m) c) and, for greedy, the first index
// of the maximum.
struct RowStat {
  float m, s;
  int i;
};
__device__ __forceinline__ float fast_exp2f(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float weight32(float x, float m, float c) {
  return x == m ? 1.f : fast_exp2f((x - m) * c);  // (inf - inf) is not taken
}
__device__ __forceinline__ RowStat join(RowStat a, RowStat b, float c) {
  RowStat r;
  r.m = fmaxf(a.m, b.m);
  r.s = (a.m == -INFINITY ? 0.f : a.s * weight32(a.m, r.m, c)) + (b.m == -INFINITY ? 0.f : b.s * weight32(b.m, r.m, c));
  r.i = a.m > b.m ? a.i : b.m > a.m ? b.i : min(a.i, b.i);
  return r;
}
template <typename T>
__device__ __forceinline__ float value(const T* p) {
  if constexpr (sizeof(T) == 4)
    return *p;
  else
    return __bfloat162float(*p);
}
template <typename T>
__device__ __forceinline__ float logit(const T* p) {
  const float x = value(p);
  return x == x ? x : -INFINITY;  // a NaN logit is never drawn
}

// An fp32 value as fp64 by its bits (the conversion instruction runs at a
// quarter of the fp64 rate): exact, but that zero, subnormal values and
// infinities come out as numbers of 2^-127 .. 2^-126 and 2^128.
__device__ __forceinline__ double wide(float x) {
  const uint32_t u = __float_as_uint(x);
  return __hiloint2double((int)((u & 0x80000000u) | (((u & 0x7FFFFFFFu) >> 3) + 0x38000000u)), (int)(u << 29));
}

// exp((x - m) / T) in fp64 by P. T. P. Tang's table-driven method: with k the
// integer next to (x - m) 256 / (T ln2), found in fp32, r = (x - m) / T - k ln2 /
// 256 (|r| < 0.0014), the value is 2^(k / 256) e^r, the first factor from a table
// and the exponent, e^r by its Taylor series to r^3: 2e-13 of the value.  Half
// the fp64 instructions of exp(), which bound the drawing.
constexpr float kTangScale = 369.32993f;  // 256 / ln2
constexpr int kTable = 256;
// The rounding of m / T is a factor of all weights, and goes with their sum.
struct Weight64 {
  float m, scale;   // the row's maximum, 256 / (T ln2)
  double inv_t, m_t;  // 1 / T, m / T
  const double* table;  // 2^(j / 256)
  __device__ __forceinline__ double operator()(float x) const {
    const float t = (x - m) * scale;
    const float kf = t + 12582912.f;  // 1.5 * 2^23: the nearest integer in the low bits
    const int k = __float_as_int(kf) - 0x4B400000;
    // 1.5 * 2^52 + 2^31 + k, for k of either sign in the low word, less its offset
    const double kd = __hiloint2double(0x43380000, (int)((uint32_t)k + 0x80000000u)) - 6755401588539392.0;
    const double r = fma(kd, -0.0027076061740622863, fma(wide(x), inv_t, -m_t));
    double p = fma(r, 1.0 / 6.0, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    p *= table[k & (kTable - 1)];
    const double v = __hiloint2double(__double2hiint(p) + ((k >> 8) << 20), __double2loint(p));
    return t > -256000.f ? v : 0.0;  // below 2^-1000, for -infinity and for NaN nothing
  }
  // with m / T so large that its rounding is no small one, the maximum's weight is
  // one (infinite logits share it)
  __device__ __forceinline__ double any(float x) const {
    return x == m && !(fabs(m_t) < 1e9) ? 1.0 : (*this)(x);
  }
};

// The sum of a row's weights in fp64, by the CTA and the same in each of its
// threads, and in every CTA: one order.  Out of line: few calls get here, and the
// kernel's registers are bounded.
template <typename T>
__device__ __noinline__ double row_weight(const T* row, int vocab, Weight64 weight, double* scratch) {
  double sum = 0.0;
  for (int i = threadIdx.x; i < vocab; i += kVfThreads) {
    const float x = value(row + i);
    sum += weight.any(x);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = sum;
  __syncthreads();
  sum = 0.0;
  for (int w = 0; w < kVfWarps; ++w) sum += scratch[w];
  __syncthreads();
  return sum;
}

// pairs of fp32 values
__device__ __forceinline__ uint64_t pair_2(float a, float b) {
  return ((uint64_t)__float_as_uint(b) << 32) | __float_as_uint(a);
}
__device__ __forceinline__ uint64_t add_2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t mul_2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// 16 bytes of logits as fp32
template <typename T, int V>
__device__ __forceinline__ void unpack16(const uint4& w, float (&x)[V]) {
  if constexpr (V == 4) {
    x[0] = __uint_as_float(w.x), x[1] = __uint_as_float(w.y), x[2] = __uint_as_float(w.z), x[3] = __uint_as_float(w.w);
  } else {
    x[0] = bf16lo(w.x), x[1] = bf16hi(w.x), x[2] = bf16lo(w.y), x[3] = bf16hi(w.y);
    x[4] = bf16lo(w.z), x[5] = bf16hi(w.z), x[6] = bf16lo(w.w), x[7] = bf16hi(w.w);
  }
}

template <typename T, bool kGreedy>
__global__ void __launch_bounds__(kVfThreads, 3) verify_kernel(const VerifyArgs a) {
  cg::cluster_group cluster = cg::this_cluster();
  __shared__ RowStat wstat[kVfRows][kVfWarps];     // this CTA's range, by warp
  __shared__ RowStat stat[kVfRows][kVfCtas];       // every CTA's range (each writes its column everywhere)
  __shared__ RowStat full[kVfRows];                // the whole row
  __shared__ double zsum[kVfCtas][kVfWarps];       // weights of p, by CTA and warp
  __shared__ double rsum[kVfCtas][kVfWarps];       // what is drawn from
  __shared__ double bsum[kVfWarps][kVfBlocks];     // of the warp's blocks of 256 values, the last told sums
  __shared__ double table[kGreedy ? 1 : kTable];   // 2^(j / 256)
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (!kGreedy && tid < kTable) table[tid] = exp2((double)tid / kTable);
  cluster.barrier_arrive();  // waited for before the first store to another CTA: it has started then
  grid_dependency_wait();
  grid_launch_dependents();
  const int rank = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks(), b = blockIdx.x / ctas;
  const T* logits = static_cast<const T*>(a.logits);
  const int begin = min(max(a.row_start[b], 0), a.n);
  const int rows = max(0, min(max(a.row_start[b + 1], 0), a.n) - begin);
  // the CTA's range of the vocabulary, in units of 8 values
  const int units = (a.vocab + 7) / 8, per_cta = (units + ctas - 1) / ctas;
  const int u0 = min(units, rank * per_cta), u1 = min(units, u0 + per_cta);
  const float c = a.inv_t_log2;

  int count = 0;        // drafts taken
  bool decided = rows == 0;
  RowStat at = {-INFINITY, 0.f, 0};  // statistics of the row that the next token comes from
  for (int r0 = 0; r0 < rows && !decided; r0 += kVfRows) {
    const int nr = min(kVfRows, rows - r0);
    // Rows side by side, 12 / nr warps each (a warp takes a row's whole share
    // of the range when there are more): few long streams instead of many short
    // ones whose latencies would add up.
    const int side = min(nr, kVfWarps), wpr = kVfWarps / side, sub = warp % wpr;
    const int per_sub = (u1 - u0 + wpr - 1) / wpr;
    const int w0 = min(a.vocab, 8 * min(u1, u0 + sub * per_sub)), w1 = min(a.vocab, 8 * min(u1, u0 + (sub + 1) * per_sub));
    for (int r = warp / wpr; r < nr && warp < side * wpr; r += side) {
      constexpr int V = 16 / (int)sizeof(T), B = 16 / V;  // values of a load, loads in flight: 16 values of a lane
      const T* row = logits + (int64_t)(begin + r0 + r) * a.ld_logits + w0;
      const int len = w1 - w0;
      // values before the first 16-byte boundary
      const int h = min(len, (int)(((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / sizeof(T)));
      const int vecs = (len - h) / V;
      const uint4* vp = reinterpret_cast<const uint4*>(row + h);
      uint4 buf[B];
      auto fetch = [&](int v0) {
#pragma unroll
        for (int e = 0; e < B; ++e)
          if (v0 + 32 * e + lane < vecs) buf[e] = __ldg(vp + v0 + 32 * e + lane);
      };
      fetch(0);
      RowStat st = {-INFINITY, 0.f, 0x7FFFFFFF};
      // values before and after the vectors
      const int odd = lane < h ? lane : h + vecs * V + (lane - h);
      const float xo = odd < len ? logit(row + odd) : -INFINITY;
      if (xo > -INFINITY) st.m = xo, st.s = 1.f, st.i = w0 + odd;
      for (int v0 = 0; v0 < vecs; v0 += 32 * B) {
        float x[B][V];
#pragma unroll
        for (int e = 0; e < B; ++e) {
          unpack16<T, V>(buf[e], x[e]);
#pragma unroll
          for (int k = 0; k < V; ++k) x[e][k] = fmaxf(x[e][k], -INFINITY);  // a NaN logit is never drawn
        }
        if (v0 + 32 * B > vecs) {
#pragma unroll
          for (int e = 0; e < B; ++e)
            if (v0 + 32 * e + lane >= vecs) {
#pragma unroll
              for (int k = 0; k < V; ++k) x[e][k] = -INFINITY;
            }
        }
        if (v0 + 32 * B < vecs) fetch(v0 + 32 * B);
        float mx = -INFINITY;
#pragma unroll
        for (int e = 0; e < B; ++e)
#pragma unroll
          for (int k = 0; k < V; ++k) mx = fmaxf(mx, x[e][k]);
        if constexpr (kGreedy) {
          if (mx >= st.m && mx > -INFINITY) {
            int first = 0x7FFFFFFF;
#pragma unroll
            for (int e = B - 1; e >= 0; --e)
#pragma unroll
              for (int k = V - 1; k >= 0; --k)
                if (x[e][k] == mx) first = w0 + h + (v0 + 32 * e + lane) * V + k;
            st.i = mx > st.m ? first : min(st.i, first);
            st.m = mx;
          }
        } else if (mx > -INFINITY) {
          if (mx > st.m) {
            st.s = st.m == -INFINITY ? 0.f : st.s * weight32(st.m, mx, c);
            st.m = mx;
          }
          if (st.m < INFINITY) {
            // (x - m) c in pairs: the difference first, which is exact where it counts
            const float nm = -st.m;
            float s0 = 0.f, s1 = 0.f;
#pragma unroll
            for (int e = 0; e < B; ++e)
#pragma unroll
              for (int k = 0; k < V; k += 2) {
                const uint64_t y = mul_2(add_2(pair_2(x[e][k], x[e][k + 1]), pair_2(nm, nm)), pair_2(c, c));
                s0 += fast_exp2f(__uint_as_float((uint32_t)y)), s1 += fast_exp2f(__uint_as_float((uint32_t)(y >> 32)));
              }
            st.s += s0 + s1;
          } else {  // an infinite logit has all the weight
#pragma unroll
            for (int e = 0; e < B; ++e)
#pragma unroll
              for (int k = 0; k < V; ++k) st.s += x[e][k] == INFINITY ? 1.f : 0.f;
          }
        }
      }
      // the warp's maximum, then sums relative to it (or the first index of it)
      RowStat wst = st;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) wst.m = fmaxf(wst.m, __shfl_xor_sync(0xffffffffu, wst.m, o));
      if constexpr (kGreedy) {
        wst.i = __reduce_min_sync(0xffffffffu, st.m == wst.m ? st.i : 0x7FFFFFFF);
      } else {
        wst.s = st.m == -INFINITY ? 0.f : st.s * weight32(st.m, wst.m, c);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) wst.s += __shfl_xor_sync(0xffffffffu, wst.s, o);
      }
      if (lane == 0) wstat[r][sub] = wst;
    }
    __syncthreads();
    if (r0 > 0)
      cluster.sync();  // everybody has read the last rows' statistics
    else
      cluster.barrier_wait();
    for (int idx = tid; idx < nr * kVfCtas; idx += kVfThreads) {  // a thread per (row, CTA to tell)
      if (idx % kVfCtas >= ctas) continue;
      RowStat st = wstat[idx / kVfCtas][0];
      for (int w = 1; w < wpr; ++w) st = join(st, wstat[idx / kVfCtas][w], c);
      *cluster.map_shared_rank(&stat[idx / kVfCtas][rank], idx % kVfCtas) = st;
    }
    cluster.sync();
    for (int r = warp; r < nr; r += kVfWarps) {  // a warp per row joins the CTAs' parts
      RowStat st = {-INFINITY, 0.f, 0x7FFFFFFF};
      if (lane < ctas) st = stat[r][lane];
#pragma unroll
      for (int o = kVfCtas / 2; o > 0; o >>= 1) {
        RowStat x;
        x.m = __shfl_xor_sync(0xffffffffu, st.m, o);
        x.s = __shfl_xor_sync(0xffffffffu, st.s, o);
        x.i = __shfl_xor_sync(0xffffffffu, st.i, o);
        st = join(st, x, c);
      }
      if (lane == 0) full[r] = st;
    }
    __syncthreads();
    // The accept decisions, a row to a lane.  The two sides are compared in fp32's
    // accuracy first; where they lie closer than its errors, in fp64's.
    for (int rb = 0; rb < nr && !decided; rb += 32) {
      const int r = rb + lane;
      bool take = false, close = false;
      if (r < nr && r0 + r < rows - 1) {
        const int rr = begin + r0 + r, x = a.drafts[rr];
        const RowStat st = full[r];
        if (x >= 0 && x < a.vocab && st.m > -INFINITY) {
          if constexpr (kGreedy) {
            take = x == st.i;
          } else {
            const float lx = logit(logits + (int64_t)rr * a.ld_logits + x);
            const float qx = a.probs ? a.probs[(int64_t)rr * a.ld_probs + x] : 1.f;
            const float e = lx == st.m ? 0.f : (lx - st.m) * c, wx = lx == -INFINITY ? 0.f : exp2f(e);
            const double ux = (double)a.accept_u[rr] * qx * st.s;
            take = ux < wx;
            close = fabs(ux - wx) <= (double)(wx * (a.tol - e * 0x1p-22f)) || (wx < 0x1p-120f && ux < 0x1p-119);
          }
        }
      }
      unsigned stop = __ballot_sync(0xffffffffu, !take);
      int k = stop ? __ffs(stop) - 1 : 32;  // the first row that is not taken (or is the last)
      if constexpr (!kGreedy) {
        for (unsigned left = __ballot_sync(0xffffffffu, close); left != 0u; left &= left - 1) {
          const int e = __ffs(left) - 1;
          if (e > k) break;
          const int rr = begin + r0 + rb + e, x = a.drafts[rr];
          const T* row = logits + (int64_t)rr * a.ld_logits;
          const float m = full[rb + e].m;
          const Weight64 weight{m, (float)a.inv_t * kTangScale, a.inv_t, (double)m * a.inv_t, table};
          const double ux = (double)a.accept_u[rr] * (a.probs ? a.probs[(int64_t)rr * a.ld_probs + x] : 1.f);
          const bool yes = ux * row_weight(row, a.vocab, weight, &bsum[0][0]) < weight.any(logit(row + x));
          stop = yes ? stop & ~(1u << e) : stop | 1u << e;
          k = stop ? __ffs(stop) - 1 : 32;
        }
      }
      const int n = min(k, nr - rb);
      count += n;
      if (n < nr - rb && n < 32) {
        decided = true;
        at = full[rb + n];
      }
    }
    __syncthreads();  // full is written again for the next rows
  }

  if (rows == 0) cluster.barrier_wait();
  int last = -1;
  if (rows > 0 && at.m > -INFINITY) {
    if constexpr (kGreedy) {
      last = at.i;
    } else {
      const int rr = begin + count;
      const bool rejected = count < rows - 1;
      const T* row = logits + (int64_t)rr * a.ld_logits;
      const int x = rejected && a.probs == nullptr ? a.drafts[rr] : -1;  // a point mass is taken out
      const float* q = rejected && a.probs != nullptr ? a.probs + (int64_t)rr * a.ld_probs : nullptr;
      const Weight64 weight{at.m, (float)a.inv_t * kTangScale, a.inv_t, (double)at.m * a.inv_t, table};
      // The warp's range in vocabulary order, in blocks of K values a lane: value
      // k of lane L is base + 32 k + L.
      constexpr int K = 8;
      const int per_warp = (per_cta + kVfWarps - 1) / kVfWarps;
      const int w0 = min(a.vocab, 8 * min(u1, u0 + warp * per_warp));
      const int w1 = min(a.vocab, 8 * min(u1, u0 + (warp + 1) * per_warp));
      if (q != nullptr)  // on its way while the weights of p are summed
        for (int i = w0 + 32 * lane; i < w1; i += 1024) asm volatile("prefetch.global.L2 [%0];" ::"l"(q + i));
      double w[K];
      auto warp_sum = [](double v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
      };
      auto lane_sum = [&]() {
        double s0 = 0.0, s1 = 0.0;
#pragma unroll
        for (int k = 0; k < K; k += 2) s0 += w[k], s1 += w[k + 1];
        return s0 + s1;
      };
      double inv_z = 1.0;
      auto weights = [&](int i0, bool of_p) {  // of p, or of what may still be drawn
        float v[K], u[K];
        const bool whole = i0 - lane + 32 * K <= w1;
        if (whole) {
#pragma unroll
          for (int k = 0; k < K; ++k) v[k] = value(row + i0 + 32 * k);
        } else {
#pragma unroll
          for (int k = 0; k < K; ++k) v[k] = i0 + 32 * k < w1 ? value(row + i0 + 32 * k) : -INFINITY;
        }
        if (!of_p && q != nullptr) {
          if (whole) {
#pragma unroll
            for (int k = 0; k < K; ++k) u[k] = __ldg(q + i0 + 32 * k);
          } else {
#pragma unroll
            for (int k = 0; k < K; ++k) u[k] = i0 + 32 * k < w1 ? __ldg(q + i0 + 32 * k) : 0.f;
          }
        }
        if (fabs(weight.m_t) < 1e9) {
#pragma unroll
          for (int k = 0; k < K; ++k) w[k] = weight(v[k]);
        } else {
#pragma unroll
          for (int k = 0; k < K; ++k) w[k] = weight.any(v[k]);
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
          if (!of_p) {
            if (q != nullptr) {
              const double d = fma(w[k], inv_z, -wide(u[k]));
              w[k] = __double2hiint(d) > 0 ? d : 0.0;
            } else if (i0 + 32 * k == x) {
              w[k] = 0.0;
            }
          }
        }
      };
      // sums of the warp's range, to every CTA, and block by block for the warp itself
      auto tell = [&](double (*sums)[kVfWarps], bool of_p) {
        double all = 0.0;
        for (int i = w0, j = 0; i < w1; i += 32 * K, ++j) {
          weights(i + lane, of_p);
          const double v = warp_sum(lane_sum());
          if (j < kVfBlocks && lane == 0) bsum[warp][j] = v;
          all += v;
        }
        if (lane < ctas) *cluster.map_shared_rank(&sums[rank][warp], lane) = all;
      };
      constexpr int P = kVfCtas * kVfWarps / 32;  // ranges of a lane, in order
      auto total = [&](const double (*sums)[kVfWarps], double (&mine)[P]) {
        double v = 0.0;
#pragma unroll
        for (int k = 0; k < P; ++k) {
          mine[k] = (P * lane + k) / kVfWarps < ctas ? (&sums[0][0])[P * lane + k] : 0.0;
          v += mine[k];
        }
        return warp_sum(v);  // (the same in every warp: one order)
      };
      double mine[P];
      tell(zsum, true);
      const double(*drawn_from)[kVfWarps] = zsum;
      if (rejected) {
        if (q != nullptr) {
          cluster.sync();
          inv_z = 1.0 / total(zsum, mine);
        }
        if (q != nullptr || (x >= w0 && x < w1)) {
          tell(rsum, false);
        } else {  // a range that the point mass does not touch
          __syncwarp();
          if (lane < ctas) *cluster.map_shared_rank(&rsum[rank][warp], lane) = zsum[rank][warp];
        }
        drawn_from = rsum;
      }
      cluster.sync();
      double all = total(drawn_from, mine);
      bool of_p = !rejected;
      const bool fallback_p = rejected && !(all > 0.0);  // p <= q everywhere: p itself is drawn from
      if (fallback_p) all = total(zsum, mine), of_p = true;
      const double goal = (double)a.sample_u[b] * all;
      // every warp finds the range that passes the goal: the first in order;
      // rounding may leave the goal beyond all of them: the last with weight then
      double before = 0.0;
#pragma unroll
      for (int k = 0; k < P; ++k) before += mine[k];
      {
        const double own = before;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double v = __shfl_up_sync(0xffffffffu, before, o);
          if (lane >= o) before += v;
        }
        before -= own;
      }
      int owner = 0x7FFFFFFF, fallback = -1;
      double base = 0.0, base_last = 0.0;
#pragma unroll
      for (int k = 0; k < P; ++k) {
        if (mine[k] > 0.0) {
          fallback = P * lane + k, base_last = before;
          if (owner == 0x7FFFFFFF && before + mine[k] > goal) owner = P * lane + k, base = before;
        }
        before += mine[k];
      }
      const int first = __reduce_min_sync(0xffffffffu, owner), end = __reduce_max_sync(0xffffffffu, fallback);
      const int chosen = first == 0x7FFFFFFF ? end : first;
      base = __shfl_sync(0xffffffffu, first == 0x7FFFFFFF ? base_last : base, max(chosen, 0) / P);
      if (chosen == rank * kVfWarps + warp) {
        int token = -1, token_last = w0;
        for (int i = w0, j = 0; i < w1 && token < 0; i += 32 * K, ++j) {
          if (j < kVfBlocks && !fallback_p && i + 32 * K < w1) {  // a block that stays below the goal
            const double v = bsum[warp][j];
            if (v > 0.0 && base + v <= goal) {
              token_last = -2 - i;  // (its last value with weight is looked for only if nothing follows)
              base += v;
              continue;
            }
            if (!(v > 0.0)) continue;
          }
          weights(i + lane, of_p);
          // sums of 32 consecutive values; the group and the value that pass the goal
          double s[K];
#pragma unroll
          for (int k = 0; k < K; ++k) s[k] = warp_sum(w[k]);
#pragma unroll
          for (int k = 0; k < K; ++k) {
            if (token < 0 && s[k] > 0.0) {
              token_last = i + 32 * k + 31 - __clz(__ballot_sync(0xffffffffu, w[k] > 0.0));
              if (base + s[k] > goal) {
                double v = w[k];
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                  const double u = __shfl_up_sync(0xffffffffu, v, o);
                  if (lane >= o) v += u;
                }
                const unsigned over = __ballot_sync(0xffffffffu, w[k] > 0.0 && base + v > goal);
                token = over ? i + 32 * k + __ffs(over) - 1 : token_last;
              }
              base += s[k];
            }
          }
        }
        if (token < 0 && token_last < 0) {  // rounding: the last value with weight of the block noted
          const int i = -2 - token_last;
          weights(i + lane, of_p);
#pragma unroll
          for (int k = 0; k < K; ++k) {
            const unsigned some = __ballot_sync(0xffffffffu, w[k] > 0.0);
            if (some) token_last = i + 32 * k + 31 - __clz(some);
          }
        }
        if (token < 0) token = token_last;
        if (lane == 0 && count < a.max_rows) a.tokens[(int64_t)b * a.ld_tokens + count] = token;
      }
    }
  }
  if (rank == 0) {
    if (tid == 0) a.accepted[b] = count;
    const bool drawn = rows > 0 && at.m > -INFINITY && !kGreedy;  // its owner writes the token
    for (int j = tid; j < a.max_rows; j += kVfThreads) {
      if (j == count && drawn) continue;
      a.tokens[(int64_t)b * a.ld_tokens + j] = j < count ? a.drafts[begin + j] : j == count ? last : -1;
    }
  }
}

// 16 CTAs a sequence while that many such clusters run at a time, else 8 (a
// portable cluster; with 16 only a whole GPC's SMs can host one).  A B200 runs 21
// of 16, three CTAs an SM.  Sequences of one row of 128000 fp32 logits: 20 take
// 21.8 us in clusters of 16; 22 take 30.7 us so and 23.2 in clusters of 8, 37
// 36.9 and 28.7; five rows with probabilities: 22 53 and 50, 37 67 and 64.
template <typename T, bool kGreedy>
static cudaError_t launch_t(const VerifyArgs& a, int n_seqs, cudaStream_t st) {
  static int clusters_of[64] = {0};  // clusters of 16 that run at a time, and one
  int dev = 0, clusters = 0;
  cudaGetDevice(&dev);
  if (dev < 64) clusters = clusters_of[dev];
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = kVfCtas;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(kVfCtas);
  cfg.blockDim = dim3(kVfThreads);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  if (clusters == 0) {
    cudaError_t e =
        cudaFuncSetAttribute(verify_kernel<T, kGreedy>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveClusters(&clusters, verify_kernel<T, kGreedy>, &cfg);
    if (e != cudaSuccess) return e;
    clusters += 1;
    if (dev < 64) clusters_of[dev] = clusters;
  }
  const int ctas = n_seqs < clusters ? kVfCtas : kVfCtas / 2;
  attr[1].val.clusterDim.x = ctas;
  cfg.gridDim = dim3((unsigned)n_seqs * ctas);
  return cudaLaunchKernelEx(&cfg, verify_kernel<T, kGreedy>, a);
}
static cudaError_t launch_verify(const VerifyArgs& a, int n_seqs, bool bf16, cudaStream_t st) {
  if (a.greedy) return bf16 ? launch_t<__nv_bfloat16, true>(a, n_seqs, st) : launch_t<float, true>(a, n_seqs, st);
  return bf16 ? launch_t<__nv_bfloat16, false>(a, n_seqs, st) : launch_t<float, false>(a, n_seqs, st);
}

int verify_launch(const draco_verify_args& v, double temperature, cudaStream_t st, char* msg, size_t ml) {
  VerifyArgs a;
  a.logits = v.logits;
  a.probs = v.draft_probs;
  a.row_start = v.row_start;
  a.drafts = v.drafts;
  a.accept_u = v.accept_u;
  a.sample_u = v.sample_u;
  a.accepted = v.accepted;
  a.tokens = v.tokens;
  a.ld_logits = v.ld_logits;
  a.ld_probs = v.ld_probs;
  a.ld_tokens = v.ld_tokens;
  a.greedy = temperature == 0.0;
  a.inv_t = a.greedy ? 1.0 : 1.0 / temperature;
  a.inv_t_log2 = (float)(a.inv_t * 1.4426950408889634);
  // In units of 2^-24: a weight is off by 2.1 |a| + 4 (a: its exponent, of three
  // roundings; exp2: two steps of 2^-23), a row's sum by 2.1 log2(vocab) + 4 for its
  // weights, 9 for a step's additions, 7 a step (512 values of a warp, in clusters
  // of 8 at least) for the running sum and its rescalings, and 6 for each of 21
  // joins: 212 + 7 steps at most together.
  a.tol = (8.f * (float)(v.vocab / (512 * (kVfCtas / 2)) + 1) + 272.f) * 0x1p-24f;
  a.n = v.n;
  a.vocab = v.vocab;
  a.max_rows = v.max_rows;
  const cudaError_t e = launch_verify(a, v.n_seqs, v.dtype == DRACO_DTYPE_BF16, st);
  if (e != cudaSuccess) {
    snprintf(msg, ml, "verify_drafts launch failed: %s", cudaGetErrorString(e));
    return DRACO_ERR_CUDA;
  }
  return DRACO_OK;
}

}  // namespace draco
