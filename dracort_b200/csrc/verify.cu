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
// Bound by bytes: the logits are read once.  One cluster of 8 CTAs per
// sequence, the vocabulary cut into one range per CTA, so that one launch does
// everything: row maxima and sums meet in distributed shared memory, every CTA
// walks the same accept decisions, and only the row that is drawn from is read
// a second time (from L2).  Sums of exponentials that decide an acceptance are
// fp32 (their error of about 1e-7 moves a decision as rarely); the cumulative
// weights of the drawn row are fp64, since an index out of 10^5 hangs on
// differences of one in 10^5 or less.
#include <cooperative_groups.h>

#include <cstdio>

#include "internal.h"
#include "paged.cuh"

namespace draco {

namespace cg = cooperative_groups;

constexpr int kVfCtas = 8;
constexpr int kVfThreads = 512;
constexpr int kVfWarps = kVfThreads / 32;
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
__device__ __forceinline__ float logit(const T* p) {
  float x;
  if constexpr (sizeof(T) == 4)
    x = *p;
  else
    x = __bfloat162float(*p);
  return x == x ? x : -INFINITY;  // a NaN logit is never drawn
}

// 2^(t / 256) for t <= 0 in fp64 (a few units in the last place), by P. T. P.
// Tang's table-driven method: t = 256 k + j + f with |f| <= 1/2, the value is
// 2^k 2^(j/256) e^r, r = f ln2 / 256, e^r by its Taylor series to r^4 (r^5 / 120 <
// 4e-17).  Half the fp64 instructions of exp(), which bound the drawing.
constexpr double kTangScale = 369.3299304675746;  // 256 / ln2
constexpr int kTable = 256;
__device__ __forceinline__ double exp2_256(double t, const double* table) {
  const double kd = t + 6755399441055744.0;  // 1.5 * 2^52: the nearest integer in the low bits
  const int n = __double2loint(kd);
  const double r = (t - (kd - 6755399441055744.0)) * 0.0027076061740622863;  // ln2 / 256
  double p = fma(r, 1.0 / 24.0, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  p *= table[n & (kTable - 1)];
  const double v = __hiloint2double(__double2hiint(p) + ((n >> 8) << 20), __double2loint(p));
  return t > -256000.0 ? v : 0.0;  // below 2^-1000 (and for -infinity): nothing
}
// exp((x - m) / T); t256 = 256 / (T ln2)
__device__ __forceinline__ double weight64(float x, double m, double t256, const double* table) {
  const double xd = (double)x;
  return xd == m ? 1.0 : exp2_256((xd - m) * t256, table);
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
__global__ void __cluster_dims__(kVfCtas, 1, 1) __launch_bounds__(kVfThreads) verify_kernel(const VerifyArgs a) {
  cg::cluster_group cluster = cg::this_cluster();
  __shared__ RowStat wstat[kVfRows][kVfWarps];     // this CTA's range, by warp
  __shared__ RowStat stat[kVfRows][kVfCtas];       // every CTA's range (each writes its column everywhere)
  __shared__ RowStat full[kVfRows];                // the whole row
  __shared__ double zsum[kVfCtas][kVfWarps];       // weights of p, by CTA and warp
  __shared__ double rsum[kVfCtas][kVfWarps];       // what is drawn from
  __shared__ double table[kGreedy ? 1 : kTable];   // 2^(j / 256)
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (!kGreedy && tid < kTable) table[tid] = exp2((double)tid / kTable);
  grid_dependency_wait();
  grid_launch_dependents();
  const int rank = (int)cluster.block_rank(), b = blockIdx.x / kVfCtas;
  const T* logits = static_cast<const T*>(a.logits);
  const int begin = min(max(a.row_start[b], 0), a.n);
  const int rows = max(0, min(max(a.row_start[b + 1], 0), a.n) - begin);
  // the CTA's range of the vocabulary, in units of 8 values
  const int units = (a.vocab + 7) / 8, per_cta = (units + kVfCtas - 1) / kVfCtas;
  const int u0 = min(units, rank * per_cta), u1 = min(units, u0 + per_cta);
  const float c = a.inv_t_log2;

  int count = 0;        // drafts taken
  bool decided = rows == 0;
  RowStat at = {-INFINITY, 0.f, 0};  // statistics of the row that the next token comes from
  for (int r0 = 0; r0 < rows && !decided; r0 += kVfRows) {
    const int nr = min(kVfRows, rows - r0);
    // Rows side by side, 16 / nr warps each (a warp takes a row's whole share
    // of the range when there are more): few long streams instead of many short
    // ones whose latencies would add up.
    const int side = min(nr, kVfWarps), wpr = kVfWarps / side, sub = warp % wpr;
    const int per_sub = (u1 - u0 + wpr - 1) / wpr;
    const int w0 = min(a.vocab, 8 * min(u1, u0 + sub * per_sub)), w1 = min(a.vocab, 8 * min(u1, u0 + (sub + 1) * per_sub));
    for (int r = warp / wpr; r < nr && warp < side * wpr; r += side) {
      constexpr int V = 16 / (int)sizeof(T), B = 32 / V;  // values of a load, loads in flight: 32 values of a lane
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
          const bool on = v0 + 32 * e + lane < vecs;
#pragma unroll
          for (int k = 0; k < V; ++k) x[e][k] = on ? x[e][k] : -INFINITY;
        }
        if (v0 + 32 * B < vecs) fetch(v0 + 32 * B);
        float mx = -INFINITY;
#pragma unroll
        for (int e = 0; e < B; ++e)
#pragma unroll
          for (int k = 0; k < V; ++k) mx = fmaxf(mx, x[e][k]);  // (passes over a NaN)
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
            float s0 = 0.f, s1 = 0.f;
#pragma unroll
            for (int e = 0; e < B; ++e)
#pragma unroll
              for (int k = 0; k < V; k += 2) {
                const float u = fast_exp2f((x[e][k] - st.m) * c), v = fast_exp2f((x[e][k + 1] - st.m) * c);
                s0 += u == u ? u : 0.f, s1 += v == v ? v : 0.f;
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
    if (r0 > 0) cluster.sync();  // everybody has read the last rows' statistics
    for (int idx = tid; idx < nr * kVfCtas; idx += kVfThreads) {  // a thread per (row, CTA to tell)
      RowStat st = wstat[idx / kVfCtas][0];
      for (int w = 1; w < wpr; ++w) st = join(st, wstat[idx / kVfCtas][w], c);
      *cluster.map_shared_rank(&stat[idx / kVfCtas][rank], idx % kVfCtas) = st;
    }
    cluster.sync();
    if (tid < nr) {
      RowStat st = stat[tid][0];
#pragma unroll
      for (int k = 1; k < kVfCtas; ++k) st = join(st, stat[tid][k], c);
      full[tid] = st;
    }
    __syncthreads();
    // the accept decisions, a row to a lane
    for (int rb = 0; rb < nr && !decided; rb += 32) {
      const int r = rb + lane;
      bool take = false;
      if (r < nr && r0 + r < rows - 1) {
        const int rr = begin + r0 + r, x = a.drafts[rr];
        const RowStat st = full[r];
        if (x >= 0 && x < a.vocab && st.m > -INFINITY) {
          if constexpr (kGreedy) {
            take = x == st.i;
          } else {
            const float lx = logit(logits + (int64_t)rr * a.ld_logits + x);
            const float qx = a.probs ? a.probs[(int64_t)rr * a.ld_probs + x] : 1.f;
            const float wx = lx == -INFINITY ? 0.f : lx == st.m ? 1.f : exp2f((lx - st.m) * c);
            take = (double)a.accept_u[rr] * qx * st.s < wx;
          }
        }
      }
      const unsigned stop = __ballot_sync(0xffffffffu, !take);
      const int k = stop ? __ffs(stop) - 1 : 32;  // the first row that is not taken (or is the last)
      const int n = min(k, nr - rb);
      count += n;
      if (n < nr - rb && n < 32) {
        decided = true;
        at = full[rb + n];
      }
    }
    __syncthreads();  // full is written again for the next rows
  }

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
      const double m64 = (double)at.m, t256 = a.inv_t * kTangScale;
      // The warp's range in vocabulary order, in blocks of 32 values a lane: value
      // k of lane L is base + 32 k + L.  Up to 2^17 entries a warp has one block,
      // whose weights stay in registers from the first sum to the draw.
      constexpr int K = 32;
      const int per_warp = (per_cta + kVfWarps - 1) / kVfWarps;
      const int w0 = min(a.vocab, 8 * min(u1, u0 + warp * per_warp));
      const int w1 = min(a.vocab, 8 * min(u1, u0 + (warp + 1) * per_warp));
      const int blocks = max(1, (w1 - w0 + 32 * K - 1) / (32 * K));
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
      auto weights = [&](int blk) {  // of p
        const int i0 = w0 + blk * 32 * K + lane;
        float v[K];
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = i0 + 32 * k < w1 ? logit(row + i0 + 32 * k) : -INFINITY;
#pragma unroll
        for (int k = 0; k < K; ++k)
          w[k] = i0 + 32 * (k & ~7) - lane >= w1 ? 0.0 : i0 + 32 * k < w1 ? weight64(v[k], m64, t256, table) : 0.0;
      };
      double inv_z = 1.0;
      auto left = [&](int blk) {  // what may still be drawn, from the weights of p
        const int i0 = w0 + blk * 32 * K + lane;
        if (q == nullptr) {
#pragma unroll
          for (int k = 0; k < K; ++k)
            if (i0 + 32 * k == x) w[k] = 0.0;
        } else {
#pragma unroll
          for (int k = 0; k < K; ++k) {
            const double d = i0 + 32 * k < w1 ? w[k] * inv_z - (double)__ldg(q + i0 + 32 * k) : 0.0;
            w[k] = d > 0.0 ? d : 0.0;
          }
        }
      };
      auto tell = [&](double (*sums)[kVfWarps], double v) {  // this warp's sum to every CTA
        v = warp_sum(v);
        if (lane < kVfCtas) *cluster.map_shared_rank(&sums[rank][warp], lane) = v;
      };
      auto total = [&](double (*sums)[kVfWarps]) {  // in one order, so that all warps have the same
        double v = 0.0;
#pragma unroll
        for (int k = 0; k < kVfCtas * kVfWarps / 32; ++k) v += (&sums[0][0])[32 * k + lane];
        return warp_sum(v);
      };
      double sp = 0.0, sd = 0.0;
      for (int blk = 0; blk < blocks; ++blk) {
        weights(blk);
        sp += lane_sum();
        if (q == nullptr) {
          left(blk);
          sd += lane_sum();
        }
      }
      tell(zsum, sp);
      if (q != nullptr) {
        cluster.sync();
        inv_z = 1.0 / total(zsum);
        for (int blk = 0; blk < blocks; ++blk) {
          if (blocks > 1) weights(blk);
          left(blk);
          sd += lane_sum();
        }
      }
      tell(rsum, sd);
      cluster.sync();
      const bool any = total(rsum) > 0.0;  // not so: p <= q everywhere, p itself is drawn from
      const double(*sums)[kVfWarps] = any ? rsum : zsum;
      const double goal = (double)a.sample_u[b] * total(const_cast<double(*)[kVfWarps]>(sums));
      // every warp finds the range that passes the goal: the first in order;
      // rounding may leave the goal beyond all of them: the last with weight then
      constexpr int P = kVfCtas * kVfWarps / 32;  // ranges of a lane
      double mine[P], before = 0.0;
#pragma unroll
      for (int k = 0; k < P; ++k) mine[k] = (&sums[0][0])[P * lane + k], before += mine[k];
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
        for (int blk = 0; blk < blocks && token < 0; ++blk) {
          if (blocks > 1 || !any) {
            weights(blk);
            if (any) left(blk);
          }
          // sums of 32 consecutive values; the group and the value that pass the goal
#pragma unroll
          for (int k = 0; k < K; ++k) {
            const double s = warp_sum(w[k]);
            if (token < 0 && s > 0.0) {
              const int i = w0 + blk * 32 * K + 32 * k;
              const unsigned some = __ballot_sync(0xffffffffu, w[k] > 0.0);
              token_last = i + 31 - __clz(some);
              if (base + s > goal) {
                double v = w[k];
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                  const double u = __shfl_up_sync(0xffffffffu, v, o);
                  if (lane >= o) v += u;
                }
                const unsigned over = __ballot_sync(0xffffffffu, w[k] > 0.0 && base + v > goal);
                token = over ? i + __ffs(over) - 1 : token_last;
              }
              base += s;
            }
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

cudaError_t launch_verify(const VerifyArgs& a, int n_seqs, bool bf16, cudaStream_t st) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)n_seqs * kVfCtas);
  cfg.blockDim = dim3(kVfThreads);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (a.greedy)
    return bf16 ? cudaLaunchKernelEx(&cfg, verify_kernel<__nv_bfloat16, true>, a)
                : cudaLaunchKernelEx(&cfg, verify_kernel<float, true>, a);
  return bf16 ? cudaLaunchKernelEx(&cfg, verify_kernel<__nv_bfloat16, false>, a)
              : cudaLaunchKernelEx(&cfg, verify_kernel<float, false>, a);
}

int verify_launch(const draco_verify_args& v, cudaStream_t st, char* msg, size_t ml) {
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
  a.greedy = v.temperature == 0.f;
  a.inv_t = a.greedy ? 1.0 : 1.0 / (double)v.temperature;
  a.inv_t_log2 = (float)(a.inv_t * 1.4426950408889634);
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
