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

// running maximum, sum of exp2((x - m) c) and first index of the maximum
struct RowStat {
  float m, s;
  int i;
};
__device__ __forceinline__ float weight32(float x, float m, float c) {
  return x == m ? 1.f : exp2f((x - m) * c);  // (inf - inf) is not taken
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
__device__ __forceinline__ double weight64(float x, float m, double inv_t) {
  return x == m ? 1.0 : x == -INFINITY ? 0.0 : exp((double)(x - m) * inv_t);
}

template <typename T>
__global__ void __cluster_dims__(kVfCtas, 1, 1) __launch_bounds__(kVfThreads) verify_kernel(const VerifyArgs a) {
  cg::cluster_group cluster = cg::this_cluster();
  __shared__ RowStat wstat[kVfRows][kVfWarps];
  __shared__ RowStat stat[kVfRows];      // this CTA's range
  __shared__ RowStat full[kVfRows];      // the whole row
  __shared__ double wsum[2][kVfWarps];   // weights of the warps' ranges: of p, and of what is drawn from
  __shared__ double csum[2];
  grid_dependency_wait();
  grid_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = (int)cluster.block_rank(), b = blockIdx.x / kVfCtas;
  const T* logits = static_cast<const T*>(a.logits);
  const int begin = min(max(a.row_start[b], 0), a.n);
  const int rows = max(0, min(max(a.row_start[b + 1], 0), a.n) - begin);
  // ranges: CTA, then warp, in vocabulary order, in units of 8 values
  const int units = (a.vocab + 7) / 8, per_cta = (units + kVfCtas - 1) / kVfCtas;
  const int per_warp = (per_cta + kVfWarps - 1) / kVfWarps;
  const int w0 = min(a.vocab, 8 * min((rank + 1) * per_cta, rank * per_cta + warp * per_warp));
  const int w1 = min(a.vocab, 8 * min((rank + 1) * per_cta, rank * per_cta + (warp + 1) * per_warp));

  int count = 0;        // drafts taken
  bool decided = rows == 0;
  RowStat at = {-INFINITY, 0.f, 0};  // statistics of the row that the next token comes from
  for (int r0 = 0; r0 < rows && !decided; r0 += kVfRows) {
    const int nr = min(kVfRows, rows - r0);
    for (int r = 0; r < nr; ++r) {
      const T* row = logits + (int64_t)(begin + r0 + r) * a.ld_logits;
      RowStat st = {-INFINITY, 0.f, 0x7FFFFFFF};
      constexpr int V = 16 / (int)sizeof(T);
      // from the first 16-byte boundary on in 16-byte loads
      const int head = min(w1, w0 + (int)(((16 - (reinterpret_cast<uintptr_t>(row + w0) & 15)) & 15) / sizeof(T)));
      const int vecs = (w1 - head) / V;
      auto take = [&](float x, int i) {
        x = x == x ? x : -INFINITY;
        if (x > st.m) {
          st.s = (st.m == -INFINITY ? 0.f : st.s * weight32(st.m, x, a.inv_t_log2)) + 1.f;
          st.m = x, st.i = i;
        } else if (x != -INFINITY) {
          st.s += weight32(x, st.m, a.inv_t_log2);
        }
      };
      if (w0 + lane < head) take(logit(row + w0 + lane), w0 + lane);
      for (int v = lane; v < vecs; v += 32) {
        const int i = head + v * V;
        const uint4 w = __ldg(reinterpret_cast<const uint4*>(row + i));
        float x[V];
        if constexpr (V == 4) {
          x[0] = __uint_as_float(w.x), x[1] = __uint_as_float(w.y), x[2] = __uint_as_float(w.z),
          x[3] = __uint_as_float(w.w);
        } else {
          x[0] = bf16lo(w.x), x[1] = bf16hi(w.x), x[2] = bf16lo(w.y), x[3] = bf16hi(w.y);
          x[4] = bf16lo(w.z), x[5] = bf16hi(w.z), x[6] = bf16lo(w.w), x[7] = bf16hi(w.w);
        }
#pragma unroll
        for (int e = 0; e < V; ++e) take(x[e], i + e);
      }
      const int tail = head + vecs * V + lane;
      if (tail < w1) take(logit(row + tail), tail);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        RowStat x;
        x.m = __shfl_xor_sync(0xffffffffu, st.m, o);
        x.s = __shfl_xor_sync(0xffffffffu, st.s, o);
        x.i = __shfl_xor_sync(0xffffffffu, st.i, o);
        st = join(st, x, a.inv_t_log2);
      }
      if (lane == 0) wstat[r][warp] = st;
    }
    __syncthreads();
    if (tid < nr) {
      RowStat st = wstat[tid][0];
      for (int w = 1; w < kVfWarps; ++w) st = join(st, wstat[tid][w], a.inv_t_log2);
      stat[tid] = st;
    }
    cluster.sync();
    if (tid < nr) {
      RowStat st = *cluster.map_shared_rank(&stat[tid], 0);
      for (int c = 1; c < kVfCtas; ++c) st = join(st, *cluster.map_shared_rank(&stat[tid], c), a.inv_t_log2);
      full[tid] = st;
    }
    cluster.sync();  // also: the ranges' statistics have been read
    for (int r = 0; r < nr; ++r) {
      const RowStat st = full[r];
      at = st;
      const int rr = begin + r0 + r;
      if (r0 + r == rows - 1) {
        decided = true;
        break;
      }
      const int x = a.drafts[rr];
      bool take = false;
      if (x >= 0 && x < a.vocab && st.m > -INFINITY) {
        if (a.greedy) {
          take = x == st.i;
        } else {
          const float lx = logit(logits + (int64_t)rr * a.ld_logits + x);
          const float qx = a.probs ? a.probs[(int64_t)rr * a.ld_probs + x] : 1.f;
          const float wx = lx == -INFINITY ? 0.f : weight32(lx, st.m, a.inv_t_log2);
          take = (double)a.accept_u[rr] * qx * st.s < wx;
        }
      }
      if (!take) {
        decided = true;
        break;
      }
      ++count;
    }
    __syncthreads();  // full is written again for the next rows
  }

  int last = -1;
  if (rows > 0 && at.m > -INFINITY) {
    if (a.greedy) {
      last = at.i;
    } else {
      const int rr = begin + count;
      const bool rejected = count < rows - 1;
      const T* row = logits + (int64_t)rr * a.ld_logits;
      const int x = rejected && a.probs == nullptr ? a.drafts[rr] : -1;  // a point mass is taken out
      const float* q = rejected && a.probs != nullptr ? a.probs + (int64_t)rr * a.ld_probs : nullptr;
      // weights of p by warp, and, without q, of what is drawn from
      double sp = 0.0, sd = 0.0, z = 1.0;
      for (int i = w0 + lane; i < w1; i += 32) {
        const double w = weight64(logit(row + i), at.m, a.inv_t);
        sp += w;
        if (i != x) sd += w;
      }
      auto warp_sum = [](double v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
      };
      auto share = [&](double p, double d) {  // warps' sums to shared memory, CTAs' sums to the cluster
        p = warp_sum(p), d = warp_sum(d);
        if (lane == 0) wsum[0][warp] = p, wsum[1][warp] = d;
        __syncthreads();
        if (tid < 2) {
          double s = 0.0;
          for (int w = 0; w < kVfWarps; ++w) s += wsum[tid][w];
          csum[tid] = s;
        }
        cluster.sync();
      };
      auto total = [&](int which) {
        double s = 0.0;
        for (int c = 0; c < kVfCtas; ++c) s += *cluster.map_shared_rank(&csum[which], c);
        return s;
      };
      auto rest = [&](int i) -> double {  // what index i may still be drawn with
        const double w = weight64(logit(row + i), at.m, a.inv_t);
        if (q == nullptr) return i == x ? 0.0 : w;
        const double d = w / z - (double)q[i];
        return d > 0.0 ? d : 0.0;
      };
      share(sp, sd);
      if (q != nullptr) {
        z = total(0);
        sd = 0.0;
        for (int i = w0 + lane; i < w1; i += 32) sd += rest(i);
        cluster.sync();  // the sums have been read
        share(sp, sd);
      }
      int which = 1;
      double sum = total(1);
      if (!(sum > 0.0)) which = 0, sum = total(0);  // p <= q everywhere: p itself
      double before = 0.0;
      for (int c = 0; c < rank; ++c) before += *cluster.map_shared_rank(&csum[which], c);
      double mine = 0.0;
      for (int w = 0; w < warp; ++w) before += wsum[which][w];
      mine = wsum[which][warp];
      const double goal = (double)a.sample_u[b] * sum;
      // the first warp in order whose range passes the goal; rounding may leave
      // the goal beyond all of them: the last range with weight then
      __shared__ int found[kVfWarps], some[kVfWarps];
      if (lane == 0) found[warp] = before + mine > goal && mine > 0.0, some[warp] = mine > 0.0;
      cluster.sync();
      int owner = -1, fallback = -1;
      for (int w = lane; w < kVfCtas * kVfWarps; w += 32) {
        if (*cluster.map_shared_rank(&found[w % kVfWarps], w / kVfWarps) && owner < 0) owner = w;
        if (*cluster.map_shared_rank(&some[w % kVfWarps], w / kVfWarps)) fallback = w;
      }
      owner = owner < 0 ? 0x7FFFFFFF : owner;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        owner = min(owner, __shfl_xor_sync(0xffffffffu, owner, o));
        fallback = max(fallback, __shfl_xor_sync(0xffffffffu, fallback, o));
      }
      if (owner == 0x7FFFFFFF) owner = fallback;
      if (owner == rank * kVfWarps + warp) {
        // this warp's range in 32 contiguous pieces, then the piece itself
        auto weight = [&](int i) { return which ? rest(i) : weight64(logit(row + i), at.m, a.inv_t); };
        auto scan = [&](double v) {
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const double u = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += u;
          }
          return v;
        };
        int lo = w0, hi = w1;
        double base = before;
        while (hi - lo > 0) {
          const int piece = (hi - lo + 31) / 32;
          const int i0 = min(hi, lo + lane * piece), i1 = min(hi, i0 + piece);
          double s = 0.0;
          for (int i = i0; i < i1; ++i) s += weight(i);
          const double upto = base + scan(s);
          const unsigned over = __ballot_sync(0xffffffffu, s > 0.0 && upto > goal);
          const unsigned any = __ballot_sync(0xffffffffu, s > 0.0);
          const int k = over ? __ffs(over) - 1 : 31 - __clz(any | 1u);
          base = __shfl_sync(0xffffffffu, upto - s, k);
          lo = __shfl_sync(0xffffffffu, i0, k);
          hi = __shfl_sync(0xffffffffu, i1, k);
          if (piece == 1) break;
        }
        if (lane == 0 && count < a.max_rows) a.tokens[(int64_t)b * a.ld_tokens + count] = lo;
      }
      cluster.sync();  // nobody leaves while others read its shared memory
    }
  }
  if (rank == 0) {
    if (tid == 0) a.accepted[b] = count;
    const bool drawn = rows > 0 && at.m > -INFINITY && !a.greedy;  // its owner writes the token
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
  return bf16 ? cudaLaunchKernelEx(&cfg, verify_kernel<__nv_bfloat16>, a)
              : cudaLaunchKernelEx(&cfg, verify_kernel<float>, a);
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
