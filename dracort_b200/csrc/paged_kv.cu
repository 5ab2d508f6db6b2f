// paged_kv.cu — writing new keys and values into the paged cache and reading
// cached rows back (draco_kv_append, draco_kv_read).
//
// Append: per token, rotate-half RoPE of the query heads and the key heads
// (x1' = x1 c - x2 s, x2' = x2 c + x1 s, every product and sum rounded once to
// fp32 as draco/runtime/cpu/ops.py:86-95 rounds them), then the key and value
// rows rounded to the cache's type: bf16 (nearest even), or Q8_0 blocks of 32
// (d = max|x| / 127 in fp32, q = rint(x / d), d stored as fp16: the encoder's
// rule of format/quantize.py).  Read: value = d * q, exact in fp32, rounded
// once when the output is bf16.
//
// Both are bound by bytes.  A thread takes 8 values of a row's lower half and
// the 8 that rotate with them, i.e. two 16-byte accesses per operand, and
// keeps the cos / sin values of its 8 angles in registers over `rows` rows of
// the token (they are read from the L2 otherwise as often as the data).
#include <cstdio>

#include "internal.h"
#include "paged.cuh"

namespace draco {

constexpr int kKvThreads = 256;

template <int HD>
struct KvShape {
  static constexpr int kLanes = HD / 16;              // threads of one row
  static constexpr int kRows = kKvThreads / kLanes;   // rows of a block at a time
  static constexpr int kChunks = HD / 8;
};

template <typename T, int HD, bool Q8>
__global__ void __launch_bounds__(kKvThreads) kv_append_kernel(
    PagedView c, const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v, T* q_out, int64_t ldq,
    int64_t ldk, int64_t ldv, int64_t ldqo, const float* __restrict__ cos_t, const float* __restrict__ sin_t,
    int64_t max_positions, const int* __restrict__ seq, const int* __restrict__ pos, int heads, int reps) {
  using S = KvShape<HD>;
  // largest magnitude of every 8 values of the rows in flight (a Q8_0 block is four of them)
  __shared__ __align__(16) float amax[Q8 ? S::kRows : 1][S::kChunks];
  grid_dependency_wait();
  grid_launch_dependents();
  const int i = blockIdx.x;
  const int slot = threadIdx.x / S::kLanes, lane = threadIdx.x % S::kLanes;
  const int total = heads + 2 * c.kv_heads;
  const bool active = slot < S::kRows;
  const int p = pos[i], s = seq[i];
  const bool turn = cos_t != nullptr && p >= 0 && p < max_positions;
  int page = -1;
  if (s >= 0 && s < c.n_seqs && p >= 0 && (turn || cos_t == nullptr)) page = page_of(c, s, p);
  const int off = p & ((1 << c.page_shift) - 1);
  float cs[8], sn[8];
  if (turn && active) {
    load8(cos_t + (int64_t)p * (HD / 2) + 8 * lane, cs);
    load8(sin_t + (int64_t)p * (HD / 2) + 8 * lane, sn);
  }
  for (int u = 0; u < reps; ++u) {
    const int r = (blockIdx.y * reps + u) * S::kRows + slot;  // q heads, then k heads, then v heads
    const bool row = active && r < total;
    float x[2][8];
    if (row) {
      const T* src;
      if (r < heads)
        src = q == nullptr ? nullptr : q + (int64_t)i * ldq + (int64_t)r * HD;
      else if (r < heads + c.kv_heads)
        src = k + (int64_t)i * ldk + (int64_t)(r - heads) * HD;
      else
        src = v + (int64_t)i * ldv + (int64_t)(r - heads - c.kv_heads) * HD;
      if (src != nullptr) {
        load8(src + 8 * lane, x[0]);
        load8(src + HD / 2 + 8 * lane, x[1]);
      }
      if (turn && r < heads + c.kv_heads) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float a = x[0][j], b = x[1][j];
          x[0][j] = __fsub_rn(__fmul_rn(a, cs[j]), __fmul_rn(b, sn[j]));
          x[1][j] = __fadd_rn(__fmul_rn(b, cs[j]), __fmul_rn(a, sn[j]));
        }
      }
      if (r < heads && q_out != nullptr) {
        T* dst = q_out + (int64_t)i * ldqo + (int64_t)r * HD;
        store8(dst + 8 * lane, x[0]);
        store8(dst + HD / 2 + 8 * lane, x[1]);
      }
    }
    const bool keep = row && r >= heads && page >= 0;
    const int kvr = r - heads;
    uint8_t* blk = nullptr;
    if (keep)
      blk = (kvr < c.kv_heads ? c.k : c.v) + ((int64_t)page * c.kv_heads + kvr % c.kv_heads) * c.block_bytes;
    if constexpr (!Q8) {
      if (keep) {
        __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(blk) + (int64_t)off * HD;
        store8(dst + 8 * lane, x[0]);
        store8(dst + HD / 2 + 8 * lane, x[1]);
      }
    } else {
      if (keep) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float m = 0.f;
          bool bad = false;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            bad |= x[h][j] != x[h][j];
            x[h][j] = fminf(fmaxf(x[h][j], -kKvLimit), kKvLimit);
            m = fmaxf(m, fabsf(x[h][j]));
          }
          // a NaN makes its whole block NaN (scale NaN, quants 0)
          amax[slot][lane + h * S::kLanes] = bad ? __int_as_float(0x7FC00000) : m;
        }
      }
      __syncthreads();
      if (keep) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int chunk = lane + h * S::kLanes;
          const float4 a = *reinterpret_cast<const float4*>(&amax[slot][chunk & ~3]);
          const float m = fmaxf(fmaxf(a.x, a.y), fmaxf(a.z, a.w));
          const bool bad = a.x != a.x || a.y != a.y || a.z != a.z || a.w != a.w;
          const float d = bad ? __int_as_float(0x7FC00000) : __fdiv_rn(fmaxf(m, 1e-12f), 127.f);
          uint32_t w[2] = {0u, 0u};
          if (!bad) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const int n = max(-127, min(127, __float2int_rn(__fdiv_rn(x[h][j], d))));
              w[j >> 2] |= (uint32_t)(n & 0xFF) << (8 * (j & 3));
            }
          }
          *reinterpret_cast<uint2*>(blk + (int64_t)off * HD + 8 * chunk) = make_uint2(w[0], w[1]);
          if ((chunk & 3) == 0)
            reinterpret_cast<__half*>(blk + ((int64_t)HD << c.page_shift))[off * (HD / 32) + chunk / 4] =
                __float2half_rn(d);
        }
      }
      __syncthreads();  // amax is written again for the next rows
    }
  }
}

// rows of the given positions, keys to k_out and values to v_out
// [n, kv_heads, head_dim]; a thread takes 16 values
template <typename T, int HD, bool Q8>
__global__ void __launch_bounds__(kKvThreads) kv_read_kernel(PagedView c, const int* __restrict__ seq,
                                                             const int* __restrict__ pos, T* k_out, T* v_out,
                                                             int64_t ldk, int64_t ldv, int reps) {
  using S = KvShape<HD>;
  grid_dependency_wait();
  grid_launch_dependents();
  const int i = blockIdx.x;
  const int slot = threadIdx.x / S::kLanes, lane = threadIdx.x % S::kLanes;
  if (slot >= S::kRows) return;
  const int p = pos[i], s = seq[i];
  const int page = s >= 0 && s < c.n_seqs && p >= 0 ? page_of(c, s, p) : -1;
  const int off = p & ((1 << c.page_shift) - 1);
  for (int u = 0; u < reps; ++u) {
    const int r = (blockIdx.y * reps + u) * S::kRows + slot;
    if (r >= 2 * c.kv_heads) return;
    const bool is_k = r < c.kv_heads;
    const int h = is_k ? r : r - c.kv_heads;
    T* dst = (is_k ? k_out + (int64_t)i * ldk : v_out + (int64_t)i * ldv) + (int64_t)h * HD + 16 * lane;
    float x[2][8] = {};
    if (page >= 0) {  // a row outside the cache reads as zeros
      const uint8_t* blk = (is_k ? c.k : c.v) + ((int64_t)page * c.kv_heads + h) * c.block_bytes;
      if constexpr (Q8) {
        const uint4 w = __ldg(reinterpret_cast<const uint4*>(blk + (int64_t)off * HD + 16 * lane));
        const float d = __half2float(reinterpret_cast<const __half*>(
            blk + ((int64_t)HD << c.page_shift))[off * (HD / 32) + lane / 2]);
        const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int j = 0; j < 16; ++j)
          x[j >> 3][j & 7] = d * (float)(int8_t)((ws[j >> 2] >> (8 * (j & 3))) & 0xFF);
      } else {
        const __nv_bfloat16* src = reinterpret_cast<const __nv_bfloat16*>(blk) + (int64_t)off * HD + 16 * lane;
        load8(src, x[0]);
        load8(src + 8, x[1]);
      }
    }
    store8(dst, x[0]);
    store8(dst + 8, x[1]);
  }
}

// Rows of one token per block and repetitions: enough blocks to fill the GPU
// come first; then up to 4 rows per thread.
static void rows_grid(int n, int rows, int per_block, int* reps, unsigned* gy) {
  const int need = (rows + per_block - 1) / per_block;
  const int64_t want = 16LL * device_sm_count();  // 8 blocks of 256 threads fit an SM
  int u = 1;
  while (u < 4 && u < need && (int64_t)n * ((need + 2 * u - 1) / (2 * u)) >= want) u *= 2;
  *reps = u;
  *gy = (unsigned)((need + u - 1) / u);
}

template <typename T, int HD, bool Q8>
static cudaError_t append_t(const PagedView& c, const draco_kv_append_args& a, cudaStream_t st) {
  int reps;
  unsigned gy;
  rows_grid(a.n, a.heads + 2 * c.kv_heads, KvShape<HD>::kRows, &reps, &gy);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.n, gy);
  cfg.blockDim = dim3(kKvThreads);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kv_append_kernel<T, HD, Q8>, c, (const T*)a.q, (const T*)a.k, (const T*)a.v,
                            (T*)a.q_out, a.ldq, a.ldk, a.ldv, a.ldqo, a.cos_table, a.sin_table, a.max_positions,
                            a.seq, a.pos, a.heads, reps);
}

template <typename T, int HD, bool Q8>
static cudaError_t read_t(const PagedView& c, const int* seq, const int* pos, int n, void* k_out, void* v_out,
                          int64_t ldk, int64_t ldv, cudaStream_t st) {
  int reps;
  unsigned gy;
  rows_grid(n, 2 * c.kv_heads, KvShape<HD>::kRows, &reps, &gy);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(n, gy);
  cfg.blockDim = dim3(kKvThreads);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kv_read_kernel<T, HD, Q8>, c, seq, pos, (T*)k_out, (T*)v_out, ldk, ldv, reps);
}

#define DRACO_HD_SWITCH(hd, CALL) \
  switch (hd) {                   \
    case 32: return CALL(32);     \
    case 64: return CALL(64);     \
    case 96: return CALL(96);     \
    case 128: return CALL(128);   \
    default: return CALL(256);    \
  }

template <typename T, bool Q8>
static cudaError_t append_hd(int hd, const PagedView& c, const draco_kv_append_args& a, cudaStream_t st) {
#define CALL(H) append_t<T, H, Q8>(c, a, st)
  DRACO_HD_SWITCH(hd, CALL)
#undef CALL
}
template <typename T, bool Q8>
static cudaError_t read_hd(int hd, const PagedView& c, const int* seq, const int* pos, int n, void* ko, void* vo,
                           int64_t ldk, int64_t ldv, cudaStream_t st) {
#define CALL(H) read_t<T, H, Q8>(c, seq, pos, n, ko, vo, ldk, ldv, st)
  DRACO_HD_SWITCH(hd, CALL)
#undef CALL
}

cudaError_t launch_kv_append(const PagedView& c, int hd, int dtype, const draco_kv_append_args& a, cudaStream_t st) {
  const bool q8 = c.type == DRACO_KV_Q8_0;
  if (dtype == DRACO_DTYPE_F32) return q8 ? append_hd<float, true>(hd, c, a, st) : append_hd<float, false>(hd, c, a, st);
  return q8 ? append_hd<__nv_bfloat16, true>(hd, c, a, st) : append_hd<__nv_bfloat16, false>(hd, c, a, st);
}

cudaError_t launch_kv_read(const PagedView& c, int hd, int dtype, const int* seq, const int* pos, int n, void* ko,
                           void* vo, int64_t ldk, int64_t ldv, cudaStream_t st) {
  const bool q8 = c.type == DRACO_KV_Q8_0;
  if (dtype == DRACO_DTYPE_F32)
    return q8 ? read_hd<float, true>(hd, c, seq, pos, n, ko, vo, ldk, ldv, st)
              : read_hd<float, false>(hd, c, seq, pos, n, ko, vo, ldk, ldv, st);
  return q8 ? read_hd<__nv_bfloat16, true>(hd, c, seq, pos, n, ko, vo, ldk, ldv, st)
            : read_hd<__nv_bfloat16, false>(hd, c, seq, pos, n, ko, vo, ldk, ldv, st);
}

}  // namespace draco
