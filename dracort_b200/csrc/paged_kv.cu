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
// Both are bound by bytes, and short of that by latency: position -> block table
// -> row is a chain of loads.  A block walks a run of tokens: it looks all their
// pages up first, then its groups (the threads of a row, in one warp) take U
// rows of a token at a time with the next rows' loads already in flight.  A
// thread takes 8 values of a row's lower half and the 8 that rotate with them
// (append), or groups of 16 output bytes (read): 16-byte accesses that lie next
// to the neighbour's, and as many rows in a block as make whole waves.  A Q8_0
// block's maximum goes through shuffles.
//
// Measured: 8.4k prompt tokens (bf16, 32 query and 8 key/value heads of 128) to
// Q8_0 and back as fp32 56 us (5.1 TB/s); 20011 rows of 8 heads read from Q8_0
// as bf16 23 us (5.4 TB/s); one token of 32 heads written and read 4.8 us.
#include <algorithm>
#include <cstdio>

#include "internal.h"
#include "paged.cuh"

namespace draco {

constexpr int kKvThreads = 256;
constexpr int kKvTokens = 512;  // tokens whose pages a block looks up at most

template <int HD>
struct KvShape {
  static constexpr int kLanes = HD / 16;              // threads of one row
  static constexpr int kPerWarp = 32 / kLanes;        // rows of a warp (HD 96: five, two lanes idle)
  static constexpr int kRows = kKvThreads / 32 * kPerWarp;
};

// The groups of a call in one sequence: token by token, group g of a token's
// `step` takes its rows g, g + step, g + 2 step, ... (U of them).  A block takes
// the `span` groups from blockIdx.x * span on, kRows at a time.
struct KvWalk {
  int n, rows, step, span;
  unsigned total;
};
struct KvItem {
  int token, row;
  bool on;
};
template <int HD>
__device__ __forceinline__ KvItem kv_item(const KvWalk& w, int k) {  // step k of the block
  using S = KvShape<HD>;
  const int lane = threadIdx.x & 31, at = k * S::kRows + (threadIdx.x >> 5) * S::kPerWarp + lane / S::kLanes;
  const unsigned idx = blockIdx.x * (unsigned)w.span + at;
  KvItem it;
  it.on = lane / S::kLanes < S::kPerWarp && at < w.span && idx < w.total;
  it.token = it.on ? (int)(idx / (unsigned)w.step) : (int)(blockIdx.x * (unsigned)w.span / (unsigned)w.step);
  it.row = (int)(idx % (unsigned)w.step);
  return it;
}
// pages and positions of the block's tokens (page -1: outside); returns the first token
__device__ __forceinline__ int kv_lookup(const PagedView& c, const KvWalk& w, const int* seq, const int* pos,
                                         int64_t max_positions, int* s_page, int* s_pos) {
  const unsigned g0 = blockIdx.x * (unsigned)w.span, g1 = min(g0 + (unsigned)w.span, w.total);
  const int t0 = (int)(g0 / (unsigned)w.step), t1 = (int)((g1 - 1) / (unsigned)w.step);
  for (int t = t0 + threadIdx.x; t <= t1; t += kKvThreads) {
    const int p = pos[t], s = seq[t];
    s_pos[t - t0] = p;
    s_page[t - t0] = s >= 0 && s < c.n_seqs && p >= 0 && p < max_positions ? page_of(c, s, p) : -1;
  }
  __syncthreads();
  return t0;
}

__device__ __forceinline__ float max_nan2(float a, float b) {  // keeps a NaN
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// largest of the values m[2] (lower chunk, upper chunk) over the four chunks of
// each chunk's Q8_0 block; a row's lanes are l0 .. l0 + kLanes - 1
template <int HD>
__device__ __forceinline__ void block_max(float (&m)[2], int lane, int l0) {
  constexpr int L = HD / 16;
  if constexpr (L % 4 == 0) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      m[h] = max_nan2(m[h], __shfl_xor_sync(0xffffffffu, m[h], 1));
      m[h] = max_nan2(m[h], __shfl_xor_sync(0xffffffffu, m[h], 2));
    }
  } else {
    float r[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int blk = (lane - l0 + h * L) / 4;
      r[h] = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int chunk = 4 * blk + e;
        const float a = __shfl_sync(0xffffffffu, m[0], (l0 + chunk % L) & 31);
        const float b = __shfl_sync(0xffffffffu, m[1], (l0 + chunk % L) & 31);
        r[h] = max_nan2(r[h], chunk < L ? a : b);
      }
    }
    m[0] = r[0], m[1] = r[1];
  }
}

// a thread's 16 values of a row as loaded: 8 of each half
template <typename T>
struct KvRaw {
  uint4 w[sizeof(T) == 4 ? 4 : 2];
};
template <typename T>
__device__ __forceinline__ void unpack_half(const KvRaw<T>& r, int h, float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    const uint4 a = r.w[2 * h], b = r.w[2 * h + 1];
    x[0] = __uint_as_float(a.x), x[1] = __uint_as_float(a.y), x[2] = __uint_as_float(a.z), x[3] = __uint_as_float(a.w);
    x[4] = __uint_as_float(b.x), x[5] = __uint_as_float(b.y), x[6] = __uint_as_float(b.z), x[7] = __uint_as_float(b.w);
  } else {
    const uint4 a = r.w[h];
    x[0] = bf16lo(a.x), x[1] = bf16hi(a.x), x[2] = bf16lo(a.y), x[3] = bf16hi(a.y);
    x[4] = bf16lo(a.z), x[5] = bf16hi(a.z), x[6] = bf16lo(a.w), x[7] = bf16hi(a.w);
  }
}

struct KvAppend {
  const void *q, *k, *v;
  void* q_out;
  int64_t ldq, ldk, ldv, ldqo;
  const float *cos_t, *sin_t;
  int64_t max_positions;
  const int *seq, *pos;
  int heads;
};

template <typename T, int HD, bool Q8, int U>
__global__ void __launch_bounds__(kKvThreads) kv_append_kernel(const PagedView c, const KvAppend a, const KvWalk wk) {
  using S = KvShape<HD>;
  __shared__ int s_page[kKvTokens], s_pos[kKvTokens];
  grid_dependency_wait();
  grid_launch_dependents();
  const int lane32 = threadIdx.x & 31, lane = lane32 % S::kLanes;
  const int heads = a.heads, kend = heads + c.kv_heads;
  const int t0 = kv_lookup(c, wk, a.seq, a.pos, a.cos_t ? a.max_positions : 0x7FFFFFFFFFFFFFFFll, s_page, s_pos);
  KvRaw<T> raw[U];
  auto fetch = [&](const KvItem& it) {
    const int64_t i = it.token;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = it.row + u * wk.step;
      if (!it.on || r >= wk.rows) continue;
      const T* src = r < heads  ? static_cast<const T*>(a.q) + i * a.ldq + (int64_t)r * HD
                     : r < kend ? static_cast<const T*>(a.k) + i * a.ldk + (int64_t)(r - heads) * HD
                                : static_cast<const T*>(a.v) + i * a.ldv + (int64_t)(r - kend) * HD;
      constexpr int N = sizeof(T) == 4 ? 2 : 1;  // 16-byte words of 8 values
      const uint4* lo = reinterpret_cast<const uint4*>(src + 8 * lane);
      const uint4* hi = reinterpret_cast<const uint4*>(src + HD / 2 + 8 * lane);
#pragma unroll
      for (int e = 0; e < N; ++e) raw[u].w[e] = lo[e], raw[u].w[N + e] = hi[e];
    }
  };
  const int steps = (wk.span + S::kRows - 1) / S::kRows;
  KvItem it = kv_item<HD>(wk, 0);
  fetch(it);
#pragma unroll 1
  for (int st = 0; st < steps; ++st) {
    const int64_t i = it.token;
    const int p = s_pos[it.token - t0], page = it.on ? s_page[it.token - t0] : -1;
    const int off = p & ((1 << c.page_shift) - 1);
    const bool turn = a.cos_t != nullptr && p >= 0 && p < a.max_positions;
    float cs[8], sn[8];
    if (turn) {
      load8(a.cos_t + (int64_t)p * (HD / 2) + 8 * lane, cs);
      load8(a.sin_t + (int64_t)p * (HD / 2) + 8 * lane, sn);
    }
    KvRaw<T> now[U];
#pragma unroll
    for (int u = 0; u < U; ++u) now[u] = raw[u];
    const KvItem next = kv_item<HD>(wk, st + 1);
    if (st + 1 < steps) fetch(next);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = it.row + u * wk.step;
      const bool row = it.on && r < wk.rows;
      float x[2][8];
      unpack_half<T>(now[u], 0, x[0]);
      unpack_half<T>(now[u], 1, x[1]);
      if (turn && r < kend) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float y = x[0][j], z = x[1][j];
          x[0][j] = __fsub_rn(__fmul_rn(y, cs[j]), __fmul_rn(z, sn[j]));
          x[1][j] = __fadd_rn(__fmul_rn(z, cs[j]), __fmul_rn(y, sn[j]));
        }
      }
      if (row && r < heads) {
        T* dst = static_cast<T*>(a.q_out) + i * a.ldqo + (int64_t)r * HD;
        store8(dst + 8 * lane, x[0]);
        store8(dst + HD / 2 + 8 * lane, x[1]);
      }
      const bool keep = row && r >= heads && page >= 0;
      uint8_t* blk = nullptr;
      if (keep)
        blk = (r < kend ? c.k : c.v) + ((int64_t)page * c.kv_heads + (r < kend ? r - heads : r - kend)) * c.block_bytes;
      if constexpr (!Q8) {
        if (keep) {
          __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(blk) + (int64_t)off * HD;
          store8(dst + 8 * lane, x[0]);
          store8(dst + HD / 2 + 8 * lane, x[1]);
        }
      } else if (__any_sync(0xffffffffu, keep)) {
        float m[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          m[h] = fabsf(x[h][0]);
#pragma unroll
          for (int j = 1; j < 8; ++j) m[h] = max_nan2(m[h], fabsf(x[h][j]));
        }
        block_max<HD>(m, lane32, lane32 - lane);
        if (keep) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int chunk = lane + h * S::kLanes;
            const bool bad = m[h] != m[h];  // a NaN makes its whole block NaN (scale NaN, quants 0)
            if (m[h] > kKvLimit) {
              m[h] = kKvLimit;
#pragma unroll
              for (int j = 0; j < 8; ++j) x[h][j] = fminf(fmaxf(x[h][j], -kKvLimit), kKvLimit);
            }
            const float d = bad ? m[h] : __fdiv_rn(fmaxf(m[h], 1e-12f), 127.f);
            // rint(x / d) with the quotient rounded to fp32: by Markstein's theorem
            // q + (x - q d) y is the rounded quotient when y is the rounded 1 / d and
            // q = x y (values from the block's largest down to 0: nothing underflows
            // that matters); then 1.5 * 2^23 leaves the nearest integer in the low bits
            const float y = 1.f / d;
            uint32_t b[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float z = x[h][j] * y;
              b[j] = __float_as_uint(fmaf(fmaf(-z, d, x[h][j]), y, z) + 12582912.f);
            }
            uint32_t w0 = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
            uint32_t w1 = __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410);
            if (bad) w0 = w1 = 0u;
            *reinterpret_cast<uint2*>(blk + (int64_t)off * HD + 8 * chunk) = make_uint2(w0, w1);
            if ((chunk & 3) == 0)
              reinterpret_cast<__half*>(blk + ((int64_t)HD << c.page_shift))[off * (HD / 32) + chunk / 4] =
                  __float2half_rn(d);
          }
        }
      }
    }
    it = next;
  }
}

// rows of the given positions, keys to k_out and values to v_out
// [n, kv_heads, head_dim]; a thread takes 16 values of each of its rows, in groups
// whose 16-byte stores touch those of the next lane
template <typename T, int HD, bool Q8, int U>
__global__ void __launch_bounds__(kKvThreads) kv_read_kernel(const PagedView c, const int* __restrict__ seq,
                                                             const int* __restrict__ pos, T* k_out, T* v_out,
                                                             int64_t ldk, int64_t ldv, const KvWalk wk) {
  using S = KvShape<HD>;
  __shared__ int s_page[kKvTokens], s_pos[kKvTokens];
  grid_dependency_wait();
  grid_launch_dependents();
  const int lane = (threadIdx.x & 31) % S::kLanes;
  const int t0 = kv_lookup(c, wk, seq, pos, 0x7FFFFFFFFFFFFFFFll, s_page, s_pos);
  constexpr int V = 16 / (int)sizeof(T), G = 16 / V, W = Q8 ? V / 4 : V / 2;  // values and words of a group, groups
  uint32_t w[U][G][W], d[U][G];
  auto fetch = [&](const KvItem& it) {
    const int page = it.on ? s_page[it.token - t0] : -1, off = s_pos[it.token - t0] & ((1 << c.page_shift) - 1);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = it.row + u * wk.step, h = r < c.kv_heads ? r : r - c.kv_heads;
      const uint8_t* blk = (r < c.kv_heads ? c.k : c.v) + ((int64_t)max(page, 0) * c.kv_heads + h) * c.block_bytes;
      const bool have = page >= 0 && r < wk.rows;  // a row outside the cache reads as zeros
#pragma unroll
      for (int e = 0; e < G; ++e) {
        const int at = V * (lane + e * S::kLanes);
        const uint32_t* p = reinterpret_cast<const uint32_t*>(blk + ((int64_t)off * HD + at) * (Q8 ? 1 : 2));
#pragma unroll
        for (int j = 0; j < W; ++j) w[u][e][j] = 0u;
        d[u][e] = 0u;
        if (have) {
          if constexpr (W == 4) {
            const uint4 x = __ldg(reinterpret_cast<const uint4*>(p));
            w[u][e][0] = x.x, w[u][e][1] = x.y, w[u][e][2] = x.z, w[u][e][3] = x.w;
          } else if constexpr (W == 2) {
            const uint2 x = __ldg(reinterpret_cast<const uint2*>(p));
            w[u][e][0] = x.x, w[u][e][1] = x.y;
          } else {
            w[u][e][0] = __ldg(p);
          }
          if constexpr (Q8)
            d[u][e] = __ldg(reinterpret_cast<const uint16_t*>(blk + ((int64_t)HD << c.page_shift)) + off * (HD / 32) + at / 32);
        }
      }
    }
  };
  const int steps = (wk.span + S::kRows - 1) / S::kRows;
  KvItem it = kv_item<HD>(wk, 0);
  fetch(it);
#pragma unroll 1
  for (int st = 0; st < steps; ++st) {
    const int64_t i = it.token;
    uint32_t now[U][G][W];
    float sc[U][G];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < G; ++e) {
#pragma unroll
        for (int j = 0; j < W; ++j) now[u][e][j] = w[u][e][j];
        sc[u][e] = f16_bits_to_f32(d[u][e]);
      }
    const KvItem next = kv_item<HD>(wk, st + 1);
    if (st + 1 < steps) fetch(next);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = it.row + u * wk.step, h = r < c.kv_heads ? r : r - c.kv_heads;
      if (!it.on || r >= wk.rows) continue;
      T* dst = (r < c.kv_heads ? k_out + i * ldk : v_out + i * ldv) + (int64_t)h * HD + V * lane;
#pragma unroll
      for (int e = 0; e < G; ++e) {
        float x[V];
        if constexpr (Q8) {
#pragma unroll
          for (int j = 0; j < V; ++j)  // 2^23 + (quant + 128), exact
            x[j] = sc[u][e] * (__uint_as_float(__byte_perm(now[u][e][j >> 2] ^ 0x80808080u, 0x4B000000u,
                                                           0x7440u | (j & 3))) - 8388736.f);
        } else {
#pragma unroll
          for (int j = 0; j < V; j += 2) x[j] = bf16lo(now[u][e][j / 2]), x[j + 1] = bf16hi(now[u][e][j / 2]);
        }
        uint4 o;
        if constexpr (sizeof(T) == 4)
          o = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
        else if constexpr (!Q8)
          o = make_uint4(now[u][e][0], now[u][e][1], now[u][e][2], now[u][e][3]);
        else
          o = make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
        *reinterpret_cast<uint4*>(dst + V * e * S::kLanes) = o;
      }
    }
    it = next;
  }
}

// CTAs of a kernel that an SM holds
template <auto Kernel>
static int kv_ctas() {
  static int ctas_of[64] = {0};
  int dev = 0, ctas = 0;
  cudaGetDevice(&dev);
  if (dev < 64) ctas = ctas_of[dev];
  if (ctas == 0) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&ctas, Kernel, kKvThreads, 0) != cudaSuccess) ctas = 1;
    ctas = std::max(ctas, 1);
    if (dev < 64) ctas_of[dev] = ctas;
  }
  return ctas;
}

// U rows of a thread at a time: one while the call does not fill the GPU
// (latency counts), else `most`.
static int kv_unroll(int n, int rows, int lanes, int most) {
  return (int64_t)n * rows * lanes > 2048LL * device_sm_count() ? most : 1;
}
// A block's span: up to 16 steps and kKvTokens tokens, as many as make whole
// waves of blocks (20000 prompt tokens to Q8_0 and back: 140 us with 16 steps
// each, 128 in whole waves; 13500: 114 and 89).
static KvWalk kv_walk(int n, int rows, int per_step, int unroll, int ctas) {
  KvWalk w;
  w.n = n;
  w.rows = rows;
  w.step = (rows + unroll - 1) / unroll;
  const int64_t total = (int64_t)n * w.step;
  w.total = (unsigned)total;
  const int64_t all = (total + per_step - 1) / per_step, slots = (int64_t)ctas * device_sm_count();
  int64_t most = 16;
  while (most > 1 && most * per_step / w.step + 2 > kKvTokens) most /= 2;
  const int64_t waves = std::max<int64_t>(1, (all + most * slots - 1) / (most * slots));
  w.span = (int)(std::max<int64_t>(1, (all + waves * slots - 1) / (waves * slots)) * per_step);
  return w;
}
static_assert(kKvThreads / 2 + 2 <= kKvTokens, "one step's tokens");

template <typename Kernel, typename... Args>
static cudaError_t launch_walk(Kernel kernel, const KvWalk& w, cudaStream_t st, Args... args) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((w.total + (unsigned)w.span - 1) / (unsigned)w.span);
  cfg.blockDim = dim3(kKvThreads);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args..., w);
}

template <typename T, int HD, bool Q8>
static cudaError_t append_t(const PagedView& c, const draco_kv_append_args& a, cudaStream_t st) {
  using S = KvShape<HD>;
  constexpr int kMost = sizeof(T) == 4 ? 2 : 4;  // 32 registers of loads in flight (bf16, 8.4k tokens to Q8_0 and back: one row 65 us, two 64, four 56)
  const int rows = a.heads + 2 * c.kv_heads, u = kv_unroll(a.n, rows, S::kLanes, kMost);
  const KvWalk w = kv_walk(a.n, rows, S::kRows, u,
                           u == 1 ? kv_ctas<kv_append_kernel<T, HD, Q8, 1>>() : kv_ctas<kv_append_kernel<T, HD, Q8, kMost>>());
  const KvAppend k = {a.q,   a.k,    a.v,         a.q_out,     a.ldq,           a.ldk, a.ldv,
                      a.ldqo, a.cos_table, a.sin_table, a.max_positions, a.seq, a.pos, a.heads};
  return launch_walk(u == 1 ? kv_append_kernel<T, HD, Q8, 1> : kv_append_kernel<T, HD, Q8, kMost>, w, st, c, k);
}

template <typename T, int HD, bool Q8>
static cudaError_t read_t(const PagedView& c, const int* seq, const int* pos, int n, void* k_out, void* v_out,
                          int64_t ldk, int64_t ldv, cudaStream_t st) {
  using S = KvShape<HD>;
  constexpr int kMost = 2;  // (20011 rows of Q8_0: one 23.9 us, two 23.0, four 23.0 with half the warps)
  const int rows = 2 * c.kv_heads, u = kv_unroll(n, rows, S::kLanes, kMost);
  const KvWalk w = kv_walk(n, rows, S::kRows, u,
                           u == 1 ? kv_ctas<kv_read_kernel<T, HD, Q8, 1>>() : kv_ctas<kv_read_kernel<T, HD, Q8, kMost>>());
  return launch_walk(u == 1 ? kv_read_kernel<T, HD, Q8, 1> : kv_read_kernel<T, HD, Q8, kMost>, w, st, c, seq, pos,
                     (T*)k_out, (T*)v_out, ldk, ldv);
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
