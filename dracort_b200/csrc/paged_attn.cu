// paged_attn.cu — causal attention of a sequence's newest tokens over its
// paged, possibly quantised cache, on the warp-level tensor-core MMA: decode
// steps, drafted tokens, chunks and prompts in fp32 or bf16
// (draco_attention_paged; large bf16 chunks go to paged_attn_tc.cu).
//
// Row (token i, query head) of a sequence sees keys 0..kv_len - new + i:
// out = softmax(scale q K^T) V with one pass over the keys: running maximum m
// and sum l, O rescaled when m grows (by more than 8 in the exponent's log2:
// up to there the old reference only makes the summands larger).
//
// What bounds it: few rows share a key, so bytes: every key and value is read
// once per row tile.  The query heads of a key/value head and the new tokens
// are the rows of one MMA (m16n8k16), so that a key's fragment serves all of
// them, and the keys go through 16 at a time: a group of WM warps (one row tile
// of 16 rows each) fills its own ring of 16 * WM keys per stage with
// cp.async and never waits for the other groups.  4 / WM groups of a CTA take
// the key blocks of the CTA's key range in turn and merge in shared memory;
// long ranges are split over CTAs (blockIdx.y) and merged, in split order, by
// the last CTA to arrive.
//
// Precision.  fp32 activations keep 22-24 bits: operands go into the MMAs as
// sums of 16-bit terms.
//   bf16 cache: keys and values are bf16 already.  q and P are one bf16 each
//     for bf16 activations, or three (8 + 8 + 8 bits) for fp32.
//   Q8_0 cache: d * quant has 18 bits, and fp16 takes 11 of them: one fp16 for
//     bf16 activations (relative error 2^-12, against 2^-9 of the output), or
//     two, exact, for fp32, with q and P as two fp16 (22 bits) and the
//     smallest cross product left out.  A row of q is scaled by a power of
//     two to at most 1 and P to at most 2^14, so that fp16's range does not cut
//     either.
// m, l, O and the scores are fp32.
//
// A key or value outside [0, kv_len) and a row of a page outside the cache is
// zero-filled in shared memory, never read.  A NaN or infinity in a value row
// that some rows of the tile do not see (a later token of the same chunk)
// must not reach them as 0 * NaN: such a step multiplies row by row.
#include <algorithm>
#include <cstdio>

#include "internal.h"
#include "paged_attn.cuh"

namespace draco {

constexpr int kPaThreads = 128;
constexpr float kPaLazy = 8.f;
constexpr int kPaMinSplit = 256;   // keys of a split at least (16 blocks per warp group at WM 1)

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool on) {
  const int n = on ? 16 : 0;  // 0: the 16 bytes are filled with zeros and src is not read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma_bf16_16816_acc(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool Q8>
__device__ __forceinline__ void mma_acc(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (Q8)
    mma_f16_16816_acc(d, a[0], a[1], a[2], a[3], b0, b1);
  else
    mma_bf16_16816_acc(d, a, b0, b1);
}
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t hmul2_(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2_rn(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t hsub2_(uint32_t a, uint32_t b) {
  const __half2 r = __hsub2_rn(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// a * b - c
__device__ __forceinline__ uint32_t hfms2_(uint32_t a, uint32_t b, uint32_t c) {
  const __half2 r = __hfma2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b),
                            __hneg2(*reinterpret_cast<__half2*>(&c)));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// the 16-bit terms of two fp32 values, NT of them, most significant first
template <bool Q8, int NT>
__device__ __forceinline__ void split2(float a, float b, uint32_t (&t)[NT]) {
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    if constexpr (Q8) {
      t[i] = pack_f16(a, b);
      if (i + 1 < NT) {
        const float2 f = __half22float2(*reinterpret_cast<__half2*>(&t[i]));
        a -= f.x, b -= f.y;
      }
    } else {
      t[i] = pack_bf16(a, b);
      if (i + 1 < NT) a -= bf16lo(t[i]), b -= bf16hi(t[i]);
    }
  }
}

// ---------------------------------------------------------------------------
// geometry
// ---------------------------------------------------------------------------
template <int HD, bool Q8, bool F32, int WM>
struct PaCfg {
  static constexpr int kTerms = F32 ? (Q8 ? 2 : 3) : 1;   // 16-bit terms of q and P
  static constexpr int kGroups = 4 / WM;                  // warp groups of the CTA
  static constexpr int kKeys = 16 * WM;                   // keys of a stage
  static constexpr int kRowsTile = 16 * WM;
  static constexpr int kRowBytes = Q8 ? HD : HD * 2;
  // row strides in shared memory without bank conflicts: ldmatrix wants the 8
  // rows of a matrix 16 bytes apart (mod 128), the Q8_0 loads want 4 rows 32
  // or 96 bytes apart
  static constexpr int kStride = Q8 ? HD + (HD % 64 == 0 ? 32 : 0) : HD * 2 + 16;
  static constexpr int kScale = Q8 ? HD / 16 : 0;         // scale bytes of a row
  static constexpr int kTile = kKeys * (kStride + kScale);  // keys, or values, of a stage
  static constexpr int kStage = 2 * kTile;
  static constexpr int kQBytes = kTerms * (HD / 16) * 32 * 16 * WM;
  static constexpr int kMerge = kGroups * kRowsTile * HD * 4;  // partial O of the groups
  static constexpr int stages() {
    int s = (104 * 1024 - kQBytes) / (kStage * kGroups);  // two CTAs per SM where that leaves two stages
    return s < 2 ? 2 : s > 6 ? 6 : s;
  }
  static constexpr int kStages = stages();
  static constexpr int kRing = kStages * kStage * kGroups;
  static constexpr int smem() { return kQBytes + (kRing > kMerge ? kRing : kMerge); }
  static_assert(kRowBytes % 16 == 0 && kStride % 16 == 0 && (kKeys * kScale) % 16 == 0, "16-byte copies");
};

// the key (0..7) of an 8-key MMA tile behind the tile's column n: for Q8_0 an
// order in which both the key loads (lanes n = 0..3 and 4..7 together) and the
// value loads (n even, n odd) touch rows that differ mod 4
template <bool Q8>
__device__ __forceinline__ int key_of_col(int n) {
  if constexpr (!Q8) return n;
  return (0x57463120 >> (4 * n)) & 0xF;
}

template <int HD, bool Q8, bool F32, int WM>
__global__ void __launch_bounds__(kPaThreads) paged_attn_kernel(const __grid_constant__ PagedAttnArgs a) {
  using C = PaCfg<HD, Q8, F32, WM>;
  using T = typename std::conditional<F32, float, __nv_bfloat16>::type;
  constexpr int NT = C::kTerms, KS = C::kStride;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float row_scale[C::kRowsTile];
  __shared__ float gm[C::kGroups][C::kRowsTile], gl[C::kGroups][C::kRowsTile];
  __shared__ int last_flag;
  grid_dependency_wait();
  grid_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  // the last tiles of a prompt see the most keys: they start first
  const int tile_id = gridDim.x - 1 - blockIdx.x;
  const RowTile tile = find_tile(a, tile_id, C::kRowsTile);
  if (tile.s < 0) return;
  const int kvh = blockIdx.z;
  const int rows = min(C::kRowsTile, tile.rows - tile.row0);
  // keys that the tile's last row sees, and this CTA's share of them
  const int kend = max(0, min(tile.kv, row_limit(a, tile, tile.row0 + rows - 1)));
  int ck = (kend + a.n_splits - 1) / a.n_splits;
  ck = max(kPaMinSplit, (ck + 63) & ~63);
  const int active = max(1, (kend + ck - 1) / ck);
  const int split = blockIdx.y;
  if (split >= active) return;
  const int kbeg = split * ck, kfin = min(kend, kbeg + ck);

  const int grp = warp / WM, wrow = (warp % WM) * 16, gt = tid % (32 * WM);
  uint8_t* ring = smem + C::kQBytes + grp * (C::kStages * C::kStage);
  const uint32_t ring_u = smem_u32(ring);

  // --- the group's loader: blocks of kKeys keys, group `grp` takes every kGroups-th
  const int n_blocks = (kfin - kbeg + C::kKeys - 1) / C::kKeys;
  const int my_blocks = n_blocks > grp ? (n_blocks - grp + C::kGroups - 1) / C::kGroups : 0;
  auto block_page = [&](int b) -> int {  // lane j < WM: the page of the block's j-th 16 keys
    const int key = kbeg + (grp + b * C::kGroups) * C::kKeys + 16 * (lane % WM);
    return b < my_blocks && key < kfin ? page_of(a.c, tile.s, key) : -1;
  };
  auto load_block = [&](int b, int stage, int page_l) {
    const int key0 = kbeg + (grp + b * C::kGroups) * C::kKeys;
    constexpr int CPR = C::kRowBytes / 16;                 // 16-byte chunks of a row
    constexpr int N = C::kKeys * CPR / (32 * WM);          // chunks of a thread
    const uint32_t dst0 = ring_u + stage * C::kStage;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int idx = i * (32 * WM) + gt, r = idx / CPR, ch = idx % CPR;
      const int page = __shfl_sync(0xffffffffu, page_l, r >> 4);
      const int key = key0 + r;
      const bool on = page >= 0 && key < kfin;
      const int64_t at = ((int64_t)(on ? page : 0) * a.c.kv_heads + kvh) * a.c.block_bytes +
                         (int64_t)(on ? key & ((1 << a.c.page_shift) - 1) : 0) * C::kRowBytes + 16 * ch;
      cp_async16(dst0 + r * KS + 16 * ch, a.c.k + at, on);
      cp_async16(dst0 + C::kTile + r * KS + 16 * ch, a.c.v + at, on);
    }
    if constexpr (Q8) {
      // scales: 16 keys' are HD / 16 chunks of 16 bytes, contiguous in the page
      constexpr int SN = WM * (HD / 16);
      const int sub = gt / (HD / 16), ch = gt % (HD / 16);
      const int page = __shfl_sync(0xffffffffu, page_l, sub < WM ? sub : 0);
      if (gt < SN) {
        const int key = key0 + 16 * sub;
        const bool on = page >= 0 && key < kfin;
        const int64_t at = ((int64_t)(on ? page : 0) * a.c.kv_heads + kvh) * a.c.block_bytes +
                           ((int64_t)HD << a.c.page_shift) +
                           (int64_t)(on ? key & ((1 << a.c.page_shift) - 1) : 0) * C::kScale + 16 * ch;
        const uint32_t d = dst0 + C::kKeys * KS + sub * 16 * C::kScale + 16 * ch;
        cp_async16(d, a.c.k + at, on);
        cp_async16(d + C::kTile, a.c.v + at, on);
      }
    }
  };
  int page_next = block_page(0);
#pragma unroll
  for (int b = 0; b < C::kStages - 1; ++b) {
    const int pg = page_next;
    page_next = block_page(b + 1);
    if (b < my_blocks) load_block(b, b, pg);
    cp_async_commit();
  }

  // --- q as MMA fragments in shared memory: [term][16 dims][row tile][lane]
  const T* qbase = static_cast<const T*>(a.q);
  auto q_row = [&](int r) -> const T* {  // row r of the tile
    const int rr = tile.row0 + r;
    return qbase + (int64_t)(tile.start + rr / a.group) * a.ldq + (int64_t)(kvh * a.group + rr % a.group) * HD;
  };
  if constexpr (Q8) {  // the row's power-of-two scale
    constexpr int TPR = kPaThreads / C::kRowsTile;  // 8, 4 or 2 threads of a row
    const int r = tid / TPR;
    float m = 0.f;
    if (r < rows) {
      const T* p = q_row(r);
      for (int j = tid % TPR; j < HD / 8; j += TPR) {
        float x[8];
        load8(p + 8 * j, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(x[e]));
      }
    }
#pragma unroll
    for (int o = TPR / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    // 2^(exponent + 1) > m; rows of zeros, infinities and NaN keep scale 1
    float s = 1.f;
    if (m > 1e-30f && m < 1e38f) s = __int_as_float((__float_as_int(m) & 0x7F800000) + 0x00800000);
    if (tid % TPR == 0) row_scale[r] = s;
    __syncthreads();
  }
  for (int idx = tid; idx < (HD / 16) * WM * 32; idx += kPaThreads) {
    const int ln = idx & 31, w = (idx >> 5) % WM, step = (idx >> 5) / WM;
    const int lg = ln >> 2, lt = ln & 3;
    // the step's dims behind fragment columns (2t, 2t+1) and (2t+8, 2t+9)
    const int d0 = Q8 ? 32 * (step >> 1) + 8 * lt + 4 * (step & 1) : 16 * step + 2 * lt;
    const int d1 = Q8 ? d0 + 2 : d0 + 8;
    uint32_t f[NT][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // rows lg, lg + 8
      const int r = 16 * w + lg + 8 * h;
      float x[4] = {0.f, 0.f, 0.f, 0.f};
      if (r < rows) {
        const T* p = q_row(r);
        if constexpr (F32) {
          const float2 u = *reinterpret_cast<const float2*>(p + d0), v = *reinterpret_cast<const float2*>(p + d1);
          x[0] = u.x, x[1] = u.y, x[2] = v.x, x[3] = v.y;
        } else {
          const uint32_t u = *reinterpret_cast<const uint32_t*>(p + d0), v = *reinterpret_cast<const uint32_t*>(p + d1);
          x[0] = bf16lo(u), x[1] = bf16hi(u), x[2] = bf16lo(v), x[3] = bf16hi(v);
        }
        if constexpr (Q8) {
          const float inv = 1.f / row_scale[r];  // a power of two: exact
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] *= inv;
        }
      }
      uint32_t lo[NT], hi[NT];
      split2<Q8, NT>(x[0], x[1], lo);
      split2<Q8, NT>(x[2], x[3], hi);
#pragma unroll
      for (int e = 0; e < NT; ++e) f[e][h] = lo[e], f[e][h + 2] = hi[e];
    }
#pragma unroll
    for (int e = 0; e < NT; ++e)
      *reinterpret_cast<uint4*>(smem + (((e * (HD / 16) + step) * WM + w) * 32 + ln) * 16) =
          make_uint4(f[e][0], f[e][1], f[e][2], f[e][3]);
  }
  __syncthreads();

  // --- this thread's rows
  const int r0 = wrow + g, r1 = r0 + 8;
  const int lim0 = r0 < rows ? min(tile.kv, row_limit(a, tile, tile.row0 + r0)) : 0;
  const int lim1 = r1 < rows ? min(tile.kv, row_limit(a, tile, tile.row0 + r1)) : 0;
  const int wfirst = min(tile.kv, row_limit(a, tile, tile.row0 + wrow));  // the warp's first row sees the fewest
  const int wlast = wrow < rows ? min(tile.kv, row_limit(a, tile, tile.row0 + min(wrow + 15, rows - 1))) : 0;
  float sc0 = a.scale_log2, sc1 = a.scale_log2;
  if constexpr (Q8) sc0 *= row_scale[r0], sc1 *= row_scale[r1];
  const int kc0 = key_of_col<Q8>(2 * t), kc1 = key_of_col<Q8>(2 * t + 1), krow = key_of_col<Q8>(g);
  constexpr float kShift = Q8 ? 6.f : 0.f;  // fp16 P: 2^6 at the reference, at most 2^14
  float acc[HD / 8][4];
#pragma unroll
  for (int i = 0; i < HD / 8; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
  // dims of accumulator i behind its columns 2t and 2t + 1
  auto dim_of = [&](int i, int e) -> int {
    return Q8 ? 32 * (i >> 2) + 4 * (2 * t + e) + (i & 3) : 8 * i + 2 * t + e;
  };

  for (int b = 0; b < my_blocks; ++b) {
    cp_async_wait<C::kStages - 2>();
    if constexpr (WM == 1)
      __syncwarp();
    else
      asm volatile("bar.sync %0, %1;" ::"r"(grp + 1), "n"(32 * WM) : "memory");
    // the next block into the stage that block b - 1 has left
    {
      const int nb = b + C::kStages - 1, pg = page_next;
      page_next = block_page(nb + 1);
      if (nb < my_blocks) load_block(nb, nb % C::kStages, pg);
      cp_async_commit();
    }
    const int key0 = kbeg + (grp + b * C::kGroups) * C::kKeys;
    const uint8_t* kt = ring + (b % C::kStages) * C::kStage;
    const uint32_t kt_u = ring_u + (b % C::kStages) * C::kStage;
#pragma unroll 1
    for (int u = 0; u < WM; ++u) {  // 16 keys at a time
      const int k16 = key0 + 16 * u;
      if (k16 >= kfin || k16 >= wlast) break;
      const uint8_t* k_s = kt + 16 * u * KS;
      const uint8_t* v_s = k_s + C::kTile;
      const uint32_t k_u = kt_u + 16 * u * KS;
      const uint8_t* ks_s = kt + C::kKeys * KS + 16 * u * C::kScale;  // scales
      const uint8_t* vs_s = ks_s + C::kTile;
      if constexpr (Q8) {
        // scales came 16 keys at a time: those of values past the end become
        // zero (stale ones may be NaN); their scores are masked
        if (k16 + 16 > kfin) {
          for (int j = lane; j < 16 * (HD / 32); j += 32)
            if (k16 + j / (HD / 32) >= kfin) reinterpret_cast<uint16_t*>(const_cast<uint8_t*>(vs_s))[j] = 0;
          __syncwarp();
        }
      }
      float s[2][4] = {};
#pragma unroll
      for (int kk = 0; kk < HD / 32; ++kk) {
        uint32_t qf[NT][2][4];
#pragma unroll
        for (int e = 0; e < NT; ++e)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint4 w = *reinterpret_cast<const uint4*>(
                smem + (((e * (HD / 16) + 2 * kk + h) * WM + warp % WM) * 32 + lane) * 16);
            qf[e][h][0] = w.x, qf[e][h][1] = w.y, qf[e][h][2] = w.z, qf[e][h][3] = w.w;
          }
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          if constexpr (!Q8) {
            uint32_t kf[4];
            ldsm4(kf, k_u + (8 * n + (lane & 7)) * KS + (4 * kk + (lane >> 3)) * 16);
#pragma unroll
            for (int e = 0; e < NT; ++e) {
              mma_acc<Q8>(s[n], qf[e][0], kf[0], kf[1]);
              mma_acc<Q8>(s[n], qf[e][1], kf[2], kf[3]);
            }
          } else {
            const uint2 w = *reinterpret_cast<const uint2*>(k_s + (8 * n + krow) * KS + 32 * kk + 8 * t);
            const uint32_t d1 = *reinterpret_cast<const uint16_t*>(ks_s + (8 * n + krow) * C::kScale + 2 * kk);
            const uint32_t dd = d1 * 0x10001u;
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t x = (h ? w.y : w.x) ^ 0x80808080u;  // quant + 128
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                // fp16 1024 + byte, minus 1152: the quant
                const uint32_t i2 = hsub2_(__byte_perm(x, 0x64646464u, j ? 0x4342 : 0x4140), 0x64806480u);
                hi[2 * h + j] = hmul2_(i2, dd);
                if constexpr (F32) lo[2 * h + j] = hfms2_(i2, dd, hi[2 * h + j]);
              }
            }
            mma_acc<Q8>(s[n], qf[0][0], hi[0], hi[1]);
            mma_acc<Q8>(s[n], qf[0][1], hi[2], hi[3]);
            if constexpr (F32) {
              mma_acc<Q8>(s[n], qf[1][0], hi[0], hi[1]);
              mma_acc<Q8>(s[n], qf[1][1], hi[2], hi[3]);
              mma_acc<Q8>(s[n], qf[0][0], lo[0], lo[1]);
              mma_acc<Q8>(s[n], qf[0][1], lo[2], lo[3]);
            }
          }
        }
      }
      // scores in log2, masked
      const bool edge = k16 + 16 > wfirst;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        s[n][0] *= sc0, s[n][1] *= sc0, s[n][2] *= sc1, s[n][3] *= sc1;
        if (edge) {
          const int ka = k16 + 8 * n + kc0, kb = k16 + 8 * n + kc1;
          if (ka >= lim0) s[n][0] = -INFINITY;
          if (kb >= lim0) s[n][1] = -INFINITY;
          if (ka >= lim1) s[n][2] = -INFINITY;
          if (kb >= lim1) s[n][3] = -INFINITY;
        }
      }
      float x0 = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1]));
      float x1 = fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3]));
      if (__any_sync(0xffffffffu, x0 > m0 + kPaLazy || x1 > m1 + kPaLazy)) {
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
          x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, o));
          x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, o));
        }
        const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
        const float f0 = n0 == -INFINITY ? 1.f : fast_exp2(m0 - n0), f1 = n1 == -INFINITY ? 1.f : fast_exp2(m1 - n1);
        m0 = n0, m1 = n1, l0 *= f0, l1 *= f1;
#pragma unroll
        for (int i = 0; i < HD / 8; ++i) acc[i][0] *= f0, acc[i][1] *= f0, acc[i][2] *= f1, acc[i][3] *= f1;
      }
      const float ref0 = m0 == -INFINITY ? 0.f : m0 - kShift, ref1 = m1 == -INFINITY ? 0.f : m1 - kShift;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        s[n][0] = fast_exp2(s[n][0] - ref0), s[n][1] = fast_exp2(s[n][1] - ref0);
        s[n][2] = fast_exp2(s[n][2] - ref1), s[n][3] = fast_exp2(s[n][3] - ref1);
        l0 += s[n][0] + s[n][1], l1 += s[n][2] + s[n][3];
      }
      if (edge) {
        // values that are not finite and that some rows of the warp do not see
        bool bad = false;
        if constexpr (Q8) {
          for (int j = lane; j < 16 * (HD / 32); j += 32)
            bad |= (reinterpret_cast<const uint16_t*>(vs_s)[j] & 0x7C00u) == 0x7C00u;
        } else {
          for (int j = lane; j < 16 * (HD / 2); j += 32) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(v_s + (j / (HD / 2)) * KS + 4 * (j % (HD / 2)));
            bad |= (w & 0x7F80u) == 0x7F80u || (w & 0x7F800000u) == 0x7F800000u;
          }
        }
        if (__any_sync(0xffffffffu, bad)) {
#pragma unroll 1
          for (int j = 0; j < 16; ++j) {
            // P of key j: column c of tile j / 8, held by lane c / 2 of the quad
            int c = 0;
            for (int n = 0; n < 8; ++n)
              if (key_of_col<Q8>(n) == (j & 7)) c = n;
            const int src = (lane & ~3) | (c >> 1);
            const float pa = j < 8 ? (c & 1 ? s[0][1] : s[0][0]) : (c & 1 ? s[1][1] : s[1][0]);
            const float pb = j < 8 ? (c & 1 ? s[0][3] : s[0][2]) : (c & 1 ? s[1][3] : s[1][2]);
            const float p0 = __shfl_sync(0xffffffffu, pa, src), p1 = __shfl_sync(0xffffffffu, pb, src);
            const bool on0 = k16 + j < lim0, on1 = k16 + j < lim1;
#pragma unroll
            for (int i = 0; i < HD / 8; ++i)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int d = dim_of(i, e);
                float v;
                if constexpr (Q8)
                  v = __half2float(reinterpret_cast<const __half*>(vs_s + j * C::kScale)[d >> 5]) *
                      (float)reinterpret_cast<const int8_t*>(v_s + j * KS)[d];
                else
                  v = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(v_s + j * KS)[d]);
                if (on0) acc[i][e] = fmaf(p0, v, acc[i][e]);
                if (on1) acc[i][e + 2] = fmaf(p1, v, acc[i][e + 2]);
              }
          }
          continue;
        }
      }
      // P as the A operand: (row g, keys of columns 2t, 2t+1), (row g+8, same), then tile 1
      uint32_t pf[NT][4];
      {
        uint32_t x[NT];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            split2<Q8, NT>(s[n][2 * h], s[n][2 * h + 1], x);
#pragma unroll
            for (int e = 0; e < NT; ++e) pf[e][2 * n + h] = x[e];
          }
      }
      if constexpr (!Q8) {
#pragma unroll
        for (int i = 0; i < HD / 8; i += 2) {
          uint32_t vf[4];  // dims 8i..8i+7: keys 0-7, 8-15; dims 8i+8..: keys 0-7, 8-15
          ldsm4t(vf, k_u + C::kTile + (lane & 15) * KS + (8 * i + 8 * (lane >> 4)) * 2);
#pragma unroll
          for (int e = 0; e < NT; ++e) {
            mma_acc<Q8>(acc[i], pf[e], vf[0], vf[1]);
            mma_acc<Q8>(acc[i + 1], pf[e], vf[2], vf[3]);
          }
        }
      } else {
#pragma unroll
        for (int blk = 0; blk < HD / 32; ++blk) {
          uint32_t hi[2][4], lo[2][4];  // [keys 0-7 / 8-15][dim 4g + j of the block]
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const int ka = 8 * n + kc0, kb = 8 * n + kc1;
            const uint32_t wa = *reinterpret_cast<const uint32_t*>(v_s + ka * KS + 32 * blk + 4 * g) ^ 0x80808080u;
            const uint32_t wb = *reinterpret_cast<const uint32_t*>(v_s + kb * KS + 32 * blk + 4 * g) ^ 0x80808080u;
            const uint32_t da = *reinterpret_cast<const uint16_t*>(vs_s + ka * C::kScale + 2 * blk);
            const uint32_t db = *reinterpret_cast<const uint16_t*>(vs_s + kb * C::kScale + 2 * blk);
            const uint32_t dd = da | (db << 16);
            const uint32_t ab[2] = {__byte_perm(wa, wb, 0x5140), __byte_perm(wa, wb, 0x7362)};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint32_t i2 =
                  hsub2_(__byte_perm(ab[j >> 1], 0x64646464u, (j & 1) ? 0x4342 : 0x4140), 0x64806480u);
              hi[n][j] = hmul2_(i2, dd);
              if constexpr (F32) lo[n][j] = hfms2_(i2, dd, hi[n][j]);
            }
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            mma_acc<Q8>(acc[4 * blk + j], pf[0], hi[0][j], hi[1][j]);
            if constexpr (F32) {
              mma_acc<Q8>(acc[4 * blk + j], pf[NT - 1], hi[0][j], hi[1][j]);
              mma_acc<Q8>(acc[4 * blk + j], pf[0], lo[0][j], lo[1][j]);
            }
          }
        }
      }
    }
  }
  cp_async_wait<0>();
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    l0 += __shfl_xor_sync(0xffffffffu, l0, o);
    l1 += __shfl_xor_sync(0xffffffffu, l1, o);
  }
  __syncthreads();  // the ring is free: partial O of the groups go over it
  if (t == 0) gm[grp][r0] = m0, gm[grp][r1] = m1, gl[grp][r0] = l0, gl[grp][r1] = l1;
  float* part = reinterpret_cast<float*>(smem + C::kQBytes);  // [group][row][HD]
#pragma unroll
  for (int i = 0; i < HD / 8; ++i)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int d = dim_of(i, e);
      part[(grp * C::kRowsTile + r0) * HD + d] = acc[i][e];
      part[(grp * C::kRowsTile + r1) * HD + d] = acc[i][e + 2];
    }
  __syncthreads();
  // merge the groups; one split: normalise and write
  constexpr int kRec = C::kRowsTile * (HD + 2);
  const int64_t unit = (int64_t)tile_id * a.c.kv_heads + kvh;
  float* rec = active > 1 ? a.recs + (unit * a.n_splits + split) * kRec : nullptr;
  T* obase = static_cast<T*>(a.out);
  auto out_row = [&](int r) -> T* {
    const int rr = tile.row0 + r;
    return obase + (int64_t)(tile.start + rr / a.group) * a.ldo + (int64_t)(kvh * a.group + rr % a.group) * HD;
  };
  for (int idx = tid; idx < rows * (HD / 8); idx += kPaThreads) {
    const int r = idx / (HD / 8), d = 8 * (idx % (HD / 8));
    float M = gm[0][r], L = 0.f, o[8] = {};
#pragma unroll
    for (int w = 1; w < C::kGroups; ++w) M = fmaxf(M, gm[w][r]);
#pragma unroll
    for (int w = 0; w < C::kGroups; ++w) {
      const float f = gm[w][r] == -INFINITY ? 0.f : fast_exp2(gm[w][r] - M);
      if (gm[w][r] == -INFINITY && !(gl[w][r] != gl[w][r])) continue;  // no key seen by this group
      L = fmaf(f, gl[w][r], L);
      const float4 p0 = *reinterpret_cast<const float4*>(part + (w * C::kRowsTile + r) * HD + d);
      const float4 p1 = *reinterpret_cast<const float4*>(part + (w * C::kRowsTile + r) * HD + d + 4);
      o[0] = fmaf(f, p0.x, o[0]), o[1] = fmaf(f, p0.y, o[1]), o[2] = fmaf(f, p0.z, o[2]), o[3] = fmaf(f, p0.w, o[3]);
      o[4] = fmaf(f, p1.x, o[4]), o[5] = fmaf(f, p1.y, o[5]), o[6] = fmaf(f, p1.z, o[6]), o[7] = fmaf(f, p1.w, o[7]);
    }
    if (rec == nullptr) {
      const float inv = L == 0.f ? 0.f : 1.f / L;  // a row that sees no key is zero
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = L == 0.f ? 0.f : o[e] * inv;
      store8(out_row(r) + d, o);
    } else {
      __stcg(reinterpret_cast<float4*>(rec + 2 * C::kRowsTile + r * HD + d), make_float4(o[0], o[1], o[2], o[3]));
      __stcg(reinterpret_cast<float4*>(rec + 2 * C::kRowsTile + r * HD + d + 4), make_float4(o[4], o[5], o[6], o[7]));
      if (d == 0) __stcg(reinterpret_cast<float2*>(rec + 2 * r), make_float2(M, L));
    }
  }
  if (active == 1) return;
  __threadfence();  // this thread's record before the arrival
  __syncthreads();
  if (tid == 0) {
    const int prev = atomicAdd(a.counters + unit, 1);
    last_flag = prev == active - 1;
    if (last_flag) {
      atomicExch(a.counters + unit, 0);  // ready for the next launch
      __threadfence();
    }
  }
  __syncthreads();
  if (!last_flag) return;
  const float* recs = a.recs + unit * a.n_splits * kRec;
  for (int idx = tid; idx < rows * (HD / 8); idx += kPaThreads) {
    const int r = idx / (HD / 8), d = 8 * (idx % (HD / 8));
    float M = -INFINITY;
    for (int sp = 0; sp < active; ++sp) M = fmaxf(M, __ldcg(recs + (int64_t)sp * kRec + 2 * r));
    float L = 0.f, o[8] = {};
#pragma unroll 2
    for (int sp = 0; sp < active; ++sp) {
      const float* rc = recs + (int64_t)sp * kRec;
      const float2 ml = __ldcg(reinterpret_cast<const float2*>(rc + 2 * r));
      const float4 p0 = __ldcg(reinterpret_cast<const float4*>(rc + 2 * C::kRowsTile + r * HD + d));
      const float4 p1 = __ldcg(reinterpret_cast<const float4*>(rc + 2 * C::kRowsTile + r * HD + d + 4));
      if (ml.x == -INFINITY && ml.y == ml.y) continue;
      const float f = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - M);
      L = fmaf(f, ml.y, L);
      o[0] = fmaf(f, p0.x, o[0]), o[1] = fmaf(f, p0.y, o[1]), o[2] = fmaf(f, p0.z, o[2]), o[3] = fmaf(f, p0.w, o[3]);
      o[4] = fmaf(f, p1.x, o[4]), o[5] = fmaf(f, p1.y, o[5]), o[6] = fmaf(f, p1.z, o[6]), o[7] = fmaf(f, p1.w, o[7]);
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = L == 0.f ? 0.f : o[e] * inv;
    store8(out_row(r) + d, o);
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
// Row tiles of 16, 32 or 64 rows (WM 1, 2, 4): the smallest that holds the rows
// of the longest chunk, since a sequence's keys are read once per row tile.
// (fp32 rows of 256 over a bf16 cache stop at 32: 64 do not fit shared memory).
static int pick_wm(int max_q, int group, int hd, bool q8, bool f32) {
  const int64_t rows = (int64_t)max_q * group;
  return rows <= 16 ? 1 : rows <= 32 || (hd == 256 && f32 && !q8) ? 2 : 4;
}
// Splits of the keys: about three CTAs for each of the two that an SM holds, so
// that sequences of different lengths even out, none shorter than kPaMinSplit.
static int pick_splits(int64_t units, int max_kv) {
  if (units > kPagedCounters || units < 1) return 1;
  const int64_t want = 6LL * device_sm_count();
  int64_t s = std::min((want + units - 1) / units, ((int64_t)max_kv + kPaMinSplit - 1) / kPaMinSplit);
  return (int)std::max<int64_t>(1, std::min<int64_t>(s, 128));
}
struct PaPlan {
  int wm, splits;
  int64_t tiles, units;
  size_t bytes;  // of partial results
};
static PaPlan plan_of(int n, int n_seqs, int group, int kv_heads, int hd, int max_q, int max_kv, bool q8, bool f32) {
  PaPlan p;
  p.wm = pick_wm(max_q, group, hd, q8, f32);
  p.tiles = (int64_t)n * group / (16 * p.wm) + n_seqs;
  p.units = p.tiles * kv_heads;
  p.splits = pick_splits(p.units, max_kv);
  p.bytes = p.splits > 1 ? (size_t)p.units * p.splits * 16 * p.wm * (hd + 2) * sizeof(float) : 0;
  return p;
}

// New tokens from which a sequence goes to the tensor-memory kernel, or 0: none
// does.  Its CTA takes 256 rows at a time however few there are.
constexpr int kTcMinRows = 64;
static int tc_from(const PagedView& c, int hd, int dtype, int group, int max_q) {
  if (!paged_attn_tc_takes(c, hd, dtype, group, 1 << c.page_shift)) return 0;
  const int from = kTcMinRows / group + 1;
  return max_q >= from ? from : 0;
}

size_t paged_attn_workspace_bytes(const PagedView& c, int n, int group, int hd, int dtype, int max_q, int max_kv) {
  const bool q8 = c.type == DRACO_KV_Q8_0, f32 = dtype == DRACO_DTYPE_F32;
  const int from = tc_from(c, hd, dtype, group, max_q);
  size_t bytes = plan_of(n, c.n_seqs, group, c.kv_heads, hd, from ? from - 1 : max_q, max_kv, q8, f32).bytes;
  if (from) bytes = std::max(bytes, paged_attn_tc_plan(n, c.n_seqs, group, c.kv_heads, hd, max_kv).bytes);
  return kPagedHead + bytes;
}

template <int HD, bool Q8, bool F32, int WM>
static cudaError_t launch_t(const PagedAttnArgs& a, const PaPlan& p, cudaStream_t st) {
  using C = PaCfg<HD, Q8, F32, WM>;
  static int attr_set[64] = {0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !attr_set[dev]) {
    cudaError_t e = cudaFuncSetAttribute(paged_attn_kernel<HD, Q8, F32, WM>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, C::smem());
    if (e != cudaSuccess) return e;
    if (dev < 64) attr_set[dev] = 1;
  }
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)p.tiles, (unsigned)p.splits, (unsigned)a.c.kv_heads);
  cfg.blockDim = dim3(kPaThreads);
  cfg.dynamicSmemBytes = C::smem();
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_attn_kernel<HD, Q8, F32, WM>, a);
}
template <int HD, bool Q8, bool F32>
static cudaError_t launch_wm(const PagedAttnArgs& a, const PaPlan& p, cudaStream_t st) {
  if (p.wm == 1) return launch_t<HD, Q8, F32, 1>(a, p, st);
  if (p.wm == 2) return launch_t<HD, Q8, F32, 2>(a, p, st);
  if constexpr (HD == 256 && F32 && !Q8)
    return cudaErrorInvalidValue;  // pick_wm never asks for it
  else
    return launch_t<HD, Q8, F32, 4>(a, p, st);
}
template <bool Q8, bool F32>
static cudaError_t launch_hd(int hd, const PagedAttnArgs& a, const PaPlan& p, cudaStream_t st) {
  switch (hd) {
    case 32: return launch_wm<32, Q8, F32>(a, p, st);
    case 64: return launch_wm<64, Q8, F32>(a, p, st);
    case 96: return launch_wm<96, Q8, F32>(a, p, st);
    case 128: return launch_wm<128, Q8, F32>(a, p, st);
    default: return launch_wm<256, Q8, F32>(a, p, st);
  }
}

int paged_attn_launch(PagedAttnArgs a, int hd, int dtype, int max_q, int max_kv, void* ws, size_t ws_bytes,
                      cudaStream_t st, char* msg, size_t ml) {
  const bool q8 = a.c.type == DRACO_KV_Q8_0, f32 = dtype == DRACO_DTYPE_F32;
  const size_t need = paged_attn_workspace_bytes(a.c, a.n, a.group, hd, dtype, max_q, max_kv);
  if (ws == nullptr || ws_bytes < need || (reinterpret_cast<uintptr_t>(ws) & 15)) {
    snprintf(msg, ml, "attention_paged: workspace of %zu bytes given (16-byte aligned), %zu needed", ws_bytes, need);
    return DRACO_ERR_WORKSPACE;
  }
  a.counters = static_cast<int*>(ws);
  a.recs = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + kPagedHead);
  // long sequences to the tensor-memory kernel, the others (any that a batch
  // holds beside them: the lengths are on the device) to the warp MMA
  const int from = tc_from(a.c, hd, dtype, a.group, max_q);
  a.min_new = 0;
  a.max_new = from ? from : 0x7FFFFFFF;
  const PaPlan p = plan_of(a.n, a.n_seqs, a.group, a.c.kv_heads, hd, from ? from - 1 : max_q, max_kv, q8, f32);
  a.n_splits = p.splits;
  const cudaError_t e = q8 ? (f32 ? launch_hd<true, true>(hd, a, p, st) : launch_hd<true, false>(hd, a, p, st))
                           : (f32 ? launch_hd<false, true>(hd, a, p, st) : launch_hd<false, false>(hd, a, p, st));
  if (e != cudaSuccess) {
    snprintf(msg, ml, "attention_paged launch failed: %s", cudaGetErrorString(e));
    return DRACO_ERR_CUDA;
  }
  if (!from) return DRACO_OK;
  a.min_new = from;
  a.max_new = 0x7FFFFFFF;
  const TcPlan t = paged_attn_tc_plan(a.n, a.n_seqs, a.group, a.c.kv_heads, hd, max_kv);
  return paged_attn_tc_launch(a, hd, t, a.counters + kPagedCounters, st, msg, ml);
}

}  // namespace draco
