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
// What bounds it: few rows share a key, so bytes; for Q8_0 the conversion of its
// quants and the latency between its steps.  Both products have the keys (and values) as the MMA's A
// operand and the rows as its 8-column B operand, S^T = K Q^T and O^T = V^T
// P^T (m16n8k16): a decode step's rows (the heads of a group) fill 8 columns
// where they would leave 16 rows half empty, S and O take half the registers,
// and a converted fragment serves all NN column tiles of the warp.  P^T comes
// out of the first product as a C fragment and goes into the second as a B
// fragment through two 8x8 transposes (movmatrix).
// A warp takes the 16-key blocks of the CTA's key range in turn with the three
// others, fills its own ring with cp.async and waits for nobody; the warps
// merge in shared memory.  Long ranges are split over CTAs (blockIdx.z) and
// merged, in split order, by the last CTA to arrive.
//
// Precision.  fp32 activations keep 22-24 bits: operands go into the MMAs as
// sums of 16-bit terms, and products go through accumulators of their own of
// at most 32 dims or 16 keys, added in fp32 (the tensor core's accumulation
// truncates).
//   bf16 cache: keys and values are bf16 already.  q and P are one bf16 each
//     for bf16 activations, or three (8 + 8 + 8 bits) for fp32.
//   Q8_0 cache, keys: the quants are exact in fp16; the products of a block of
//     32 are scaled by its scale in fp32.  A byte quant + 128 in the low half
//     of a word is the fp16 subnormal (quant + 128) 2^-24, as it stands; the
//     2^24 goes into the row's scale, the 128 sum(q) into the accumulator's
//     start (fp32 activations subtract it beforehand, exactly).
//     Values: scale * quant has 18 bits, and fp16 takes 11 of them: one fp16 for
//     bf16 activations (relative error 2^-11, against 2^-8 of the output), or
//     two, exact, for fp32.  q and P are one fp16, or two (22 bits); the
//     smallest cross product is left out.  A row of q is scaled by a power of
//     two to at most 1 and P to at most 2^14, so that fp16's range does not cut
//     either.
// m, l, O and the scores are fp32.
//
// A key or value outside [0, kv_len) and a row of a page outside the cache is
// zero-filled in shared memory, never read.  A NaN or infinity in a value row
// that some rows of the tile do not see (a later token of the same chunk)
// must not reach them as 0 * NaN: such a step multiplies key by key.
//
// Measured, 32 query heads over 8 of 128 unless said otherwise: 40 decode steps
// over 500-8000 bf16 positions 136 us (6.0 TB/s); 48 over 900-8000 Q8_0
// positions 105 us (4.6 TB/s: about 380 instructions for a block of 16 keys; neither
// their issue, at 59 % of the rate, nor DRAM, at 55 %, is full with four CTAs an SM,
// so that a part is latency that 16 warps leave open); nine sequences of 4-7 drafts,
// fp32 over up to 6000 Q8_0 positions 56 us (840 instructions a block, two terms of
// everything, and each page converted by the two row tiles of its sequence); one
// fp32 step of 32 heads over 1024 bf16 positions 11 us, most of it the chain
// lengths -> page -> keys and the splits' merge; 32 fp32 tokens of one sequence over
// 8160 positions 76 us (bf16) and 61 (Q8_0), in eight row tiles that each load and
// convert all keys; head_dim 256, 512 bf16 tokens of 16 heads over 4 and 8192
// positions 1045 us, in 256 row tiles of 8 rows a head.
#include <algorithm>
#include <cstdio>

#include "internal.h"
#include "paged_attn.cuh"

namespace draco {

constexpr int kPaThreads = 128;
constexpr int kPaMinSplit = 128;  // keys of a split at least: 2 blocks of each warp
constexpr int kPaMaxSplits = 64;  // two a lane of the merging warp
constexpr float kPaFixed = 250.f;  // keys' worth of time that a CTA's beginning and merge take (12k clocks at 45-60 a key)
constexpr int kPaLookSeqs = 256;  // sequences whose lengths every CTA looks at

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
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
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
template <int HD, bool Q8, bool F32, int NN>
struct PaCfg {
  static constexpr int kTerms = F32 ? (Q8 ? 2 : 3) : 1;   // 16-bit terms of q and P
  static constexpr int kRows = 8 * NN;                    // rows of a tile
  static constexpr int kWarps = kPaThreads / 32;
  static constexpr int kRowBytes = Q8 ? HD : HD * 2;
  // rows 16 bytes apart (mod 128) in shared memory: what ldmatrix wants of the 8
  // rows of a matrix.  The Q8_0 loads take 32 bytes of 4 rows, which 32 bytes
  // apart would not collide in any bank, but were slower (the 48 steps above: 112
  // us, 105 so).
  static constexpr int kStride = kRowBytes + 16;
  static constexpr int kScale = Q8 ? HD / 16 : 0;           // scale bytes of a row
  static constexpr int kTile = 16 * (kStride + kScale);     // 16 keys, or values
  static constexpr int kStage = 2 * kTile;
  static constexpr int kQBytes = kTerms * (HD / 32) * NN * 512;
  static constexpr int kInit = Q8 && !F32 ? (HD / 32) * kRows * 4 : 0;  // -128 sum(q) of every block
  static constexpr int kHead = kQBytes + kInit;
  static constexpr int kMerge = kWarps * kRows * (HD + 4) * 4;    // partial O of the warps
  // shared memory for four CTAs per SM over Q8_0, whose warps compute, three
  // over bf16 (40 steps over 500-8000: 146 us with two, 135 with three; drafts 46
  // and 40), where that leaves two stages
  static constexpr int stages() {
    int s = ((Q8 ? 56 : 74) * 1024 - kHead) / (kStage * kWarps);
    return s < 2 ? 2 : s > 6 ? 6 : s;
  }
  static constexpr int kStages = stages();
  static constexpr int kRing = kStages * kStage * kWarps;
  static constexpr int smem() { return kHead + (kRing > kMerge ? kRing : kMerge); }
  static constexpr int kMinCtas = NN == 1 && HD <= 128 ? 4 : 3;  // bounds the registers
  static_assert(kRowBytes % 16 == 0 && kStride % 16 == 0 && (16 * kScale) % 16 == 0, "16-byte copies");
  static_assert(smem() <= 220 * 1024, "shared memory");
  static_assert(kRing + kMerge > 0 && (kRing > kMerge ? kRing : kMerge) >= (kRows * kPaMaxSplits + 8 * kPaThreads) * 4,
                "the merge's weights and sums");
};

// Keys of a split: the same for all tiles of the batch, so that all CTAs but a
// tile's last run equally long, and so many that the batch makes one or two
// whole waves of a.want CTAs of a head: with T tiles, whose lengths end
// anywhere in their last split, total / ck + T / 2 CTAs.  A wave takes as long
// as a split's keys and the kPaFixed that its beginning and its merge are worth.
// fresh0, kv0: new tokens and keys of sequence `lane`, loaded beforehand.
template <int R>
__device__ __forceinline__ int split_keys(const PagedAttnArgs& a, int kend, int fresh0, int kv0) {
  int longest = kend;
  float tiles = (float)gridDim.x, total = tiles * (float)kend;  // many sequences: as if all were alike
  if (a.n_seqs <= kPaLookSeqs) {
    const int64_t cap = (int64_t)a.c.max_pages << a.c.page_shift;
    total = tiles = 0.f;
    int fresh = fresh0, kv = kv0;
    for (int i = threadIdx.x & 31;;) {
      if (fresh > 0 && fresh >= a.min_new && fresh < a.max_new) {
        kv = (int)min((int64_t)max(kv, 0), cap);
        const float t = (float)((fresh * a.group + R - 1) / R);
        longest = max(longest, kv);
        total += t * (float)kv, tiles += t;
      }
      i += 32;
      if (i >= a.n_seqs) break;
      fresh = seq_begin(a, i + 1) - seq_begin(a, i), kv = __ldg(a.kv_len + i);
    }
    longest = __reduce_max_sync(0xffffffffu, longest);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {  // the same sums in every lane of every CTA
      total += __shfl_xor_sync(0xffffffffu, total, o);
      tiles += __shfl_xor_sync(0xffffffffu, tiles, o);
    }
  }
  float aim = fminf(total / fmaxf(a.want - 0.5f * tiles, 0.25f * a.want), (float)longest);
  if (a.waves > 1) {
    const float two = total / fmaxf(2.f * a.want - 0.5f * tiles, 0.5f * a.want);
    if (2.f * (two + kPaFixed) < aim + kPaFixed) aim = two;
  }
  aim = fminf(aim, 1073741824.f);  // (rounded up below; two splits hold any sequence)
  const int ck = max((int)aim, (longest + a.n_splits - 1) / a.n_splits);
  return max(kPaMinSplit, (ck + 63) & ~63);
}

template <int HD, bool Q8, bool F32, int NN>
__global__ void __launch_bounds__(kPaThreads, (PaCfg<HD, Q8, F32, NN>::kMinCtas)) paged_attn_kernel(const __grid_constant__ PagedAttnArgs a) {
  using C = PaCfg<HD, Q8, F32, NN>;
  using T = typename std::conditional<F32, float, __nv_bfloat16>::type;
  constexpr int NT = C::kTerms, KS = C::kStride, NB = HD / 32, W = C::kWarps;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float row_scale[C::kRows], row_max[NB][C::kRows];
  __shared__ float gm[W][C::kRows], gl[W][C::kRows];
  __shared__ int last_flag;
  grid_dependency_wait();
  grid_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  // the last tiles of a prompt see the most keys: they start first
  const int tile_id = gridDim.x - 1 - blockIdx.x;
  int fresh0 = 0, kv0 = 0;
  if (lane < a.n_seqs && a.n_splits > 1) {
    fresh0 = seq_begin(a, lane + 1) - seq_begin(a, lane);
    kv0 = __ldg(a.kv_len + lane);
  }
  const RowTile tile = find_tile(a, tile_id, C::kRows);
  if (tile.s < 0) return;
  const int kvh = blockIdx.y;
  const int rows = min(C::kRows, tile.rows - tile.row0);
  // Keys that the tile's last row sees, and this CTA's share of them.
  const int kend = max(0, min(tile.kv, row_limit(a, tile, tile.row0 + rows - 1)));
  const int ck = a.n_splits > 1 ? split_keys<C::kRows>(a, kend, fresh0, kv0) : max(kend, 1);
  const int active = split_count(kend, ck);
  const int split = blockIdx.z;  // slowest: CTAs without keys start last
  if (split >= active) return;
  const int kbeg = split * ck, kfin = split_end(kbeg, kend, ck);

  // --- the warp's ring: 16-key blocks, warp w takes every W-th (a block lies in one page)
  uint8_t* ring = smem + C::kHead + warp * (C::kStages * C::kStage);
  const uint32_t ring_u = smem_u32(ring);
  const int n_blocks = (kfin - kbeg + 15) / 16;
  const int my_blocks = n_blocks > warp ? (n_blocks - warp + W - 1) / W : 0;
  const int page_mask = (1 << a.c.page_shift) - 1;
  auto block_key = [&](int b) { return kbeg + (warp + b * W) * 16; };
  auto block_page = [&](int b) { return b < my_blocks ? page_of(a.c, tile.s, block_key(b)) : -1; };
  auto load_block = [&](int b, int stage, int page) {
    constexpr int CPR = C::kRowBytes / 16;  // 16-byte chunks of a row
    constexpr int N = 16 * CPR / 32;        // chunks of a lane
    const int key0 = block_key(b);
    const int have = page >= 0 ? min(16, kfin - key0) : 0;
    const int64_t at = ((int64_t)max(page, 0) * a.c.kv_heads + kvh) * a.c.block_bytes;
    const int off = key0 & page_mask;
    const uint8_t* kp = a.c.k + at + (int64_t)off * C::kRowBytes + 16 * lane;
    const uint8_t* vp = a.c.v + at + (int64_t)off * C::kRowBytes + 16 * lane;
    const uint32_t dst0 = ring_u + stage * C::kStage;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int idx = i * 32 + lane, r = idx / CPR, ch = idx % CPR;
      const uint32_t dst = dst0 + r * KS + 16 * ch;
      cp_async16(dst, kp + 512 * i, r < have);
      cp_async16(dst + C::kTile, vp + 512 * i, r < have);
    }
    if constexpr (Q8) {  // the scales of 16 keys: HD / 16 chunks, contiguous in the page
      if (lane < HD / 16) {
        const int64_t sc = ((int64_t)HD << a.c.page_shift) - (int64_t)off * C::kRowBytes + (int64_t)off * C::kScale;
        const uint32_t dst = dst0 + 16 * KS + 16 * lane;
        cp_async16(dst, kp + sc, have > 0);
        cp_async16(dst + C::kTile, vp + sc, have > 0);
      }
    }
  };
  // --- q: read ahead of the keys; a thread holds 8 dims of a row and 32-dim block, kQItems times
  constexpr int kQItems = (NB * NN * 32 + kPaThreads - 1) / kPaThreads;
  const T* qbase = static_cast<const T*>(a.q);
  constexpr int QW = F32 ? 8 : 4;  // words of 8 dims
  uint32_t raw[kQItems][QW];
#pragma unroll
  for (int i = 0; i < kQItems; ++i) {
    const int idx = tid + i * kPaThreads, lg = (idx & 31) >> 2, lt = idx & 3;
    const int nt = (idx >> 5) % NN, blk = (idx >> 5) / NN, r = 8 * nt + lg;
#pragma unroll
    for (int e = 0; e < QW; ++e) raw[i][e] = 0u;
    if (blk < NB && r < rows) {
      const int rr = tile.row0 + r;
      const T* p = qbase + (int64_t)(tile.start + rr / a.group) * a.ldq +
                   (int64_t)(kvh * a.group + rr % a.group) * HD + 32 * blk;
      if constexpr (Q8) {
#pragma unroll
        for (int e = 0; e < QW; e += 4) {
          const uint4 u = *reinterpret_cast<const uint4*>(p + 8 * lt + e);
          raw[i][e] = u.x, raw[i][e + 1] = u.y, raw[i][e + 2] = u.z, raw[i][e + 3] = u.w;
        }
      } else {
        // the dims behind (2t, 2t+1) and (2t+8, 2t+9) of the block's two steps
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const T* u = p + 16 * (e >> 1) + 8 * (e & 1) + 2 * lt;
          if constexpr (F32) {
            const uint2 w = *reinterpret_cast<const uint2*>(u);
            raw[i][2 * e] = w.x, raw[i][2 * e + 1] = w.y;
          } else {
            raw[i][e] = *reinterpret_cast<const uint32_t*>(u);
          }
        }
      }
    }
  }
  int page_next = block_page(0);
#pragma unroll
  for (int b = 0; b < C::kStages - 1; ++b) {
    const int pg = page_next;
    page_next = block_page(b + 1);
    if (b < my_blocks) load_block(b, b, pg);
    cp_async_commit();
  }

  // --- q as B fragments in shared memory: [term][32 dims][column tile][lane] of two MMA steps
  float* init = reinterpret_cast<float*>(smem + C::kQBytes);  // [32 dims][row]
  float x[kQItems][8];
#pragma unroll
  for (int i = 0; i < kQItems; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (F32)
        x[i][2 * e] = __uint_as_float(raw[i][2 * e]), x[i][2 * e + 1] = __uint_as_float(raw[i][2 * e + 1]);
      else
        x[i][2 * e] = bf16lo(raw[i][e]), x[i][2 * e + 1] = bf16hi(raw[i][e]);
    }
  if constexpr (Q8) {  // the rows' largest values
#pragma unroll
    for (int i = 0; i < kQItems; ++i) {
      const int idx = tid + i * kPaThreads, nt = (idx >> 5) % NN, blk = (idx >> 5) / NN;
      float big = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) big = fmaxf(big, fabsf(x[i][e]));
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
      if (t == 0 && blk < NB) row_max[blk][8 * nt + g] = big;
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < kQItems; ++i) {
    const int idx = tid + i * kPaThreads, nt = (idx >> 5) % NN, blk = (idx >> 5) / NN, r = 8 * nt + g;
    if (blk >= NB) break;
    if constexpr (Q8) {  // the row's power-of-two scale
      float big = row_max[0][r];
#pragma unroll
      for (int e = 1; e < NB; ++e) big = fmaxf(big, row_max[e][r]);
      // 2^(exponent + 1) > big; rows of zeros, infinities and NaN keep scale 1
      float s = 1.f;
      if (big > 1e-30f && big < 1e38f) s = __int_as_float((__float_as_int(big) & 0x7F800000) + 0x00800000);
      if (t == 0 && blk == 0) row_scale[r] = s;
      const float inv = 1.f / s;  // exact
#pragma unroll
      for (int e = 0; e < 8; ++e) x[i][e] *= inv;
    }
    uint32_t f[4][NT];
#pragma unroll
    for (int e = 0; e < 4; ++e) split2<Q8, NT>(x[i][2 * e], x[i][2 * e + 1], f[e]);
#pragma unroll
    for (int e = 0; e < NT; ++e)
      *reinterpret_cast<uint4*>(smem + (((e * NB + blk) * NN + nt) * 32 + lane) * 16) =
          make_uint4(f[0][e], f[1][e], f[2][e], f[3][e]);
    if constexpr (C::kInit > 0) {
      float q = 0.f;  // of the fp16 values
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 u = __half22float2(*reinterpret_cast<__half2*>(&f[e][0]));
        q += u.x + u.y;
      }
      q += __shfl_xor_sync(0xffffffffu, q, 1);
      q += __shfl_xor_sync(0xffffffffu, q, 2);
      if (t == 0) init[blk * C::kRows + r] = q * (-128.f / 16777216.f);
    }
  }
  __syncthreads();

  // --- this thread's columns: rows 8 nt + 2t, + 1; its keys: g, g + 8 of a block
  int lim[NN][2];
  float sc[NN][2];
  const int first = min(tile.kv, row_limit(a, tile, tile.row0));  // the first row sees the fewest keys
#pragma unroll
  for (int n = 0; n < NN; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = 8 * n + 2 * t + e;
      // (columns behind the last row hold q = 0 and are not stored)
      lim[n][e] = min(tile.kv, row_limit(a, tile, tile.row0 + min(r, rows - 1)));
      sc[n][e] = a.scale_log2;
      if constexpr (Q8) sc[n][e] *= row_scale[r] * (F32 ? 1.f : 16777216.f);
    }
  constexpr float kShift = Q8 ? 6.f : 0.f;  // fp16 P: 2^6 at the reference, at most 2^14
  float acc[HD / 16][NN][4];
#pragma unroll
  for (int i = 0; i < HD / 16; ++i)
#pragma unroll
    for (int n = 0; n < NN; ++n) acc[i][n][0] = acc[i][n][1] = acc[i][n][2] = acc[i][n][3] = 0.f;
  float m[NN][2], l[NN][2];
#pragma unroll
  for (int n = 0; n < NN; ++n) m[n][0] = m[n][1] = -INFINITY, l[n][0] = l[n][1] = 0.f;
  bool huge = false;
  // dim behind accumulator i, elements 0/1 (h = 0) or 2/3 (h = 1)
  auto dim_of = [&](int i, int h) -> int { return Q8 ? 32 * (i >> 1) + 4 * g + 2 * (i & 1) + h : 16 * i + g + 8 * h; };

#pragma unroll 1
  for (int b = 0; b < my_blocks; ++b) {
    cp_async_wait<C::kStages - 2>();
    __syncwarp();  // everybody's copies are there, and block b - 1 has been read
    {
      const int nb = b + C::kStages - 1, pg = page_next;
      page_next = block_page(nb + 1);
      if (nb < my_blocks) load_block(nb, nb % C::kStages, pg);
      cp_async_commit();
    }
    const int k16 = block_key(b);
    const int at = (b % C::kStages) * C::kStage;
    const uint8_t* k_s = ring + at;
    const uint8_t* v_s = k_s + C::kTile;
    const uint32_t k_u = ring_u + at;
    const uint8_t* ks_s = k_s + 16 * KS;  // scales
    const uint8_t* vs_s = ks_s + C::kTile;
    if constexpr (Q8) {
      // scales came 16 keys at a time: those of values past the end become
      // zero (stale ones may be NaN); their scores are masked
      if (k16 + 16 > kfin) {
        for (int j = lane; j < 16 * NB; j += 32)
          if (k16 + j / NB >= kfin) reinterpret_cast<uint16_t*>(const_cast<uint8_t*>(vs_s))[j] = 0;
        __syncwarp();
      }
    }
    float s[NN][4];
#pragma unroll
    for (int n = 0; n < NN; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
    // scales of keys g and g + 8, all blocks
    uint32_t dk[2][(NB + 1) / 2];
    if constexpr (Q8) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint8_t* p = ks_s + (g + 8 * h) * C::kScale;
        if constexpr (NB == 1)
          dk[h][0] = *reinterpret_cast<const uint16_t*>(p);
        else if constexpr (NB == 3)
          dk[h][0] = *reinterpret_cast<const uint16_t*>(p) | ((uint32_t)*reinterpret_cast<const uint16_t*>(p + 2) << 16),
          dk[h][1] = *reinterpret_cast<const uint16_t*>(p + 4);
        else
#pragma unroll
          for (int e = 0; e < NB / 2; ++e) dk[h][e] = *reinterpret_cast<const uint32_t*>(p + 4 * e);
      }
    }
#pragma unroll
    for (int blk = 0; blk < NB; ++blk) {
      uint32_t kf[2][4];  // two steps of 16 dims: (key g, key g + 8) x (dims 2t, dims 2t + 8)
      if constexpr (!Q8) {
        const uint32_t p = k_u + ((lane & 7) + 8 * ((lane >> 3) & 1)) * KS + (4 * blk + (lane >> 4)) * 16;
        ldsm4(kf[0], p);
        ldsm4(kf[1], p + 32);
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint2 w = *reinterpret_cast<const uint2*>(k_s + (g + 8 * h) * KS + 32 * blk + 8 * t);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t x = (e ? w.y : w.x) ^ 0x80808080u;  // quant + 128
            if constexpr (F32) {
              // fp16 1024 + byte, minus 1152: the quant
              kf[e][h] = hsub2_(__byte_perm(x, 0x64646464u, 0x4140), 0x64806480u);
              kf[e][h + 2] = hsub2_(__byte_perm(x, 0x64646464u, 0x4342), 0x64806480u);
            } else {
              kf[e][h] = __byte_perm(x, 0u, 0x4140);
              kf[e][h + 2] = __byte_perm(x, 0u, 0x4342);
            }
          }
        }
      }
      float d0 = 1.f, d1 = 1.f;
      if constexpr (Q8) {
        d0 = f16_bits_to_f32(dk[0][blk / 2] >> (16 * (blk & 1)));
        d1 = f16_bits_to_f32(dk[1][blk / 2] >> (16 * (blk & 1)));
      }
#pragma unroll
      for (int n = 0; n < NN; ++n) {
        if constexpr (!Q8 && !F32) {
          const uint4 w = *reinterpret_cast<const uint4*>(smem + ((blk * NN + n) * 32 + lane) * 16);
          mma_acc<Q8>(s[n], kf[0], w.x, w.y);
          mma_acc<Q8>(s[n], kf[1], w.z, w.w);
        } else {
          float u[4] = {0.f, 0.f, 0.f, 0.f};
          if constexpr (C::kInit > 0) {
            const float2 i2 = *reinterpret_cast<const float2*>(init + blk * C::kRows + 8 * n + 2 * t);
            u[0] = u[2] = i2.x, u[1] = u[3] = i2.y;
          }
#pragma unroll
          for (int e = NT - 1; e >= 0; --e) {  // the smallest terms first
            const uint4 w = *reinterpret_cast<const uint4*>(smem + (((e * NB + blk) * NN + n) * 32 + lane) * 16);
            mma_acc<Q8>(u, kf[0], w.x, w.y);
            mma_acc<Q8>(u, kf[1], w.z, w.w);
          }
          if constexpr (Q8) {
            s[n][0] = fmaf(u[0], d0, s[n][0]), s[n][1] = fmaf(u[1], d0, s[n][1]);
            s[n][2] = fmaf(u[2], d1, s[n][2]), s[n][3] = fmaf(u[3], d1, s[n][3]);
          } else {
            s[n][0] += u[0], s[n][1] += u[1], s[n][2] += u[2], s[n][3] += u[3];
          }
        }
      }
    }
    const bool edge = k16 + 16 > first;
    bool grow = false;
#pragma unroll
    for (int n = 0; n < NN; ++n) {
      if (edge) {
        const int ka = k16 + g, kb = ka + 8;
        if (ka >= lim[n][0]) s[n][0] = -INFINITY;
        if (ka >= lim[n][1]) s[n][1] = -INFINITY;
        if (kb >= lim[n][0]) s[n][2] = -INFINITY;
        if (kb >= lim[n][1]) s[n][3] = -INFINITY;
      }
      grow |= fmaxf(s[n][0], s[n][2]) * sc[n][0] > m[n][0] + kPaLazy;
      grow |= fmaxf(s[n][1], s[n][3]) * sc[n][1] > m[n][1] + kPaLazy;
    }
    if (__any_sync(0xffffffffu, grow)) {
      huge = false;
#pragma unroll
      for (int n = 0; n < NN; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = fmaxf(s[n][e], s[n][e + 2]) * sc[n][e];
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
          const float nm = fmaxf(m[n][e], x);
          const float f = nm == -INFINITY ? 1.f : fast_exp2(m[n][e] - nm);
          m[n][e] = nm, l[n][e] *= f;
          huge |= is_huge(nm);
#pragma unroll
          for (int i = 0; i < HD / 16; ++i) acc[i][n][e] *= f, acc[i][n][e + 2] *= f;
        }
      huge = __any_sync(0xffffffffu, huge);
    }
    if (huge) {
#pragma unroll
      for (int n = 0; n < NN; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[n][e] = fast_exp2(huge_exponent(s[n][e], sc[n][e & 1], m[n][e & 1]) + kShift);
          l[n][e & 1] += s[n][e];
        }
    } else {
#pragma unroll
      for (int n = 0; n < NN; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float ref = m[n][e] == -INFINITY ? 0.f : m[n][e] - kShift;
          s[n][e] = fast_exp2(fmaf(s[n][e], sc[n][e], -ref));
          s[n][e + 2] = fast_exp2(fmaf(s[n][e + 2], sc[n][e], -ref));
          l[n][e] += s[n][e] + s[n][e + 2];
        }
    }
    if (edge) {
      // values that are not finite and that some rows of the tile do not see
      bool bad = false;
      if constexpr (Q8) {
        for (int j = lane; j < 16 * NB; j += 32)
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
          const int src = 4 * (j & 7) + t;  // holds P of key j
#pragma unroll
          for (int n = 0; n < NN; ++n) {
            const float p0 = __shfl_sync(0xffffffffu, j < 8 ? s[n][0] : s[n][2], src);
            const float p1 = __shfl_sync(0xffffffffu, j < 8 ? s[n][1] : s[n][3], src);
            const bool on0 = k16 + j < lim[n][0], on1 = k16 + j < lim[n][1];
#pragma unroll
            for (int i = 0; i < HD / 16; ++i)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int d = dim_of(i, h);
                float v;
                if constexpr (Q8)
                  v = __half2float(reinterpret_cast<const __half*>(vs_s + j * C::kScale)[d >> 5]) *
                      (float)reinterpret_cast<const int8_t*>(v_s + j * KS)[d];
                else
                  v = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(v_s + j * KS)[d]);
                if (on0) acc[i][n][2 * h] = fmaf(p0, v, acc[i][n][2 * h]);
                if (on1) acc[i][n][2 * h + 1] = fmaf(p1, v, acc[i][n][2 * h + 1]);
              }
          }
        }
        continue;
      }
    }
    // P^T as B operands: (keys of rows 2t, 2t+1; column g), (the same + 8)
    uint32_t pf[NN][NT][2];
#pragma unroll
    for (int n = 0; n < NN; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t x[NT];
        split2<Q8, NT>(s[n][2 * h], s[n][2 * h + 1], x);
#pragma unroll
        for (int e = 0; e < NT; ++e) pf[n][e][h] = transpose8x8(x[e]);
      }
    if constexpr (!Q8) {
#pragma unroll
      for (int i = 0; i < HD / 16; ++i) {
        uint32_t vf[4];  // (dim g, dim g + 8) x (keys 2t, keys 2t + 8)
        ldsm4t(vf, k_u + C::kTile + ((lane & 7) + 8 * (lane >> 4)) * KS + (2 * i + ((lane >> 3) & 1)) * 16);
#pragma unroll
        for (int n = 0; n < NN; ++n) {
          if constexpr (!F32) {
            mma_acc<Q8>(acc[i][n], vf, pf[n][0][0], pf[n][0][1]);
          } else {
            float u[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int e = NT - 1; e >= 0; --e) mma_acc<Q8>(u, vf, pf[n][e][0], pf[n][e][1]);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][n][e] += u[e];
          }
        }
      }
    } else {
      // scales of keys 2t, 2t + 1 and those + 8: neighbours, NB words
      uint32_t dv[2][NB];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint8_t* p = vs_s + (8 * h + 2 * t) * C::kScale;
        if constexpr (NB % 4 == 0) {
#pragma unroll
          for (int e = 0; e < NB; e += 4) {
            const uint4 w = *reinterpret_cast<const uint4*>(p + 4 * e);
            dv[h][e] = w.x, dv[h][e + 1] = w.y, dv[h][e + 2] = w.z, dv[h][e + 3] = w.w;
          }
        } else if constexpr (NB == 2) {
          const uint2 w = *reinterpret_cast<const uint2*>(p);
          dv[h][0] = w.x, dv[h][1] = w.y;
        } else {
#pragma unroll
          for (int e = 0; e < NB; ++e) dv[h][e] = *reinterpret_cast<const uint32_t*>(p + 4 * e);
        }
      }
#pragma unroll
      for (int blk = 0; blk < NB; ++blk) {
        uint32_t hi[2][4], lo[2][4];  // [keys 2t.. / 2t + 8..][dim 4g + j of the block]
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int ka = 8 * h + 2 * t, kb = ka + 1;
          const uint32_t wa = *reinterpret_cast<const uint32_t*>(v_s + ka * KS + 32 * blk + 4 * g) ^ 0x80808080u;
          const uint32_t wb = *reinterpret_cast<const uint32_t*>(v_s + kb * KS + 32 * blk + 4 * g) ^ 0x80808080u;
          // (key 2t's is half blk of the words, key 2t + 1's half NB + blk)
          const uint32_t dd = __byte_perm(dv[h][blk / 2], dv[h][(NB + blk) / 2],
                                          (blk & 1 ? 0x32 : 0x10) | ((NB + blk) & 1 ? 0x7600 : 0x5400));
          const uint32_t ab[2] = {__byte_perm(wa, wb, 0x5140), __byte_perm(wa, wb, 0x7362)};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t i2 = hsub2_(__byte_perm(ab[j >> 1], 0x64646464u, (j & 1) ? 0x4342 : 0x4140), 0x64806480u);
            hi[h][j] = hmul2_(i2, dd);
            if constexpr (F32) lo[h][j] = hfms2_(i2, dd, hi[h][j]);
          }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t vh[4] = {hi[0][2 * i], hi[0][2 * i + 1], hi[1][2 * i], hi[1][2 * i + 1]};
#pragma unroll
          for (int n = 0; n < NN; ++n) {
            if constexpr (!F32) {
              mma_acc<Q8>(acc[2 * blk + i][n], vh, pf[n][0][0], pf[n][0][1]);
            } else {
              const uint32_t vl[4] = {lo[0][2 * i], lo[0][2 * i + 1], lo[1][2 * i], lo[1][2 * i + 1]};
              float u[4] = {0.f, 0.f, 0.f, 0.f};
              mma_acc<Q8>(u, vl, pf[n][0][0], pf[n][0][1]);
              mma_acc<Q8>(u, vh, pf[n][NT - 1][0], pf[n][NT - 1][1]);
              mma_acc<Q8>(u, vh, pf[n][0][0], pf[n][0][1]);
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[2 * blk + i][n][e] += u[e];
            }
          }
        }
      }
    }
  }
  cp_async_wait<0>();
#pragma unroll
  for (int n = 0; n < NN; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], o);
  __syncthreads();  // the rings are free: partial O of the warps go over them
  constexpr int PS = HD + 4;  // a row's stride: the stores below touch every bank once
  float* part = reinterpret_cast<float*>(smem + C::kHead);  // [warp][row][PS]
#pragma unroll
  for (int n = 0; n < NN; ++n) {
    if (g == 0) {
      *reinterpret_cast<float2*>(&gm[warp][8 * n + 2 * t]) = make_float2(m[n][0], m[n][1]);
      *reinterpret_cast<float2*>(&gl[warp][8 * n + 2 * t]) = make_float2(l[n][0], l[n][1]);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float* p = part + (warp * C::kRows + 8 * n + 2 * t + e) * PS;
      if constexpr (Q8) {
#pragma unroll
        for (int i = 0; i < HD / 16; i += 2)
          *reinterpret_cast<float4*>(p + dim_of(i, 0)) =
              make_float4(acc[i][n][e], acc[i][n][e + 2], acc[i + 1][n][e], acc[i + 1][n][e + 2]);
      } else {
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) p[dim_of(i, 0)] = acc[i][n][e], p[dim_of(i, 1)] = acc[i][n][e + 2];
      }
    }
  }
  __syncthreads();
  // merge the warps; one split: normalise and write
  constexpr int kRec = C::kRows * (HD + 2);
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
    for (int w = 1; w < W; ++w) M = fmaxf(M, gm[w][r]);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (gm[w][r] == -INFINITY && gl[w][r] == gl[w][r]) continue;  // no key seen by this warp
      const float f = gm[w][r] == -INFINITY ? 0.f : fast_exp2(gm[w][r] - M);
      L = fmaf(f, gl[w][r], L);
      const float4 p0 = *reinterpret_cast<const float4*>(part + (w * C::kRows + r) * PS + d);
      const float4 p1 = *reinterpret_cast<const float4*>(part + (w * C::kRows + r) * PS + d + 4);
      o[0] = fmaf(f, p0.x, o[0]), o[1] = fmaf(f, p0.y, o[1]), o[2] = fmaf(f, p0.z, o[2]), o[3] = fmaf(f, p0.w, o[3]);
      o[4] = fmaf(f, p1.x, o[4]), o[5] = fmaf(f, p1.y, o[5]), o[6] = fmaf(f, p1.z, o[6]), o[7] = fmaf(f, p1.w, o[7]);
    }
    if (rec == nullptr) {
      const float inv = L == 0.f ? 0.f : 1.f / L;  // a row that sees no key is zero
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = L == 0.f ? 0.f : o[e] * inv;
      store8(out_row(r) + d, o);
    } else {
      __stcg(reinterpret_cast<float4*>(rec + 2 * C::kRows + r * HD + d), make_float4(o[0], o[1], o[2], o[3]));
      __stcg(reinterpret_cast<float4*>(rec + 2 * C::kRows + r * HD + d + 4), make_float4(o[4], o[5], o[6], o[7]));
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
  // Merge in split order.  A warp per row turns the splits' (m, l) into weights
  // (lanes over splits); then the threads go over the rows' values, and, where
  // those leave threads idle, over parts of the splits.
  const float* recs = a.recs + unit * a.n_splits * kRec;
  float* wts = reinterpret_cast<float*>(smem + C::kHead);  // [row][split]
  constexpr int RW = C::kRows / W;
  float2 ml[RW][2];  // of two splits a lane (kPaMaxSplits): all rows' loads together
#pragma unroll
  for (int i = 0; i < RW; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = warp + i * W, sp = lane + 32 * h;
      ml[i][h] = make_float2(-INFINITY, 0.f);
      if (r < rows && sp < active) ml[i][h] = __ldcg(reinterpret_cast<const float2*>(recs + (int64_t)sp * kRec + 2 * r));
    }
#pragma unroll
  for (int i = 0; i < RW; ++i) {
    const int r = warp + i * W;
    float M = fmaxf(ml[i][0].x, ml[i][1].x), L = 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      // (m -infinity: no key seen, unless l is NaN)
      const float f = ml[i][h].x == -INFINITY ? 0.f : fast_exp2(ml[i][h].x - M);
      L += ml[i][h].x == -INFINITY && ml[i][h].y == ml[i][h].y ? 0.f : f * ml[i][h].y;
      if (r < rows && lane + 32 * h < active) wts[r * a.n_splits + lane + 32 * h] = f;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    if (lane == 0) gl[0][r] = L;
  }
  __syncthreads();
  const int items = rows * (HD / 8), parts = max(1, min(kPaThreads / items, 8));
  float* sums = wts + ((rows * a.n_splits + 3) & ~3);  // [part][item][8]
  for (int idx = tid; idx < items * parts; idx += kPaThreads) {
    const int part_i = idx / items, it = idx % items, r = it / (HD / 8), d = 8 * (it % (HD / 8));
    float o[8] = {};
#pragma unroll 8
    for (int sp = part_i; sp < active; sp += parts) {
      const float* rc = recs + (int64_t)sp * kRec + 2 * C::kRows + r * HD + d;
      const float f = wts[r * a.n_splits + sp];
      const float4 p0 = __ldcg(reinterpret_cast<const float4*>(rc)), p1 = __ldcg(reinterpret_cast<const float4*>(rc + 4));
      o[0] = fmaf(f, p0.x, o[0]), o[1] = fmaf(f, p0.y, o[1]), o[2] = fmaf(f, p0.z, o[2]), o[3] = fmaf(f, p0.w, o[3]);
      o[4] = fmaf(f, p1.x, o[4]), o[5] = fmaf(f, p1.y, o[5]), o[6] = fmaf(f, p1.z, o[6]), o[7] = fmaf(f, p1.w, o[7]);
    }
    if (parts == 1) {
      const float L = gl[0][r], inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = L == 0.f ? 0.f : o[e] * inv;
      store8(out_row(r) + d, o);
    } else {
      *reinterpret_cast<float4*>(sums + 8 * idx) = make_float4(o[0], o[1], o[2], o[3]);
      *reinterpret_cast<float4*>(sums + 8 * idx + 4) = make_float4(o[4], o[5], o[6], o[7]);
    }
  }
  if (parts == 1) return;
  __syncthreads();
  for (int it = tid; it < items; it += kPaThreads) {
    const int r = it / (HD / 8), d = 8 * (it % (HD / 8));
    float o[8] = {};
    for (int p = 0; p < parts; ++p)
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] += sums[8 * (p * items + it) + e];
    const float L = gl[0][r], inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = L == 0.f ? 0.f : o[e] * inv;
    store8(out_row(r) + d, o);
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
// Column tiles of a warp (NN: 1, 2 or 4): the fewest that hold the rows of the
// longest chunk, since a sequence's keys are read and converted once per row
// tile; but O's HD * NN / 4 registers leave room for other warps (drafts over
// Q8_0 in fp32, 16-28 rows of 128: 62 us with one tile of NN 4, 56 with two of NN
// 2, 58 with NN 1; bf16 over bf16 pages 42, 40 and 57).
static int pick_nn(int max_q, int group, int hd) {
  const int64_t rows = (int64_t)max_q * group;
  const int most = hd <= 64 ? 4 : hd <= 128 ? 2 : 1;
  int nn = 1;
  while (nn < most && rows > 8 * nn) nn *= 2;
  return nn;
}
// Splits of the keys at most, none shorter than kPaMinSplit: the grid's; the
// kernel, which sees the lengths, uses those that it needs (split_keys).  Twice
// what two waves take of sequences that are alike.  `ctas`: CTAs an SM holds.
static int pick_splits(int64_t units, int max_kv, int ctas) {
  if (units > kPagedCounters || units < 1) return 1;
  const int64_t slots = (int64_t)ctas * device_sm_count();
  const int64_t s = std::min(4 * slots / units, ((int64_t)max_kv + kPaMinSplit - 1) / kPaMinSplit);
  return (int)std::max<int64_t>(1, std::min<int64_t>(s, kPaMaxSplits));
}
struct PaPlan {
  int nn, splits, per_seq;
  int64_t tiles, units;
  size_t bytes;  // of partial results
};
static PaPlan plan_of(int n, int n_seqs, int group, int kv_heads, int hd, int max_q, int max_kv,
                      bool q8) {
  PaPlan p;
  p.nn = pick_nn(max_q, group, hd);
  const int R = 8 * p.nn;
  p.tiles = (int64_t)n * group / R + n_seqs;
  // short chunks: as many tiles for every sequence
  const int64_t per = ((int64_t)max_q * group + R - 1) / R;
  p.per_seq = per > 0 && per * n_seqs <= p.tiles ? (int)per : 0;
  if (p.per_seq) p.tiles = per * n_seqs;
  p.units = p.tiles * kv_heads;
  p.splits = pick_splits(p.units, max_kv, q8 ? 4 : 3);
  p.bytes = p.splits > 1 ? (size_t)p.units * p.splits * 8 * p.nn * (hd + 2) * sizeof(float) : 0;
  return p;
}

// New tokens from which a sequence goes to the tensor-memory kernel, or 0: none
// does.
static int tc_from(const PagedView& c, int n, int hd, int dtype, int group, int max_q, int max_kv) {
  if (!paged_attn_tc_takes(c, hd, dtype, group, 1 << c.page_shift)) return 0;
  const int from = tc_min_tokens(group);
  if (max_q < from) return 0;
  // (its tiles are the grid's y)
  return paged_attn_tc_plan(n, c.n_seqs, group, c.kv_heads, hd, max_kv).tiles <= 65535 ? from : 0;
}

size_t paged_attn_workspace_bytes(const PagedView& c, int n, int group, int hd, int dtype, int max_q, int max_kv) {
  const int from = tc_from(c, n, hd, dtype, group, max_q, max_kv);
  size_t bytes = plan_of(n, c.n_seqs, group, c.kv_heads, hd, from ? from - 1 : max_q, max_kv, c.type == DRACO_KV_Q8_0).bytes;
  if (from) bytes = std::max(bytes, paged_attn_tc_plan(n, c.n_seqs, group, c.kv_heads, hd, max_kv).bytes);
  return kPagedHead + bytes;
}

template <int HD, bool Q8, bool F32, int NN>
static cudaError_t launch_t(PagedAttnArgs a, const PaPlan& p, cudaStream_t st) {
  using C = PaCfg<HD, Q8, F32, NN>;
  static int ctas_of[64] = {0};  // CTAs an SM holds
  int dev = 0, ctas = 0;
  cudaGetDevice(&dev);
  if (dev < 64) ctas = ctas_of[dev];
  if (ctas == 0) {
    cudaError_t e = cudaFuncSetAttribute(paged_attn_kernel<HD, Q8, F32, NN>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, C::smem());
    if (e == cudaSuccess)
      e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&ctas, paged_attn_kernel<HD, Q8, F32, NN>, kPaThreads,
                                                        C::smem());
    if (e != cudaSuccess) return e;
    ctas = std::max(ctas, 1);
    if (dev < 64) ctas_of[dev] = ctas;
  }
  const int64_t slots = (int64_t)ctas * device_sm_count();
  // A few units (one sequence) are all alike: two CTAs an SM, more only add to
  // the merge (16384 Q8_0 positions, 8 heads: 24.8 us with one, 19.8 with two,
  // 20.0 with three).  Others have different lengths, which two waves of smaller
  // pieces may even out (48 sequences of 900-8000 positions: 117 us with one
  // wave, 105 with two; drafts of nine: 56 and 64): the kernel chooses.
  const bool few = p.units * 8 <= slots;
  a.want = (float)(few ? 2LL * device_sm_count() : slots) / (float)a.c.kv_heads;
  a.waves = few ? 1 : 2;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)p.tiles, (unsigned)a.c.kv_heads, (unsigned)p.splits);
  cfg.blockDim = dim3(kPaThreads);
  cfg.dynamicSmemBytes = C::smem();
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_attn_kernel<HD, Q8, F32, NN>, a);
}
template <int HD, bool Q8, bool F32>
static cudaError_t launch_nn(const PagedAttnArgs& a, const PaPlan& p, cudaStream_t st) {
  if (p.nn == 1) return launch_t<HD, Q8, F32, 1>(a, p, st);
  if constexpr (HD <= 64) {
    if (p.nn == 4) return launch_t<HD, Q8, F32, 4>(a, p, st);
  }
  if constexpr (HD <= 128) return launch_t<HD, Q8, F32, 2>(a, p, st);
  return cudaErrorInvalidValue;  // pick_nn gives no more
}
template <bool Q8, bool F32>
static cudaError_t launch_hd(int hd, const PagedAttnArgs& a, const PaPlan& p, cudaStream_t st) {
  switch (hd) {
    case 32: return launch_nn<32, Q8, F32>(a, p, st);
    case 64: return launch_nn<64, Q8, F32>(a, p, st);
    case 96: return launch_nn<96, Q8, F32>(a, p, st);
    case 128: return launch_nn<128, Q8, F32>(a, p, st);
    default: return launch_nn<256, Q8, F32>(a, p, st);
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
  const int from = tc_from(a.c, a.n, hd, dtype, a.group, max_q, max_kv);
  a.min_new = 0;
  a.max_new = from ? from : 0x7FFFFFFF;
  const PaPlan p = plan_of(a.n, a.n_seqs, a.group, a.c.kv_heads, hd, from ? from - 1 : max_q, max_kv, q8);
  a.n_splits = p.splits;
  a.per_seq = p.per_seq;
  const cudaError_t e = q8 ? (f32 ? launch_hd<true, true>(hd, a, p, st) : launch_hd<true, false>(hd, a, p, st))
                           : (f32 ? launch_hd<false, true>(hd, a, p, st) : launch_hd<false, false>(hd, a, p, st));
  if (e != cudaSuccess) {
    snprintf(msg, ml, "attention_paged launch failed: %s", cudaGetErrorString(e));
    return DRACO_ERR_CUDA;
  }
  if (!from) return DRACO_OK;
  a.per_seq = 0;
  a.min_new = from;
  a.max_new = 0x7FFFFFFF;
  const TcPlan t = paged_attn_tc_plan(a.n, a.n_seqs, a.group, a.c.kv_heads, hd, max_kv);
  return paged_attn_tc_launch(a, hd, t, a.counters + kPagedCounters, st, msg, ml);
}

}  // namespace draco
