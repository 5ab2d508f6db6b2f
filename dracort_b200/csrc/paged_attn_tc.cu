// paged_attn_tc.cu — causal attention of long chunks and prompts over the paged
// cache on the 5th-generation tensor cores (tcgen05): bf16 activations,
// head_dim up to 128, bf16 or Q8_0 pages (draco_attention_paged chooses).
//
// Mathematics as in paged_attn.cu: one pass over the keys, S = Q K^T, P =
// exp2(c S - m), O += P V, the reference m raised (and O rescaled) only when
// the row's maximum outgrows it by 2^8.
//
// A CTA holds two tiles of 128 rows (a row is a (token, query head) pair of one
// key/value head, so the heads of a group share the key tiles) and takes the
// keys in steps of 64: while one tile's scores of a step go through the softmax
// warps, the MMAs of the other tile and of the next step run.
//   warps 0-3, 4-7   softmax of tile 0 and 1: a thread owns a row: it reads the
//                    step's 64 scores from tensor memory, forms P and stores it
//                    over them as the A operand of the second product, so P
//                    never goes through shared memory;
//   warp 8           issues the MMAs: per step and row tile P V, then the scores
//                    of the step after next into the columns that P leaves;
//   bf16 pages:      warp 9 loads key and value tiles of 128 page by page with TMA
//                    (128-byte swizzle; a bad page is loaded from past the
//                    end: zeros), warps 10-11 clean the value tiles at the
//                    causal edge (below);
//   Q8_0 pages:      warps 12-19 load quants and scales, and write d * quant as
//                    fp16 (11 bits of its 18) into the same swizzled tiles.
// Tensor memory: two 64-column S / P buffers and an O tile for each row tile;
// shared memory: two Q tiles, two stages of key and value tiles; one CTA per SM.
// Key tiles are read from the L2 by the CTAs of a head, whose row tiles run side
// by side.
//
// What bounds it, head_dim 128: a step of both tiles is 1280 clocks of MMAs (the
// scores' MMAs, 64 columns wide, are fed by shared memory at 48 clocks each where
// 32 would do) and about as many of softmax per tile (64 exponentials a row, a
// quarter of them on the FMA pipe, and the loads and stores of tensor memory);
// with the barriers between the two it takes 1660.  Steps of 128 keys would feed
// the MMAs better, but leave no second buffer of scores.  Four softmax
// warpgroups, turns between the tiles and P formed before the maximum is known
// were no faster.  32 query heads over 8, bf16: four
// prompts of 700-4000 tokens 257 us (805 TFLOP/s of unmasked products); 512
// tokens over 16384 cached 163 us, over Q8_0 210 us, whose tiles are converted
// once per 256 rows; 8192 tokens, 32 heads 521-534 us (1040 TFLOP/s).
//
// Q8_0: operands are fp16, q is scaled per row by a power of two and P by 2^6,
// as in paged_attn.cu.
//
// Rows that see no key of a tile multiply its values by P = 0, so values past
// the end, and values that are not finite in tiles with masked pairs, are
// replaced by zeros in shared memory; the latter are marked, and the rows that
// do see them add their products at the end, element by element.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <cstdio>

#include "internal.h"
#include "paged_attn.cuh"

namespace draco {

constexpr int kTcRows = 128;            // rows of a tile (fewer when the group does not divide 128)
constexpr int kTcKeys = 128;            // keys of a shared-memory tile
constexpr int kTcStep = 64;             // keys of a step: scores, P, second product
constexpr int kTcPoly = 2;              // bf16 pages: of kTcPoly pairs of exponentials one is on the FMA pipe
constexpr uint64_t kTcWaitNs = 2000000000ull;  // 2 s: far beyond any legitimate wait
constexpr int kTcBadWords = 32;         // marks of 1024 keys from the first edge tile on

struct __align__(64) TcParams {
  CUtensorMap qmap, kmap, vmap;
  PagedAttnArgs a;
  int rt;        // rows of a row tile: group * (128 / group)
  int hd;
  int box_rows;  // rows of a TMA box: min(page_size, 128)
  int page_rows; // rows in the key (or value) buffer: pages * kv_heads * page_size
  int by_tokens; // partial results by record_place (else by tile)
  int* status;
};

template <int HDP, bool Q8>
struct TcCfg {
  static constexpr int kBoxes = HDP / 64;
  static constexpr int kHalf = 128 * 128;                 // 128 rows x 64 values
  static constexpr int kTile = kBoxes * kHalf;            // 32 or 16 KB
  static constexpr int kStages = 2;
  static constexpr int kSmem = 1024 + 2 * kTile + kStages * 2 * kTile;
  static constexpr int kThreads = Q8 ? 640 : 384;
  static constexpr int kProducers = 8;                    // Q8_0: converting warps
  // registers of a thread: softmax warpgroups, the MMA / load warpgroup, converting warpgroups
  static constexpr int kRegsSoftmax = Q8 ? 136 : 208, kRegsOne = Q8 ? 64 : 80, kRegsConvert = 72;
  static constexpr int kRegsBlock = 256 * kRegsSoftmax + 128 * kRegsOne + (kThreads - 384) * kRegsConvert;
};

__device__ __forceinline__ void tca_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tca_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tca_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tca_commit(uint32_t one, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
      "r"(one)
      : "memory");
}
// Shared-memory operand with the 128-byte swizzle, rows of 64 values at 128
// bytes, 8-row groups at 1024 (version 1, layout 2).  K-major: rows are M / N,
// values K; MN-major: rows are K, values N, and `lbo` is the distance between
// 64-value groups of N.
__device__ __forceinline__ uint64_t tca_desc(uint32_t addr, uint32_t lbo) {
  return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// the descriptor behind its low word (tca_desc's high word is constant)
__device__ __forceinline__ uint64_t tca_desc_of(uint32_t lo) {
  constexpr uint32_t hi = (1024 >> 4) | (1u << 14) | (2u << 29);
  return ((uint64_t)hi << 32) | lo;
}
// fp32 D; A and B bf16 (format 1) or fp16 (0); bit 16: B is MN-major
__host__ __device__ constexpr uint32_t tca_idesc(bool bf16, int m, int n, bool b_mn) {
  return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(m >> 4) << 24);
}
// (`one`: the lane that issues.  The predicate sits on the instruction, not on a
// branch: in warp-uniform code the operands are computed in uniform registers,
// where a branch of one lane would move each there; 55 clocks an MMA.)
__device__ __forceinline__ void tca_mma_ss(uint32_t one, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(one)
      : "memory");
}
__device__ __forceinline__ void tca_mma_ts(uint32_t one, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(one)
      : "memory");
}
__device__ __forceinline__ void tca_ld32(uint32_t addr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
// waits for this thread's loads; ties 32 of the loaded registers to the wait
__device__ __forceinline__ void tca_ld_wait(float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                 "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31])::"memory");
}
__device__ __forceinline__ void tca_st32(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
      "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
      "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tca_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tca_load_2d(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tca_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ float tca_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void tca_st16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(
          r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(addr)
      : "memory");
}
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t x;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(x));
  return x;
}
// maximum that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// pairs of fp32 values in one register pair
__device__ __forceinline__ uint64_t pair2(float a, float b) {
  return ((uint64_t)__float_as_uint(b) << 32) | __float_as_uint(a);
}
__device__ __forceinline__ float lo_2(uint64_t x) { return __uint_as_float((uint32_t)x); }
__device__ __forceinline__ float hi_2(uint64_t x) { return __uint_as_float((uint32_t)(x >> 32)); }
__device__ __forceinline__ uint64_t fma_2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
// 2^x on the FMA pipe: x = n + f with n the nearest integer (added to 1.5 * 2^23
// it sits in the low bits), 2^f by a cubic fitted to |f| <= 1/2 for the least
// relative error (7.5e-5; P keeps 8 or 11 bits), n added to the exponent (the
// argument reduction of Cody and Waite).  x is raised to -126 at least; not
// for NaN.
constexpr float kP0 = 0.99992806f, kP1 = 0.69326097f, kP2 = 0.24261115f, kP3 = 0.05517165f;
__device__ __forceinline__ float exp2_poly(float x) {
  x = fmaxf(x, -126.f);
  const float n = x + 12582912.f;
  const float f = x - (n - 12582912.f);
  float p = fmaf(kP3, f, kP2);
  p = fmaf(p, f, kP1);
  p = fmaf(p, f, kP0);
  return __uint_as_float(__float_as_uint(p) + (__float_as_uint(n) << 23));
}
template <int N>
__device__ __forceinline__ void regs_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// What a wait that ran out leaves, beside the workspace's word: a workspace may be
// dropped, or zeroed by the next replay of a graph, before anybody asks.
__device__ int tc_status;

struct TcBars {
  uint64_t q_full, q_ready;
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], v_clean[2];
  uint64_t s_full[2][2], p_full[2][2], pv_done[2][2], o_full[2], drain;  // [row tile][step & 1]
};

template <int HDP, bool Q8>
__global__ void __launch_bounds__(TcCfg<HDP, Q8>::kThreads, 1)
    paged_attn_tc_kernel(const __grid_constant__ TcParams P) {
  using C = TcCfg<HDP, Q8>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) TcBars bars;
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort, s_last;
  __shared__ uint32_t s_bad[kTcBadWords];
  const PagedAttnArgs& a = P.a;
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint8_t* q_s = smem;                       // [2] Q tiles
  uint8_t* k_s = smem + 2 * C::kTile;        // [stage] key tiles
  uint8_t* v_s = k_s + C::kStages * C::kTile;
  // (lane 0's values: the compiler sees that the warp shares them)
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  grid_dependency_wait();
  // the tiles with the most keys first, of all heads
  const int tile_id = gridDim.y - 1 - blockIdx.y;
  const RowTile tile = find_tile(a, tile_id, 2 * P.rt);
  if (tile.s < 0) return;
  const int kvh = blockIdx.x % a.c.kv_heads, hd = P.hd;
  const int rows = min(2 * P.rt, tile.rows - tile.row0);
  const int kend = max(0, min(tile.kv, row_limit(a, tile, tile.row0 + rows - 1)));
  int ck = (kend + a.n_splits - 1) / a.n_splits;
  ck = max(kTcKeys, (ck + kTcKeys - 1) & ~(kTcKeys - 1));
  const int active = split_count(kend, ck);
  const int split = blockIdx.x / a.c.kv_heads;
  if (split >= active) return;
  const int kbeg = split * ck, kfin = split_end(kbeg, kend, ck);
  const int nj = __shfl_sync(0xffffffffu, (kfin - kbeg + kTcKeys - 1) / kTcKeys, 0);  // key tiles
  const int ns = __shfl_sync(0xffffffffu, (kfin - kbeg + kTcStep - 1) / kTcStep, 0);  // steps
  // the first tile in which some row is masked (or keys end)
  const int first_lim = max(0, min(tile.kv, row_limit(a, tile, tile.row0)));
  const int jedge = max(0, min(nj, first_lim <= kbeg ? 0 : (first_lim - kbeg) / kTcKeys));

  if (tid == 0) {
    mbar_init(&bars.q_full, 1);
    mbar_init(&bars.q_ready, 8);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.k_full[i], Q8 ? C::kProducers : 1);
      mbar_init(&bars.v_full[i], Q8 ? C::kProducers : 1);
      mbar_init(&bars.k_empty[i], 1);
      mbar_init(&bars.v_empty[i], 1);
      for (int h = 0; h < 2; ++h) {
        mbar_init(&bars.s_full[i][h], 1);
        mbar_init(&bars.p_full[i][h], 4);
        mbar_init(&bars.pv_done[i][h], 1);
      }
      mbar_init(&bars.o_full[i], 1);
      mbar_init(&bars.v_clean[i], 2);
    }
    mbar_init(&bars.drain, 1);
    fence_mbar_init();
    s_abort = 0;
  }
  if (tid < kTcBadWords) s_bad[tid] = 0;
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tca_before();
  __syncthreads();
  tca_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0);

  // a wait that gives up: the role leaves its loop, the others' waits run out
  // too.  (A wait names a phase by its parity: no barrier completes two phases
  // more before the waiting side has passed.)
  auto wait = [&](uint64_t* bar, int phase) -> bool {
    if (mbar_wait_bounded(bar, (uint32_t)phase & 1u, kTcWaitNs)) return true;
    s_abort = 1;
    return false;
  };
  auto wait_fast = [&](uint64_t* bar, int phase) -> bool {  // the whole warp; one vote when the phase is over
    const bool done = mbar_try_wait(bar, (uint32_t)phase & 1u);
    if (__all_sync(0xffffffffu, done)) return true;
    return __all_sync(0xffffffffu, wait(bar, phase));
  };
  auto wait_warp = [&](uint64_t* bar, int phase) -> bool {
    return __all_sync(0xffffffffu, wait(bar, phase));
  };

  // registers by warpgroup: the sums stay within what the block is launched with
  if (warp < 8)
    regs_up<C::kRegsSoftmax>();
  else if (warp < 12)
    regs_down<C::kRegsOne>();
  else
    regs_down<C::kRegsConvert>();

  if (warp < 8) {
    // ------------------------------------------------------------- softmax
    const int w = warp >> 2, rw = 32 * (warp & 3) + lane;  // row of the tile
    const int r = w * P.rt + rw;                           // row of the CTA
    const bool valid = rw < P.rt && r < rows;
    const int lim = valid ? max(0, min(tile.kv, row_limit(a, tile, tile.row0 + r))) : 0;
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t s_t = tmem + 128 * w + lanes, o_t = tmem + 256 + HDP * w + lanes;
    float sc = a.scale_log2;
    bool ok = true;
    if constexpr (Q8) {
      // q as fp16, scaled by a power of two to at most 1 per row
      ok = nj == 0 || wait_warp(&bars.q_full, 0);
      if (ok && nj > 0) {
        uint8_t* row = q_s + w * C::kTile + rw * 128;
        float m = 0.f;
#pragma unroll 1
        for (int c = 0; c < HDP / 8; ++c) {
          const uint4 u = *reinterpret_cast<const uint4*>(row + (c >> 3) * C::kHalf + (((c & 7) ^ (rw & 7)) << 4));
          m = fmaxf(fmaxf(fmaxf(m, fmaxf(fabsf(bf16lo(u.x)), fabsf(bf16hi(u.x)))),
                          fmaxf(fabsf(bf16lo(u.y)), fabsf(bf16hi(u.y)))),
                    fmaxf(fmaxf(fabsf(bf16lo(u.z)), fabsf(bf16hi(u.z))),
                          fmaxf(fabsf(bf16lo(u.w)), fabsf(bf16hi(u.w)))));
        }
        float s = 1.f;
        if (m > 1e-30f && m < 1e38f) s = __int_as_float((__float_as_int(m) & 0x7F800000) + 0x00800000);
        const float inv = 1.f / s;
        sc *= s;
#pragma unroll 1
        for (int c = 0; c < HDP / 8; ++c) {
          uint4* p = reinterpret_cast<uint4*>(row + (c >> 3) * C::kHalf + (((c & 7) ^ (rw & 7)) << 4));
          const uint4 u = *p;
          *p = make_uint4(pack_f16(bf16lo(u.x) * inv, bf16hi(u.x) * inv), pack_f16(bf16lo(u.y) * inv, bf16hi(u.y) * inv),
                          pack_f16(bf16lo(u.z) * inv, bf16hi(u.z) * inv), pack_f16(bf16lo(u.w) * inv, bf16hi(u.w) * inv));
        }
        tca_proxy();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.q_ready);
      }
    }
    constexpr float kShift = Q8 ? 6.f : 0.f;
    float m = -INFINITY, l = 0.f;
    // the exponents are slope s - ref, and m grows when scores outgrow `most`: what
    // follows from m, set where m is
    float ref = 0.f, slope = sc, most = -INFINITY;
    for (int i = 0; i < ns && ok; ++i) {
      if (!(ok = wait_warp(&bars.s_full[w][i & 1], i >> 1))) break;
      tca_after();
      const uint32_t s_i = s_t + kTcStep * (i & 1);
      const int vis = lim - (kbeg + i * kTcStep);  // columns that the row sees
      float s[kTcStep];
      tca_ld32(s_i, s);
      tca_ld32(s_i + 32, s + 32);
      tca_ld_wait(s);
      tca_ld_wait(s + 32);
      const bool edge = __any_sync(0xffffffffu, vis < kTcStep);
      if (edge) {
#pragma unroll
        for (int e = 0; e < kTcStep; ++e) s[e] = e < vis ? s[e] : -INFINITY;
      }
      float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
      for (int e = 0; e < kTcStep; e += 4) {
        x0 = max_nan(x0, s[e], s[e + 1]);
        x1 = max_nan(x1, s[e + 2], s[e + 3]);
      }
      const float mx = max_nan(x0, x1, x1) * sc;
      if (__any_sync(0xffffffffu, !(mx <= most))) {
        const float n = max_nan(m, mx, mx);
        const float f = n == -INFINITY ? 1.f : tca_exp2(m - n);
        m = n;
        l *= f;
        // (a row with an infinite score is NaN, as inf - inf)
        ref = m == -INFINITY ? 0.f : m == INFINITY ? __int_as_float(0x7FC00000) : m - kShift;
        slope = sc, most = m + kPaLazy;
        if (__any_sync(0xffffffffu, is_huge(m))) {  // ... and so on every step from here
#pragma unroll
          for (int e = 0; e < kTcStep; ++e) s[e] = huge_exponent(s[e], sc, m);
          ref = -kShift, slope = 1.f, most = __int_as_float(0x7FC00000);
        }
        if (i > 0) {  // O of the steps so far, once their products are done
          if (!(ok = wait_warp(&bars.pv_done[w][(i - 1) & 1], (i - 1) >> 1))) break;
          tca_after();
#pragma unroll 1
          for (int c = 0; c < HDP / 32; ++c) {
            float o[32];
            tca_ld32(o_t + 32 * c, o);
            tca_ld_wait(o);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] *= f;
            tca_st32(o_t + 32 * c, reinterpret_cast<uint32_t*>(o));
          }
        }
      }
      const uint64_t sc2 = pair2(slope, slope), ref2 = pair2(-ref, -ref);
      float l0 = 0.f, l1 = 0.f;
      // P.  A quarter of the exponentials go to the FMA pipe over bf16 pages (four
      // prompts 268 -> 257 us); over Q8_0, whose converters use that pipe, none
      // (512 tokens over 16384: 210 us, 228 with a quarter).
      auto form = [&](auto poly) {
#pragma unroll
        for (int c = 0; c < kTcStep / 32; ++c) {
          uint32_t p[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const uint64_t x = fma_2(pair2(s[32 * c + 2 * e], s[32 * c + 2 * e + 1]), sc2, ref2);
            const float u = tca_exp2(lo_2(x));
            const float v = decltype(poly)::value && !Q8 && e % kTcPoly == 1 ? exp2_poly(hi_2(x)) : tca_exp2(hi_2(x));
            l0 += u, l1 += v;
            p[e] = Q8 ? pack_f16(u, v) : pack_bf16(u, v);
          }
          tca_st16(s_i + 16 * c, p);
        }
      };
      if (edge)
        form(std::false_type());
      else
        form(std::true_type());
      l += l0 + l1;
      tca_st_wait();
      tca_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.p_full[w][i & 1]);
    }
    if (ok && ns > 0) ok = wait_warp(&bars.o_full[w], 0);
    tca_after();
    // marked values: what the rows that see them add
    uint32_t any_bad = 0;
#pragma unroll 1
    for (int i = 0; i < kTcBadWords; ++i) any_bad |= s_bad[i];
    const int rr = tile.row0 + r;
    const int64_t place = P.by_tokens ? record_place(tile.start, tile.row0, a.group, 2 * P.rt, a.min_new) : tile_id;
    const int64_t unit = place * a.c.kv_heads + kvh;
    float* rec = a.recs + (unit * a.n_splits + split) * (int64_t)(2 * P.rt) * (hd + 2);
    __nv_bfloat16* orow = static_cast<__nv_bfloat16*>(a.out) + (int64_t)(tile.start + rr / a.group) * a.ldo +
                          (int64_t)(kvh * a.group + rr % a.group) * hd;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (ok) {
#pragma unroll 1
      for (int c = 0; c < HDP / 32 && 32 * c < hd; ++c) {
        __syncwarp();
        float o[32];
        if (nj > 0) {
          tca_ld32(o_t + 32 * c, o);
          tca_ld_wait(o);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0.f;
        }
        if (any_bad != 0 && valid) {
          const uint8_t* qrow = q_s + w * C::kTile + rw * 128;
#pragma unroll 1
          for (int b = 0; b < kTcBadWords * 32; ++b) {
            if (!((s_bad[b >> 5] >> (b & 31)) & 1u)) continue;
            const int key = kbeg + jedge * kTcKeys + b;
            if (key >= lim) break;
            const int page = page_of(a.c, tile.s, key), off = key & ((1 << a.c.page_shift) - 1);
            const int64_t at = ((int64_t)page * a.c.kv_heads + kvh) * a.c.block_bytes;
            float dot = 0.f;
#pragma unroll 1
            for (int d = 0; d < hd; ++d) {
              const uint16_t qb = *reinterpret_cast<const uint16_t*>(
                  qrow + (d >> 6) * C::kHalf + ((((d >> 3) & 7) ^ (rw & 7)) << 4) + 2 * (d & 7));
              float kv;
              if constexpr (Q8)
                kv = __half2float(reinterpret_cast<const __half*>(a.c.k + at + ((int64_t)hd << a.c.page_shift))
                                      [off * (hd / 32) + d / 32]) *
                     (float)reinterpret_cast<const int8_t*>(a.c.k + at)[off * hd + d];
              else
                kv = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(a.c.k + at)[off * hd + d]);
              dot = fmaf(Q8 ? __half2float(__ushort_as_half(qb)) : __uint_as_float((uint32_t)qb << 16), kv, dot);
            }
            const float p = tca_exp2(fmaf(dot, sc, -(m == -INFINITY ? 0.f : m - kShift)));
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const int d = 32 * c + i;
              float v;
              if constexpr (Q8)
                v = __half2float(reinterpret_cast<const __half*>(a.c.v + at + ((int64_t)hd << a.c.page_shift))
                                     [off * (hd / 32) + d / 32]) *
                    (float)reinterpret_cast<const int8_t*>(a.c.v + at)[off * hd + d];
              else
                v = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(a.c.v + at)[off * hd + d]);
              if (!(fabsf(v) < INFINITY)) o[i] = fmaf(p, v, o[i]);
            }
          }
        }
        if (valid && active == 1) {
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = l == 0.f ? 0.f : o[i + e] * inv;
            store8(orow + 32 * c + i, x);
          }
        } else if (valid) {
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            __stcg(reinterpret_cast<float4*>(rec + 4 * P.rt + (int64_t)r * hd + 32 * c + i),
                   make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]));
          if (c == 0) __stcg(reinterpret_cast<float2*>(rec + 2 * r), make_float2(m, l));
        }
      }
    }
    if (active > 1) {
      __threadfence();  // this thread's record before the arrival
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (tid == 0) {
        s_last = 0;
        if (!s_abort) {
          const int prev = atomicAdd(a.counters + unit, 1);
          s_last = prev == active - 1;
          if (s_last) {
            atomicExch(a.counters + unit, 0);
            __threadfence();
          }
        }
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");
      {
        if (s_last && valid) {
          const int64_t rsz = (int64_t)(2 * P.rt) * (hd + 2);
          const float* recs = a.recs + unit * a.n_splits * rsz;
          float M = -INFINITY, L = 0.f;
          for (int sp = 0; sp < active; ++sp) M = fmaxf(M, __ldcg(recs + sp * rsz + 2 * r));
          for (int sp = 0; sp < active; ++sp) {
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(recs + sp * rsz + 2 * r));
            if (ml.x == -INFINITY && ml.y == ml.y) continue;
            L = fmaf(ml.x == -INFINITY ? 0.f : tca_exp2(ml.x - M), ml.y, L);
          }
          const float iv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll 1
          for (int d = 0; d < hd; d += 8) {
            float x[8] = {};
#pragma unroll 1
            for (int sp = 0; sp < active; ++sp) {
              const float* rc = recs + sp * rsz;
              const float2 ml = __ldcg(reinterpret_cast<const float2*>(rc + 2 * r));
              if (ml.x == -INFINITY && ml.y == ml.y) continue;
              const float f = ml.x == -INFINITY ? 0.f : tca_exp2(ml.x - M);
              const float4 u = __ldcg(reinterpret_cast<const float4*>(rc + 4 * P.rt + (int64_t)r * hd + d));
              const float4 v = __ldcg(reinterpret_cast<const float4*>(rc + 4 * P.rt + (int64_t)r * hd + d + 4));
              x[0] = fmaf(f, u.x, x[0]), x[1] = fmaf(f, u.y, x[1]), x[2] = fmaf(f, u.z, x[2]), x[3] = fmaf(f, u.w, x[3]);
              x[4] = fmaf(f, v.x, x[4]), x[5] = fmaf(f, v.y, x[5]), x[6] = fmaf(f, v.z, x[6]), x[7] = fmaf(f, v.w, x[7]);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = L == 0.f ? 0.f : x[e] * iv;
            store8(orow + d, x);
          }
        }
      }
    }
    tca_before();
  } else if (warp == 8) {
    // ------------------------------------------------------------- MMA
    // the whole warp runs the loop, one lane issues: operands stay warp-uniform
    // (a lane of its own would move each to a uniform register first)
    if (nj > 0) {
      const uint32_t one = elect_one();
      constexpr uint32_t ids = tca_idesc(!Q8, 128, kTcStep, false), ido = tca_idesc(!Q8, 128, HDP, true);
      // low words of the operand descriptors (address / 16 and the leading offset);
      // the high word is the same for all
      const uint32_t q_d = (uint32_t)tca_desc(smem_u32(q_s), 16), k_d = (uint32_t)tca_desc(smem_u32(k_s), 16),
                     v_d = (uint32_t)tca_desc(smem_u32(v_s), C::kHalf);
      constexpr uint32_t kTile16 = C::kTile >> 4, kStep16 = kTcStep * 128 >> 4;
      // The loop is written out by step parity and row tile: what a step needs
      // beside its MMAs is a dozen instructions, since this one warp's
      // instruction latency would otherwise be what the tensor core waits for.
      auto scores = [&](auto wc, auto hc, int j, bool last) {  // half h of key tile j
        constexpr int w = decltype(wc)::value, h = decltype(hc)::value;
        const uint32_t ka = k_d + (j & 1) * kTile16 + h * kStep16;
#pragma unroll
        for (int k = 0; k < HDP / 16; ++k) {
          const uint32_t at = ((k >> 2) * C::kHalf + (k & 3) * 32) >> 4;
          tca_mma_ss(one, tmem + 128 * w + kTcStep * h, tca_desc_of(q_d + w * kTile16 + at), tca_desc_of(ka + at), ids,
                     k > 0);
        }
        tca_commit(one, &bars.s_full[w][h]);
        if (w == 1 && (h == 1 || last)) tca_commit(one, &bars.k_empty[j & 1]);
      };
      auto outputs = [&](auto wc, auto hc, int j, bool last) {
        constexpr int w = decltype(wc)::value, h = decltype(hc)::value;
        const uint32_t va = v_d + (j & 1) * kTile16 + h * kStep16;
#pragma unroll
        for (int k = 0; k < kTcStep / 16; ++k)
          tca_mma_ts(one, tmem + 256 + HDP * w, tmem + 128 * w + kTcStep * h + 8 * k, tca_desc_of(va + k * (2048 >> 4)),
                     ido, h > 0 || k > 0 || j > 0);
        tca_commit(one, &bars.pv_done[w][h]);
        if (last) tca_commit(one, &bars.o_full[w]);
        if (w == 1 && (h == 1 || last)) tca_commit(one, &bars.v_empty[j & 1]);
      };
      using I0 = std::integral_constant<int, 0>;
      using I1 = std::integral_constant<int, 1>;
      bool ok = wait_fast(Q8 ? &bars.q_ready : &bars.q_full, 0) && wait_fast(&bars.k_full[0], 0);
      if (ok) {
        tca_after();
        scores(I0(), I0(), 0, ns == 1), scores(I1(), I0(), 0, ns == 1);
        if (ns > 1) scores(I0(), I1(), 0, false), scores(I1(), I1(), 0, false);
      }
      auto step = [&](auto wc, auto hc, int j) -> bool {
        constexpr int w = decltype(wc)::value, h = decltype(hc)::value;
        const int i = 2 * j + h;
        if (!wait_fast(&bars.p_full[w][h], j)) return false;
        tca_after();
        outputs(wc, hc, j, i == ns - 1);
        if (i + 2 < ns) {
          if (w == 0 && h == 0 && !wait_fast(&bars.k_full[(j + 1) & 1], (j + 1) >> 1)) return false;
          scores(wc, hc, j + 1, i + 2 == ns - 1);
        }
        return true;
      };
#pragma unroll 1
      for (int j = 0; j < nj && ok; ++j) {
        ok = wait_fast(Q8 ? &bars.v_full[j & 1] : &bars.v_clean[j & 1], j >> 1) && step(I0(), I0(), j) &&
             step(I1(), I0(), j);
        if (ok && 2 * j + 1 < ns) ok = step(I0(), I1(), j) && step(I1(), I1(), j);
      }
      if (!ok) {
        // the MMAs issued so far finish before shared and tensor memory are given up
        tca_commit(one, &bars.drain);
        mbar_wait_bounded(&bars.drain, 0, kTcWaitNs);
      }
    }
    __syncwarp();
    tca_before();
  } else if (warp < 12) {
    if (warp == 9) {
      // ----------------------------------------------------------- loads
      if (lane == 0 && nj > 0) {
        mbar_arrive_expect_tx(&bars.q_full, 2 * C::kBoxes * P.rt * 128);
        const int tok = tile.start + tile.row0 / a.group;
        for (int w = 0; w < 2; ++w)
          for (int b = 0; b < C::kBoxes; ++b)
            tca_load_3d(q_s + w * C::kTile + b * C::kHalf, &P.qmap, 64 * b, kvh * a.group,
                        tok + w * (P.rt / a.group), &bars.q_full);
      }
      if constexpr (!Q8) {
        // lane i holds the page of the tile's i-th box
        const int per = kTcKeys / P.box_rows;
        bool ok = true;
        int j = 0;
        for (; j < nj; ++j) {
          const int st = j & 1, k0 = kbeg + j * kTcKeys;
          const int key = k0 + lane * P.box_rows;
          int row = P.page_rows;  // past the end: zeros
          if (lane < per && key < kfin) {
            const int page = page_of(a.c, tile.s, key);
            if (page >= 0)
              row = ((page * a.c.kv_heads + kvh) << a.c.page_shift) + (key & ((1 << a.c.page_shift) - 1));
          }
          if (j >= 2) ok = wait_warp(&bars.k_empty[st], (j >> 1) - 1);
          if (!ok) break;
          if (lane == 0) mbar_arrive_expect_tx(&bars.k_full[st], C::kTile);
          __syncwarp();
          if (lane < per)
            for (int b = 0; b < C::kBoxes; ++b)
              tca_load_2d(k_s + st * C::kTile + b * C::kHalf + lane * P.box_rows * 128, &P.kmap, 64 * b, row,
                          &bars.k_full[st]);
          if (j >= 2) ok = wait_warp(&bars.v_empty[st], (j >> 1) - 1);
          if (!ok) break;
          if (lane == 0) mbar_arrive_expect_tx(&bars.v_full[st], C::kTile);
          __syncwarp();
          if (lane < per)
            for (int b = 0; b < C::kBoxes; ++b)
              tca_load_2d(v_s + st * C::kTile + b * C::kHalf + lane * P.box_rows * 128, &P.vmap, 64 * b, row,
                          &bars.v_full[st]);
        }
        if (!ok && lane == 0) {  // copies in flight land before the CTA leaves
          for (int jj = max(0, j - 1); jj <= j; ++jj) {
            mbar_wait_bounded(&bars.k_full[jj & 1], (jj >> 1) & 1, kTcWaitNs);
            if (jj < j) mbar_wait_bounded(&bars.v_full[jj & 1], (jj >> 1) & 1, kTcWaitNs);
          }
        }
      }
      __syncwarp();
    } else if constexpr (!Q8) {
      // ----------------------------------------------------------- value tiles at the edge
      bool ok = true;
      const int t = tid - 320;  // 64 threads: two rows each
      for (int j = 0; j < nj && ok; ++j) {
        if (!(ok = wait_warp(&bars.v_full[j & 1], j >> 1))) break;
        if (j < jedge) {
          if (lane == 0) mbar_arrive(&bars.v_clean[j & 1]);
          continue;
        }
        const int k0 = kbeg + j * kTcKeys;
        uint8_t* tile_s = v_s + (j & 1) * C::kTile;
#pragma unroll 1
        for (int rr = t; rr < kTcKeys; rr += 64) {
          bool bad = false;
#pragma unroll 1
          for (int c = 0; c < HDP / 8; ++c) {
            uint4* p = reinterpret_cast<uint4*>(tile_s + (c >> 3) * C::kHalf + rr * 128 + (((c & 7) ^ (rr & 7)) << 4));
            if (k0 + rr >= kfin) {
              *p = make_uint4(0, 0, 0, 0);
              continue;
            }
            uint4 u = *p;
            bool hit = false;
            auto clean = [&](uint32_t& x) {
              if ((x & 0x7F80u) == 0x7F80u) x &= 0xFFFF0000u, hit = true;
              if ((x & 0x7F800000u) == 0x7F800000u) x &= 0xFFFFu, hit = true;
            };
            clean(u.x), clean(u.y), clean(u.z), clean(u.w);
            if (hit) *p = u, bad = true;
          }
          const int b = (j - jedge) * kTcKeys + rr;
          if (bad && b < kTcBadWords * 32) atomicOr(&s_bad[b >> 5], 1u << (b & 31));
        }
        tca_proxy();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.v_clean[j & 1]);
      }
    }
  } else {
    // --------------------------------------------------------------- Q8_0 tiles
    if constexpr (Q8) {
      // 16 values of a key per lane, the lanes of a warp on contiguous keys: 16-byte
      // loads of whole lines, and 16-byte stores of which eight lanes cover all
      // banks (a lane's two chunks go in the order that its place asks for)
      constexpr int kPer = HDP / 16;               // lanes of a key
      constexpr int kKeysPass = 256 / kPer;        // keys that the 8 warps take at a time
      constexpr int kPass = kTcKeys / kKeysPass;   // 4 or 2
      const int pt = tid - 384, piece = pt % kPer, d0 = 16 * piece, key_l = pt / kPer;
      const bool on_d = d0 < hd;
      // keys and values in registers of their own, loaded a tile ahead, and the
      // tile's pages before that: a tile's conversion never waits for a chain of
      // loads
      uint4 kq[kPass], vq[kPass];
      uint32_t ksc[kPass], vsc[kPass];
      int pages[kPass];
      auto look = [&](int j) {
#pragma unroll
        for (int i = 0; i < kPass; ++i) {
          const int key = kbeg + j * kTcKeys + i * kKeysPass + key_l;
          pages[i] = on_d && j < nj && key < kfin ? page_of(a.c, tile.s, key) : -1;
        }
      };
      auto fetch = [&](const uint8_t* base, int j, uint4 (&qv)[kPass], uint32_t (&sv)[kPass]) {
#pragma unroll
        for (int i = 0; i < kPass; ++i) {
          qv[i] = make_uint4(0, 0, 0, 0);
          sv[i] = 0;
          if (pages[i] >= 0) {
            const int off = (kbeg + j * kTcKeys + i * kKeysPass + key_l) & ((1 << a.c.page_shift) - 1);
            const uint8_t* blk = base + ((int64_t)pages[i] * a.c.kv_heads + kvh) * a.c.block_bytes;
            qv[i] = __ldg(reinterpret_cast<const uint4*>(blk + off * hd + d0));
            sv[i] = __ldg(reinterpret_cast<const uint16_t*>(blk + (hd << a.c.page_shift)) + off * (hd / 32) + (d0 >> 5));
          }
        }
      };
      auto put = [&](uint8_t* tile_s, const uint4 (&qv)[kPass], const uint32_t (&sv)[kPass]) {
        const int c0 = (d0 >> 3) & 7, flip = (piece ^ (piece >> 2)) & 1;
#pragma unroll
        for (int i = 0; i < kPass; ++i) {
          const uint32_t d = sv[i] * 0x10001u;
          const __half2 d2 = *reinterpret_cast<const __half2*>(&d);
          const uint32_t ws[4] = {qv[i].x ^ 0x80808080u, qv[i].y ^ 0x80808080u, qv[i].z ^ 0x80808080u,
                                  qv[i].w ^ 0x80808080u};
          uint32_t o[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint32_t x = __byte_perm(ws[e >> 1], 0x64646464u, (e & 1) ? 0x4342 : 0x4140), c = 0x64806480u;
            const __half2 h = __hmul2_rn(__hsub2_rn(*reinterpret_cast<const __half2*>(&x),
                                                    *reinterpret_cast<const __half2*>(&c)), d2);
            o[e] = *reinterpret_cast<const uint32_t*>(&h);
          }
          const int row = i * kKeysPass + key_l;
          uint8_t* base = tile_s + (d0 >> 6) * C::kHalf + row * 128;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int second = e ^ flip;
            *reinterpret_cast<uint4*>(base + (((c0 + second) ^ (row & 7)) << 4)) =
                second ? make_uint4(o[4], o[5], o[6], o[7]) : make_uint4(o[0], o[1], o[2], o[3]);
          }
        }
      };
      bool ok = true;
      look(0);
      fetch(a.c.k, 0, kq, ksc);
      fetch(a.c.v, 0, vq, vsc);
      look(1);
      for (int j = 0; j < nj && ok; ++j) {
        const int st = j & 1;
        if (j >= 2 && !(ok = wait_warp(&bars.k_empty[st], (j >> 1) - 1))) break;
        put(k_s + st * C::kTile, kq, ksc);
        fetch(a.c.k, j + 1, kq, ksc);
        tca_proxy();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.k_full[st]);
        if (j >= 2 && !(ok = wait_warp(&bars.v_empty[st], (j >> 1) - 1))) break;
        if (j >= jedge) {
#pragma unroll
          for (int i = 0; i < kPass; ++i) {
            const int b = (j - jedge) * kTcKeys + i * kKeysPass + key_l;
            if ((vsc[i] & 0x7C00u) == 0x7C00u) {
              vsc[i] = 0;
              if (b < kTcBadWords * 32) atomicOr(&s_bad[b >> 5], 1u << (b & 31));
            }
          }
        }
        put(v_s + st * C::kTile, vq, vsc);
        fetch(a.c.v, j + 1, vq, vsc);
        look(j + 2);
        tca_proxy();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.v_full[st]);
      }
    }
  }
  __syncthreads();
  if (s_abort && tid == 0) {
    atomicExch(P.status, DRACO_ERR_TIMEOUT);
    atomicExch(&tc_status, DRACO_ERR_TIMEOUT);
    if (nj > 0) mbar_wait_bounded(&bars.q_full, 0, kTcWaitNs);
  }
  if (warp == 8) {
    tca_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
static PFN_cuTensorMapEncodeTiled_v12000 tc_encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  if (!fn) {
    cudaDriverEntryPointQueryResult q;
    void* p = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }
  return fn;
}

bool paged_attn_tc_takes(const PagedView& c, int hd, int dtype, int group, int page_size) {
  if (dtype != DRACO_DTYPE_BF16 || hd > 128 || group > kTcRows) return false;
  // TMA row coordinates are 32-bit
  return c.type == DRACO_KV_Q8_0 || (int64_t)c.n_pages * c.kv_heads * page_size < 0x7FFFFF00ll;
}

TcPlan paged_attn_tc_plan(int n, int n_seqs, int group, int kv_heads, int hd, int max_kv) {
  TcPlan p;
  p.rt = group * (kTcRows / group);
  p.tiles = (int64_t)n * group / (2 * p.rt) + n_seqs;
  // Partial results take 256 rows of fp32 a place: of many sequences few are long
  // enough for this kernel (200 steps beside a chunk of 512 tokens, 8 heads of 128:
  // 115 MB, where a place for every tile would take 1.95 GB).
  const int64_t by_tokens = record_places(n, group, 2 * p.rt, tc_min_tokens(group));
  p.by_tokens = by_tokens < p.tiles;
  p.units = std::min(by_tokens, p.tiles) * kv_heads;
  // One CTA per SM: when the row tiles leave SMs idle, as many splits as fit
  // one wave.  A split's partial rows cost a round trip through the L2, so a
  // second wave of splits never pays.
  const int64_t full = (int64_t)n * group / (2 * p.rt) * kv_heads;  // tiles that surely have rows
  int64_t s = full > 0 ? device_sm_count() / full : 1;
  s = std::min<int64_t>(s, ((int64_t)max_kv + 4 * kTcKeys - 1) / (4 * kTcKeys));
  p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(s, 32));
  if (p.units > kPagedCounters) p.splits = 1;
  p.bytes = p.splits > 1 ? (size_t)p.units * p.splits * (2 * p.rt) * (hd + 2) * sizeof(float) : 0;
  return p;
}

cudaError_t paged_attn_status(int replace, int* status) {
  cudaError_t e = cudaMemcpyFromSymbol(status, tc_status, sizeof(int));
  if (e == cudaSuccess && *status != replace) e = cudaMemcpyToSymbol(tc_status, &replace, sizeof(int));
  return e;
}

template <int HDP, bool Q8>
static cudaError_t tc_launch(const TcParams& P, const TcPlan& p, cudaStream_t st) {
  using C = TcCfg<HDP, Q8>;
  static int attr_set[64] = {0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !attr_set[dev]) {
    cudaError_t e = cudaFuncSetAttribute(paged_attn_tc_kernel<HDP, Q8>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         C::kSmem);
    if (e != cudaSuccess) return e;
    // the warpgroups' register counts are drawn from the block's: with fewer
    // registers than that the increase would wait for good
    cudaFuncAttributes fa;
    e = cudaFuncGetAttributes(&fa, paged_attn_tc_kernel<HDP, Q8>);
    if (e != cudaSuccess) return e;
    if (fa.numRegs * C::kThreads < C::kRegsBlock) return cudaErrorInvalidConfiguration;
    if (dev < 64) attr_set[dev] = 1;
  }
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(P.a.c.kv_heads * p.splits), (unsigned)p.tiles);
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_attn_tc_kernel<HDP, Q8>, P);
}

int paged_attn_tc_launch(const PagedAttnArgs& a, int hd, const TcPlan& p, int* status, cudaStream_t st, char* msg,
                         size_t ml) {
  auto enc = tc_encode_fn();
  if (!enc) {
    snprintf(msg, ml, "attention_paged: cuTensorMapEncodeTiled unavailable");
    return DRACO_ERR_CUDA;
  }
  TcParams P;
  P.a = a;
  P.a.n_splits = p.splits;
  P.by_tokens = p.by_tokens;
  P.rt = p.rt;
  P.hd = hd;
  P.status = status;
  const int page_size = 1 << a.c.page_shift;
  P.box_rows = std::min(page_size, kTcKeys);
  const bool q8 = a.c.type == DRACO_KV_Q8_0;
  // q [n][heads][hd]: 64 values x the group's heads x the tile's tokens
  cuuint64_t qdim[3] = {(cuuint64_t)hd, (cuuint64_t)a.heads, (cuuint64_t)a.n};
  cuuint64_t qstr[2] = {(cuuint64_t)hd * 2, (cuuint64_t)a.ldq * 2};
  cuuint32_t qbox[3] = {64, (cuuint32_t)a.group, (cuuint32_t)(p.rt / a.group)};
  cuuint32_t one[3] = {1, 1, 1};
  CUresult r = enc(&P.qmap, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(a.q), qdim, qstr, qbox, one,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  P.page_rows = 0;
  if (!q8 && r == CUDA_SUCCESS) {
    P.page_rows = a.c.n_pages * a.c.kv_heads * page_size;
    cuuint64_t dim[2] = {(cuuint64_t)hd, (cuuint64_t)P.page_rows};
    cuuint64_t str[1] = {(cuuint64_t)hd * 2};
    cuuint32_t box[2] = {64, (cuuint32_t)P.box_rows};
    for (int i = 0; i < 2 && r == CUDA_SUCCESS; ++i)
      r = enc(i ? &P.vmap : &P.kmap, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, i ? a.c.v : a.c.k, dim, str, box, one,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  } else {
    P.kmap = P.qmap;
    P.vmap = P.qmap;
  }
  if (r != CUDA_SUCCESS) {
    snprintf(msg, ml, "attention_paged: cuTensorMapEncodeTiled failed (%d)", (int)r);
    return DRACO_ERR_ARG;
  }
  const cudaError_t e = hd <= 64 ? (q8 ? tc_launch<64, true>(P, p, st) : tc_launch<64, false>(P, p, st))
                                 : (q8 ? tc_launch<128, true>(P, p, st) : tc_launch<128, false>(P, p, st));
  if (e != cudaSuccess) {
    snprintf(msg, ml, "attention_paged launch failed: %s", cudaGetErrorString(e));
    return DRACO_ERR_CUDA;
  }
  return DRACO_OK;
}

}  // namespace draco
