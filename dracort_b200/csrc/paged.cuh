// paged.cuh — device view of one layer's paged key/value cache (draco_kv_cache)
// and the 16-byte / 8-byte row accesses shared by its kernels.
//
// A page holds page_size rows of each key/value head, heads outermost:
//   bf16 : [page][kv_head][page_size][head_dim] bf16
//   Q8_0 : per (page, kv_head) page_size * head_dim int8 quants, then
//          page_size * (head_dim / 32) fp16 scales; value = scale * quant.
// Keeping a page's scales behind its quants leaves both 16-byte aligned (a
// 34-byte block is not), so that they move with 16-byte copies.
#pragma once

#include "common.cuh"

namespace draco {

struct PagedView {
  uint8_t* k;
  uint8_t* v;
  const int* table;
  int64_t table_stride;  // entries between two sequences' rows
  int64_t block_bytes;   // bytes of one (page, kv_head)
  int n_seqs, max_pages, n_pages, kv_heads, page_shift, type;
};

__host__ __device__ inline int64_t paged_block_bytes(int type, int page_size, int hd) {
  return type == DRACO_KV_Q8_0 ? (int64_t)page_size * (hd + hd / 16) : (int64_t)page_size * hd * 2;
}

// page of position p of sequence s (p >= 0), or -1: outside the table's width,
// or an entry outside the cache
__device__ __forceinline__ int page_of(const PagedView& c, int s, int p) {
  const int idx = p >> c.page_shift;
  if (idx >= c.max_pages) return -1;
  const int pg = __ldg(c.table + (int64_t)s * c.table_stride + idx);
  return pg >= 0 && pg < c.n_pages ? pg : -1;
}

// values the Q8_0 cache holds are clamped to +-127 * 512, so that scale * quant
// always fits fp16
constexpr float kKvLimit = 65024.f;

__device__ __forceinline__ float bf16lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}

// 8 consecutive activations as fp32 (16 bytes of bf16 or 32 of fp32)
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    x[0] = bf16lo(a.x), x[1] = bf16hi(a.x), x[2] = bf16lo(a.y), x[3] = bf16hi(a.y);
    x[4] = bf16lo(a.z), x[5] = bf16hi(a.z), x[6] = bf16lo(a.w), x[7] = bf16hi(a.w);
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
  }
}

}  // namespace draco
