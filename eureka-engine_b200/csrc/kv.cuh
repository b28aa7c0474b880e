// kv.cuh -- the paged key-value cache on the device: where a slot lies, which rows a call has, what a row sees.
#pragma once
#include <cuda_bf16.h>

#include "common.cuh"

// bits of the error word (llb_b200_kv_errors)
#define KV_ERR_PAGE 1u
#define KV_ERR_LEN 2u
#define KV_ERR_ROWS 4u

struct KvDev {
  uint16_t *k, *v;             // [n_pages][KV][page][hd]
  const int *table, *lens;
  int KV, page_sh, n_pages, seqs, tstride;
  int cap;                     // the most slots of a sequence
  unsigned int *err;
};
struct KvRows { const int *start; int rows, max_rows; };

// 16-bit types: a value, and two in a word
template <typename T> struct KvEl;
template <> struct KvEl<__half> {
  static __device__ __forceinline__ float to(uint16_t v) { return __half2float(__ushort_as_half(v)); }
  static __device__ __forceinline__ uint16_t of(float v) { return __half_as_ushort(__float2half_rn(v)); }
  static __device__ __forceinline__ float2 to2(uint32_t v) { return __half22float2(*(const __half2 *)&v); }
  static __device__ __forceinline__ uint32_t of2(float a, float b) { const __half2 h = __floats2half2_rn(a, b); return *(const uint32_t *)&h; }
};
template <> struct KvEl<__nv_bfloat16> {
  static __device__ __forceinline__ float to(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
  static __device__ __forceinline__ uint16_t of(float v) { return __bfloat16_as_ushort(__float2bfloat16_rn(v)); }
  static __device__ __forceinline__ float2 to2(uint32_t v) { return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u)); }
  static __device__ __forceinline__ uint32_t of2(float a, float b) { const __nv_bfloat162 h = __floats2bfloat162_rn(a, b); return *(const uint32_t *)&h; }
};

// slots of sequence b, cut to what the table (or the call) holds
__device__ __forceinline__ int kv_len(const KvDev &c, int b) {
  const int n = __ldcg(c.lens + b);
  if (n >= 0 && n <= c.cap) return n;
  atomicOr(c.err, KV_ERR_LEN);
  return n < 0 ? 0 : c.cap;
}
// the page with entry i of sequence b, or -1 where the entry is no page of the pool
__device__ __forceinline__ int kv_page(const KvDev &c, int b, int i) {
  const int id = __ldcg(c.table + (size_t)b * c.tstride + i);
  if ((unsigned)id < (unsigned)c.n_pages) return id;
  atomicOr(c.err, KV_ERR_PAGE);
  return -1;
}
// elements from the pool's start to the first slot of kv head g in a page
__device__ __forceinline__ size_t kv_at(const KvDev &c, int id, int g, int hd) { return (((size_t)id * c.KV + g) << c.page_sh) * hd; }
// first row and number of rows of sequence b; none where they do not lie within the call's
__device__ __forceinline__ int kv_rows(const KvDev &c, const KvRows &r, int b, int &first) {
  const int a = __ldcg(r.start + b), z = __ldcg(r.start + b + 1);
  first = a;
  if (a >= 0 && z >= a && z <= r.rows) return z - a;
  atomicOr(c.err, KV_ERR_ROWS);
  return 0;
}
// The sequence that row r belongs to, or -1: 32 candidates a step, the whole warp.  (Where row_start falls the search ends somewhere; what it
// ends at is checked.)
__device__ __forceinline__ int kv_find(const KvRows &rw, int seqs, int r, int lane) {
  int lo = 0, n = seqs;
  while (n > 1) {
    const int step = (n + 31) >> 5, i = lane * step;
    const unsigned on = __ballot_sync(0xffffffffu, i < n && __ldcg(rw.start + lo + i) <= r);
    if (!on) return -1;
    const int at = (__popc(on) - 1) * step;
    lo += at;
    n = min(step, n - at);
  }
  const int a = __ldcg(rw.start + lo), z = __ldcg(rw.start + lo + 1);
  return a <= r && r < z && a >= 0 && z <= rw.rows ? lo : -1;
}
// by the threads of one block of a kernel that goes by rows: what no row shows
__device__ __forceinline__ void kv_check_rows(const KvDev &c, const KvRows &r) {
  for (int b = threadIdx.x; b < c.seqs; b += blockDim.x) {
    int first;
    if (kv_rows(c, r, b, first) > r.max_rows) atomicOr(c.err, KV_ERR_ROWS);
  }
}
// what the row at slot e sees
__device__ __forceinline__ bool kv_sees(int j, int e, int window, int sinks) { return j <= e && (!window || j > e - window || j < sinks); }
__device__ __forceinline__ int kv_first(int e, int window) { return window && e >= window ? e - window + 1 : 0; }   // first slot of its window
