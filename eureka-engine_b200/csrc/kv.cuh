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
  static __device__ __forceinline__ uint16_t of(float v) { return __half_as_ushort(__float2half_rn(v)); }
  static __device__ __forceinline__ float2 to2(uint32_t v) { return __half22float2(*(const __half2 *)&v); }
  static __device__ __forceinline__ uint32_t of2(float a, float b) { const __half2 h = __floats2half2_rn(a, b); return *(const uint32_t *)&h; }
};
template <> struct KvEl<__nv_bfloat16> {
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
__device__ __forceinline__ int kv_first(int e, int window) { return window && e >= window ? e - window + 1 : 0; }   // first slot of its window

// last slot before its window, or some slot below 0.  Rows at slots below 0 see nothing: what several rows see begins with the first at slot 0 or above (and the
// difference stays an int for every window)
__device__ __forceinline__ int kv_before(int e, int window) { return max(e, 0) - window; }

// ---- a call's attention ----------------------------------------------------------------------------
struct KvAttn {
  const uint16_t *q;
  void *out;
  long long qs, os;            // elements between rows
  int H, G, window, sinks, out32;   // G: query heads a kv head
  unsigned inv;                // 2^32 / G, rounded up
  float scale2;                // times log2(e): probabilities are powers of two
  const float *w_in;
  float *w_out;
  int wstride;
};
// row of a query i G + h: exact for fewer than 2^26 queries (kv_attn_check), G at most 64
__device__ __forceinline__ int kv_row_of(const KvAttn &a, int q) { return a.G == 1 ? q : (int)__umulhi((unsigned)q, a.inv); }
// one sequence's share of a call.  What its rows see is cut into chunks of `1 << sh` slots: cs of first tokens, then those from slot lo's on.
struct KvSeq {
  int first, n, len;           // first row, rows; slots
  int nc;                      // rows that are computed: max_rows at most
  int e0;                      // slot of the first row
  int lo, cs, chunks;
};
__device__ __forceinline__ KvSeq kv_seq(const KvDev &c, const KvRows &r, int b, int window, int sinks, int sh) {
  KvSeq s;
  const int a = __ldcg(r.start + b), z = __ldcg(r.start + b + 1), n = __ldcg(c.lens + b);   // (all on their way before any is looked at)
  s.first = a;
  s.n = a >= 0 && z >= a && z <= r.rows ? z - a : 0;
  s.len = min(max(n, 0), c.cap);
  if (s.n != z - a || a < 0) atomicOr(c.err, KV_ERR_ROWS);
  if (s.len != n) atomicOr(c.err, KV_ERR_LEN);
  s.nc = min(s.n, r.max_rows);
  if (s.n > r.max_rows) atomicOr(c.err, KV_ERR_ROWS);
  s.e0 = s.len - s.n;
  const int last = s.e0 + s.nc - 1;
  s.lo = kv_first(max(s.e0, 0), window);
  s.cs = min((min(sinks, s.lo) + (1 << sh) - 1) >> sh, s.lo >> sh);
  s.chunks = !s.nc ? 0 : last < 0 ? 1 : s.cs + (last >> sh) - (s.lo >> sh) + 1;   // (rows that see nothing: one chunk with nothing in it)
  return s;
}
__device__ __forceinline__ int kv_chunk_slot(const KvSeq &s, int ch, int sh) { return (ch < s.cs ? ch : (s.lo >> sh) + ch - s.cs) << sh; }
// whether some row of the sequence sees slot j
__device__ __forceinline__ bool kv_any_sees(const KvSeq &s, int j, int window, int sinks) {
  return j <= s.e0 + s.nc - 1 && (!window || j > kv_before(s.e0, window) || j < sinks);
}

template <int W> __device__ __forceinline__ void kv_words(const void *p, uint32_t (&w)[W]) {
  if constexpr (W == 1) w[0] = __ldcg((const uint32_t *)p);
  else if constexpr (W == 2) { const uint2 t = __ldcg((const uint2 *)p); w[0] = t.x; w[1] = t.y; }
  else { const uint4 t = __ldcg((const uint4 *)p); w[0] = t.x; w[1] = t.y; w[2] = t.z; w[3] = t.w; }
}
template <typename T, int E> __device__ __forceinline__ void kv_row_in(const T *p, float (&x)[E]) {
  uint32_t w[E / 2];
  kv_words<E / 2>(p, w);
#pragma unroll
  for (int i = 0; i < E / 2; i++) { const float2 f = KvEl<T>::to2(w[i]); x[2 * i] = f.x; x[2 * i + 1] = f.y; }
}
template <typename T, int E> __device__ __forceinline__ void kv_row_out(uint16_t *p, bool wide, const float (&x)[E]) {
  if (wide) {
    uint32_t w[E / 2];
#pragma unroll
    for (int i = 0; i < E / 2; i++) w[i] = KvEl<T>::of2(x[2 * i], x[2 * i + 1]);
    if constexpr (E == 2) *(uint32_t *)p = w[0];
    else if constexpr (E == 4) *(uint2 *)p = make_uint2(w[0], w[1]);
    else *(uint4 *)p = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < E; i++) p[i] = KvEl<T>::of(x[i]);
  }
}
__device__ __forceinline__ float kv_warp_sum(float v) {
#pragma unroll
  for (int m = 16; m; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  return v;
}
// Whether a sum of products may be none of the row's: NaN, and in bf16 infinity too (V near 2^127 times probabilities relative to an old maximum; f16 has no
// values whose sums overflow, an infinity comes from a slot that the row sees)
template <typename T> __device__ __forceinline__ bool kv_again(float x) { return __is_same(T, __half) ? x != x : !(fabsf(x) < INFINITY); }
// Chunks c0 .. c1 - 1, of 1 << sh slots, of what several rows see: the first cs of them of first tokens, then those from number lo on (KvSeq, KpTiles).
struct KvSpan { int c0, c1, cs, lo, sh; };
// What the row at slot e and head h sees of a span, slot after slot, by a warp; lane's dimensions E lane ..  o, m, l: the sums, relative to 2^m.
// The attention kernels take a row to it, or the part of it that one block had, whose sum of probabilities is a number and whose result is none: their products multiply
// V by a probability of zero where a row does not see a slot that another one does, which is NaN where that slot holds an infinity or NaN.  (Where the sum is no number, a
// score that the row sees is NaN or plus infinity, and so is every dimension of the result: nothing to do again.)
// A token behind 100000 slots, 4 heads of 128: a NaN key, or an infinite V in f16, 37 us as without it (58 and 60 ms when such rows were done again, wholly).
// Inlined: as a function of its own, though no row comes to it, it cost the kernels the registers and the order of their code that a call asks for (48 sequences of up to 6000
// slots with weights 159 us for 134, 3011 rows of 24 heads of 256 106 for 102, 4 x up to 2000 rows of 32 heads of 128 148 for 133).
template <typename T, int HD>
__device__ __forceinline__ void kv_attn_row(const KvDev &c, const KvAttn &a, int b, int r, int h, int e, const KvSpan &sp, int lane, float (&o)[HD / 32], float &m, float &l) {
  constexpr int E = HD / 32;
  const int g = h / a.G, pm = (1 << c.page_sh) - 1, lw = a.window ? kv_before(e, a.window) + 1 : 0;
  float q[E];
  kv_row_in<T, E>((const T *)a.q + r * a.qs + (long long)h * HD + lane * E, q);
#pragma unroll
  for (int i = 0; i < E; i++) { q[i] *= a.scale2; o[i] = 0.0f; }
  m = -INFINITY; l = 0.0f;
  int id = -1, at = -1;
#pragma unroll 1
  for (int ch = sp.c0; ch < sp.c1; ch++) {
    const int j0 = (ch < sp.cs ? ch : sp.lo + ch - sp.cs) << sp.sh;
#pragma unroll 1
    for (int j = j0; j < j0 + (1 << sp.sh); j++) {
      if (j > e || (j < lw && j >= a.sinks)) continue;
      if (j >> c.page_sh != at) { at = j >> c.page_sh; id = kv_page(c, b, at); }
      if (id < 0) continue;
      const size_t p = kv_at(c, id, g, HD) + (size_t)(j & pm) * HD + lane * E;
      float k[E], v[E];
      kv_row_in<T, E>((const T *)c.k + p, k);
      kv_row_in<T, E>((const T *)c.v + p, v);
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < E; i++) s += q[i] * k[i];
      s = kv_warp_sum(s);
      const float mn = fmaxf(m, s), cf = m == -INFINITY ? 0.0f : exp2f(m - mn), w = s == -INFINITY ? 0.0f : exp2f(s - mn);
      l = l * cf + w;
      // (0 times an infinity is no number either: a slot that is seen and whose probability is 0 counts as in the definition, exp(s) V)
#pragma unroll
      for (int i = 0; i < E; i++) o[i] = o[i] * cf + w * v[i];
      m = mn;
    }
  }
}
// a row's result, normalised, by a warp
template <typename T, int HD> __device__ __forceinline__ void kv_store(const KvAttn &a, int r, int h, int lane, float (&o)[HD / 32], float l) {
  constexpr int E = HD / 32;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;   // (nothing seen: zeros)
#pragma unroll
  for (int i = 0; i < E; i++) o[i] *= inv;
  const long long at = r * a.os + (long long)h * HD + lane * E;
  if (a.out32) {
    float *p = (float *)a.out + at;
#pragma unroll
    for (int i = 0; i < E; i += 2) *(float2 *)(p + i) = make_float2(o[i], o[i + 1]);
  } else kv_row_out<T, E>((uint16_t *)a.out + at, true, o);
}
// one more part's sums (relative to 2^pm) to a row's
template <int E> __device__ __forceinline__ void kv_add_part(float (&o)[E], float &m, float &l, const float (&v)[E], float pm, float pl) {
  const float t = fmaxf(m, pm), ref = t == -INFINITY ? 0.0f : t, f = exp2f(m - ref), fp = exp2f(pm - ref);
  l = l * f + pl * fp;
  m = t;
#pragma unroll
  for (int i = 0; i < E; i++) o[i] = o[i] * f + v[i] * fp;
}
// whether a row's sums may be none of its own (l a number, o none): the whole warp
template <typename T, int E> __device__ __forceinline__ bool kv_again_any(const float (&o)[E], float l) {
  bool again = false;
#pragma unroll
  for (int i = 0; i < E; i++) again |= kv_again<T>(o[i]);
  return __any_sync(0xffffffffu, again) && l == l;
}
