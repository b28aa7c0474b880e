// kvpf.cuh -- attention of many rows (prompts and pieces of them) over the paged cache, on tcgen05: bound by the matrix products.
//
// A block has 128 queries of one kv head (query i G + h is row i, head h of the kv head's G) at head dimension 256, two times 128 below (two
// streams), and the slots that they see, 64 at a time.  A stream has the scores of two tiles of slots in tensor memory, so that the tensor core works
// on the next tile's while the softmax of one runs.
//   S[query][slot] = Q K^T     Q in shared memory, or in tensor memory at head dimension 256, where reading it from shared memory beside 64 slots of K
//                              would take longer than the product
//   P = exp(S - m)             a thread a query; in 16 bits over S's columns
//   O[query][dim] += P V       V as it lies in the cache (MN-major)
// m is the maximum of a query's scores as of the last step in which it grew by more than 2^8: O and the sum are only then rescaled, and P stays below 2^8.
// The second product takes 16-bit operands, so that P is rounded to the cache's type; the sum takes it unrounded.  (P in two such numbers would be a second product and
// as much tensor memory again.  Errors against 64 bits: bf16 2.1e-3 where the output's own rounding makes 1.6e-3, f16 2.9e-4 and 2.1e-4.)  In f16 P is taken times 2^7,
// in the sum and O alike: below 2^15, and what is lost of a slot is 2^-32 of the maximum's weight; without it 2^-25, which 131072 slots make 2^-8.
// K and V come by TMA, a page's part of a tile each, in rows of 128 swizzled bytes.  A slot that no row of the block sees is zeroed in V before
// the product (whatever the page holds there, 0 times it has to be 0).
//
// Warps: softmax (4 a query tile), one that loads K, one that loads V, one a stream that issues its MMAs: an MMA is issued when the one before has
// begun, so that a warp's time between two products (its waits, its commits) is the tensor core's too, unless the other stream's warp has
// products in line.  Every wait is bounded.
//
// Measured, cycles of a step of 64 slots: at head dimension 256 about 1370, of which the products are 16 x 33 + 4 x 130; at 128 (two streams) about 1700, products 2 x (8 x 48 + 4 x 64):
// there the two streams' softmax warps share an SM quarter.  3011 rows of 24 heads of 256 on 4: 120 us, 0.93 PFLOP/s at 1.69 GHz under the power limit; 4 x up to 2000 rows, window 1024, 32
// heads of 128 on 8: 143 us.  A block takes some 6000 cycles to its first scores and 4000 from its last to its results.
#pragma once
#include "kvatt.cuh"

template <int HD> struct Kp {
  static constexpr int NQT = HD == 256 ? 1 : 2;            // query tiles: streams
  static constexpr int TILE = 64, SH = 6;                  // slots
  static constexpr int GB = TILE * HD * 2;                 // bytes of a tile of K or V
  static constexpr int QB = HD == 256 ? 0 : NQT * 128 * HD * 2;
  static constexpr int NK = HD == 256 ? 3 : HD == 128 ? 5 : 6, NV = HD == 256 ? 4 : NK;   // tiles of K and of V that have room
  static constexpr int SMEM = 1024 + QB + (NK + NV) * GB;
  static constexpr int SOFT = 4 * NQT, THREADS = 32 * (SOFT + 2 + NQT);
  static constexpr uint32_t O = 0, S = HD == 256 ? 384 : 256, Q = 256;   // tensor memory's columns; S: two tiles a stream
};
static_assert(Kp<256>::SMEM <= 232448 && Kp<128>::SMEM <= 232448 && Kp<64>::SMEM <= 232448, "shared memory");

template <typename T> constexpr float kp_up = __is_same(T, __half) ? 7.0f : 0.0f;   // P, and so a stream's sums, are taken times two to this

struct KvPfPlan {
  int splits;                  // blocks a unit's tiles of slots are spread over
  float *pm, *pl, *po;         // [seqs][KV][queries][splits](, [hd]), where there are several; queries: G max_rows
  unsigned int *err;
};
// a unit's tiles of slots: those of first tokens, then those from the first row's window on
struct KpTiles { int lo, cs, n; };
template <int SH> __device__ __forceinline__ KpTiles kp_tiles(int ea, int ez, int window, int sinks) {
  KpTiles t;
  t.lo = kv_first(max(ea, 0), window) >> SH;
  t.cs = min((min(sinks, kv_first(max(ea, 0), window)) + (1 << SH) - 1) >> SH, t.lo);
  t.n = ez < 0 ? 0 : t.cs + (ez >> SH) - t.lo + 1;
  return t;
}
__device__ __forceinline__ void kp_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// D f32, A and B of type T, M = 128; mn: B is MN-major
template <typename T> __host__ __device__ constexpr uint32_t kp_idesc(int N, bool mn) {
  return 0x08000010u | (sizeof(T) == 2 && !__is_same(T, __half) ? (1u << 7) | (1u << 10) : 0u) | (mn ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17);
}
// rows of 128 swizzled bytes, eight of them 1024 bytes on from the next eight; step: from 64 columns of an MN-major operand to the next 64
__device__ __forceinline__ uint64_t kp_desc(uint32_t addr_s, uint32_t step) { return g3_desc(addr_s, step, 1024) | (2ull << 61); }
__device__ __forceinline__ void kp_ld32(uint32_t taddr, float *v) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
        "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 32; i++) v[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ uint32_t kp_below(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }   // the n lowest bits

// 2^y of two numbers by the FMA pipe (y <= 127): the whole part makes a power of two, 2^f on [-1/2, 1/2] is the polynomial of degree four whose largest relative
// error is smallest (2.7e-6 in f32; coefficients by Remez's exchange).  NaN stays NaN through the clamp, the polynomial and the last product.  At -127, where the
// clamp takes what is below it, a masked slot's minus infinity too, the power of two is an exact 0: 2^-126 would be a number in bf16, and a slot that a row
// does not see would have a weight.  The special
// function unit takes a warp's 32 in eight cycles; where two streams' softmax warps share one, every fourth pair goes this way: 4 x up to
// 2000 rows, window 1024, 32 heads of 128 on 8, called again and again, take 133 us with it and 140 without
// (pages of 64: 131 and 140; of 16, where copies bound it, 145 and 140).
// Every second pair: 144 (135, 156).  One stream (head dimension 256) gains nothing: 108 for 108 us at pages of 64, 142 for 138 at 16.
__device__ __forceinline__ float kp_max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ void kp_exp2_fma(f32x2 y, float &r0, float &r1) {
  float a, b;
  x2_unpack(y, a, b);
  y = x2_pack(kp_max_nan(a, -127.0f), kp_max_nan(b, -127.0f));
  const f32x2 big = x2_pack(12582912.0f, 12582912.0f), one = x2_pack(-1.0f, -1.0f);
  const f32x2 t = x2_add(y, big), f = x2_add(y, x2_fma(t, one, big));      // (t's low bits: the whole part)
  f32x2 v = x2_fma(x2_pack(0.009570102207362652f, 0.009570102207362652f), f, x2_pack(0.05591785907745361f, 0.05591785907745361f));
  v = x2_fma(v, f, x2_pack(0.240247443318367f, 0.240247443318367f));
  v = x2_fma(v, f, x2_pack(0.6931217908859253f, 0.6931217908859253f));
  v = x2_fma(v, f, x2_pack(0.9999992847442627f, 0.9999992847442627f));
  x2_unpack(t, a, b);
  const f32x2 e = x2_pack(__int_as_float((__float_as_int(a) << 23) + 0x3f800000), __int_as_float((__float_as_int(b) << 23) + 0x3f800000));
  x2_unpack(x2_mul(v, e), r0, r1);
}

template <typename T, int HD>
__global__ void __launch_bounds__(Kp<HD>::THREADS, 1) k_kv_pf(const KvDev c, const KvRows rw, const KvAttn a, const KvPfPlan p, int tiles, const __grid_constant__ CUtensorMap km,
                                                              const __grid_constant__ CUtensorMap vm) {
  using C = Kp<HD>;
  constexpr int NQT = C::NQT, TILE = C::TILE, SH = C::SH, GB = C::GB, NK = C::NK, NV = C::NV, QT = 128 * NQT, BLK = TILE * 128;   // BLK: 64 dims of a tile
  extern __shared__ __align__(1024) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t bar_s = smem_u32(smem), q_s = bar_s + 1024, ring_s = q_s + C::QB, ringv_s = ring_s + NK * GB;
  auto full = [&](bool v, int s) { return bar_s + (v ? 96u : 0u) + 8u * (uint32_t)s; };
  auto empty = [&](bool v, int s) { return bar_s + (v ? 144u : 48u) + 8u * (uint32_t)s; };
  auto s_full = [&](int x, int i) { return bar_s + 192u + 8u * (uint32_t)(2 * x + (i & 1)); };
  auto p_full = [&](int x, int i) { return bar_s + 224u + 8u * (uint32_t)(2 * x + (i & 1)); };
  auto pv_done = [&](int x) { return bar_s + 256u + 8u * (uint32_t)x; };
  // a stream's last product has a barrier of its own: both phases of the last two products could pass before a warp that did not have to rescale looks for either
  auto pv_last = [&](int x) { return bar_s + 352u + 8u * (uint32_t)x; };
  const uint32_t q_full = bar_s + 272u;
  uint32_t *tmem_slot = (uint32_t *)(smem + 280);
  volatile uint32_t *dead = (volatile uint32_t *)(smem + 284);
  volatile uint32_t *badm = (volatile uint32_t *)(smem + 288);   // [tile & 15]: 16-slot groups whose page is no page
  // (what needs nothing of the call: barriers, each of its own thread; a tile's places are given back by both streams)
  if (tid < 12) { mbar_init(full(tid >= 6, tid % 6), 1); mbar_init(empty(tid >= 6, tid % 6), NQT); }
  if (tid < 4) { mbar_init(s_full(tid >> 1, tid), 1); mbar_init(p_full(tid >> 1, tid), 4); }
  if (tid < 4) mbar_init(tid < 2 ? pv_done(tid) : pv_last(tid - 2), 1);
  if (tid == 0) { mbar_init(q_full, C::SOFT); *dead = 0; }
  if (tid < 12) asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  pdl_wait();
  if (warp == C::SOFT + 2) {                     // tensor memory, while the others look their rows up
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  auto leave = [&]() {                           // nothing to do here
    t5_fence_before();
    __syncthreads();
    if (warp == C::SOFT + 2) {
      t5_fence_after();
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(*tmem_slot), "r"(512u) : "memory");
    }
  };
  // ---- which unit: the last query tiles first, they see the most ----
  const int split = blockIdx.y, u = blockIdx.x, g = u % c.KV, b = u / c.KV % c.seqs, tile = tiles - 1 - u / c.KV / c.seqs;
  const KvSeq s = kv_seq(c, rw, b, a.window, a.sinks, SH);
  const int NQ = a.G * s.nc, q0 = tile * QT;
  if (q0 >= NQ) { leave(); return; }
  const int ea = s.e0 + kv_row_of(a, q0), ez = s.e0 + kv_row_of(a, min(q0 + QT - 1, NQ - 1));   // slots of the first and the last row
  const KpTiles kt = kp_tiles<SH>(ea, ez, a.window, a.sinks);
  const int per = (kt.n + p.splits - 1) / p.splits, t0 = min(kt.n, split * per), n = min(kt.n, t0 + per) - t0;
  auto slot_of = [&](int i) { i += t0; return (i < kt.cs ? i : kt.lo + i - kt.cs) << SH; };
  auto seen = [&](int j) { return j <= ez && (!a.window || j > kv_before(ea, a.window) || j < a.sinks); };   // by some row of the block
  auto part_of = [&](int qi) { return (((size_t)b * c.KV + g) * ((size_t)a.G * rw.max_rows) + qi) * p.splits + split; };
  if (!n) {
    for (int qi = q0 + tid; qi < min(q0 + QT, NQ); qi += C::THREADS) {
      if (p.splits > 1) { p.pm[part_of(qi)] = -INFINITY; p.pl[part_of(qi)] = 0.0f; continue; }
      const long long at = (long long)(s.first + kv_row_of(a, qi)) * a.os + (long long)(g * a.G + qi - kv_row_of(a, qi) * a.G) * HD;
      for (int d = 0; d < HD * (a.out32 ? 4 : 2); d += 16) *(uint4 *)((uint8_t *)a.out + at * (a.out32 ? 4 : 2) + d) = make_uint4(0, 0, 0, 0);
    }
    leave();
    return;
  }
  const int streams = NQT == 2 && q0 + 128 < NQ ? 2 : 1;
  // a softmax warp's 32 queries are asked for before the block meets: four rows of 128 bytes a load
  uint4 qw[HD / 64][8];
  if (warp < 4 * streams) {
#pragma unroll
    for (int k = 0; k < 8; k++) {
      const int qk = q0 + 32 * warp + 4 * k + (lane >> 3);
      const uint16_t *src = a.q + (long long)(s.first + kv_row_of(a, qk)) * a.qs + (long long)(g * a.G + qk - kv_row_of(a, qk) * a.G) * HD + 8 * (lane & 7);
#pragma unroll
      for (int d = 0; d < HD / 64; d++) {
        qw[d][k] = make_uint4(0, 0, 0, 0);                 // (a choice between the load and zeros would wait for the load)
        if (qk < NQ)
          asm volatile("ld.global.nc.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(qw[d][k].x), "=r"(qw[d][k].y), "=r"(qw[d][k].z), "=r"(qw[d][k].w) : "l"(src + 64 * d));
      }
    }
  }
  const int bs = min(c.page_sh, SH), boxes = TILE >> bs;   // slots of a page's part of a tile, and how many parts
  // a loading lane's entry of tile i's pages, asked for a tile before its use; on: some row sees some of it
  struct Entry { int id; bool on; };
  auto entry = [&](int i) {
    Entry x = {-1, false};
    if (lane < boxes && i < n) {
      const int j = slot_of(i) + (lane << bs);
      x.on = j <= ez && (!a.window || j + (1 << bs) - 1 > kv_before(ea, a.window) || j < a.sinks);   // (what is seen is one run of slots and the first ones)
      if (x.on) asm volatile("ld.global.cg.s32 %0, [%1];" : "=r"(x.id) : "l"(c.table + (size_t)b * c.tstride + (j >> c.page_sh)));
    }
    return x;
  };
  Entry first = {-1, false};
  if (warp == C::SOFT || warp == C::SOFT + 1) first = entry(0);
  t5_fence_before();
  __syncthreads();
  t5_fence_after();
  pdl_trigger();                                 // (tensor memory is taken: a later kernel's block cannot sit on it while it waits for this one)
  const uint32_t tmem = *tmem_slot;
  auto wait = [&](uint32_t bar, uint32_t parity) {   // gives up for the whole block
    for (uint32_t k = 0; !mbar_wait(bar, parity, 4); k += 4) {
      if (*dead) return;
      if (k >= T5_WAIT_LIMIT) { *dead = 1; atomicExch(p.err, 1u); return; }
    }
  };

  if (warp < 4 * streams) {
    // ---- softmax: a thread a query ----
    const int x0 = warp >> 2, qi = q0 + 128 * x0 + (tid & 127), e = s.e0 + kv_row_of(a, min(qi, NQ - 1)), lw = a.window ? kv_before(e, a.window) + 1 : 0;
    const uint32_t lq = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
    // the queries: into shared memory as the product reads them, or through the last place of V's ring into tensor memory, 128 dims at a time
    {
      constexpr int PART = HD == 256 ? 2 : HD / 64;        // 64 dims at a time
      const uint32_t to = HD == 256 ? ringv_s + (NV - 1) * GB + (uint32_t)warp * 8192u : q_s + x0 * (128 * HD * 2) + (uint32_t)(warp & 3) * 4096u;
#pragma unroll
      for (int d0 = 0; d0 < HD / 64; d0 += PART) {
#pragma unroll
        for (int d = 0; d < PART; d++)
#pragma unroll
          for (int k = 0; k < 8; k++) {
            const int r = 4 * k + (lane >> 3);
            const uint4 w = qw[d0 + d][k];
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to + d * (HD == 256 ? 4096 : 128 * 128) + r * 128 + (((lane & 7) ^ (r & 7)) << 4)), "r"(w.x), "r"(w.y), "r"(w.z),
                         "r"(w.w)
                         : "memory");
          }
        if constexpr (HD == 256) {
          __syncwarp();
#pragma unroll
          for (int d = 0; d < 2; d++) {
            uint32_t v[32];
#pragma unroll
            for (int i = 0; i < 8; i++)
              asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[4 * i]), "=r"(v[4 * i + 1]), "=r"(v[4 * i + 2]), "=r"(v[4 * i + 3])
                           : "r"(to + d * 4096 + lane * 128 + ((i ^ (lane & 7)) << 4)) : "memory");
            t5_st32(lq + C::Q + 32 * (d0 + d), v);
          }
          __syncwarp();
        }
      }
      if constexpr (HD == 256) { t5_wait_st(); t5_fence_before(); }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
    }
    float m = -INFINITY, l = 0.0f;
    // slots of this query tile's first and last row: a tile between what they see is seen whole by every row
    const int qa = q0 + 128 * x0, ra = s.e0 + kv_row_of(a, qa), rz = s.e0 + kv_row_of(a, min(qa + 127, NQ - 1));
#pragma unroll 1
    for (int i = 0; i < n; i++) {
      const int slot = slot_of(i);
      const uint32_t S = lq + C::S + (uint32_t)(TILE * (2 * x0 + (i & 1)));
      float v[TILE];
      wait(s_full(x0, i), (uint32_t)(i >> 1) & 1u);
      __syncwarp();
      t5_fence_after();
#pragma unroll
      for (int k = 0; k < TILE; k += 32) kp_ld32(S + k, v + k);
      t5_wait_ld();
      const uint32_t bm = badm[i & 15];
      if (bm || slot + TILE - 1 > ra || (a.window && slot <= kv_before(rz, a.window) && slot + TILE - 1 >= a.sinks)) {
#pragma unroll
        for (int k0 = 0; k0 < TILE; k0 += 32) {            // a bit a slot: seen
          const int j = slot + k0;
          uint32_t on = kp_below(e + 1 - j) & (~kp_below(lw - j) | kp_below(a.sinks - j));
          if (bm >> (k0 >> 4) & 1) on &= 0xffff0000u;
          if (bm >> (k0 >> 4) & 2) on &= 0x0000ffffu;
          if (!__any_sync(0xffffffffu, on != 0xffffffffu)) continue;
#pragma unroll
          for (int k = 0; k < 32; k++) v[k0 + k] = on & (1u << k) ? v[k0 + k] : -INFINITY;
        }
      }
      float mx[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
      for (int k = 4; k < TILE; k += 8) {
#pragma unroll
        for (int w = 0; w < 4; w++) mx[w] = k + 4 + w < TILE ? fmaxf(mx[w], fmaxf(v[k + w], v[k + 4 + w])) : fmaxf(mx[w], v[k + w]);
      }
      const float t = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale2;
      const bool grow = t > m + 8.0f;                      // (from minus infinity at once)
      if (__any_sync(0xffffffffu, grow)) {
        const float mn = grow ? t : m, cf = mn == -INFINITY ? 1.0f : kv_exp2(m - mn);
        m = mn;
        l *= cf;
        if (i) {
          wait(pv_done(x0), (uint32_t)(i - 1) & 1u);       // the last product into O is done
          __syncwarp();
          t5_fence_after();
#pragma unroll 1
          for (int d = 0; d < HD; d += 32) {
            float o[32];
            const uint32_t at = lq + C::O + (uint32_t)(x0 * HD + d);
            kp_ld32(at, o);
            t5_wait_ld();
            uint32_t w[32];
#pragma unroll
            for (int k = 0; k < 32; k++) w[k] = __float_as_uint(o[k] * cf);
            t5_st32(at, w);
          }
          t5_wait_st();
        }
      }
      const float ref = (m == -INFINITY ? 0.0f : -m) + kp_up<T>;
      const f32x2 sc2 = x2_pack(a.scale2, a.scale2), rf2 = x2_pack(ref, ref);
      f32x2 sum[2] = {0, 0};
#pragma unroll
      for (int k0 = 0; k0 < TILE; k0 += 64) {
        uint32_t w[32];
#pragma unroll
        for (int k = 0; k < 32; k++) {
          float y0, y1;
          const f32x2 y = x2_fma(x2_pack(v[k0 + 2 * k], v[k0 + 2 * k + 1]), sc2, rf2);
          if (NQT == 2 && k % 4 == 3) kp_exp2_fma(y, y0, y1);
          else { x2_unpack(y, y0, y1); y0 = kv_exp2(y0); y1 = kv_exp2(y1); }
          sum[k & 1] = x2_add(sum[k & 1], x2_pack(y0, y1));
          w[k] = KvEl<T>::of2(y0, y1);
        }
        t5_st32(S + k0 / 2, w);
      }
      float a0, a1;
      x2_unpack(x2_add(sum[0], sum[1]), a0, a1);
      l += a0 + a1;
      // slots that no row of the block sees: their V is taken out, whatever the page holds, before the first product with the tile
      // (every stream's warps do it: what is zero is written as zero again)
      if (bm || slot + TILE - 1 > ez || (a.window && slot <= kv_before(ea, a.window) && slot + TILE - 1 >= a.sinks)) {
        const int rs = i % NV;
        wait(full(true, rs), (uint32_t)(i / NV) & 1u);
        const uint32_t at = ringv_s + rs * GB;
        auto clear = [&](int ra, int rz) {                 // rows ra .. rz - 1, those of them that the tile has
          ra = min(max(ra, 0), TILE); rz = min(max(rz, 0), TILE);
#pragma unroll 1
          for (int w = ra * (HD / 8) + (tid & 127); w < rz * (HD / 8); w += 128) {
            const int r = w / (HD / 8), d = w % (HD / 8);  // a row's 16 bytes, in the order in which they lie
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at + (d >> 3) * BLK + r * 128 + ((d & 7) << 4)), "r"(0) : "memory");
          }
        };
        clear(ez + 1 - slot, TILE);
        if (a.window) clear(a.sinks - slot, kv_before(ea, a.window) + 1 - slot);
#pragma unroll 1
        for (int r = 0; bm && r < TILE; r += 16)
          if (bm >> (r >> 4) & 1) clear(r, r + 16);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
      t5_wait_st();
      t5_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full(x0, i));
    }
    // ---- the rows' results ----
    if (n > 1) wait(pv_done(x0), (uint32_t)(n - 2) & 1u);  // (that barrier's last phase.  Without this wait 3011 rows of 24 heads of 256 took 108.2 us for 106.9)
    wait(pv_last(x0), 0);
    __syncwarp();
    t5_fence_after();
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const f32x2 inv2 = x2_pack(inv, inv), zero2 = x2_pack(0.0f, 0.0f);
    f32x2 chk[2] = {x2_pack(l, 0.0f), zero2};
    if (p.splits > 1 && qi < NQ) { const size_t part = part_of(qi); p.pm[part] = m; p.pl[part] = l; }
    // whole 128-byte pieces of rows, turned in memory that no product reads any more: the stream's queries', or the rings where it is the only stream
    const bool wide = p.splits > 1 || a.out32;             // 32 dims a piece, or 64
    const uint32_t st = (HD == 256 ? ring_s : q_s + x0 * (128 * HD * 2)) + (uint32_t)(warp & 3) * 4096u;
    uint8_t *dst[8];                                       // rows 4 k + lane / 8 of the warp's
#pragma unroll
    for (int k = 0; k < 8; k++) {
      const int qk = q0 + 128 * x0 + 32 * (warp & 3) + 4 * k + (lane >> 3);
      dst[k] = nullptr;
      if (qk >= NQ) continue;
      if (p.splits > 1) dst[k] = (uint8_t *)(p.po + part_of(qk) * HD);
      else dst[k] = (uint8_t *)a.out + ((long long)(s.first + kv_row_of(a, qk)) * a.os + (long long)(g * a.G + qk - kv_row_of(a, qk) * a.G) * HD) * (a.out32 ? 4 : 2);
      dst[k] += 16 * (lane & 7);
    }
    auto piece = [&](int at) {
      uint32_t w[8][4];
      __syncwarp();
#pragma unroll
      for (int k = 0; k < 8; k++)
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[k][0]), "=r"(w[k][1]), "=r"(w[k][2]), "=r"(w[k][3])
                     : "r"(st + (4 * k + (lane >> 3)) * 128 + (((lane & 7) ^ ((4 * k + (lane >> 3)) & 7)) << 4)) : "memory");
#pragma unroll
      for (int k = 0; k < 8; k++)
        if (dst[k]) *(uint4 *)(dst[k] + at) = make_uint4(w[k][0], w[k][1], w[k][2], w[k][3]);
      __syncwarp();
    };
    auto put = [&](int k, uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3) {
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(st + lane * 128 + ((k ^ (lane & 7)) << 4)), "r"(w0), "r"(w1), "r"(w2), "r"(w3) : "memory");
    };
#pragma unroll 1
    for (int d = 0; d < HD; d += 64) {
      float o[64];
      kp_ld32(lq + C::O + (uint32_t)(x0 * HD + d), o);
      kp_ld32(lq + C::O + (uint32_t)(x0 * HD + d + 32), o + 32);
      t5_wait_ld();
      if (p.splits == 1) {
#pragma unroll
        for (int k = 0; k < 64; k += 2) {
          const f32x2 w = x2_pack(o[k], o[k + 1]);
          chk[(k >> 1) & 1] = x2_fma(w, zero2, chk[(k >> 1) & 1]);
          x2_unpack(x2_mul(w, inv2), o[k], o[k + 1]);
        }
      }
      if (wide) {
#pragma unroll
        for (int half = 0; half < 2; half++) {
#pragma unroll
          for (int k = 0; k < 8; k++) {
            const float *w = o + 32 * half + 4 * k;
            put(k, __float_as_uint(w[0]), __float_as_uint(w[1]), __float_as_uint(w[2]), __float_as_uint(w[3]));
          }
          piece(4 * (d + 32 * half));
        }
      } else {
#pragma unroll
        for (int k = 0; k < 8; k++) {
          const float *w = o + 8 * k;
          put(k, KvEl<T>::of2(w[0], w[1]), KvEl<T>::of2(w[2], w[3]), KvEl<T>::of2(w[4], w[5]), KvEl<T>::of2(w[6], w[7]));
        }
        piece(2 * d);
      }
    }
    // rows whose result is no number once more (kv_attn_row says why)
    float c0, c1;
    x2_unpack(x2_add(chk[0], chk[1]), c0, c1);
    bool again = p.splits == 1 && qi < NQ && l == l && !(fabsf(c0 + c1) < INFINITY);
    if (__is_same(T, __half) && __any_sync(0xffffffffu, again)) {   // (NaN, or only infinities?)
      bool nan = false;
#pragma unroll 1
      for (int d = 0; d < HD; d += 32) {
        float o[32];
        kp_ld32(lq + C::O + (uint32_t)(x0 * HD + d), o);
        t5_wait_ld();
#pragma unroll
        for (int k = 0; k < 32; k++) nan |= kv_again<T>(o[k]);
      }
      again = again && nan;
    }
    const unsigned redo = __ballot_sync(0xffffffffu, again);
#pragma unroll 1
    for (int half = 0; redo && half < 32; half += 16)
      if (redo >> half & 0xffff) kv_attn_rows16<T, HD>(c, a, b, g, s.first, s.e0, q0 + 128 * x0 + 32 * (warp & 3) + half, NQ, {0, kt.n, kt.cs, kt.lo, SH}, lane, redo >> half & 0xffff);
  } else if (warp < C::SOFT) {
    if (lane == 0) mbar_arrive(q_full);          // the second query tile is behind the last query
  } else if (warp < C::SOFT + 2) {
    // ---- K, or V: the pages' parts of a tile ----
    const bool isv = warp == C::SOFT + 1;
    const CUtensorMap *map = isv ? &vm : &km;
    const int N = isv ? NV : NK;
    const uint32_t ring = isv ? ringv_s : ring_s;
    Entry next = first;
    int slot = 0;
    uint32_t round = 0;
#pragma unroll 1
    for (int i = 0; i < n; i++) {
      asm volatile("" : "+r"(next.id));                    // (the load is not waited for before)
      const int id = !next.on ? -2 : (unsigned)next.id < (unsigned)c.n_pages ? next.id : -1;   // -2: not wanted, -1: no page
      next = entry(i + 1);
      if (round) wait(empty(isv, slot), (round - 1) & 1u);
      else if (HD == 256 && isv && slot == NV - 1) wait(q_full, 0);   // (the queries come through it)
      __syncwarp();
      const bool in = id >= 0;
      const unsigned have = __ballot_sync(0xffffffffu, in), lost = __ballot_sync(0xffffffffu, id == -1);
      const uint32_t bar = full(isv, slot), at = ring + slot * GB;
      const int j = slot_of(i) & ((1 << c.page_sh) - 1);   // (where a tile has several pages, the first slot of each)
      if (lane == 0) {
        if (lost) atomicOr(c.err, KV_ERR_PAGE);
        if (!isv) {
          uint32_t bm = 0;
          for (int k = 0; lost && k < boxes; k++) if (lost >> k & 1) bm |= ((1u << (1 << (bs - 4))) - 1) << (k << (bs - 4));
          badm[i & 15] = bm;
        }
        if (!*dead && have) kv_expect(bar, (uint32_t)__popc(have) * (HD / 64) * (128u << bs));
        else mbar_arrive(bar);
        if (!*dead && boxes == 1 && have) kv_tma(at, map, 0, j, 0, g, id, bar);              // one box of all dims
      }
      if (boxes > 1) {
        __syncwarp();
        if (in && !*dead) {
#pragma unroll
          for (int d = 0; d < HD / 64; d++) kv_tma(at + d * BLK + (lane << bs) * 128, map, 0, j, d, g, id, bar);
        }
      }
      __syncwarp();
      if (++slot == N) { slot = 0; round++; }
    }
  } else if (warp < C::SOFT + 2 + streams) {
    // ---- the tensor core, a thread a stream ----
    if (t5_elect()) {
      const int x = warp - C::SOFT - 2;
      constexpr uint32_t ids = kp_idesc<T>(TILE, false), ido = kp_idesc<T>(HD, true);
      const uint64_t k0 = kp_desc(ring_s, 16), v0 = kp_desc(ringv_s, BLK), qd = kp_desc(q_s + x * (128 * HD * 2), 16);
      const uint32_t S0 = tmem + C::S + (uint32_t)(2 * TILE * x), O = tmem + C::O + (uint32_t)(x * HD);
      int ks = 0, vs = 0;
      uint32_t kp = 0, vp = 0;                             // ring places and their phases
      auto score = [&](int i, uint32_t look, uint32_t phase) {   // (its K is there); looks at a barrier on the way
        const uint32_t D = S0 + (uint32_t)(TILE * (i & 1));
        const uint64_t kd = k0 + (uint64_t)(ks * (GB / 16));
        bool seen = false;
#pragma unroll
        for (int d = 0; d < HD / 16; d++) {
          const uint64_t kk = kd + (uint64_t)((d >> 2) * (BLK / 16) + 2 * (d & 3));
          // (an issue waits until the MMA two in front of it is done: the look fits between the last ones)
          if (d == HD / 16 - 2 && look) seen = mbar_wait(look, phase, 1);
          if constexpr (HD == 256) t5_mma_f16_ts(D, tmem + C::Q + 8 * d, kk, ids, d != 0);
          else kp_ss(D, qd + (uint64_t)((d >> 2) * (128 * 128 / 16) + 2 * (d & 3)), kk, ids, d != 0);
        }
        t5_commit(s_full(x, i));
        t5_commit(empty(false, ks));
        if (streams < NQT) t5_commit(empty(false, ks));    // (for the stream that is not)
        if (++ks == NK) { ks = 0; kp ^= 1u; }
        return seen;
      };
      wait(q_full, 0);
      wait(full(false, 0), 0);
      t5_fence_after();
      score(0, 0, 0);
      if (n > 1) { wait(full(false, ks), kp); t5_fence_after(); score(1, 0, 0); }
      wait(full(true, 0), 0);
      bool seen = false;
#pragma unroll 1
      for (int i = 0; i < n; i++) {
        if (!seen) wait(p_full(x, i), (uint32_t)(i >> 1) & 1u);   // (V's rows that nobody sees are zero by then, too)
        t5_fence_after();
        const uint64_t vd = v0 + (uint64_t)(vs * (GB / 16));
        const uint32_t P = S0 + (uint32_t)(TILE * (i & 1));
#pragma unroll
        for (int d = 0; d < TILE / 16; d++) t5_mma_f16_ts(O, P + 8 * d, vd + 128 * d, ido, i != 0 || d != 0);
        t5_commit(i + 1 < n ? pv_done(x) : pv_last(x));
        t5_commit(empty(true, vs));
        if (streams < NQT) t5_commit(empty(true, vs));
        if (++vs == NV) { vs = 0; vp ^= 1u; }
        // what comes next is waited for while this product runs; the next scores go into the columns of the probabilities that it uses
        seen = false;
        if (i + 2 < n) {
          const bool vk = mbar_wait(full(true, vs), vp, 1), kk = mbar_wait(full(false, ks), kp, 1);
          if (!vk) wait(full(true, vs), vp);
          if (!kk) wait(full(false, ks), kp);
          t5_fence_after();
          seen = score(i + 2, p_full(x, i + 1), (uint32_t)((i + 1) >> 1) & 1u);
        } else if (i + 1 < n) wait(full(true, vs), vp);
      }
    }
  }
  // after a wait ran out nothing is requested any more, but copies may be on their way
  if (*dead) for (int i = 0; i < 64; i++) __nanosleep(1000);
  __syncwarp();
  t5_fence_before();
  __syncthreads();
  if (warp == C::SOFT + 2) {
    t5_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

// the splits of a row and head put together, in their order: a warp each
template <typename T, int HD>
__global__ void __launch_bounds__(128) k_kv_pf_join(const KvDev c, const KvRows rw, const KvAttn a, const KvPfPlan p) {
  constexpr int E = HD / 32;
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, h = blockIdx.y * 4 + (threadIdx.x >> 5), r = blockIdx.x;
  const int b = kv_find(rw, c.seqs, r, lane);
  if (b < 0 || h >= a.H) return;
  int first;
  const int n = kv_rows(c, rw, b, first), i = r - first;
  if (i >= rw.max_rows) return;
  const int g = h / a.G;
  const size_t at = (((size_t)b * c.KV + g) * ((size_t)a.G * rw.max_rows) + (size_t)i * a.G + h % a.G) * p.splits;
  float M = -INFINITY;
  for (int w = lane; w < p.splits; w += 32) M = fmaxf(M, __ldcg(p.pm + at + w));
#pragma unroll
  for (int k = 16; k; k >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, k));
  float o[E], l = 0.0f;
#pragma unroll
  for (int k = 0; k < E; k++) o[k] = 0.0f;
#pragma unroll 4
  for (int w = 0; w < p.splits; w++) {
    const float pm = __ldcg(p.pm + at + w);
    if (pm == -INFINITY) continue;                         // (nothing seen there: no sums)
    const float f = exp2f(pm - M);
    l += __ldcg(p.pl + at + w) * f;
#pragma unroll
    for (int k = 0; k < E; k += 2) { const float2 v = __ldcg((const float2 *)(p.po + (at + w) * HD + lane * E + k)); o[k] += v.x * f; o[k + 1] += v.y * f; }
  }
  if (kv_again_any<T, E>(o, l)) {                          // the splits whose sums are no numbers once more, by themselves
    constexpr int QT = 128 * Kp<HD>::NQT, SH = Kp<HD>::SH;
    const int e0 = kv_len(c, b) - n, NQ = a.G * min(n, rw.max_rows), q0 = (i * a.G + h % a.G) / QT * QT;
    const KpTiles kt = kp_tiles<SH>(e0 + kv_row_of(a, q0), e0 + kv_row_of(a, min(q0 + QT - 1, NQ - 1)), a.window, a.sinks);
    const int per = (kt.n + p.splits - 1) / p.splits;
    M = -INFINITY; l = 0.0f;
#pragma unroll
    for (int k = 0; k < E; k++) o[k] = 0.0f;
#pragma unroll 1
    for (int w = 0; w < p.splits; w++) {
      float pm = __ldcg(p.pm + at + w), pl = __ldcg(p.pl + at + w), v[E];
      if (pm == -INFINITY) continue;
#pragma unroll
      for (int k = 0; k < E; k += 2) { const float2 t = __ldcg((const float2 *)(p.po + (at + w) * HD + lane * E + k)); v[k] = t.x; v[k + 1] = t.y; }
      if (kv_again_any<T, E>(v, pl)) {
        const int t0 = min(kt.n, w * per);
        kv_attn_row<T, HD>(c, a, b, r, h, e0 + i, {t0, min(kt.n, t0 + per), kt.cs, kt.lo, SH}, lane, v, pm, pl);
        pm += kp_up<T>;                                    // (as the others' sums are)
      }
      kv_add_part<E>(o, M, l, v, pm, pl);
    }
  }
  kv_store<T, HD>(a, r, h, lane, o, l);
}
