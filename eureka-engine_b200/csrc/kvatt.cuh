// kvatt.cuh -- attention of the few rows of a decode or verify step over the paged cache: bound by the cache's bytes.
//
// A unit is (sequence, kv head, 16 queries); its queries are the rows' heads side by side, query i G + h is row i, head h of the kv head's
// G.  What a unit sees is cut into groups of 32 or 64 slots, and the groups of all units, one after the other, into as many equal stretches as
// there are blocks, so that sequences of any lengths keep every SM busy to the end; a block's stretch may begin and end inside a unit.
// Two threads of the block request the groups' K and V (TMA, a box a page, rows of 128 swizzled bytes) and every unit's queries, on over the ends of units;
// the other warps take 16 slots of a group each.
//   S[query][slot] = Q K^T      m16n8k16, 16 queries x 16 slots
//   O[query][dim] += P V        P from the registers of S, rounded to the cache's type (the second product takes 16-bit operands; P in two of them would be half as
//                               many MMAs again.  Errors against 64 bits: bf16 1.9e-3 where the output's own rounding makes 1.6e-3, f16 2.5e-4 and 2.1e-4)
// with the maximum and the sum of every query kept in f32.  Where a unit ends the warps' sums are put together, some dims at a time.  A unit that one
// block has wholly is finished there; the others' sums go to the workspace, and k_kv_join, the second launch, puts them together in the order of the blocks.
//
// 16 slots are a chain of 1500 to 2000 cycles for their warp (two products with the softmax between), which is why several warps work on slots of their own; a
// request takes its thread 100 to 200 cycles a box whatever the box's size, which is why groups are 32 KB and why K and V have a thread each.
// Measured: 32 sequences of up to 8192 slots, 16 heads of 256 on 4, pages of 64: 102 us with the join, 5.9 TB/s of cache; two of 131071 and 58165, 24 heads of 256 on
// 4: 130 us, 6.0 TB/s; 48 of up to 6000, 32 heads of 128 on 8, pages of 32: 136 us, of which 19 are the slots' weights.
#pragma once
#include <cuda.h>

#include "kv.cuh"
#include "tc5.cuh"

__host__ __device__ constexpr int kf_sh(int HD) { return HD == 256 ? 5 : 6; }                         // log2 of a group's slots
__host__ __device__ constexpr int kf_parts(int HD) { return 1 << (kf_sh(HD) - 4); }                   // of 16 slots in it
__host__ __device__ constexpr int kf_warps(int HD) { return HD == 256 ? 6 : 8; }                      // that compute
__host__ __device__ constexpr int kf_ring(int HD) { return HD == 64 ? 8 : 6; }                        // groups that have room
__host__ __device__ constexpr int kf_bytes(int HD) { return 2 * HD * 2 << kf_sh(HD); }                // of a group: K, then V
__host__ __device__ constexpr int kf_qrow(int HD) { return HD * 2 + 16; }                             // bytes from a query to the next: four banks on
struct KfUnit { KvSeq s; int b, g, qt, c0, c1, last; };   // c0 .. c1 - 1: the block's groups of it; c1 < 0: no more; last: the ring is empty behind it
#define KF_ROW 40              // floats from a row of the warps' sums to the next: 32 dims, and eight banks on
struct KfHead {                // before the ring
  uint64_t full[8], empty[8], qfull[2], qempty[2];
  int sum[16], b, rem, dead;
  KvSeq s;
  KfUnit unit[2];              // what the queries that are there belong to
  int bad[8], odd[16], ids[2][32];   // bad: a bit for 16 slots of a group whose page is no page
  float m[8][16], l[8][16], M[16], L[16];
};
#define KF_HEAD 2048
static_assert(sizeof(KfHead) <= KF_HEAD, "the ring begins after it");
// 16 slots' place in the ring is one warp's: a warp that came to it after another would take the phase before the other's for its own where that one's copy is late.
static_assert(kf_ring(256) * kf_parts(256) % kf_warps(256) == 0 && kf_ring(128) * kf_parts(128) % kf_warps(128) == 0 && kf_ring(64) * kf_parts(64) % kf_warps(64) == 0, "a place is one warp's");
__host__ __device__ constexpr int kf_smem(int HD) { return KF_HEAD + kf_ring(HD) * kf_bytes(HD) + kf_warps(HD) * 16 * KF_ROW * 4 + 2 * 16 * kf_qrow(HD); }
static_assert(kf_smem(256) <= 232448 && kf_smem(128) <= 232448 && kf_smem(64) <= 232448, "shared memory");

struct KvPlan {
  int blocks;                  // of k_kv_few
  int least;                   // groups of a block's stretch, at least
  int *unit;                   // [seqs][KV][16-query tiles][2]: the first and the last block that had a part of the unit
  int2 *span;                  // [2 blocks]: the groups of its unit that a part has, from and to
  float *pm, *pl, *po;         // [2 blocks][16](, [hd])
  float *sc;                   // [seqs][KV][G max_rows][sstride]: scores, where weights are wanted
  float *lse;                  // [seqs][KV][G max_rows]: of units that one block has wholly
  int sstride;
  unsigned int *err;           // a wait ran out
};

template <typename T> __device__ __forceinline__ void kf_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void kf_mma<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) { mma16816(d, a[0], a[1], a[2], a[3], b0, b1); }
template <> __device__ __forceinline__ void kf_mma<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void kf_ldsm(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void kf_ldsm_t(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ float kv_exp2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
// a box of pool_map's: from 64 dims number d of kv head g's slot `slot` of a page on
__device__ __forceinline__ void kv_tma(uint32_t dst_s, const CUtensorMap *map, int x, int slot, int d, int g, int page, uint32_t bar_s) {
  asm volatile("cp.async.bulk.tensor.5d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst_s), "l"(map), "r"(x), "r"(slot),
               "r"(d), "r"(g), "r"(page), "r"(bar_s)
               : "memory");
}
__device__ __forceinline__ void kv_expect(uint32_t bar_s, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar_s), "r"(bytes) : "memory");
}

// so many bytes from global to shared memory, counted on a barrier
__device__ __forceinline__ void kv_bulk(uint32_t dst_s, const void *src, uint32_t bytes, uint32_t bar_s) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst_s), "l"(src), "r"(bytes), "r"(bar_s) : "memory");
}
// a block's way through its stretch: the unit it is in, and the groups c0 .. c1 - 1 of it that are the block's
template <int SH> struct KfWalk {
  KvSeq s;
  int b, g, qt, c0, c1;
  int left;                    // groups of the stretch behind this unit's
  __device__ __forceinline__ void take() {
    c1 = min(s.chunks, c0 + left);
    left -= c1 - c0;
  }
  __device__ __forceinline__ bool next(const KvDev &c, const KvRows &r, const KvAttn &a) {
    if (left <= 0) return false;
    c0 = 0;
    if (++qt >= (a.G * s.nc + 15) >> 4) {
      qt = 0;
      if (++g == c.KV) {
        g = 0;
        do {
          if (++b >= c.seqs) { left = 0; return false; }
          s = kv_seq(c, r, b, a.window, a.sinks, SH);
        } while (!s.chunks);
      }
    }
    take();
    return true;
  }
};

__device__ __forceinline__ KvSpan kf_span(const KvSeq &s, int c0, int c1, int sh) { return {c0, c1, s.cs, s.lo >> sh, sh}; }

// The same as kv_attn_row for 16 queries of kv head g from q0 on (query i G + h: row i, head h; `first` and e0: the sequence's first row and its slot), 16 slots at a time,
// stored where `rows` has the query's bit: scores by products (a key that is no number is one column of them), V added up in f32 by those that see its slot alone.
// 3000 rows of 4 heads of 256 on 2 whose middle one has a V of NaN: 5.6 ms, and 39 ms row by row and slot by slot (47 us where all is numbers).
template <typename T, int HD>
__device__ __forceinline__ void kv_attn_rows16(const KvDev &c, const KvAttn &a, int b, int g, int first, int e0, int q0, int NQ, const KvSpan &sp, int lane, unsigned rows) {
  const int gid = lane >> 2, j2 = 2 * (lane & 3), pm = (1 << c.page_sh) - 1;
  const uint16_t *q[2];
  long long at[2];                                         // the lane's two queries: gid and gid + 8
  int e[2], lw[2];
#pragma unroll
  for (int w = 0; w < 2; w++) {
    const int qi = min(q0 + gid + 8 * w, NQ - 1), row = kv_row_of(a, qi);
    const long long r = first + row, h = (long long)(g * a.G + qi - row * a.G) * HD;
    q[w] = a.q + r * a.qs + h + j2;
    at[w] = r * a.os + h + j2;
    e[w] = e0 + row;
    lw[w] = a.window ? kv_before(e[w], a.window) + 1 : 0;
  }
  auto sees = [&](int w, int j) { return j <= e[w] && (j >= lw[w] || j < a.sinks); };
  constexpr int DN = HD == 256 ? 16 : HD / 8;              // eight dims at a time: at head dimension 256 half of them (the registers are the attention kernel's too)
#pragma unroll 1
  for (int d0 = 0; d0 < HD; d0 += 8 * DN) {
    float o[DN][4] = {}, m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll 1
    for (int ch = sp.c0; ch < sp.c1; ch++) {
      const int j0 = (ch < sp.cs ? ch : sp.lo + ch - sp.cs) << sp.sh;
#pragma unroll 1
      for (int j = j0; j < j0 + (1 << sp.sh); j += 16) {
        bool on[2][4], any = false;                          // [query][slots j + j2, j + j2 + 1, and eight on]
#pragma unroll
        for (int i = 0; i < 8; i++) any |= on[i >> 2][i & 3] = sees(i >> 2, j + j2 + (i & 1) + 8 * ((i >> 1) & 1));
        if (!__any_sync(0xffffffffu, any)) continue;
        const int id = kv_page(c, b, j >> c.page_sh);        // (16 slots: one page's)
        if (id < 0) continue;
        const size_t p = kv_at(c, id, g, HD) + (size_t)(j & pm) * HD + j2;
        float x[2][4] = {};
#pragma unroll 2
        for (int d = 0; d < HD; d += 16) {
          const uint32_t qa[4] = {__ldcg((const uint32_t *)(q[0] + d)), __ldcg((const uint32_t *)(q[1] + d)), __ldcg((const uint32_t *)(q[0] + d + 8)), __ldcg((const uint32_t *)(q[1] + d + 8))};
#pragma unroll
          for (int t = 0; t < 2; t++) {
            const uint16_t *k = c.k + p + (8 * t + gid) * HD + d;
            kf_mma<T>(x[t], qa, __ldcg((const uint32_t *)k), __ldcg((const uint32_t *)(k + 8)));
          }
        }
#pragma unroll
        for (int w = 0; w < 2; w++) {
          float t = -INFINITY;
#pragma unroll
          for (int i = 0; i < 4; i++) {
            float &v = x[i >> 1][2 * w + (i & 1)];
            v = on[w][i] ? v * a.scale2 : -INFINITY;
            t = fmaxf(t, v);
          }
          t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 1));
          t = fmaxf(fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2)), m[w]);
          const float ref = t == -INFINITY ? 0.0f : t, cf = m[w] == -INFINITY ? 0.0f : exp2f(m[w] - ref);
          m[w] = t;
          l[w] *= cf;
#pragma unroll
          for (int i = 0; i < 4; i++) {
            float &v = x[i >> 1][2 * w + (i & 1)];
            v = exp2f(v - ref);
            l[w] += v;
          }
#pragma unroll
          for (int k = 0; k < DN; k++) { o[k][2 * w] *= cf; o[k][2 * w + 1] *= cf; }
        }
#pragma unroll
        for (int t = 0; t < 2; t++) {
#pragma unroll 1
          for (int i = 0; i < 8; i += 2) {                   // slots j + 8 t + i and the next: their probabilities are the quad's thread i / 2's
            float pr[4];
#pragma unroll
            for (int k = 0; k < 4; k++) pr[k] = __shfl_sync(0xffffffffu, x[t][k], (lane & ~3) | (i >> 1));
#pragma unroll
            for (int u = 0; u < 2; u++) {
              const int n = 8 * t + i + u;
              const bool s0 = sees(0, j + n), s1 = sees(1, j + n);
              const uint16_t *v = c.v + p + n * HD + d0;
#pragma unroll
              for (int k = 0; k < DN; k++) {
                const float2 f = KvEl<T>::to2(__ldcg((const uint32_t *)(v + 8 * k)));
                if (s0) { o[k][0] += pr[u] * f.x; o[k][1] += pr[u] * f.y; }
                if (s1) { o[k][2] += pr[2 + u] * f.x; o[k][3] += pr[2 + u] * f.y; }
              }
            }
          }
        }
      }
    }
#pragma unroll
    for (int w = 0; w < 2; w++) {
      l[w] += __shfl_xor_sync(0xffffffffu, l[w], 1); l[w] += __shfl_xor_sync(0xffffffffu, l[w], 2);
      if (!(rows >> (gid + 8 * w) & 1)) continue;
      const float inv = l[w] == 0.0f ? 0.0f : 1.0f / l[w];
#pragma unroll
      for (int k = 0; k < DN; k++) {
        if (a.out32) *(float2 *)((float *)a.out + at[w] + d0 + 8 * k) = make_float2(o[k][2 * w] * inv, o[k][2 * w + 1] * inv);
        else *(uint32_t *)((uint16_t *)a.out + at[w] + d0 + 8 * k) = KvEl<T>::of2(o[k][2 * w] * inv, o[k][2 * w + 1] * inv);
      }
    }
  }
}

template <typename T, int HD, bool WT>
__global__ void __launch_bounds__(32 * (kf_warps(HD) + 2), 1) k_kv_few(const KvDev c, const KvRows rw, const KvAttn a, const KvPlan p, const __grid_constant__ CUtensorMap km,
                                                                      const __grid_constant__ CUtensorMap vm) {
  constexpr int CW = kf_warps(HD), NT = 32 * (CW + 2), NG = kf_ring(HD), SB = kf_bytes(HD), KB = SB / 2, TD = HD / 8, SH = kf_sh(HD), PG = kf_parts(HD), QR = kf_qrow(HD);   // TD: tiles of eight dims
  extern __shared__ __align__(1024) uint8_t smem[];
  KfHead &hd = *(KfHead *)smem;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gid = lane >> 2, j2 = 2 * (lane & 3), lr = lane & 7, mi = lane >> 3;
  const uint32_t bar_s = smem_u32(smem), ring_s = bar_s + KF_HEAD, q_s = ring_s + NG * SB + CW * 16 * KF_ROW * 4;   // two units' queries
  float *sums = (float *)(smem + KF_HEAD + NG * SB);                     // [warp][16][KF_ROW]
  auto full = [&](int i) { return bar_s + 8u * (uint32_t)i; };
  auto empty = [&](int i) { return bar_s + 64u + 8u * (uint32_t)i; };
  auto qfull = [&](int i) { return bar_s + 128u + 8u * (uint32_t)i; };
  auto qempty = [&](int i) { return bar_s + 144u + 8u * (uint32_t)i; };
  if (tid < 8) { mbar_init(full(tid), 2); mbar_init(empty(tid), PG); }
  if (tid < 2) { mbar_init(qfull(tid), 1); mbar_init(qempty(tid), 1); }
  if (tid == 0) asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  if (tid < 16) hd.odd[tid] = 0;
  if (tid == 0) hd.dead = 0;
  pdl_trigger();
  pdl_wait();
  // ---- the block's stretch: groups of every sequence, summed over the threads' runs of sequences ----
  const int run = (c.seqs + NT - 1) / NT, ba = min(c.seqs, tid * run), bz = min(c.seqs, ba + run);
  KvSeq seq;
  auto work = [&](int b) {
    seq = kv_seq(c, rw, b, a.window, a.sinks, SH);
    return seq.chunks * c.KV * ((a.G * seq.nc + 15) >> 4);
  };
  int mine = 0;
#pragma unroll 1
  for (int b = ba; b < bz; b++) mine += work(b);
  int to = mine;
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) { const int o = __shfl_up_sync(0xffffffffu, to, m); if (lane >= m) to += o; }
  if (lane == 31) hd.sum[warp] = to;
  __syncthreads();
  int all = 0;
#pragma unroll
  for (int w = 0; w < CW + 2; w++) { if (w < warp) to += hd.sum[w]; all += hd.sum[w]; }
  const int per = max(p.least, (all + (int)gridDim.x - 1) / (int)gridDim.x);
  if (blockIdx.x >= (all + per - 1) / per) return;
  const int start = per * blockIdx.x;
  if (to - mine <= start && start < to) {
    int at = to - mine, b = ba;
#pragma unroll 1
    for (;; b++) { const int w = work(b); if (start < at + w) break; at += w; }
    hd.b = b; hd.rem = start - at; hd.s = seq;
  }
  __syncthreads();
  bool dead = false;
  const int bs = min(c.page_sh, SH), bmask = (1 << bs) - 1;   // log2 of a box's slots: a page's part of a group
  if (warp >= CW) {
    // ---- K and the queries, or V, over the ends of units.  The pages of 32 boxes are asked for at once, those of the next 32 while these are requested ----
    const bool isv = warp > CW;
    const CUtensorMap *map = isv ? &vm : &km;
    const uint32_t ring = ring_s + (isv ? KB : 0);
    KfWalk<SH> use;
    use.b = hd.b;
    use.s = hd.s;
    {
      const int qts = (a.G * use.s.nc + 15) >> 4, u = hd.rem / use.s.chunks;
      use.g = u / qts; use.qt = u % qts; use.c0 = hd.rem % use.s.chunks;
      use.left = min(per, all - start);
      use.take();
    }
    const int boxes = 1 << (SH - bs), gb = 5 - (SH - bs), pm = (1 << c.page_sh) - 1;   // of a group; log2 of the groups that 32 boxes are
    int st = 0, sp = 0;
    uint32_t round = 0;
    auto tell = [&](bool more) {                           // a unit, and its queries, a lane each; rows behind the last one stay what they are: their results go nowhere
      const int qb = sp & 1, q0 = 16 * use.qt, nq = more ? min(16, a.G * use.s.nc - q0) : 0;
      if (sp >= 2 && !dead && !mbar_wait(qempty(qb), (uint32_t)((sp >> 1) - 1) & 1u)) { dead = true; if (lane == 0) atomicExch(p.err, 1u); }
      dead = __any_sync(0xffffffffu, dead);
      if (lane == 0) {
        hd.unit[qb] = {use.s, use.b, use.g, use.qt, use.c0, more ? use.c1 : -1, use.left <= 0};
        if (dead || !more) mbar_arrive(qfull(qb));
        else kv_expect(qfull(qb), nq * HD * 2);
      }
      __syncwarp();
      if (lane < nq && !dead) {
        const int qi = q0 + lane, row = kv_row_of(a, qi);
        kv_bulk(q_s + (qb * 16 + lane) * QR, a.q + (long long)(use.s.first + row) * a.qs + (long long)(use.g * a.G + qi - row * a.G) * HD, HD * 2, qfull(qb));
      }
      sp++;
    };
    do {
      const int last = use.s.e0 + use.s.nc - 1;
      struct Entry { int id; bool on; };                   // on: some row sees some of it
      auto pages = [&](int ch) {                           // of box lane % boxes of group ch + lane / boxes
        Entry x = {-1, false};
        const int k = ch + (lane >> (SH - bs)), j = kv_chunk_slot(use.s, k, SH) + ((lane & (boxes - 1)) << bs);
        x.on = k < use.c1 && j <= last && (!a.window || j + bmask > kv_before(use.s.e0, a.window) || j < a.sinks);
        if (x.on) asm volatile("ld.global.cg.s32 %0, [%1];" : "=r"(x.id) : "l"(c.table + (size_t)use.b * c.tstride + (j >> c.page_sh)));
        return x;
      };
      Entry next = pages(use.c0);
      if (!isv) tell(true);
#pragma unroll 1
      for (int c0 = use.c0; c0 < use.c1; c0 += 1 << gb) {
        const int n = min(1 << gb, use.c1 - c0);
        __syncwarp();
        hd.ids[isv][lane] = !next.on ? -2 : (unsigned)next.id < (unsigned)c.n_pages ? next.id : -1;   // -2: not wanted, -1: no page
        __syncwarp();
        next = pages(c0 + (1 << gb));
        if (lane == 0) {                                   // one thread: a warp that walks together takes three times as long a request
#pragma unroll 1
          for (int k = 0; k < n; k++) {
            const int slot = kv_chunk_slot(use.s, c0 + k, SH) & pm;
            if (round && !dead && !mbar_wait(empty(st), (round - 1) & 1u)) { dead = true; atomicExch(p.err, 1u); }
            uint32_t bad = 0;
            int have = 0;
#pragma unroll 1
            for (int x = 0; x < boxes; x++) {
              const int id = hd.ids[isv][(k << (SH - bs)) + x];
              if (id >= 0) have++;
              else if (id == -1) bad |= ((1u << (1 << (bs - 4))) - 1) << (x << (bs - 4));
            }
            if (bad) atomicOr(c.err, KV_ERR_PAGE);
            if (!isv) hd.bad[st] = bad;
            if (have && !dead) {
              kv_expect(full(st), (uint32_t)have * (HD * 2 << bs));
#pragma unroll 1
              for (int x = 0; x < boxes; x++) {
                const int id = hd.ids[isv][(k << (SH - bs)) + x];
                if (id < 0) continue;
                kv_tma(ring + st * SB + x * (HD * 2 << bs), map, 0, slot, 0, use.g, id, full(st));
              }
            } else mbar_arrive(full(st));
            if (++st == NG) { st = 0; round++; }
          }
        }
        st = __shfl_sync(0xffffffffu, st, 0); round = __shfl_sync(0xffffffffu, round, 0); dead = __any_sync(0xffffffffu, dead);
      }
    } while (use.next(c, rw, a));
    if (!isv) tell(false);
    if (dead) for (int i = 0; i < 64; i++) __nanosleep(1000);   // copies may be on their way
    return;
  }
  auto wait = [&](uint32_t bar, uint32_t parity) {
    if (!dead && !mbar_wait(bar, parity)) { dead = true; if (lane == 0) atomicExch(p.err, 1u); }
  };
  auto meet = [&]() { asm volatile("bar.sync 1, %0;" ::"n"(32 * CW) : "memory"); };   // the warps that compute
  int n0 = 0, sp = 0;                                      // groups of the stretch before this unit's, units before it
#pragma unroll 1
  for (;;) {
    wait(qfull(sp & 1), (uint32_t)(sp >> 1) & 1u);
    const KfUnit use = hd.unit[sp & 1];
    if (dead) hd.dead = 1;
    meet();                                                // (one warp's wait that ran out is every warp's end: they meet again and again)
    if (use.c1 < 0 || hd.dead) break;
    const KvSeq &s = use.s;
    const int NQ = a.G * s.nc, q0 = 16 * use.qt, last = s.e0 + s.nc - 1;
    const uint32_t qs = q_s + (sp & 1) * 16 * QR;
    float o[TD][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < TD; i++)
#pragma unroll
      for (int k = 0; k < 4; k++) o[i][k] = 0.0f;
    // the slots that the thread's two queries see: from lw to e, and below the first tokens' end
    int e[2], lw[2];
#pragma unroll
    for (int k = 0; k < 2; k++) {
      const int qi = q0 + gid + 8 * k;
      e[k] = qi < NQ ? s.e0 + kv_row_of(a, qi) : -1;
      lw[k] = a.window ? kv_before(e[k], a.window) + 1 : 0;
    }
    const int ea = s.e0 + kv_row_of(a, q0), ez = s.e0 + kv_row_of(a, min(q0 + 15, NQ - 1));      // slots of the unit's first and last row
    const int m1 = (n0 + use.c1 - use.c0) * PG;
    int m0 = n0 * PG;                                      // 16 slots number m of the stretch are warp m % CW's
    m0 += (warp + CW - m0 % CW) % CW;
#pragma unroll 1
    for (int mm = m0; mm < m1; mm += CW) {
      const int n = mm / PG, part = mm % PG, st = n % NG, slot = kv_chunk_slot(s, use.c0 + n - n0, SH) + 16 * part;
      const uint32_t k_s = ring_s + st * SB + ((16 * part) >> bs) * (HD * 2 << bs) + ((16 * part) & bmask) * 128, v_s = k_s + KB, blk = 128u << bs;   // 64 dims of a box
      wait(full(st), (uint32_t)(n / NG) & 1u);
      // (nothing of it is seen, or it was not brought)
      const bool none = (hd.bad[st] >> part & 1) || dead || slot > last || (a.window && slot + 15 <= kv_before(s.e0, a.window) && slot >= a.sinks);
      float x[2][4];
      if (!none) {
        // slots that no row sees: their V is taken out, whatever it holds (0 times NaN is NaN)
        if (slot + 15 > last || (a.window && slot <= kv_before(s.e0, a.window) && slot + 15 >= a.sinks)) {
          for (int i = lane; i < 16 * TD; i += 32) {
            const int r = i & 15;
            if (!kv_any_sees(s, slot + r, a.window, a.sinks)) *(uint4 *)(smem + (v_s - bar_s) + (i >> 7) * blk + r * 128 + ((i >> 4) & 7) * 16) = make_uint4(0, 0, 0, 0);
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
        }
        float y[2][2][4];                                  // even and odd steps: shorter chains
#pragma unroll
        for (int i = 0; i < 16; i++) y[i >> 3][(i >> 2) & 1][i & 3] = 0.0f;
#pragma unroll
        for (int ks = 0; ks < HD / 16; ks++) {
          uint32_t qa[4], kb[4];
          // queries: matrix mi has queries 8 (mi & 1) .., dims 8 (2 ks + mi / 2) ..; keys: slots 8 (mi / 2) .., dims 8 (2 ks + (mi & 1)) ..
          kf_ldsm(qa, qs + (lr + 8 * (mi & 1)) * QR + (2 * ks + (mi >> 1)) * 16);
          const int unit = 2 * ks + (mi & 1), row = lr + 8 * (mi >> 1);
          kf_ldsm(kb, k_s + (unit >> 3) * blk + row * 128 + (((unit & 7) ^ lr) << 4));
          kf_mma<T>(y[ks & 1][0], qa, kb[0], kb[1]);
          kf_mma<T>(y[ks & 1][1], qa, kb[2], kb[3]);
        }
#pragma unroll
        for (int i = 0; i < 8; i++) x[i >> 2][i & 3] = (y[0][i >> 2][i & 3] + y[1][i >> 2][i & 3]) * a.scale2;
      }
      const bool whole = !none && slot + 15 <= ea && (!a.window || slot > kv_before(ez, a.window) || slot + 15 < a.sinks) && q0 + 15 < NQ;
      if (!whole) {
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
          for (int k = 0; k < 4; k++) {
            const int j = slot + 8 * t + j2 + (k & 1), w = k >> 1;
            if (none | (j > e[w]) | ((j < lw[w]) & (j >= a.sinks))) x[t][k] = -INFINITY;
          }
      }
      if constexpr (WT) {
#pragma unroll
        for (int w = 0; w < 2; w++)
          if (q0 + gid + 8 * w < NQ && slot <= last) {
            float *d = p.sc + (((size_t)use.b * c.KV + use.g) * (a.G * rw.max_rows) + q0 + gid + 8 * w) * p.sstride + slot + j2;
            *(float2 *)d = make_float2(x[0][2 * w], x[0][2 * w + 1]);
            *(float2 *)(d + 8) = make_float2(x[1][2 * w], x[1][2 * w + 1]);
          }
      }
      float cf[2];
#pragma unroll
      for (int w = 0; w < 2; w++) {
        float t = fmaxf(fmaxf(x[0][2 * w], x[0][2 * w + 1]), fmaxf(x[1][2 * w], x[1][2 * w + 1]));
        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 1));
        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2));
        t = fmaxf(t, m[w]);
        const float ref = t == -INFINITY ? 0.0f : t;      // (nothing seen yet: every probability is 0)
        cf[w] = kv_exp2(m[w] - ref);
        m[w] = t;
#pragma unroll
        for (int k = 0; k < 2; k++) { x[0][2 * w + k] = kv_exp2(x[0][2 * w + k] - ref); x[1][2 * w + k] = kv_exp2(x[1][2 * w + k] - ref); }
        l[w] = l[w] * cf[w] + ((x[0][2 * w] + x[0][2 * w + 1]) + (x[1][2 * w] + x[1][2 * w + 1]));
      }
      if (!none) {
        if (__any_sync(0xffffffffu, cf[0] != 1.0f || cf[1] != 1.0f)) {
#pragma unroll
          for (int i = 0; i < TD; i++) { o[i][0] *= cf[0]; o[i][1] *= cf[0]; o[i][2] *= cf[1]; o[i][3] *= cf[1]; }
        }
        const uint32_t pa[4] = {KvEl<T>::of2(x[0][0], x[0][1]), KvEl<T>::of2(x[0][2], x[0][3]), KvEl<T>::of2(x[1][0], x[1][1]), KvEl<T>::of2(x[1][2], x[1][3])};
#pragma unroll
        for (int i = 0; i < TD; i += 2) {
          uint32_t vb[4];                                  // matrix mi: slots 8 (mi & 1) .., dims 8 (i + mi / 2) ..
          const int unit = i + (mi >> 1), row = lr + 8 * (mi & 1);
          kf_ldsm_t(vb, v_s + (unit >> 3) * blk + row * 128 + (((unit & 7) ^ lr) << 4));
          kf_mma<T>(o[i], pa, vb[0], vb[1]);
          kf_mma<T>(o[i + 1], pa, vb[2], vb[3]);
        }
      }
      __syncwarp();                                        // the slots have been read
      if (lane == 0) mbar_arrive(empty(st));
    }
    n0 += use.c1 - use.c0;
    sp++;
    // ---- the warps' sums put together: everything relative to the largest maximum, then 32 dims at a time, or 64 or 128 where there are so few queries ----
#pragma unroll
    for (int w = 0; w < 2; w++) {
      l[w] += __shfl_xor_sync(0xffffffffu, l[w], 1); l[w] += __shfl_xor_sync(0xffffffffu, l[w], 2);
      if (j2 == 0) { hd.m[warp][gid + 8 * w] = m[w]; hd.l[warp][gid + 8 * w] = l[w]; }
    }
    meet();
    if (tid == 0) mbar_arrive(qempty((sp - 1) & 1));        // the queries have been read
#pragma unroll
    for (int w = 0; w < 2; w++) {
      float M = -INFINITY, L = 0.0f;
#pragma unroll
      for (int k = 0; k < CW; k++) M = fmaxf(M, hd.m[k][gid + 8 * w]);
      const float ref = M == -INFINITY ? 0.0f : M, f = kv_exp2(m[w] - ref);
      if (warp == 0) {
#pragma unroll
        for (int k = 0; k < CW; k++) L += hd.l[k][gid + 8 * w] * kv_exp2(hd.m[k][gid + 8 * w] - ref);
        if (j2 == 0) { hd.M[gid + 8 * w] = M; hd.L[gid + 8 * w] = L; }
      }
#pragma unroll
      for (int i = 0; i < TD; i++) { o[i][2 * w] *= f; o[i][2 * w + 1] *= f; }
    }
    const bool wholly = use.c0 == 0 && use.c1 == s.chunks;
    if (tid == 0) {
      int *u = p.unit + (((size_t)use.b * c.KV + use.g) * ((a.G * rw.max_rows + 15) >> 4) + use.qt) * 2;
      if (use.c0 == 0) u[0] = blockIdx.x;
      if (use.c1 == s.chunks) u[1] = blockIdx.x;
      p.span[blockIdx.x * 2 + (use.c0 == 0)] = make_int2(use.c0, use.c1);
    }
    const size_t part = ((size_t)blockIdx.x * 2 + (use.c0 == 0)) * 16;
    const int nr = min(16, NQ - q0);
    auto result = [&](int r, int dim, float2 v) {          // two dims of a query
      if (!wholly) { *(float2 *)(p.po + (part + r) * HD + dim) = v; return; }
      const int qi = q0 + r, row = kv_row_of(a, qi), h = use.g * a.G + qi - row * a.G;
      const float L = hd.L[r], inv = L == 0.0f ? 0.0f : 1.0f / L;   // (nothing seen: zeros)
      if (kv_again<T>(v.x) || kv_again<T>(v.y)) hd.odd[r] = 1;
      const long long at = (long long)(s.first + row) * a.os + (long long)h * HD + dim;
      if (a.out32) *(float2 *)((float *)a.out + at) = make_float2(v.x * inv, v.y * inv);
      else *(uint32_t *)((uint16_t *)a.out + at) = KvEl<T>::of2(v.x * inv, v.y * inv);
    };
    if (use.last) {
      // nothing is brought any more: all dims at once, in the ring's memory
      constexpr int RW = HD + 8;
      static_assert(CW * 16 * RW * 4 <= NG * SB, "the ring's memory");
      float *all_ = (float *)(smem + KF_HEAD), *d = all_ + warp * 16 * RW;
#pragma unroll
      for (int i = 0; i < TD; i++) {
        if (gid < nr) *(float2 *)(d + gid * RW + 8 * i + j2) = make_float2(o[i][0], o[i][1]);
        if (gid + 8 < nr) *(float2 *)(d + (gid + 8) * RW + 8 * i + j2) = make_float2(o[i][2], o[i][3]);
      }
      meet();
#pragma unroll 2
      for (int it = tid; it < nr * (HD / 2); it += 32 * CW) {
        const int r = it / (HD / 2), dim = 2 * (it % (HD / 2));
        float2 v = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < CW; k++) { const float2 t = *(const float2 *)(all_ + (k * 16 + r) * RW + dim); v.x += t.x; v.y += t.y; }
        result(r, dim, v);
      }
      meet();
    } else {
      const int fold = HD == 64 ? (nr <= 8) : nr <= 4 ? 2 : nr <= 8, rows = 16 >> fold;   // 32 << fold dims at a time, of `rows` rows
#pragma unroll
      for (int d0 = 0; d0 < HD; d0 += 32) {
        const int at32 = (d0 >> 5) & ((1 << fold) - 1);    // which 32 of those dims
        float *d = sums + (warp * 16 + at32 * rows) * KF_ROW;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          if (gid < rows) *(float2 *)(d + gid * KF_ROW + 8 * i + j2) = make_float2(o[d0 / 8 + i][0], o[d0 / 8 + i][1]);
          if (rows == 16) *(float2 *)(d + (gid + 8) * KF_ROW + 8 * i + j2) = make_float2(o[d0 / 8 + i][2], o[d0 / 8 + i][3]);
        }
        if (at32 != (1 << fold) - 1) continue;
        meet();
        const int first = d0 + 32 - (32 << fold);
#pragma unroll 1
        for (int it = tid; it < 256; it += 32 * CW) {      // a row, two dims
          const int pos = it >> 4, r = pos & (rows - 1), dd = 2 * (it & 15);
          if (r >= nr) continue;
          float2 v = make_float2(0.0f, 0.0f);
#pragma unroll
          for (int k = 0; k < CW; k++) { const float2 t = *(const float2 *)(sums + (k * 16 + pos) * KF_ROW + dd); v.x += t.x; v.y += t.y; }
          result(r, first + 32 * (pos >> (4 - fold)) + dd, v);
        }
        meet();
      }
    }
    if (tid < 16 && q0 + tid < NQ) {
      if (!wholly) { p.pm[part + tid] = hd.M[tid]; p.pl[part + tid] = hd.L[tid]; }
      else if (WT) p.lse[((size_t)use.b * c.KV + use.g) * (a.G * rw.max_rows) + q0 + tid] = hd.L[tid] == 0.0f ? INFINITY : hd.M[tid] + log2f(hd.L[tid]);
    }
    // rows whose result is no number once more (kv_attn_row says why)
    if (wholly && warp == 0) {
      const unsigned again = __ballot_sync(0xffffffffu, lane < 16 && hd.odd[lane & 15] && hd.L[lane & 15] == hd.L[lane & 15]);
      if (__builtin_expect(again != 0, 0)) kv_attn_rows16<T, HD>(c, a, use.b, use.g, s.first, s.e0, q0, NQ, kf_span(s, 0, s.chunks, SH), lane, again);
      if (lane < 16) hd.odd[lane] = 0;
    }
  }
}

// How many parts a unit has whose first and last block are noted so.  After a wait ran out (p.err) a unit may not be noted at all, and what stands there is whatever
// the workspace held: no part, then, or parts that exist.
__host__ __device__ __forceinline__ int kf_parts_of(int first, int last, int blocks) { return first >= 0 && last >= first && last < blocks ? last - first + 1 : 0; }
// the part of a unit that block w had, of blocks w0 .. (only the first begins with the unit's first chunk)
__device__ __forceinline__ size_t kf_part(int w, int w0) { return ((size_t)w * 2 + (w == w0)) * 16; }

// Units that several blocks had: a block a query, its four warps the parts in turn, each with what it needs of them asked for at once.  Blocks from
// `joins` on: what every slot got, KJ_SLOTS of a kv head each.
#define KJ_SLOTS 2048
template <typename T, int HD, bool WT>
__global__ void __launch_bounds__(128) k_kv_join(const KvDev c, const KvRows rw, const KvAttn a, const KvPlan p, int joins, int wblocks) {
  constexpr int E = HD / 32;
  __shared__ float sm[4], sl[4], so[4][HD], lse[64];
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, NQM = a.G * rw.max_rows, QTM = (NQM + 15) >> 4;
  if (!WT || blockIdx.x < joins) {
    const int qi = blockIdx.x % NQM, gb = blockIdx.x / NQM, g = gb % c.KV, b = gb / c.KV;
    const int2 w = __ldcg((const int2 *)p.unit + (size_t)gb * QTM + (qi >> 4));
    const KvSeq s = kv_seq(c, rw, b, a.window, a.sinks, kf_sh(HD));
    if (qi >= a.G * s.nc || kf_parts_of(w.x, w.y, p.blocks) < 2) return;
    float o[E], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int k = 0; k < E; k++) o[k] = 0.0f;
#pragma unroll 2
    for (int i = w.x + warp; i <= w.y; i += 4) {
      const size_t at = kf_part(i, w.x) + (qi & 15);
      const float pm = __ldcg(p.pm + at), pl = __ldcg(p.pl + at);
      float2 v[E / 2];
#pragma unroll
      for (int k = 0; k < E / 2; k++) v[k] = __ldcg((const float2 *)(p.po + at * HD + lane * E) + k);
      const float t = fmaxf(m, pm), ref = t == -INFINITY ? 0.0f : t, f = kv_exp2(m - ref), fp = kv_exp2(pm - ref);
      l = l * f + pl * fp;
      m = t;
#pragma unroll
      for (int k = 0; k < E / 2; k++) { o[2 * k] = o[2 * k] * f + v[k].x * fp; o[2 * k + 1] = o[2 * k + 1] * f + v[k].y * fp; }
    }
    if (lane == 0) { sm[warp] = m; sl[warp] = l; }
#pragma unroll
    for (int k = 0; k < E; k += 2) *(float2 *)&so[warp][lane * E + k] = make_float2(o[k], o[k + 1]);
    __syncthreads();
    if (warp) return;
    const float M = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3])), ref = M == -INFINITY ? 0.0f : M;
    float f[4];
    l = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) { f[i] = kv_exp2(sm[i] - ref); l += sl[i] * f[i]; }
#pragma unroll
    for (int k = 0; k < E; k++) {
      o[k] = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; i++) o[k] += so[i][lane * E + k] * f[i];
    }
    const int row = kv_row_of(a, qi), h = g * a.G + qi - row * a.G;
    if (kv_again_any<T, E>(o, l)) {                        // the parts whose sums are no numbers once more, by themselves
      m = -INFINITY; l = 0.0f;
#pragma unroll
      for (int k = 0; k < E; k++) o[k] = 0.0f;
#pragma unroll 1
      for (int i = w.x; i <= w.y; i++) {
        const size_t at = kf_part(i, w.x) + (qi & 15);
        float pm = __ldcg(p.pm + at), pl = __ldcg(p.pl + at), v[E];
#pragma unroll
        for (int k = 0; k < E; k += 2) { const float2 t = __ldcg((const float2 *)(p.po + at * HD + lane * E + k)); v[k] = t.x; v[k + 1] = t.y; }
        if (kv_again_any<T, E>(v, pl)) {
          const int2 part = __ldcg(p.span + 2 * i + (i == w.x));
          kv_attn_row<T, HD>(c, a, b, s.first + row, h, s.e0 + row, kf_span(s, max(part.x, 0), min(part.y, s.chunks), kf_sh(HD)), lane, v, pm, pl);
        }
        kv_add_part<E>(o, m, l, v, pm, pl);
      }
    }
    kv_store<T, HD>(a, s.first + row, h, lane, o, l);
    return;
  }
  if constexpr (WT) {
    const int u = blockIdx.x - joins, wb = u % wblocks, gb = u / wblocks, b = gb / c.KV;
    const KvSeq s = kv_seq(c, rw, b, a.window, a.sinks, kf_sh(HD));
    if (wb * KJ_SLOTS >= s.len) return;
    const int NQ = a.G * s.nc;
    const size_t ug = gb;
    // four slots a thread, and the first eight queries' scores of them at once; the first slots' before the queries' sums are there
    float in[4], sc[8][4];
    bool on[4], see[4];
    auto ask = [&](int j0) {
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const int j = j0 + k * 128 + tid;
        on[k] = j < s.len; see[k] = on[k] && NQ && kv_any_sees(s, j, a.window, a.sinks);
        in[k] = 0.0f;
        if (on[k] && a.w_in) asm volatile("ld.global.cg.f32 %0, [%1];" : "=f"(in[k]) : "l"(a.w_in + ug * a.wstride + j));
#pragma unroll
        for (int q = 0; q < 8; q++) {
          sc[q][k] = -INFINITY;
          if (see[k] && q < NQ) asm volatile("ld.global.cg.f32 %0, [%1];" : "=f"(sc[q][k]) : "l"(p.sc + (ug * NQM + q) * p.sstride + j));
        }
      }
    };
    ask(wb * KJ_SLOTS);
    if (tid < NQ) {
      const int2 w = __ldcg((const int2 *)p.unit + ug * QTM + (tid >> 4));
      if (kf_parts_of(w.x, w.y, p.blocks) < 2) lse[tid] = __ldcg(p.lse + ug * NQM + tid);
      else {
        float M = -INFINITY, l = 0.0f;
#pragma unroll 4
        for (int i = w.x; i <= w.y; i++) M = fmaxf(M, __ldcg(p.pm + kf_part(i, w.x) + (tid & 15)));
        const float ref = M == -INFINITY ? 0.0f : M;
#pragma unroll 4
        for (int i = w.x; i <= w.y; i++) { const size_t at = kf_part(i, w.x) + (tid & 15); l += __ldcg(p.pl + at) * exp2f(__ldcg(p.pm + at) - ref); }
        lse[tid] = l == 0.0f ? INFINITY : M + log2f(l);
      }
    }
    __syncthreads();
#pragma unroll 1
    for (int j0 = wb * KJ_SLOTS;; ) {
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int q = 0; q < 8; q++)
        if (q < NQ)
#pragma unroll
          for (int k = 0; k < 4; k++) sum[k] += kv_exp2(sc[q][k] - lse[q]);
#pragma unroll 4
      for (int q = 8; q < NQ; q++)
#pragma unroll
        for (int k = 0; k < 4; k++)
          if (see[k]) sum[k] += kv_exp2(__ldcg(p.sc + (ug * NQM + q) * p.sstride + j0 + k * 128 + tid) - lse[q]);
#pragma unroll
      for (int k = 0; k < 4; k++)
        if (on[k]) a.w_out[ug * a.wstride + j0 + k * 128 + tid] = in[k] + sum[k];
      j0 += 512;
      if (j0 >= min(s.len, (wb + 1) * KJ_SLOTS)) break;
      ask(j0);
    }
  }
}
