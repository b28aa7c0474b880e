// kv.cu -- the paged key-value cache's operators (llb_b200_kv_*): rows in, attention, eviction.
#include <algorithm>
#include <limits.h>
#include <math.h>

#include "../../include/llb_b200.h"
#include "host.cuh"
#include "kv.cuh"
#include "kvatt.cuh"
#include "kvpf.cuh"

static unsigned int *g_kv_err = nullptr;   // what the kernels met (KV_ERR_*)
static decltype(&cuTensorMapEncodeTiled) g_kv_map = nullptr;

// ---- rows in ------------------------------------------------------------------------------------
// A warp a row, or a few heads of one where there are few rows: it finds the row's place, makes its sines, and takes the heads, 512 / head_dim at a
// time and the next ones on their way.  A lane has eight dimensions in each half of a head and reads their partners of the rotation too (the line is
// there), so that nothing but the sum of squares crosses lanes.  Angles in turns and 64 bits: at position 200,000 a 32-bit product is 0.008
// off; what is left of whole turns fits a float.  8926 rows of 24 + 2 x 4 heads of 256, bf16: 78 us, 3.7 TB/s; with registers held down
// for three blocks an SM instead of two, 89 us.
struct KvAppend {
  const void *q, *k, *v;
  long long qs, ks, vs;
  int qhs;
  const float *qn, *kn;
  const double *invfreq;
  const int *pos;
  uint16_t *qo;
  long long qos;
  int H, rope;
  float eps;
  int wide;                    // q, k, v and q_out: eight elements lie on a multiple of 16 bytes
};
// eight values of a row of the caller's, as they lie there
template <typename X> struct KaIn { uint32_t w[2 * sizeof(X)]; };
template <typename X> __device__ __forceinline__ KaIn<X> ka_load(const X *p, bool wide) {
  constexpr int W = 2 * sizeof(X);
  KaIn<X> r;
  if (wide) {
#pragma unroll
    for (int i = 0; i < W; i += 4) { const uint4 t = __ldcs((const uint4 *)p + i / 4); r.w[i] = t.x; r.w[i + 1] = t.y; r.w[i + 2] = t.z; r.w[i + 3] = t.w; }
  } else if constexpr (sizeof(X) == 4) {
#pragma unroll
    for (int i = 0; i < W; i++) r.w[i] = __ldcs((const uint32_t *)p + i);
  } else {
#pragma unroll
    for (int i = 0; i < W; i++) r.w[i] = (uint32_t)__ldcs((const uint16_t *)p + 2 * i) | ((uint32_t)__ldcs((const uint16_t *)p + 2 * i + 1) << 16);
  }
  return r;
}
// as pairs
template <typename X> __device__ __forceinline__ void ka_values(const KaIn<X> &r, f32x2 (&x)[4]) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if constexpr (sizeof(X) == 4) x[i] = x2_pack(__uint_as_float(r.w[2 * i]), __uint_as_float(r.w[2 * i + 1]));
    else { const float2 f = KvEl<X>::to2(r.w[i]); x[i] = x2_pack(f.x, f.y); }
  }
}
template <typename T, typename X, int HD, bool ROW>
__global__ void __launch_bounds__(256, ROW ? 2 : 1) k_kv_append(const KvDev c, const KvRows rw, const KvAppend a) {
  constexpr int LPH = HD / 16, HPW = 32 / LPH, H2 = HD / 2;   // lanes a head, heads a warp
  __shared__ float2 turn[8][H2];
  pdl_trigger();
  pdl_wait();
  if (!blockIdx.x && !blockIdx.y) kv_check_rows(c, rw);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, half = a.rope >> 1, r = ROW ? blockIdx.x * 8 + warp : blockIdx.x;
  const int b = r < rw.rows ? kv_find(rw, c.seqs, r, lane) : -1;
  if (b < 0) return;                           // behind the last row, or row_start is not what it should be
  const int slot = kv_len(c, b) - __ldcg(rw.start + b + 1) + r;
  const double pos = a.pos ? (double)__ldcg(a.pos + b) + (r - __ldcg(rw.start + b)) : slot;   // (a first position near 2^31 has later ones above it)
  const int id = slot >= 0 ? kv_page(c, b, slot >> c.page_sh) : -1;
#pragma unroll 1
  for (int p = lane; p < half; p += 32) {
    const double n = pos * __ldg(a.invfreq + p) * 0.15915494309189533577;   // turns
    float s, co;
    sincospif((float)(2.0 * (n - rint(n))), &s, &co);
    turn[warp][p] = make_float2(co, s);
  }
  __syncwarp();
  const int sub = lane / LPH, l8 = 8 * (lane % LPH);   // the lane's head of the warp's; its dimensions l8 .. and HD / 2 + l8 ..
  const bool lanes = half % 8 == 0;                    // eight dimensions' partners lie side by side
  const size_t at = id < 0 ? 0 : kv_at(c, id, 0, HD) + (size_t)(slot & ((1 << c.page_sh) - 1)) * HD, head_step = (size_t)HD << c.page_sh;
  // heads ha .. n - 1 of one kind (the warp's first HPW of them where the warp has no row of its own)
  auto heads = [&](const X *src, long long step, int ha, int n, const float *norm, uint16_t *dst, size_t dstep, bool wide, bool turns) {
    f32x2 A[2][4], B[2][4];                    // a dimension becomes x A + partner B, divided by the root of the mean square
    bool roll[2];                              // the warp: this half of the heads has turned dimensions
#pragma unroll
    for (int h = 0; h < 2; h++) {
      roll[h] = turns && a.rope > h * H2;
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        float p[2], q[2];
#pragma unroll
        for (int k = 0; k < 2; k++) {
          const int d = h * H2 + l8 + j + k;
          const bool low = d < half, in = roll[h] && d < a.rope;
          const float2 t = in ? turn[warp][low ? d : d - half] : make_float2(1.0f, 0.0f);
          p[k] = (norm ? __ldg(norm + d) : 1.0f) * t.x;
          q[k] = (norm && in ? __ldg(norm + (low ? d + half : d - half)) : 1.0f) * (low ? -t.y : t.y);
        }
        A[h][j / 2] = x2_pack(p[0], p[1]); B[h][j / 2] = x2_pack(q[0], q[1]);
      }
    }
    KaIn<X> nin[2], npr[2];                    // the next heads, on their way while these are worked on
    auto ask = [&](int h0) {
      const X *q = src + min(h0 + sub, n - 1) * step + l8;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        nin[h] = ka_load<X>(q + h * H2, a.wide);
        if (!roll[h]) continue;
        const int d = h * H2 + l8;
        if (lanes) npr[h] = ka_load<X>(d < a.rope ? q + h * H2 + (d < half ? half : -half) : q + h * H2, a.wide);
        else if constexpr (sizeof(X) == 4) {
#pragma unroll
          for (int j = 0; j < 8; j++) npr[h].w[j] = __ldcs((const uint32_t *)(q + h * H2) + j + (d + j < half ? half : d + j < a.rope ? -half : 0));
        } else {
#pragma unroll
          for (int j = 0; j < 8; j += 2) {
            uint32_t v[2];
#pragma unroll
            for (int k = 0; k < 2; k++) v[k] = __ldcs((const uint16_t *)(q + h * H2) + j + k + (d + j + k < half ? half : d + j + k < a.rope ? -half : 0));
            npr[h].w[j / 2] = v[0] | v[1] << 16;
          }
        }
      }
    };
    ask(ha);
#pragma unroll 1
    for (int h0 = ha; h0 < n; h0 += HPW) {
      f32x2 x[2][4], y[2][4];
#pragma unroll
      for (int h = 0; h < 2; h++) {
        ka_values<X>(nin[h], x[h]);
        if (roll[h]) ka_values<X>(npr[h], y[h]);
      }
      if (ROW && h0 + HPW < n) ask(h0 + HPW);
      float sc = 1.0f;
      if (norm) {
        f32x2 q = x2_mul(x[0][0], x[0][0]), q2 = x2_mul(x[1][0], x[1][0]);
#pragma unroll
        for (int j = 1; j < 4; j++) { q = x2_fma(x[0][j], x[0][j], q); q2 = x2_fma(x[1][j], x[1][j], q2); }
        float q0, q1;
        x2_unpack(x2_add(q, q2), q0, q1);
        float ss = q0 + q1;
#pragma unroll
        for (int m = LPH / 2; m; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
        sc = rsqrtf(ss * (1.0f / HD) + a.eps);
      }
      const f32x2 sc2 = x2_pack(sc, sc);
      uint16_t *to = dst + (h0 + sub) * dstep + l8;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        float o[8];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          f32x2 v = x[h][j];
          if (turns) {
            if (roll[h]) v = x2_fma(v, A[h][j], x2_mul(y[h][j], B[h][j]));
            else v = x2_mul(v, A[h][j]);
            v = x2_mul(v, sc2);
          }
          x2_unpack(v, o[2 * j], o[2 * j + 1]);
        }
        if (h0 + sub < n) kv_row_out<T, 8>(to + h * H2, wide, o);
      }
      if (!ROW) break;
    }
  };
  // query heads, then keys, then values; where the warp has no row of its own, its HPW of one of them
  const int u = blockIdx.y * 8 + warp, qu = (a.H + HPW - 1) / HPW, ku = (c.KV + HPW - 1) / HPW, kh = u - qu, vh = kh - ku;
  if (a.q && (ROW || u < qu)) heads((const X *)a.q + r * a.qs, a.qhs, ROW ? 0 : u * HPW, a.H, a.qn, a.qo + r * a.qos, HD, a.wide, true);
  if (id < 0) return;
  if (ROW || (kh >= 0 && kh < ku)) heads((const X *)a.k + r * a.ks, HD, ROW ? 0 : kh * HPW, c.KV, a.kn, c.k + at, head_step, true, true);
  if (ROW || (vh >= 0 && vh < ku)) heads((const X *)a.v + r * a.vs, HD, ROW ? 0 : vh * HPW, c.KV, nullptr, c.v + at, head_step, true, false);
}

// ---- eviction -------------------------------------------------------------------------------------
struct KvEvict {
  int budget, sinks, recent;
  const float *w;
  int wstride;
  float *w_out;
  int w_out_stride;
  int *kept;
  int kept_stride;             // (kept: the caller's, or the workspace)
  int *dst_lens;
};
// order-preserving key of a weight; NaN below every number, zeros alike
__device__ __forceinline__ uint32_t kv_key(float w) {
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
// Which slots stay: CL blocks, a cluster, a kv head of a sequence, each with its run of the slots.  The weight that the last one has, by passes over the keys' digits
// (eleven, eleven and ten bits; counts in shared memory, summed over the cluster; a warp's zeros are counted together, and so are those that are like its first other
// weight: many are zero, or all alike), then the slots above it and the first of those that equal it, in order.  The keys are kept in shared memory where they have
// room, so that the weights are read once. A cluster of four against one block, with the
// copies: 4 sequences of up to 60000 slots, 4 heads of 256, 54 us and 158; 16 of 20000 119 and 126; 16 of 8000 45 and 40, so that shorter ones take one block.  (The rule looks at the
// length alone.  One sequence of 10000 slots, 2 heads of 128: 17 and 20; 64 of 10000, 8 heads: 326 and 238.)
#define KE_THREADS 1024
#define KE_CLUSTER 4           // blocks of a head where sequences may have more than
#define KE_LONG 12288          // slots
#define KE_KEYS 49152          // most slots of a block whose keys have room
#define KE_HIST (4 * 2048)     // words: the passes' counts, and their sum over the cluster
#define KE_SMEM ((KE_HIST + KE_KEYS) * 4)
static_assert(KE_LONG <= KE_KEYS, "one block's keys always have room");
template <bool ROOM, int CL>
__global__ void __cluster_dims__(CL, 1, 1) __launch_bounds__(KE_THREADS, 2) k_kv_pick(const KvDev c, const KvEvict e) {
  constexpr int NT = KE_THREADS;
  extern __shared__ __align__(16) int dyn[];
  uint32_t *keys = (uint32_t *)(dyn + KE_HIST);
  __shared__ int part[32][2], pick[2], total[2];
  pdl_trigger();
  pdl_wait();
  const int g = blockIdx.x / CL, rank = blockIdx.x % CL, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int len = kv_len(c, b), now = min(len, e.budget);
  int *kept = e.kept + ((size_t)b * c.KV + g) * e.kept_stride;
  if (g == 0 && rank == 0 && tid == 0) e.dst_lens[b] = now;
  if (len <= e.budget) {
    for (int i = rank * NT + tid; i < len; i += CL * NT) kept[i] = i;
    return;
  }
  int lo = e.sinks;
  const int hi = len - e.recent, all = hi - lo;
  int want = e.budget - e.sinks - e.recent;    // of them, more than it
  for (int i = rank * NT + tid; i < lo; i += CL * NT) kept[i] = i;
  for (int i = rank * NT + tid; i < e.recent; i += CL * NT) kept[e.budget - e.recent + i] = hi + i;
  if (!want) return;                           // (as the return before: the whole cluster)
  // from word `at` of this block's shared memory to the same of block r's
  auto of_rank = [&](const int *at, int r) {
    int v;
    asm volatile("{.reg .u32 a; mapa.shared::cluster.u32 a, %1, %2; ld.shared::cluster.s32 %0, [a];}" : "=r"(v) : "r"(smem_u32(at)), "r"(r) : "memory");
    return v;
  };
  auto meet = [&]() {
    if constexpr (CL > 1) asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
    else __syncthreads();
  };
  const int each = (all + CL - 1) / CL, n = max(0, min(each, all - rank * each)), first = lo;   // the block's: n from `lo` on
  lo += rank * each;
  const float *w = e.w + ((size_t)b * c.KV + g) * e.wstride + lo;
  for (int i = tid; i < 3 * 2048; i += NT) dyn[i] = 0;
  __syncthreads();
  auto key_at = [&](int i) { return ROOM ? keys[i] : kv_key(__ldcg(w + i)); };
  uint32_t key = 0, known = 0;                 // the digits so far, and which bits they are
#pragma unroll 1
  for (int pass = 0; pass < 3; pass++) {
    const int sh = pass == 0 ? 21 : pass == 1 ? 10 : 0, mask = pass == 2 ? 1023 : 2047;
    int *hist = dyn + 2048 * pass;
#pragma unroll 1
    for (int i0 = 0; i0 < n; i0 += 4 * NT) {
      uint32_t u[4];
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const int i = i0 + k * NT + tid;
        u[k] = 0;
        if (i < n) {
          u[k] = ROOM && pass == 0 ? kv_key(__ldcg(w + i)) : key_at(i);
          if (ROOM && pass == 0) keys[i] = u[k];
        }
      }
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const bool on = i0 + k * NT + tid < n && (u[k] & known) == key;
        const bool zero = on && u[k] == 0x80000000u;
        const int d = (u[k] >> sh) & mask;
        const unsigned zeros = __ballot_sync(0xffffffffu, zero), act = __ballot_sync(0xffffffffu, on && !zero);
        if (zeros && lane == 0) atomicAdd(hist + ((0x80000000u >> sh) & mask), __popc(zeros));
        if (!act) continue;
        const int d0 = __shfl_sync(0xffffffffu, d, __ffs(act) - 1);
        const unsigned same = __ballot_sync(0xffffffffu, on && !zero && d == d0);
        if (lane == __ffs(act) - 1) atomicAdd(hist + d0, __popc(same));
        else if (on && !zero && d != d0) atomicAdd(hist + d, 1);
      }
    }
    meet();
    if constexpr (CL > 1) {
      for (int i = tid; i < 2048; i += NT) {
        int t = 0;
#pragma unroll
        for (int r = 0; r < CL; r++) t += of_rank(hist + i, r);
        dyn[3 * 2048 + i] = t;
      }
      hist = dyn + 3 * 2048;
      __syncthreads();
    }
    if (warp == 0) {                           // from the top: a lane 64 digits, then the lane's own
      int s = 0;
      const int d1 = 2047 - 64 * lane;         // the lane's: d1 down to d1 - 63
#pragma unroll 8
      for (int k = 0; k < 64; k++) s += hist[d1 - ((k + lane) & 63)];   // (a bank of its own for every lane)
      int to = s;
#pragma unroll
      for (int m = 1; m < 32; m <<= 1) { const int o = __shfl_up_sync(0xffffffffu, to, m); if (lane >= m) to += o; }
      const bool mine = to >= want && to - s < want;
      const int who = __ffs(__ballot_sync(0xffffffffu, mine)) - 1, left0 = want - __shfl_sync(0xffffffffu, to - s, who), base = 2047 - 64 * who;
      // the 64 digits of that lane, two a lane
      const int a0 = hist[base - 2 * lane], a1 = hist[base - 2 * lane - 1], t2 = a0 + a1;
      int up = t2;
#pragma unroll
      for (int m = 1; m < 32; m <<= 1) { const int o = __shfl_up_sync(0xffffffffu, up, m); if (lane >= m) up += o; }
      if (up >= left0 && up - t2 < left0) {
        const int left = left0 - (up - t2);
        const bool first = a0 >= left;
        pick[0] = base - 2 * lane - (first ? 0 : 1); pick[1] = first ? left : left - a0;
      }
    }
    __syncthreads();
    key |= (uint32_t)pick[0] << sh;
    known |= (uint32_t)mask << sh;
    want = pick[1];                            // of those that equal the key so far
  }
  // a thread a run of slots (an odd number of them: banks), counted, then written
  const int run = ((n + NT - 1) / NT) | 1, ra = min(n, tid * run), rz = min(n, ra + run);
  int no = 0, ne = 0;
#pragma unroll 4
  for (int i = ra; i < rz; i++) { const uint32_t u = key_at(i); no += u > key; ne += u == key; }
  int so = no, se = ne;
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, so, m), q = __shfl_up_sync(0xffffffffu, se, m);
    if (lane >= m) { so += o; se += q; }
  }
  if (lane == 31) { part[warp][0] = so; part[warp][1] = se; }
  __syncthreads();
  so -= no; se -= ne;
  {
    int po = lane < warp ? part[lane][0] : 0, pe = lane < warp ? part[lane][1] : 0;   // of the warps before
#pragma unroll
    for (int m = 16; m; m >>= 1) { po += __shfl_xor_sync(0xffffffffu, po, m); pe += __shfl_xor_sync(0xffffffffu, pe, m); }
    so += po; se += pe;
  }
  if constexpr (CL > 1) {                      // of the blocks before
    if (tid == NT - 1) { total[0] = so + no; total[1] = se + ne; }
    meet();
    for (int r = 0; r < rank; r++) { so += of_rank(total, r); se += of_rank(total + 1, r); }
    meet();                                    // (nobody's memory goes before it was read)
  }
#pragma unroll 1
  for (int i = ra; i < rz; i++) {
    const uint32_t u = key_at(i);
    if (u > key) { kept[first + so + min(se, want)] = lo + i; so++; }
    else if (u == key) { if (se < want) kept[first + so + se] = lo + i; se++; }
  }
}
// K, V and weights of the kept slots into their new pages: 16 bytes of K and of V a thread.  A thread's way is a chain of three trips (which slot, its page, its
// row), so that many threads with one piece each keep more on its way than few with several: 16 sequences of 4096 slots, 4 heads of 256, take 119 us with the picking
// at one piece and six blocks an SM, 5 us more at two and five, 30 at four and three.
template <int HD>
__global__ void __launch_bounds__(256, 6) k_kv_move(const KvDev c, const KvDev d, const KvEvict e) {
  pdl_trigger();
  pdl_wait();
  constexpr int P = HD / 8;    // pieces of a row
  const int g = blockIdx.y, b = blockIdx.z, now = min(kv_len(c, b), e.budget);
  const size_t head = (size_t)b * c.KV + g;
  // (counted by slots: a sequence may have more pieces than an int holds)
  const int p = threadIdx.x % P;
  for (unsigned i = blockIdx.x * (256 / P) + threadIdx.x / P; i < (unsigned)now; i += gridDim.x * (256 / P)) {
    const int j = __ldcg(e.kept + head * e.kept_stride + i);
    const int from = kv_page(c, b, j >> c.page_sh), to = kv_page(d, b, i >> d.page_sh);
    const bool on = from >= 0 && to >= 0;
    const size_t x = kv_at(c, on ? from : 0, g, HD) + (size_t)(j & ((1 << c.page_sh) - 1)) * HD + 8 * p, y = kv_at(d, on ? to : 0, g, HD) + (size_t)(i & ((1 << d.page_sh) - 1)) * HD + 8 * p;
    uint4 k = {}, v = {};
    if (on) { k = __ldcs((const uint4 *)(c.k + x)); v = __ldcs((const uint4 *)(c.v + x)); }
    if (p == 0 && e.w_out) e.w_out[head * e.w_out_stride + i] = __ldcg(e.w + head * e.wstride + j);
    if (on) { *(uint4 *)(d.k + y) = k; *(uint4 *)(d.v + y) = v; }
  }
}

// ---- what the agents of k_kv_pf do with their barriers ----------------------------------------------
// (llb_b200_pf_trace.)  form, bits: 1 the second query tile is empty, 2 every step rescales, 4 every step takes V out; n tiles.  Agents: the softmax warps, the loaders of K and
// V, a thread a stream that issues MMAs.  Barriers: full K 0, V 6; empty K 12, V 18; s_full 24, p_full 28 (+ 2 stream + tile parity); pv_done 32; q_full 34; pv_last 35.
template <int HD> static int kp_trace(PfTrace &t, int form, int n, int agent) {
  using C = Kp<HD>;
  const int streams = C::NQT == 2 && !(form & 1) ? 2 : 1, q_full = 34;
  if (agent >= C::SOFT + 2 + C::NQT || n < 1) return -1;
  if (agent < C::SOFT) {
    const int x = agent >> 2;
    t.arrive(q_full);
    if (x >= streams) return t.n;
    for (int i = 0; i < n; i++) {
      t.wait(24 + 2 * x + (i & 1), i >> 1);
      if ((form & 2) && i) t.wait(32 + x, i - 1);
      if (form & 4) t.wait(6 + i % C::NV, i / C::NV);
      t.arrive(28 + 2 * x + (i & 1));
    }
    if (n > 1) t.wait(32 + x, n - 2);
    t.wait(35 + x, 0);
  } else if (agent < C::SOFT + 2) {
    const bool isv = agent > C::SOFT;
    const int N = isv ? C::NV : C::NK;
    for (int i = 0; i < n; i++) {
      t.free_again((isv ? 18 : 12) + i % N, i / N);
      if (HD == 256 && isv && i == N - 1) t.wait(q_full, 0);
      t.later((isv ? 6 : 0) + i % N);
    }
  } else if (agent < C::SOFT + 2 + streams) {
    const int x = agent - C::SOFT - 2;
    auto give = [&](int b) { for (int k = 0; k < (streams < C::NQT ? 2 : 1); k++) t.later(b); };
    auto score = [&](int i) { t.wait(i % C::NK, i / C::NK); t.later(24 + 2 * x + (i & 1)); give(12 + i % C::NK); };
    t.wait(q_full, 0);
    score(0);
    if (n > 1) score(1);
    t.wait(6, 0);
    for (int i = 0; i < n; i++) {
      t.wait(28 + 2 * x + (i & 1), i >> 1);
      if (i + 1 < n) { t.later(32 + x); t.wait(32 + x, i); }
      else t.later(35 + x);
      give(18 + i % C::NV);
      if (i + 1 < n) t.wait(6 + (i + 1) % C::NV, (i + 1) / C::NV);
      if (i + 2 < n) score(i + 2);
    }
  }
  return t.n;
}
int kv_pf_trace(PfTrace &t, int hd, int form, int n, int agent) {
  return hd == 64 ? kp_trace<64>(t, form, n, agent) : hd == 128 ? kp_trace<128>(t, form, n, agent) : hd == 256 ? kp_trace<256>(t, form, n, agent) : -1;
}
int kv_pf_bar_count(int hd, int bar) {
  const int nqt = hd == 256 ? 1 : 2;
  return bar >= 12 && bar < 24 ? nqt : bar >= 28 && bar < 32 ? 4 : bar == 34 ? 4 * nqt : 1;
}

// ---- host -----------------------------------------------------------------------------------------
// Every kernel is loaded here: one that is first met while a stream is being captured may not be.  (78 instances: llb_b200_init takes 30 ms for 12, and 4 MiB more of the
// device's memory.)
template <typename K> static int kv_load(K k, int smem = 0) {
  if (smem) CU_OK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  cudaFuncAttributes at;
  CU_OK(cudaFuncGetAttributes(&at, k));
  return 0;
}
template <typename T, typename X, int HD> static int load_append() { return kv_load(k_kv_append<T, X, HD, false>) || kv_load(k_kv_append<T, X, HD, true>); }
template <typename T, int HD> static int load_of() {
  return kv_load(k_kv_few<T, HD, false>, kf_smem(HD)) || kv_load(k_kv_few<T, HD, true>, kf_smem(HD)) || kv_load(k_kv_join<T, HD, false>) || kv_load(k_kv_join<T, HD, true>) ||
         kv_load(k_kv_pf<T, HD>, Kp<HD>::SMEM) || kv_load(k_kv_pf_join<T, HD>) || load_append<T, float, HD>() || load_append<T, __half, HD>() || load_append<T, __nv_bfloat16, HD>();
}
template <int HD> static int load_hd() { return load_of<__half, HD>() || load_of<__nv_bfloat16, HD>() || kv_load(k_kv_move<HD>); }
int kv_setup(void) {
  if (load_hd<64>() || load_hd<128>() || load_hd<256>() || kv_load(k_kv_pick<true, 1>, KE_SMEM) || kv_load(k_kv_pick<true, KE_CLUSTER>, KE_SMEM) || kv_load(k_kv_pick<false, KE_CLUSTER>)) return -1;
  if (!g_kv_map) {
    cudaDriverEntryPointQueryResult found;
    CU_OK(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", (void **)&g_kv_map, 12000, cudaEnableDefault, &found));
    if (!g_kv_map) return llb_fail("the driver has no cuTensorMapEncodeTiled");
  }
  if (!g_kv_err) {
    CU_OK(cudaMalloc(&g_kv_err, 4));
    CU_OK(cudaMemset(g_kv_err, 0, 4));
  }
  return 0;
}
// A call's scope: the library's device for the calling thread, no launch recording, and no engine capturing meanwhile
namespace {
struct KvScope {
  int was = -1;
  std::lock_guard<std::recursive_mutex> hold{llb_enqueue_lock()};
  KvScope() {
    int d = 0;
    if (cudaGetDevice(&d) == cudaSuccess && d != g_llb.device) { was = d; cudaSetDevice(g_llb.device); }
  }
  ~KvScope() { if (was >= 0) cudaSetDevice(was); }
};
}
#define KV_BEGIN \
  if (!g_llb.stream) return llb_fail("llb_b200_init has not been called"); \
  KvScope scope; \
  if (backend_graph_bail()) return -1

static bool off(llb_b200_dptr p, unsigned n) { return p % n != 0; }
// Whether `rows` rows of wa bytes, sa bytes apart from a on, may share a byte with rows of wb bytes, sb apart from b on.  Rows that lie beside each other in one buffer (equal
// strides) do not.
static bool rows_meet(llb_b200_dptr a, long long sa, long long wa, llb_b200_dptr b, long long sb, long long wb, long long rows) {
  if (!a || !b || rows < 1 || wa < 1 || wb < 1) return false;
  if (a + (unsigned long long)((rows - 1) * sa + wa) <= b || b + (unsigned long long)((rows - 1) * sb + wb) <= a) return false;
  if (rows == 1 || sa != sb || wa > sa || wb > sb) return true;
  const long long d = (long long)((b > a ? b - a : a - b) % (unsigned long long)sa), from_a = b > a || !d ? d : sa - d;   // where b's rows begin in a's
  return from_a < wa || from_a + wb > sa;
}
static int kv_check(const llb_kv *kv, const char *what) {
  if (!kv) return llb_fail("%s: no cache", what);
  if (kv->el != LLB_EL_F16 && kv->el != LLB_EL_BF16) return llb_fail("%s: el %d (a cache is of f16 or bf16)", what, kv->el);
  if (kv->head_dim != 64 && kv->head_dim != 128 && kv->head_dim != 256) return llb_fail("%s: head_dim %d (64, 128 or 256)", what, kv->head_dim);
  if (kv->kv_heads < 1 || kv->kv_heads > 1024) return llb_fail("%s: %d kv heads", what, kv->kv_heads);
  if (kv->page != 16 && kv->page != 32 && kv->page != 64 && kv->page != 128) return llb_fail("%s: pages of %d slots (16, 32, 64 or 128)", what, kv->page);
  if (kv->n_pages < 1) return llb_fail("%s: %d pages", what, kv->n_pages);
  if (kv->seqs < 1 || kv->seqs > 65535) return llb_fail("%s: %d sequences (1 .. 65535)", what, kv->seqs);
  if (kv->table_stride < 1) return llb_fail("%s: table_stride %d", what, kv->table_stride);
  if (!kv->k || !kv->v || off(kv->k, 16) || off(kv->v, 16)) return llb_fail("%s: k and v lie on multiples of 16 bytes", what);
  if (!kv->table || !kv->lens || off(kv->table, 4) || off(kv->lens, 4)) return llb_fail("%s: table and lens are int32 on the device", what);
  return 0;
}
// the most slots of a sequence: a slot's number, rounded up to the 2048 that a joining block has or 32 boxes on, is an int
#define KV_MOST (INT_MAX - 4095)
static long long kv_most(const llb_kv *kv) { return std::min((long long)kv->table_stride * kv->page, (long long)KV_MOST); }
// ... and of a call that bounds them by max_len: what a call's sizes go by (max_len itself may be anything up to INT_MAX)
static int kv_slots(const llb_kv *kv, int max_len) { return (int)std::min(kv_most(kv), (long long)max_len); }
static KvDev kv_dev(const llb_kv *kv, long long cap) {
  KvDev c;
  c.k = (uint16_t *)(uintptr_t)kv->k; c.v = (uint16_t *)(uintptr_t)kv->v;
  c.table = (const int *)(uintptr_t)kv->table; c.lens = (const int *)(uintptr_t)kv->lens;
  c.KV = kv->kv_heads; c.page_sh = kv->page == 16 ? 4 : kv->page == 32 ? 5 : kv->page == 64 ? 6 : 7;
  c.n_pages = kv->n_pages; c.seqs = kv->seqs; c.tstride = kv->table_stride;
  c.cap = (int)std::min(kv_most(kv), cap);
  c.err = g_kv_err;
  return c;
}
static int heads_check(const llb_kv *kv, int heads, const char *what) {
  if (heads < 1 || heads % kv->kv_heads || heads / kv->kv_heads > 64) return llb_fail("%s: %d heads on %d kv heads", what, heads, kv->kv_heads);
  return 0;
}

// A warp 512 / head_dim heads where that leaves SMs free (a step of a few tokens is as long as a warp's chain of latencies: place, sines, a head), else a warp a row.
template <typename T, typename X, int HD> static int append_hd(const KvDev &c, const KvRows &rw, const KvAppend &a) {
  constexpr int HPW = 512 / HD;
  const int groups = ((a.H + HPW - 1) / HPW + 2 * ((c.KV + HPW - 1) / HPW) + 7) / 8;
  if ((long long)rw.rows * groups <= 8LL * g_llb.sms) CU_OK(llb_launch(k_kv_append<T, X, HD, false>, dim3(rw.rows, groups), dim3(256), (size_t)0, g_llb.stream, c, rw, a));
  else CU_OK(llb_launch(k_kv_append<T, X, HD, true>, dim3((unsigned)(((long long)rw.rows + 7) / 8)), dim3(256), (size_t)0, g_llb.stream, c, rw, a));
  return 0;
}
template <typename T, typename X> static int append_go(const KvDev &c, const KvRows &rw, const KvAppend &a, int hd) {
  return hd == 64 ? append_hd<T, X, 64>(c, rw, a) : hd == 128 ? append_hd<T, X, 128>(c, rw, a) : append_hd<T, X, 256>(c, rw, a);
}
// pages as [page][kv head][64 dims][slot][dim], in boxes of `slots` slots and `blocks` times 64 dims of a kv head of a page
static int pool_map(CUtensorMap *map, const llb_kv *kv, llb_b200_dptr base, int slots, int blocks) {
  const cuuint64_t row = (cuuint64_t)kv->head_dim * 2;
  const cuuint64_t dim[5] = {64, (cuuint64_t)kv->page, (cuuint64_t)kv->head_dim / 64, (cuuint64_t)kv->kv_heads, (cuuint64_t)kv->n_pages};
  const cuuint64_t step[4] = {row, 128, row * kv->page, row * kv->page * kv->kv_heads};
  const cuuint32_t box[5] = {64, (cuuint32_t)slots, (cuuint32_t)blocks, 1, 1}, one[5] = {1, 1, 1, 1, 1};
  const CUresult r = g_kv_map(map, kv->el == LLB_EL_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, (void *)(uintptr_t)base, dim, step, box, one,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : llb_fail("kv: tensor map of %d pages: error %d", kv->n_pages, (int)r);
}
// ---- which kernel, and its workspace ----
// Queries a kv head up to which a call goes to k_kv_few, which alone gives slots' weights (64 queries at most).  It brings K and V once for every 16 queries, k_kv_pf once for 128
// or 256.  Both kernels, us, k_kv_few first; 8 queries a kv head, 16, 32, 64:
//   16 sequences of 8000 slots, 8 kv heads of 128, pages of 64:      92, 92   92, 93   172, 94   328, 99      window 2048: 35, 34   38, 35   61, 35   105, 36
//   2 of 30000, the same heads:                                      49, 58   50, 57    85, 55   124, 56
//   16 of 8000, 2 kv heads of 256, pages of 64:                      53, 51   56, 52    93, 53   167, 60      window 2048: 23, 20   25, 21   33, 22    46, 27
//   1 of 1500, 8 kv heads of 128; 2 of 256:                          11, 19   12, 19    12, 19    14, 19                   20, 19   23, 19   23, 19    21, 19
// Up to 16 queries the two are near each other, and k_kv_few is ahead where few blocks have work; for 17 to 64 queries without weights a border at 16 would be faster but for short
// contexts.
#define KV_FEW 64
// Fewest groups of a block's stretch.  One token, us, with one, two and four: 700 slots, 2 kv heads of 128: 8.9, 11.0, 12.2; 4 of 256: 16.1, 12.6, 15.1; 4000 slots 16.5, 12.5, 13.1
// and 22.7, 22.6, 22.6; four sequences of 300, 2 of 128: 9.2, 11.4, 12.7; 4 of 256: 11.6, 11.6, 14.9
#define KF_LEAST 2
static int most_rows(const llb_kv_attn *a) { return std::min(a->max_rows, std::max(a->rows, 1)); }
static bool attn_few(const llb_kv *kv, const llb_kv_attn *a) { return (long long)a->heads / kv->kv_heads * most_rows(a) <= KV_FEW; }
static_assert(KJ_SLOTS <= 2048 && (KV_MOST + 2047LL) / 2048 * 2048 <= INT_MAX, "a joining block's last slot");
static int few_grid(void) { return g_llb.sms ? g_llb.sms : 148; }
// its parts, one behind the other; the size where `base` is 0
static size_t few_plan(const llb_kv *kv, const llb_kv_attn *a, uintptr_t base, KvPlan *p) {
  const size_t blocks = few_grid(), queries = (size_t)kv->seqs * a->heads * most_rows(a);
  size_t at = 0;
  auto take = [&](size_t bytes) { const size_t was = at; at += (bytes + 15) & ~(size_t)15; return base + was; };
  p->blocks = (int)blocks; p->least = KF_LEAST;
  p->unit = (int *)take((size_t)kv->seqs * kv->kv_heads * (((size_t)(a->heads / kv->kv_heads) * most_rows(a) + 15) / 16) * 8);
  p->span = (int2 *)take(blocks * 2 * 8);
  p->pm = (float *)take(blocks * 2 * 16 * 4);
  p->pl = (float *)take(blocks * 2 * 16 * 4);
  p->po = (float *)take(blocks * 2 * 16 * kv->head_dim * 4);
  p->sstride = std::max(16, (kv_slots(kv, a->max_len) + 15) & ~15);
  p->lse = (float *)take(a->w_out ? queries * 4 : 0);
  p->sc = (float *)take(a->w_out ? queries * p->sstride * 4 : 0);
  return at;
}
template <typename T, int HD> static int few_go(const llb_kv *kv, const llb_kv_attn *call, const KvDev &c, const KvRows &rw, const KvAttn &a) {
  KvPlan p;
  few_plan(kv, call, (uintptr_t)call->ws, &p);
  p.err = gemm_err_word();
  CUtensorMap km, vm;
  const int slots = std::min(kv->page, 1 << kf_sh(HD));
  if (pool_map(&km, kv, kv->k, slots, HD / 64) || pool_map(&vm, kv, kv->v, slots, HD / 64)) return -1;
  const dim3 grid(p.blocks), block(32 * (kf_warps(HD) + 2));
  const int joins = c.seqs * c.KV * a.G * rw.max_rows, wblocks = (c.cap + KJ_SLOTS - 1) / KJ_SLOTS;   // (attn_check: they fit)
  if (a.w_out) {
    CU_OK(llb_launch(k_kv_few<T, HD, true>, grid, block, (size_t)kf_smem(HD), g_llb.stream, c, rw, a, p, km, vm));
    CU_OK(llb_launch(k_kv_join<T, HD, true>, dim3(joins + wblocks * c.KV * c.seqs), dim3(128), (size_t)0, g_llb.stream, c, rw, a, p, joins, wblocks));
  } else {
    CU_OK(llb_launch(k_kv_few<T, HD, false>, grid, block, (size_t)kf_smem(HD), g_llb.stream, c, rw, a, p, km, vm));
    CU_OK(llb_launch(k_kv_join<T, HD, false>, dim3(joins), dim3(128), (size_t)0, g_llb.stream, c, rw, a, p, joins, 0));
  }
  return 0;
}
// many rows: query tiles of the longest sequence's rows, and how many blocks share a tile's slots where there are fewer units than SMs
static int pf_queries(const llb_kv *kv) { return kv->head_dim == 256 ? 128 : 256; }
static int pf_tiles(const llb_kv *kv, const llb_kv_attn *a) {
  return (int)(((long long)a->heads / kv->kv_heads * most_rows(a) + pf_queries(kv) - 1) / pf_queries(kv));
}
static size_t pf_plan(const llb_kv *kv, const llb_kv_attn *a, uintptr_t base, KvPfPlan *p) {
  const long long sms = g_llb.sms ? g_llb.sms : 148, units = (long long)pf_tiles(kv, a) * kv->kv_heads * kv->seqs;
  const int len = kv_slots(kv, a->max_len), slots = a->window ? (int)std::min((long long)len, (long long)a->window + a->sinks + most_rows(a)) : len;   // that a unit sees, at most
  p->splits = (int)std::max(1LL, std::min(sms / std::max(units, 1LL), (long long)slots / 512));
  size_t at = 0;
  auto take = [&](size_t bytes) { const size_t was = at; at += (bytes + 15) & ~(size_t)15; return base + was; };
  const size_t parts = p->splits > 1 ? (size_t)kv->seqs * a->heads * most_rows(a) * p->splits : 0;
  p->pm = (float *)take(parts * 4);
  p->pl = (float *)take(parts * 4);
  p->po = (float *)take(parts * 4 * kv->head_dim);
  return std::max(at, (size_t)16);
}
template <typename T, int HD> static int attn_go(const llb_kv *kv, const llb_kv_attn *call, const KvDev &c, const KvRows &rw, const KvAttn &a) {
  if (attn_few(kv, call)) return few_go<T, HD>(kv, call, c, rw, a);
  KvPfPlan p;
  pf_plan(kv, call, (uintptr_t)call->ws, &p);
  p.err = gemm_err_word();
  const int slots = std::min(kv->page, Kp<HD>::TILE), blocks = slots == Kp<HD>::TILE ? HD / 64 : 1, tiles = pf_tiles(kv, call);
  CUtensorMap km, vm;
  if (pool_map(&km, kv, kv->k, slots, blocks) || pool_map(&vm, kv, kv->v, slots, blocks)) return -1;
  CU_OK(llb_launch(k_kv_pf<T, HD>, dim3(tiles * c.KV * c.seqs, p.splits), dim3(Kp<HD>::THREADS), (size_t)Kp<HD>::SMEM, g_llb.stream, c, rw, a, p, tiles, km, vm));
  if (p.splits > 1) CU_OK(llb_launch(k_kv_pf_join<T, HD>, dim3(rw.rows, (a.H + 3) / 4), dim3(128), (size_t)0, g_llb.stream, c, rw, a, p));
  return 0;
}

static int attn_check(const llb_kv *kv, const llb_kv_attn *a) {
  const char *const me = "kv_attn";
  if (kv_check(kv, me)) return -1;
  if (!a) return llb_fail("kv_attn: no call");
  if (heads_check(kv, a->heads, me)) return -1;
  if (a->rows < 0) return llb_fail("kv_attn: %d rows", a->rows);
  if (a->max_rows < 1 || a->max_len < 0) return llb_fail("kv_attn: max_rows %d, max_len %d", a->max_rows, a->max_len);
  if (a->window < 0 || a->sinks < 0) return llb_fail("kv_attn: window %d, sinks %d", a->window, a->sinks);
  if (a->sinks && !a->window) return llb_fail("kv_attn: sinks without a window (every first slot is seen anyway)");
  if (!(a->scale >= 0.0f) || a->scale > 3.0e38f) return llb_fail("kv_attn: scale %g", (double)a->scale);
  if (a->el_out != LLB_EL_F32 && a->el_out != kv->el) return llb_fail("kv_attn: el_out %d (f32 or the cache's type)", a->el_out);
  const long long row = (long long)a->heads * kv->head_dim;
  if ((a->rows && (!a->q || !a->out)) || off(a->q, 16) || off(a->out, 16)) return llb_fail("kv_attn: q and out lie on multiples of 16 bytes");
  if (a->rows && a->q == a->out) return llb_fail("kv_attn: out is q");
  if (a->q_stride < row || a->q_stride % 8) return llb_fail("kv_attn: q_stride %lld for rows of %lld", a->q_stride, row);
  if (a->out_stride < row || a->out_stride % (a->el_out == LLB_EL_F32 ? 4 : 8)) return llb_fail("kv_attn: out_stride %lld for rows of %lld", a->out_stride, row);
  if (!a->row_start || off(a->row_start, 4)) return llb_fail("kv_attn: row_start is int32 on the device");
  if (a->w_in && !a->w_out) return llb_fail("kv_attn: w_in without w_out");
  const long long queries = (long long)a->heads / kv->kv_heads * most_rows(a), pairs = (long long)kv->seqs * kv->kv_heads;
  const int len = kv_slots(kv, a->max_len);
  if (queries <= KV_FEW && pairs * ((queries + 15) / 16) > INT_MAX / 2 / (len / 32 + 3))
    return llb_fail("kv_attn: %d sequences of %d kv heads with up to %d slots: more than are counted (max_len bounds it)", kv->seqs, kv->kv_heads, len);
  if (queries >= 1 << 26 || pairs * (std::min(queries, (queries + 127) / 128 + KV_FEW) + (a->w_out ? (len + 511) / 512 : 0)) > INT_MAX)
    return llb_fail("kv_attn: %d sequences of %d kv heads, %d rows, %d slots: more than one launch holds", kv->seqs, kv->kv_heads, most_rows(a), len);
  if (a->w_out) {
    if (off(a->w_in, 4) || off(a->w_out, 4)) return llb_fail("kv_attn: weights are f32 on the device");
    if (a->w_stride < a->max_len) return llb_fail("kv_attn: w_stride %d for %d slots", a->w_stride, a->max_len);
    if ((long long)a->heads / kv->kv_heads * a->max_rows > 64) return llb_fail("kv_attn: weights of %d rows of %d heads a kv head (64 together at most)", a->max_rows, a->heads / kv->kv_heads);
  }
  return 0;
}
static size_t attn_ws(const llb_kv *kv, const llb_kv_attn *a) {
  KvPlan p;
  KvPfPlan f;
  return attn_few(kv, a) ? few_plan(kv, a, 0, &p) : pf_plan(kv, a, 0, &f);
}
static int evict_check(const llb_kv *src, const llb_kv_evict *e) {
  if (kv_check(src, "kv_evict")) return -1;
  if (!e) return llb_fail("kv_evict: no call");
  if (e->budget < 1 || e->sinks < 0 || e->recent < 0 || (long long)e->sinks + e->recent > e->budget)
    return llb_fail("kv_evict: budget %d with %d first and %d last slots", e->budget, e->sinks, e->recent);
  if (e->max_len < 0) return llb_fail("kv_evict: max_len %d", e->max_len);
  const int most = std::min(e->budget, e->max_len);
  if (!e->w || off(e->w, 4) || e->w_stride < e->max_len) return llb_fail("kv_evict: weights of %d slots a head for %d", e->w_stride, e->max_len);
  if (e->w_out && (off(e->w_out, 4) || e->w_out == e->w || e->w_out_stride < most)) return llb_fail("kv_evict: w_out is not w and has %d slots a head or more", most);
  if (e->kept && (off(e->kept, 4) || e->kept_stride < most)) return llb_fail("kv_evict: kept has %d slots a head or more", most);
  return 0;
}
static size_t evict_ws(const llb_kv *src, const llb_kv_evict *e) { return 16 + (e->kept ? 0 : (size_t)src->seqs * src->kv_heads * std::min(e->budget, kv_slots(src, e->max_len)) * 4); }

extern "C" {

int llb_b200_kv_errors(void) {
  KV_BEGIN;
  unsigned int v = 0;
  CU_OK(cudaMemcpyAsync(&v, g_kv_err, 4, cudaMemcpyDeviceToHost, g_llb.stream));
  CU_OK(cudaStreamSynchronize(g_llb.stream));
  return (int)v;
}
int llb_b200_kv_errors_clear(void) {
  KV_BEGIN;
  CU_OK(cudaMemsetAsync(g_kv_err, 0, 4, g_llb.stream));
  return 0;
}

int llb_b200_kv_join_parts(int first, int last) { return kf_parts_of(first, last, few_grid()); }

int llb_b200_kv_append(const llb_kv *kv, const llb_kv_append *a) {
  const char *const me = "kv_append";
  if (kv_check(kv, me)) return -1;
  if (!a) return llb_fail("kv_append: no call");
  if (heads_check(kv, a->heads, me)) return -1;
  const int hd = kv->head_dim;
  if (a->rows < 0) return llb_fail("kv_append: %d rows", a->rows);
  if (a->el_in < LLB_EL_F32 || a->el_in > LLB_EL_BF16) return llb_fail("kv_append: el_in %d", a->el_in);
  if (a->rope_dim < 0 || a->rope_dim > hd || a->rope_dim % 2) return llb_fail("kv_append: rope_dim %d with head_dim %d", a->rope_dim, hd);
  if (!(a->eps > 0.0f) || a->eps > 3.0e38f) return llb_fail("kv_append: eps %g", (double)a->eps);
  const unsigned es = a->el_in == LLB_EL_F32 ? 4 : 2;
  if ((a->rows && (!a->k || !a->v)) || off(a->q, es) || off(a->k, es) || off(a->v, es)) return llb_fail("kv_append: q, k and v lie on multiples of their elements");
  if (a->q && (a->q_head_stride < hd || a->q_stride < (long long)(a->heads - 1) * a->q_head_stride + hd)) return llb_fail("kv_append: heads of q %d apart, rows %lld", a->q_head_stride, a->q_stride);
  if (a->k_stride < (long long)kv->kv_heads * hd || a->v_stride < (long long)kv->kv_heads * hd) return llb_fail("kv_append: k_stride %lld, v_stride %lld", a->k_stride, a->v_stride);
  if (a->q && (!a->q_out || off(a->q_out, 2) || a->q_out_stride < (long long)a->heads * hd)) return llb_fail("kv_append: q_out with rows %lld apart", a->q_out_stride);
  if (off(a->q_norm, 4) || off(a->k_norm, 4)) return llb_fail("kv_append: norm weights are f32 on the device");
  if (a->rope_dim && (!a->invfreq || off(a->invfreq, 8))) return llb_fail("kv_append: invfreq is f64 on the device");
  if (!a->row_start || off(a->row_start, 4) || off(a->pos, 4)) return llb_fail("kv_append: row_start and pos are int32 on the device");
  KV_BEGIN;
  if (!a->rows) return 0;
  const long long heads_w = (long long)kv->kv_heads * hd * es, qo_w = 2LL * a->heads * hd, qo_s = 2 * a->q_out_stride;
  if (a->q && (rows_meet(a->q, a->q_stride * es, ((a->heads - 1LL) * a->q_head_stride + hd) * es, a->q_out, qo_s, qo_w, a->rows) ||
               rows_meet(a->k, a->k_stride * es, heads_w, a->q_out, qo_s, qo_w, a->rows) || rows_meet(a->v, a->v_stride * es, heads_w, a->q_out, qo_s, qo_w, a->rows)))
    return llb_fail("kv_append: q_out overlaps q, k or v");
  const KvDev c = kv_dev(kv, LLONG_MAX);
  const KvRows rw{(const int *)(uintptr_t)a->row_start, a->rows, a->rows};
  KvAppend k;
  k.q = (const void *)(uintptr_t)a->q; k.k = (const void *)(uintptr_t)a->k; k.v = (const void *)(uintptr_t)a->v;
  k.qs = a->q_stride; k.ks = a->k_stride; k.vs = a->v_stride; k.qhs = a->q_head_stride;
  k.qn = (const float *)(uintptr_t)a->q_norm; k.kn = (const float *)(uintptr_t)a->k_norm;
  k.invfreq = (const double *)(uintptr_t)a->invfreq; k.pos = (const int *)(uintptr_t)a->pos;
  k.qo = (uint16_t *)(uintptr_t)a->q_out; k.qos = a->q_out_stride;
  k.H = a->heads; k.rope = a->rope_dim; k.eps = a->eps;
  // eight elements as 16-byte words, where all of q, k, v and q_out have them there
  k.wide = !off(a->q, 16) && !off(a->k, 16) && !off(a->v, 16) && !off(a->q_out, 16) && a->q_stride % 8 == 0 && a->k_stride % 8 == 0 && a->v_stride % 8 == 0 && a->q_head_stride % 8 == 0 &&
           a->q_out_stride % 8 == 0;
  if (kv->el == LLB_EL_F16) {
    if (a->el_in == LLB_EL_F32) return append_go<__half, float>(c, rw, k, hd);
    if (a->el_in == LLB_EL_F16) return append_go<__half, __half>(c, rw, k, hd);
    return append_go<__half, __nv_bfloat16>(c, rw, k, hd);
  }
  if (a->el_in == LLB_EL_F32) return append_go<__nv_bfloat16, float>(c, rw, k, hd);
  if (a->el_in == LLB_EL_F16) return append_go<__nv_bfloat16, __half>(c, rw, k, hd);
  return append_go<__nv_bfloat16, __nv_bfloat16>(c, rw, k, hd);
}

size_t llb_b200_kv_attn_ws(const llb_kv *kv, const llb_kv_attn *a) { return attn_check(kv, a) ? 0 : attn_ws(kv, a); }
int llb_b200_kv_attn(const llb_kv *kv, const llb_kv_attn *a) {
  if (attn_check(kv, a)) return -1;
  const size_t need = attn_ws(kv, a);
  if (!a->ws || off(a->ws, 16) || a->ws_bytes < need) return llb_fail("kv_attn: a workspace of %zu bytes (%zu are needed, on a multiple of 16)", a->ws_bytes, need);
  KV_BEGIN;
  if (!a->rows && !a->w_out) return 0;
  const KvDev c = kv_dev(kv, a->max_len);
  const long long row = (long long)a->heads * kv->head_dim, ow = a->el_out == LLB_EL_F32 ? 4 : 2;
  if (rows_meet(a->q, 2 * a->q_stride, 2 * row, a->out, ow * a->out_stride, ow * row, a->rows)) return llb_fail("kv_attn: out overlaps q");
  if (a->w_in != a->w_out && rows_meet(a->w_in, 4LL * a->w_stride, 4LL * c.cap, a->w_out, 4LL * a->w_stride, 4LL * c.cap, (long long)kv->seqs * kv->kv_heads))
    return llb_fail("kv_attn: w_out overlaps w_in and is not w_in");
  const KvRows rw{(const int *)(uintptr_t)a->row_start, a->rows, most_rows(a)};
  KvAttn k;
  k.q = (const uint16_t *)(uintptr_t)a->q; k.out = (void *)(uintptr_t)a->out;
  k.qs = a->q_stride; k.os = a->out_stride; k.H = a->heads; k.G = a->heads / kv->kv_heads; k.inv = (unsigned)(((1ull << 32) + k.G - 1) / k.G); k.window = a->window; k.sinks = a->sinks; k.out32 = a->el_out == LLB_EL_F32;
  k.scale2 = (float)((a->scale > 0.0f ? (double)a->scale : 1.0 / sqrt((double)kv->head_dim)) * 1.4426950408889634);
  k.w_in = (const float *)(uintptr_t)a->w_in; k.w_out = (float *)(uintptr_t)a->w_out; k.wstride = a->w_stride;
  if (kv->el == LLB_EL_F16) return kv->head_dim == 64 ? attn_go<__half, 64>(kv, a, c, rw, k) : kv->head_dim == 128 ? attn_go<__half, 128>(kv, a, c, rw, k) : attn_go<__half, 256>(kv, a, c, rw, k);
  return kv->head_dim == 64 ? attn_go<__nv_bfloat16, 64>(kv, a, c, rw, k) : kv->head_dim == 128 ? attn_go<__nv_bfloat16, 128>(kv, a, c, rw, k) : attn_go<__nv_bfloat16, 256>(kv, a, c, rw, k);
}

size_t llb_b200_kv_evict_ws(const llb_kv *src, const llb_kv_evict *e) { return evict_check(src, e) ? 0 : evict_ws(src, e); }
int llb_b200_kv_evict(const llb_kv *src, const llb_kv *dst, const llb_kv_evict *e) {
  if (evict_check(src, e) || kv_check(dst, "kv_evict: dst")) return -1;
  if (dst->el != src->el || dst->kv_heads != src->kv_heads || dst->head_dim != src->head_dim || dst->seqs != src->seqs)
    return llb_fail("kv_evict: dst has another type, other heads or other sequences than src");
  if (dst->table == src->table || dst->lens == src->lens) return llb_fail("kv_evict: dst has a table and lens of its own");
  const int len = kv_slots(src, e->max_len), most = std::min(e->budget, len);
  if (kv_most(dst) < most) return llb_fail("kv_evict: dst holds %lld slots a sequence, %d may be kept", kv_most(dst), most);
  const size_t need = evict_ws(src, e);
  if (!e->kept && (!e->ws || off(e->ws, 16) || e->ws_bytes < need)) return llb_fail("kv_evict: a workspace of %zu bytes (%zu are needed, on a multiple of 16)", e->ws_bytes, need);
  KV_BEGIN;
  if (rows_meet(src->lens, 4LL * src->seqs, 4LL * src->seqs, dst->lens, 4LL * src->seqs, 4LL * src->seqs, 1)) return llb_fail("kv_evict: dst's lens overlap src's");
  if (rows_meet(e->w, 4LL * e->w_stride, 4LL * len, e->w_out, 4LL * e->w_out_stride, 4LL * most, (long long)src->seqs * src->kv_heads)) return llb_fail("kv_evict: w_out overlaps w");
  const KvDev c = kv_dev(src, e->max_len), d = kv_dev(dst, LLONG_MAX);
  KvEvict k;
  k.budget = e->budget; k.sinks = e->sinks; k.recent = e->recent;
  k.w = (const float *)(uintptr_t)e->w; k.wstride = e->w_stride;
  k.w_out = (float *)(uintptr_t)e->w_out; k.w_out_stride = e->w_out_stride;
  k.kept = (int *)(uintptr_t)(e->kept ? e->kept : e->ws); k.kept_stride = e->kept ? e->kept_stride : most;
  k.dst_lens = (int *)(uintptr_t)dst->lens;
  // (keys of a block's slots; a block with few of them leaves room for others on its SM)
  const int blocks = len > KE_LONG ? KE_CLUSTER : 1, own = std::max((len + blocks - 1) / blocks, 1);
  const dim3 heads((unsigned)c.KV * blocks, c.seqs);
  if (blocks == 1) CU_OK(llb_launch(k_kv_pick<true, 1>, heads, dim3(KE_THREADS), (size_t)(KE_HIST + own) * 4, g_llb.stream, c, k));
  else if (own <= KE_KEYS) CU_OK(llb_launch(k_kv_pick<true, KE_CLUSTER>, heads, dim3(KE_THREADS), (size_t)(KE_HIST + own) * 4, g_llb.stream, c, k));
  else CU_OK(llb_launch(k_kv_pick<false, KE_CLUSTER>, heads, dim3(KE_THREADS), (size_t)KE_HIST * 4, g_llb.stream, c, k));
  if (!most) return 0;
  // blocks of a head: one trip each, as long as there are not more blocks than 64 an SM (eight: 6 % slower; one trip whatever the number: 7 %)
  const long long pieces = (long long)most * (src->head_dim / 8), room = std::max(1LL, 64LL * g_llb.sms / ((long long)c.KV * c.seqs));
  const dim3 grid((unsigned)std::max(1LL, std::min(room, (pieces + 255) / 256)), c.KV, c.seqs);
  if (src->head_dim == 64) CU_OK(llb_launch(k_kv_move<64>, grid, dim3(256), (size_t)0, g_llb.stream, c, d, k));
  else if (src->head_dim == 128) CU_OK(llb_launch(k_kv_move<128>, grid, dim3(256), (size_t)0, g_llb.stream, c, d, k));
  else CU_OK(llb_launch(k_kv_move<256>, grid, dim3(256), (size_t)0, g_llb.stream, c, d, k));
  return 0;
}

}  // extern "C"
