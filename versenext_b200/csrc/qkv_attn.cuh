// Attention of a step's rows over the 8-bit cache: the committed positions and the rows that the step has appended.
//
// o = sum_j p_j s_j c_j / sum_j p_j,  p_j = exp2(t_j r - m),  t_j = (q' . k_j) a_j: k_j, c_j codes of keys and values, a_j, s_j their
// scales, q' the query times a power of two that brings its largest channel to [2^13, 2^14), r what undoes that times
// scale * log2(e).  Codes are whole numbers or e4m3, both exact in 16-bit floats, so the products run on the tensor cores
// (mma.sync m16n8k16, fp32 sums) with no rounding of keys and values; queries and weights are rounded to 11 bits for bf16 rows and
// split into two halves of 11 bits for fp32 rows.  A weight p_j s_j is taken relative to a power of two R above every s_j met so
// far, times 2^15, so that a half holds weights down to 2^-39 of the largest.
//
// What bounds it is the memory of the codes (few rows) or the mma.sync rate and the conversions (many): one warp reads and converts a
// block of 32 positions for 8 NT rows (tokens x heads of a group), four warps of a CTA take every fourth block.  Positions are the
// rows of the products and queries their columns (8 at a time): S = K q^T, O = V^T p^T, with p transposed by movmatrix between.  The blocks of
// all (entry, rows, head) units form one line that is cut into equal shares for the CTAs, whatever the lengths; a unit that several
// CTAs have is merged, in their order, by the one that ends last.
#pragma once
#include "qkv.cuh"

namespace qkv_detail {

using bf16 = __nv_bfloat16;
constexpr int WARPS = 4, THREADS = 32 * WARPS;
constexpr int MIN_SHARE = WARPS;                    // blocks of a CTA at least
constexpr unsigned long long WAIT_CYCLES = 4000000000ull;   // a copy that has not come after about two seconds never will

template <typename T, int P, int NT>
struct AttnCfg {
  static constexpr int NQ = sizeof(T) == 4 ? 2 : 1;           // halves of a query or weight
  static constexpr int RT = 8 * NT, CH = P / 16, BLOCK = QKV_BLOCK * (2 * P + 8);
  static constexpr int QP = 2 * P + ((2 * P) % 64 == 0 ? 32 : 0);   // bytes of a staged query row: four rows' 32-byte pieces in 128 bytes of banks
  static constexpr int STAGES = P <= 64 ? 4 : P <= 128 && NT >= 2 && NT * NQ <= 2 ? 3 : 2;
  static constexpr bool QREG = NT * NQ <= 2 && NT * NQ * P <= 256;      // query fragments in registers
  static constexpr int SUB = NT >= 4 ? 1 : 2;                 // chunks of 16 channels that are merged at a time
  static constexpr int MP = 20;                               // pitch of a merged row: 16 lanes' pairs in different banks
  static constexpr int CTAS = P > 192 || (P > 128 && NQ * NT > 1) ? 1 : P * NT <= 128 ? 3 : 2;
  static constexpr int RING = 0, Q = RING + WARPS * STAGES * BLOCK, MERGE = Q + NQ * RT * QP, MERGE_BYTES = SUB * WARPS * RT * MP * 4, ML = MERGE + MERGE_BYTES,
                       ROWS = ML + WARPS * RT * 8, RF = ROWS + RT * 16, BARS = RF + RT * 8, SMEM = BARS + WARPS * STAGES * 8, PLAN = MERGE;
  static_assert(MERGE_BYTES >= (THREADS + 1) * 8, "the plan is read before anything is merged, from the same place");
  static_assert(RT * P <= QKV_PART, "a part fits its place");
};

struct RowInfo { int t, away; unsigned long long seen; };    // t < 0: no row

__device__ __forceinline__ void mbar_init1(unsigned bar) { asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bar)); }
__device__ __forceinline__ bool mbar_try1(unsigned bar, unsigned parity) {
  unsigned ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
static __device__ __noinline__ bool mbar_wait_long(unsigned bar, unsigned parity, unsigned long long limit) {
  const long long t0 = clock64();
  while (!mbar_try1(bar, parity))
    if ((unsigned long long)(clock64() - t0) > limit) return false;
  return true;
}
// one block of the cache into shared memory (src 16-byte aligned)
__device__ __forceinline__ void fetch_block(unsigned dst, const void* src, unsigned bytes, unsigned bar) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

__device__ __forceinline__ void mma_f16(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const unsigned*>(&h);
}
__device__ __forceinline__ float2 unpack_f16(unsigned u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
__device__ __forceinline__ unsigned transposed(unsigned u) {
  unsigned v;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(v) : "r"(u));
  return v;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float pow2(int biased) { return __uint_as_float((unsigned)min(max(biased, 0), 254) << 23); }   // 2^(biased - 127), 0 below

// two codes of a register as halves.  int8: a code plus 128 is put under the exponent of 1024, from which 1152 is taken off (BIAS: it
// is left there).  e4m3: the type's own conversion.
// PAIR: bytes 0 and 1 (0), 2 and 3 (1); e4m3 takes neighbours only, so 0 and 2, 1 and 3 are brought together first
__device__ __forceinline__ unsigned halves_of_e4m3(unsigned short u) {
  unsigned r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(u));
  return r;
}
template <int SCHEME, bool EVERY_OTHER, bool BIAS> __device__ __forceinline__ void halves_of(unsigned u, unsigned& lo, unsigned& hi) {
  if (SCHEME == QKV_I8) {
    lo = __byte_perm(u, 0x64646464u, EVERY_OTHER ? 0x4240 : 0x4140);
    hi = __byte_perm(u, 0x64646464u, EVERY_OTHER ? 0x4341 : 0x4342);
    if (BIAS) return;
    const __half2 off = __half2half2(__ushort_as_half(0x6480));
    const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&lo), off), y = __hsub2(*reinterpret_cast<const __half2*>(&hi), off);
    lo = *reinterpret_cast<const unsigned*>(&x);
    hi = *reinterpret_cast<const unsigned*>(&y);
  } else {
    if (EVERY_OTHER) u = __byte_perm(u, 0u, 0x3120);
    lo = halves_of_e4m3((unsigned short)u);
    hi = halves_of_e4m3((unsigned short)(u >> 16));
  }
}

// what a unit -- RT rows of an entry and one head -- reads
struct Unit {
  int slot, r0, n, len, f0, nf;              // rows f0 .. of nf = tokens x heads of the group
  int lo, hi, full_lo, full_hi;              // positions any row sees; positions all rows see
  int tile0, tiles;                          // blocks of 32 positions
};

template <int RT>
__device__ __forceinline__ bool unit_of(const QkvAttnArgs& a, int rts, long long z, Unit& u) {
  const int e = (int)(z / rts), rt = (int)(z % rts), G = a.v.H / a.v.KH;
  u.tiles = 0;
  if (!a.step.entry(a.v, e, &u.slot, &u.r0, &u.n)) return false;
  u.f0 = rt * RT;
  u.nf = u.n * G;
  if (u.f0 >= u.nf) return false;
  const int t0 = u.f0 / G, t1 = (min(u.f0 + RT, u.nf) - 1) / G;
  u.len = a.v.len(u.slot);
  const bool tree = a.tree.seen != nullptr;
  u.hi = min(u.len + (tree ? u.n : t1 + 1), a.v.capacity());
  u.full_hi = min(u.len + (tree ? 0 : t0 + 1), u.hi);
  u.lo = u.full_lo = 0;
  if (a.window > 0) {
    u.lo = max(0, u.len + (tree ? 0 : t0) - a.window + 1);
    u.full_lo = max(0, u.len + (tree ? QKV_MAX_DRAFT - 1 : t1) - a.window + 1);
    if (tree) u.lo = min(u.lo, u.len);
  }
  u.tile0 = u.lo / QKV_BLOCK;
  u.tiles = (u.hi + QKV_BLOCK - 1) / QKV_BLOCK - u.tile0;
  if (u.tiles <= 0) { u.tile0 = 0; u.tiles = 1; }            // rows that see nothing still get their zeros
  return true;
}

template <typename T, int SCHEME, int P, int NT>
__global__ void __launch_bounds__(THREADS, (AttnCfg<T, P, NT>::CTAS)) qkv_attn_kernel(QkvAttnArgs a, int rts) {
  using C = AttnCfg<T, P, NT>;
  constexpr int RT = C::RT, CH = C::CH, ST = C::STAGES, NQ = C::NQ;
  constexpr bool BIAS = SCHEME == QKV_I8 && NQ == 1;         // keys 1152 too large: taken off the sums instead, at the cost of some bits of them
  extern __shared__ __align__(128) unsigned char smem[];
  const QkvView& v = a.v;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rg = lane >> 2, rc = lane & 3;
  const int G = v.H / v.KH;
  const unsigned s_base = (unsigned)__cvta_generic_to_shared(smem);
  unsigned char* ring = smem + C::RING + warp * ST * C::BLOCK;
  const unsigned ring_s = s_base + C::RING + warp * ST * C::BLOCK, bars = s_base + C::BARS + warp * ST * 8;
  RowInfo* s_rows = reinterpret_cast<RowInfo*>(smem + C::ROWS);
  float2* s_rf = reinterpret_cast<float2*>(smem + C::RF);    // r of a row, and what its sums begin with
  float2* s_ml = reinterpret_cast<float2*>(smem + C::ML);
  float* s_merge = reinterpret_cast<float*>(smem + C::MERGE);
  long long* s_plan = reinterpret_cast<long long*>(smem + C::PLAN);

  if (lane < ST) mbar_init1(bars + 8 * lane);
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  // ---- the line of blocks and this CTA's share
  const long long Z = (long long)a.step.n_ent * rts, zc = (Z + THREADS - 1) / THREADS;
  Unit u;
  {
    long long sum = 0;
    for (long long z = tid * zc; z < min(Z, (tid + 1) * zc); ++z) {
      unit_of<RT>(a, rts, z, u);
      sum += (long long)u.tiles * v.KH;
    }
    long long up = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long t = __shfl_up_sync(0xffffffffu, up, o);
      if (lane >= o) up += t;
    }
    long long* s_tot = s_plan + THREADS - WARPS + 1;          // overwritten below
    if (lane == 31) s_tot[warp] = up;
    __syncthreads();
    for (int w = 0; w < warp; ++w) up += s_tot[w];
    __syncthreads();
    s_plan[tid + 1] = up;
    if (tid == 0) s_plan[0] = 0;
    __syncthreads();
  }
  const long long W = s_plan[THREADS];
  const long long share = max((W + gridDim.x - 1) / gridDim.x, (long long)MIN_SHARE);
  long long at = blockIdx.x * share;
  const long long end = min(W, at + share);
  if (at >= end) return;
  long long z;
  int head, tile;                                            // where the share begins
  {
    int j = 0;
#pragma unroll
    for (int o = THREADS / 2; o > 0; o >>= 1)
      if (s_plan[j + o] <= at) j += o;
    z = j * zc;
    long long rem = at - s_plan[j];
    for (;; ++z) {
      unit_of<RT>(a, rts, z, u);
      const long long n = (long long)u.tiles * v.KH;
      if (rem < n) break;
      rem -= n;
    }
    head = (int)(rem / u.tiles);
    tile = (int)(rem % u.tiles);
  }

  unsigned it = 0, put = 0;                                  // blocks taken and asked for
  bool dead = false;                                         // a copy did not come: nothing is computed any more
  int page_cur = -1, page_nxt = -1;                          // pages of the warp's next 32 and 64 blocks of a segment
  int seg_a = 0, seg_b = 0;
  auto pages_of = [&](int k0) {
    const int i = seg_a + warp + WARPS * (k0 + lane);
    return i < seg_b ? v.page(u.slot, i * QKV_BLOCK / KV_PAGE) : -1;
  };
  auto ask = [&](int k, int page) {                          // block k of the warp's in this segment
    if (lane == 0) {
      const unsigned s = put % ST, bar = bars + 8 * s;
      const int i = seg_a + warp + WARPS * k;
      if (page >= 0 && !dead) fetch_block(ring_s + s * C::BLOCK, v.block(page, head, i & 1), C::BLOCK, bar);
      else asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
    }
    ++put;
  };
  auto begin_segment = [&]() {
    seg_a = u.tile0 + tile;
    seg_b = (int)min((long long)(u.tile0 + u.tiles), seg_a + (end - at));
    page_cur = pages_of(0);
    page_nxt = pages_of(32);
#pragma unroll
    for (int k = 0; k < ST; ++k)
      if (seg_a + warp + WARPS * k < seg_b) ask(k, __shfl_sync(0xffffffffu, page_cur, k));
  };
  auto stage_queries = [&]() {
    for (int r = warp; r < RT; r += WARPS) {
      const int f = u.f0 + r, t = f / G;
      const bool ok = f < u.nf;
      const T* q = reinterpret_cast<const T*>(a.q) + ((long long)(u.r0 + (ok ? t : 0)) * v.H + head * G + (ok ? f % G : 0)) * v.d;
      float4 x[P > 128 ? 2 : 1];
      unsigned top = 0;
#pragma unroll
      for (int y = 0; y < (P > 128 ? 2 : 1); ++y) {
        const int c = 4 * lane + 128 * y;
        x[y] = ok && c < v.d ? load4(q + c) : make_float4(0.f, 0.f, 0.f, 0.f);
        top = max(top, max(max(__float_as_uint(x[y].x) & 0x7fffffffu, __float_as_uint(x[y].y) & 0x7fffffffu),
                           max(__float_as_uint(x[y].z) & 0x7fffffffu, __float_as_uint(x[y].w) & 0x7fffffffu)));
      }
      top = __reduce_max_sync(0xffffffffu, top);
      const int e = top >= 0x7f800000u ? 140 : min(max((int)(top >> 23), 27), 254);      // a row that is not finite is left as it is
      const float up = pow2(267 - e);
      float sum = 0.f;
#pragma unroll
      for (int y = 0; y < (P > 128 ? 2 : 1); ++y) {
        const int c = 4 * lane + 128 * y;
        if (c >= P) break;
        const float4 w = scaled(x[y], up);
        uint2 h = make_uint2(pack_f16(w.x, w.y), pack_f16(w.z, w.w));
        unsigned char* to = smem + C::Q + r * C::QP + 2 * c;
        *reinterpret_cast<uint2*>(to) = h;
        if (BIAS) {
          const float2 p0 = unpack_f16(h.x), p1 = unpack_f16(h.y);
          sum += (p0.x + p0.y) + (p1.x + p1.y);
        }
        if (NQ == 2) {
          const float2 p0 = unpack_f16(h.x), p1 = unpack_f16(h.y);
          *reinterpret_cast<uint2*>(to + RT * C::QP) = make_uint2(pack_f16(w.x - p0.x, w.y - p0.y), pack_f16(w.z - p1.x, w.w - p1.y));
        }
      }
      if (BIAS) sum = warp_sum(sum);
      if (lane == 0) {
        s_rf[r] = make_float2(fmaxf(a.scale * 1.4426950408889634f * pow2(e - 13), 1.17549435e-38f), -1152.f * sum);
        RowInfo info = {-1, 0, 0};
        if (ok) {
          info.t = t;
          info.away = a.tree.away(u.r0 + t, t);
          if (a.tree.seen) info.seen = a.tree.seen[a.tree.per_row ? u.r0 + t : t];
        }
        s_rows[r] = info;
      }
    }
  };

  begin_segment();
  stage_queries();
  __syncthreads();
  while (true) {
    // ---- the warp's blocks of this segment.  A thread's rows are 8 nt + 2 rc + x (x = 0, 1), its positions 8 j + rg of a block
    float acc[CH][NT][4], m_run[NT][2], l_run[NT][2], rf[NT][2], first[NT][2];
    unsigned qf[C::QREG ? CH : 1][NT * NQ][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int k = 0; k < CH; ++k)
#pragma unroll
        for (int x = 0; x < 4; ++x) acc[k][nt][x] = 0.f;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        m_run[nt][x] = -CUDART_INF_F;
        l_run[nt][x] = 0.f;
        const float2 r = s_rf[8 * nt + 2 * rc + x];
        rf[nt][x] = r.x;
        first[nt][x] = r.y;
      }
    }
    auto query = [&](int nt, int half, int k, unsigned (&q)[2]) {
      const uint2 x = *reinterpret_cast<const uint2*>(smem + C::Q + half * RT * C::QP + (8 * nt + rg) * C::QP + 32 * k + 8 * rc);
      q[0] = x.x; q[1] = x.y;
    };
    if (C::QREG)
#pragma unroll
      for (int k = 0; k < CH; ++k)
#pragma unroll
        for (int j = 0; j < NT * NQ; ++j) query(j / NQ, j % NQ, k, qf[C::QREG ? k : 0][j]);
    int R = 16;                                              // biased exponent of the largest scale of values met
    for (int k = 0, i = seg_a + warp; i < seg_b; ++k, i += WARPS, ++it) {
      if ((k & 31) == 0 && k) { page_cur = page_nxt; page_nxt = pages_of(k + 32); }
      const int page = __shfl_sync(0xffffffffu, page_cur, k & 31);
      const unsigned s = it % ST;
      if (!mbar_try1(bars + 8 * s, (it / ST) & 1) && !mbar_wait_long(bars + 8 * s, (it / ST) & 1, dead ? 1000000ull : WAIT_CYCLES)) dead = true;
      dead = __any_sync(0xffffffffu, dead);
      const unsigned char* blk = ring + s * C::BLOCK;
      if (page < 0 || dead) {
        if (lane == 0) v.status[dead ? 2 : 0] = 1;
      } else {
        const float* sc = reinterpret_cast<const float*>(blk + 2 * QKV_BLOCK * P);
        const unsigned row_s = ring_s + s * C::BLOCK + lane * P;
        const int turn = qkv_turn(CH, lane);
        const int k0 = i * QKV_BLOCK;
        const bool full = k0 >= u.full_lo && k0 + QKV_BLOCK <= u.full_hi;
        // ---- scores: register j of a read holds channels 4 rc .. + 3 of position 8 j + rg
        float t[2][NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int x = 0; x < 4; ++x) t[0][nt][x] = t[1][nt][x] = BIAS ? first[nt][x & 1] : 0.f;
#pragma unroll
        for (int kc = 0; kc < CH; ++kc) {
          unsigned r[4], ka[2][4];
          asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(row_s + ((kc ^ turn) << 4)));
#pragma unroll
          for (int j = 0; j < 4; ++j) halves_of<SCHEME, false, BIAS>(r[j], ka[j >> 1][j & 1], ka[j >> 1][2 + (j & 1)]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int half = 0; half < NQ; ++half) {
              unsigned q[2];
              if (C::QREG) { q[0] = qf[C::QREG ? kc : 0][nt * NQ + half][0]; q[1] = qf[C::QREG ? kc : 0][nt * NQ + half][1]; }
              else query(nt, half, kc, q);
              mma_f16(t[0][nt], ka[0], q[0], q[1]);
              mma_f16(t[1][nt], ka[1], q[0], q[1]);
            }
        }
        // ---- scales of the block: the largest of the values' that count
        {
          const unsigned b = __float_as_uint(sc[QKV_BLOCK + lane]);
          const bool counts = (full || (k0 + lane >= u.lo && k0 + lane < u.hi)) && b < 0x7f800000u;
          const int e = (int)(__reduce_max_sync(0xffffffffu, counts ? b : 0u) >> 23);
          if (e > R) {
            const float f = pow2(127 + R - e);
            R = e;
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int x = 0; x < 4; ++x) acc[c][nt][x] *= f;
          }
        }
        const float rs = pow2(268 - R);
        float ks[4], vs[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) { ks[j] = sc[8 * j + rg]; vs[j] = sc[QKV_BLOCK + 8 * j + rg] * rs; }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int x = 0; x < 2; ++x) t[j >> 1][nt][2 * (j & 1) + x] *= ks[j];
        if (!full) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const RowInfo row = s_rows[8 * nt + 2 * rc + x];
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const int key = k0 + 8 * j + rg, n = key - u.len;
                bool see;
                if (n < 0) see = a.window == 0 || u.len + row.away - key < a.window;
                else if (a.tree.seen) see = n < u.n && ((row.seen >> n) & 1);
                else see = n <= row.t && (a.window == 0 || row.t - n < a.window);
                if (row.t < 0 || !see || key >= u.hi) t[j >> 1][nt][2 * (j & 1) + x] = -CUDART_INF_F;
              }
            }
        }
        // ---- weights
        unsigned pb[NT][NQ][4];                              // of positions 8 j + 2 rc, + 1 and row 8 nt + rg
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float f[2], base[2];
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float mx = fmaxf(fmaxf(t[0][nt][x], t[0][nt][2 + x]), fmaxf(t[1][nt][x], t[1][nt][2 + x]));
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            const float m = fmaxf(m_run[nt][x], mx * rf[nt][x]);
            base[x] = m == -CUDART_INF_F ? 0.f : m;          // nothing seen yet: every weight becomes exp2(-inf) = 0
            f[x] = ex2(m_run[nt][x] - base[x]);
            m_run[nt][x] = m;
          }
          if (__any_sync(0xffffffffu, f[0] != 1.f || f[1] != 1.f)) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              l_run[nt][x] *= f[x];
#pragma unroll
              for (int c = 0; c < CH; ++c) { acc[c][nt][x] *= f[x]; acc[c][nt][2 + x] *= f[x]; }
            }
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float w[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const float s1 = t[j >> 1][nt][2 * (j & 1) + x], p = ex2(fmaf(s1, rf[nt][x], -base[x]));
              l_run[nt][x] += p;                             // this lane's share; the eight lanes of a row are summed at the end
              w[x] = p * vs[j];
              if (!full && s1 == -CUDART_INF_F) w[x] = 0.f;  // what a row does not see may have any scale, NaN too
            }
            const unsigned hi = pack_f16(w[0], w[1]);
            pb[nt][0][j] = transposed(hi);
            if (NQ == 2) {
              const float2 g = unpack_f16(hi);
              pb[nt][NQ - 1][j] = transposed(pack_f16(w[0] - g.x, w[1] - g.y));
            }
          }
        }
        // ---- values: register j of a transposed read holds channels 2 rg, 2 rg + 1 of positions 8 j + 2 rc, + 1; row m of the
        // product is channel 2 m (m < 8) or 2 (m - 8) + 1
#pragma unroll
        for (int kc = 0; kc < CH; ++kc) {
          unsigned r[4], va[2][4];
          asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(row_s + QKV_BLOCK * P + ((kc ^ turn) << 4)));
#pragma unroll
          for (int j = 0; j < 4; ++j) halves_of<SCHEME, true, false>(r[j], va[j >> 1][2 * (j & 1)], va[j >> 1][2 * (j & 1) + 1]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int half = 0; half < NQ; ++half)
#pragma unroll
              for (int ks2 = 0; ks2 < 2; ++ks2) mma_f16(acc[kc][nt], va[ks2], pb[nt][half][2 * ks2], pb[nt][half][2 * ks2 + 1]);
        }
      }
      __syncwarp();                                          // all lanes are done with the stage
      if (i + WARPS * ST < seg_b) {
        const int kn = k + ST;
        ask(kn, __shfl_sync(0xffffffffu, (kn >> 5) == (k >> 5) ? page_cur : page_nxt, kn & 31));
      }
    }
    // ---- the next segment's first blocks are on their way while this one is merged
    const Unit du = u;
    const int d_head = head;
    const long long u_begin = at - tile, seg_n = seg_b - seg_a;
    const bool whole = seg_n == du.tiles;
    const int cta0 = (int)(u_begin / share), cta1 = (int)((u_begin + du.tiles - 1) / share);
    at += seg_n;
    const bool more = at < end;
    if (more) {
      tile = 0;
      if (++head == v.KH) {
        head = 0;
        do { ++z; unit_of<RT>(a, rts, z, u); } while (u.tiles == 0);
      }
      begin_segment();
    }
    // ---- the four warps' results of a row
    const float r_inv = pow2(R - 14);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        float l = l_run[nt][x];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        if (rg == 0) s_ml[warp * RT + 8 * nt + 2 * rc + x] = make_float2(m_run[nt][x], l);
      }
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int r = 8 * nt + 2 * rc + x;
        float m = -CUDART_INF_F;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) m = fmaxf(m, s_ml[w * RT + r].x);
        const float f = m_run[nt][x] == -CUDART_INF_F ? 0.f : ex2(m_run[nt][x] - m) * r_inv;
#pragma unroll
        for (int c = 0; c < CH; ++c) { acc[c][nt][x] *= f; acc[c][nt][2 + x] *= f; }
      }
    constexpr int SUB = C::SUB, MP = C::MP;
    const int o_sub = tid / (RT * 4), o_row = tid / 4 % RT, o_c = 4 * (tid % 4), f = du.f0 + o_row;
    const int part = 2 * (int)blockIdx.x + ((int)blockIdx.x == cta0 ? 1 : 0);
    float m_all = -CUDART_INF_F, l_all = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) m_all = fmaxf(m_all, s_ml[w * RT + o_row].x);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float2 x = s_ml[w * RT + o_row];
      if (x.x != -CUDART_INF_F) l_all += x.y * ex2(x.x - m_all);
    }
    const float inv = l_all == 0.f ? 0.f : 1.f / l_all;      // nothing seen: zero
    T* out = reinterpret_cast<T*>(a.out) + ((long long)(du.r0 + f / G) * v.H + d_head * G + f % G) * v.d;
    float* part_o = a.part_o + ((long long)part * RT + o_row) * P;
#pragma unroll
    for (int c0 = 0; c0 < CH; c0 += SUB) {
#pragma unroll
      for (int sub = 0; sub < SUB; ++sub) {
        if (c0 + sub >= CH) break;
        const int cc = c0 + sub < CH ? c0 + sub : 0;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int x = 0; x < 2; ++x)
            *reinterpret_cast<float2*>(s_merge + ((sub * WARPS + warp) * RT + 8 * nt + 2 * rc + x) * MP + 2 * rg) = make_float2(acc[cc][nt][x], acc[cc][nt][2 + x]);
      }
      __syncthreads();
      const int c = 16 * (c0 + o_sub) + o_c;
      if (o_sub < SUB && f < du.nf && c < P) {
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
          const float4 y = *reinterpret_cast<const float4*>(s_merge + ((o_sub * WARPS + w) * RT + o_row) * MP + o_c);
          x = make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w);
        }
        if (!whole) store4(part_o + c, x);
        else if (c < v.d) store4(out + c, scaled(x, inv));
      }
      __syncthreads();
    }
    // ---- a unit of several CTAs
    if (!whole) {
      if (f < du.nf && tid % 4 == 0 && o_sub == 0) a.part_ml[part * RT + o_row] = make_float2(m_all, l_all);
      __shared__ int s_last;
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        s_last = atomicAdd(&a.tickets[cta0], 1) == cta1 - cta0;
        if (s_last) a.tickets[cta0] = 0;
      }
      __syncthreads();
      if (s_last) {
        __threadfence();
        const int n = cta1 - cta0 + 1, rows = min(RT, du.nf - du.f0);
        auto slot_of = [&](int j) { return 2 * (cta0 + j) + (j == 0 ? 1 : 0); };
        for (int x = tid; x < rows * (P / 4); x += THREADS) {
          const int r = x / (P / 4), c = x % (P / 4) * 4, ff = du.f0 + r;
          float m = -CUDART_INF_F, l = 0.f;
          for (int j = 0; j < n; ++j) m = fmaxf(m, __ldcg(&a.part_ml[slot_of(j) * RT + r]).x);
          float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
          for (int j = 0; j < n; ++j) {
            const float2 ml = __ldcg(&a.part_ml[slot_of(j) * RT + r]);
            const float4 y = __ldcg(reinterpret_cast<const float4*>(a.part_o + ((long long)slot_of(j) * RT + r) * P + c));
            const float w = ml.x == -CUDART_INF_F ? 0.f : ex2(ml.x - m);
            l = fmaf(ml.y, w, l);
            o = make_float4(fmaf(y.x, w, o.x), fmaf(y.y, w, o.y), fmaf(y.z, w, o.z), fmaf(y.w, w, o.w));
          }
          if (c < v.d)
            store4(reinterpret_cast<T*>(a.out) + ((long long)(du.r0 + ff / G) * v.H + d_head * G + ff % G) * v.d + c, scaled(o, l == 0.f ? 0.f : 1.f / l));
        }
      }
    }
    if (!more) break;
    stage_queries();
    __syncthreads();
  }
}

template <typename T, int SCHEME, int P, int NT>
int32_t launch(vn_qkv* c, const QkvAttnArgs& a) {
  using C = AttnCfg<T, P, NT>;
  vn_ctx* ctx = c->ctx;
  auto kernel = qkv_attn_kernel<T, SCHEME, P, NT>;
  static int per_sm[64] = {};
  int& occ = per_sm[ctx->device & 63];
  if (!occ) {
    VN_CUDA(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    int n = 0;
    VN_CUDA(ctx, cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, THREADS, C::SMEM));
    VN_REQUIRE(ctx, n > 0, "qkv_attn_kernel does not fit an SM");
    occ = min(n, QKV_MAX_CTAS);
  }
  const long long rts = ceil_div((long long)a.step.T * (a.v.H / a.v.KH), (long long)C::RT);
  VN_REQUIRE(ctx, rts < (1ll << 31), "too many rows");
  // no more CTAs than there can be shares of blocks
  const double most = (double)a.step.n_ent * (double)rts * a.v.KH * (a.v.capacity() / QKV_BLOCK) / MIN_SHARE + 1;
  const unsigned grid = (unsigned)min((double)occ * ctx->sm_count, most);
  VN_LAUNCH_NAMED(ctx, "qkv_attn_kernel", kernel, grid, THREADS, C::SMEM, a, (int)rts);
  return VN_OK;
}

template <int SCHEME>
int32_t pick(vn_qkv* c, const QkvAttnArgs& a) {
  // as few columns as hold the rows of an entry; 32 share the conversions of a block where there are more than 16
  const long long rows = (long long)a.step.T * (a.v.H / a.v.KH);
#define GO(P, NT) return c->dtype == VN_F32 ? launch<float, SCHEME, P, NT>(c, a) : launch<bf16, SCHEME, P, NT>(c, a)
#define GO2(P) do { if (rows <= 8) GO(P, 1); else GO(P, 2); } while (0)
#define GO4(P) do { if (rows <= 8) GO(P, 1); else if (rows <= 16) GO(P, 2); else GO(P, 4); } while (0)
  switch (a.v.P) {
    case 32: GO4(32);
    case 64: GO4(64);
    case 80: GO4(80);
    case 96: GO4(96);
    case 128: GO4(128);
    case 192: GO2(192);
    case 256: GO2(256);
    default: return vn_fail(c->ctx, VN_ERR_UNSUPPORTED, "pitch %d", a.v.P);
  }
#undef GO4
#undef GO2
#undef GO
}

}  // namespace qkv_detail
