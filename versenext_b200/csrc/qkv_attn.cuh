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
// block of 32 positions for 16 MT rows (tokens x heads of a group), four warps of a CTA take every fourth block.  The blocks of
// all (entry, rows, head) units form one line that is cut into equal shares for the CTAs, whatever the lengths; a unit that several
// CTAs have is merged, in their order, by the one that ends last.
#pragma once
#include "qkv.cuh"

namespace qkv_detail {

using bf16 = __nv_bfloat16;
constexpr int WARPS = 4, THREADS = 32 * WARPS;
constexpr int MIN_SHARE = WARPS;                    // blocks of a CTA at least
constexpr unsigned long long WAIT_CYCLES = 4000000000ull;   // a copy that has not come after about two seconds never will

template <typename T, int P, int MT>
struct AttnCfg {
  static constexpr int NQ = sizeof(T) == 4 ? 2 : 1;           // halves of a query or weight
  static constexpr int RT = 16 * MT, CH = P / 16, BLOCK = QKV_BLOCK * (2 * P + 8);
  static constexpr int QP = 2 * P + ((2 * P) % 64 == 0 ? 32 : 0);   // bytes of a staged query row: four rows' 32-byte pieces in 128 bytes of banks
  static constexpr int STAGES = P <= 64 ? 4 : P <= 128 && MT * NQ == 1 ? 3 : 2;
  static constexpr bool QREG = MT * NQ == 1 && P <= 128;      // query fragments in registers
  static constexpr int RING = 0, Q = RING + WARPS * STAGES * BLOCK, MERGE = Q + NQ * RT * QP, ML = MERGE + 8192, ROWS = ML + WARPS * RT * 8,
                       RF = ROWS + RT * 16, BARS = RF + RT * 4, SMEM = BARS + WARPS * STAGES * 8, PLAN = MERGE;   // the plan is read before anything is merged
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
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float pow2(int biased) { return __uint_as_float((unsigned)min(max(biased, 0), 254) << 23); }   // 2^(biased - 127), 0 below

// two codes of a register as halves.  int8: with the sign bit flipped a code plus 128 is put under the exponent of 1024, from which
// 1152 is taken off.  e4m3: sign, exponent and mantissa moved to a half's places, 2^8 too small (the factors r and R allow for it).
// PAIR: bytes 0 and 1 (0), 2 and 3 (1), 0 and 2 (2), 1 and 3 (3); u: the register, for int8 with its sign bits flipped
template <int SCHEME, int PAIR> __device__ __forceinline__ unsigned halves_of(unsigned u) {
  if (SCHEME == QKV_I8) {
    constexpr unsigned sel = PAIR == 0 ? 0x4140 : PAIR == 1 ? 0x4342 : PAIR == 2 ? 0x4240 : 0x4341;
    const unsigned x = __byte_perm(u, 0x64646464u, sel);
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const unsigned*>(&h);
  }
  constexpr unsigned sel = PAIR == 0 ? 0x1404 : PAIR == 1 ? 0x3424 : PAIR == 2 ? 0x2404 : 0x3414;
  const unsigned x = __byte_perm(u, 0u, sel);
  return ((x >> 1) & 0x3f803f80u) | (x & 0x80008000u);
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

template <typename T, int SCHEME, int P, int MT>
__global__ void __launch_bounds__(THREADS, P > 192 ? 1 : 2) qkv_attn_kernel(QkvAttnArgs a, int rts) {
  using C = AttnCfg<T, P, MT>;
  static_assert(C::RT * P <= QKV_PART, "a part fits its place");
  constexpr int RT = C::RT, CH = C::CH, ST = C::STAGES, NQ = C::NQ;
  extern __shared__ __align__(128) unsigned char smem[];
  const QkvView& v = a.v;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rg = lane >> 2, rc = lane & 3;
  const int G = v.H / v.KH;
  const unsigned s_base = (unsigned)__cvta_generic_to_shared(smem);
  unsigned char* ring = smem + C::RING + warp * ST * C::BLOCK;
  const unsigned ring_s = s_base + C::RING + warp * ST * C::BLOCK, bars = s_base + C::BARS + warp * ST * 8;
  RowInfo* s_rows = reinterpret_cast<RowInfo*>(smem + C::ROWS);
  float* s_rf = reinterpret_cast<float*>(smem + C::RF);
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
#pragma unroll
      for (int y = 0; y < (P > 128 ? 2 : 1); ++y) {
        const int c = 4 * lane + 128 * y;
        if (c >= P) break;
        const float4 w = scaled(x[y], up);
        uint2 h = make_uint2(pack_f16(w.x, w.y), pack_f16(w.z, w.w));
        unsigned char* to = smem + C::Q + r * C::QP + 2 * c;
        *reinterpret_cast<uint2*>(to) = h;
        if (NQ == 2) {
          const float2 p0 = unpack_f16(h.x), p1 = unpack_f16(h.y);
          *reinterpret_cast<uint2*>(to + RT * C::QP) = make_uint2(pack_f16(w.x - p0.x, w.y - p0.y), pack_f16(w.z - p1.x, w.w - p1.y));
        }
      }
      if (lane == 0) {
        s_rf[r] = fmaxf(a.scale * 1.4426950408889634f * pow2(e - 13 + (SCHEME == QKV_E4M3 ? 8 : 0)), 1.17549435e-38f);
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
    // ---- the warp's blocks of this segment
    float acc[MT][CH][2][4], m_run[MT][2], l_run[MT][2], rf[MT][2];
    unsigned qf[C::QREG ? CH : 1][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int k = 0; k < CH; ++k)
#pragma unroll
        for (int x = 0; x < 4; ++x) acc[mt][k][0][x] = acc[mt][k][1][x] = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        m_run[mt][h] = -CUDART_INF_F;
        l_run[mt][h] = 0.f;
        rf[mt][h] = s_rf[16 * mt + rg + 8 * h];
      }
    }
    auto query = [&](int mt, int half, int k, unsigned (&q)[4]) {
      const unsigned char* p = smem + C::Q + half * RT * C::QP + (16 * mt + rg) * C::QP + 32 * k + 8 * rc;
      const uint2 x = *reinterpret_cast<const uint2*>(p), y = *reinterpret_cast<const uint2*>(p + 8 * C::QP);
      q[0] = x.x; q[1] = y.x; q[2] = x.y; q[3] = y.y;
    };
    if (C::QREG)
#pragma unroll
      for (int k = 0; k < CH; ++k) query(0, 0, k, qf[C::QREG ? k : 0]);
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
        // ---- scores
        float t[MT][4][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int nb = 0; nb < 4; ++nb)
#pragma unroll
            for (int x = 0; x < 4; ++x) t[mt][nb][x] = 0.f;
#pragma unroll
        for (int kc = 0; kc < CH; ++kc) {
          unsigned r[4];
          asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(row_s + ((kc ^ turn) << 4)));
          unsigned b[4][2];
#pragma unroll
          for (int nb = 0; nb < 4; ++nb) {
            if (SCHEME == QKV_I8) r[nb] ^= 0x80808080u;
            b[nb][0] = halves_of<SCHEME, 0>(r[nb]);
            b[nb][1] = halves_of<SCHEME, 1>(r[nb]);
          }
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int half = 0; half < NQ; ++half) {
              unsigned q[4];
              if (C::QREG) {
#pragma unroll
                for (int x = 0; x < 4; ++x) q[x] = qf[C::QREG ? kc : 0][x];
              } else {
                query(mt, half, kc, q);
              }
#pragma unroll
              for (int nb = 0; nb < 4; ++nb) mma_f16(t[mt][nb], q, b[nb][0], b[nb][1]);
            }
        }
        // ---- scales of the block: the largest of the values' that count
        {
          const float vs = sc[QKV_BLOCK + lane];
          const unsigned b = __float_as_uint(vs);
          const bool counts = (full || (k0 + lane >= u.lo && k0 + lane < u.hi)) && b < 0x7f800000u;
          const int e = (int)(__reduce_max_sync(0xffffffffu, counts ? b : 0u) >> 23);
          if (e > R) {
            const float f = pow2(127 + R - e);
            R = e;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
              for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int x = 0; x < 4; ++x) { acc[mt][c][0][x] *= f; acc[mt][c][1][x] *= f; }
          }
        }
        const float rs = pow2(268 - R);
#pragma unroll
        for (int nb = 0; nb < 4; ++nb) {
          const float2 ks = *reinterpret_cast<const float2*>(sc + 8 * nb + 2 * rc);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int x = 0; x < 4; ++x) t[mt][nb][x] *= x & 1 ? ks.y : ks.x;
        }
        if (!full) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const RowInfo row = s_rows[16 * mt + rg + 8 * h];
#pragma unroll
              for (int nb = 0; nb < 4; ++nb)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                  const int key = k0 + 8 * nb + 2 * rc + x, j = key - u.len;
                  bool see;
                  if (j < 0) see = a.window == 0 || u.len + row.away - key < a.window;
                  else if (a.tree.seen) see = j < u.n && ((row.seen >> j) & 1);
                  else see = j <= row.t && (a.window == 0 || row.t - j < a.window);
                  if (row.t < 0 || !see || key >= u.hi) t[mt][nb][2 * h + x] = -CUDART_INF_F;
                }
            }
        }
        // ---- weights
        unsigned pa[MT][NQ][2][4];                           // halves of the weights of 16 keys, as the product takes them
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          float f[2], base[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float mx = t[mt][0][2 * h];
#pragma unroll
            for (int nb = 0; nb < 4; ++nb) mx = fmaxf(mx, fmaxf(t[mt][nb][2 * h], t[mt][nb][2 * h + 1]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const float m = fmaxf(m_run[mt][h], mx * rf[mt][h]);
            base[h] = m == -CUDART_INF_F ? 0.f : m;          // nothing seen yet: every weight becomes exp2(-inf) = 0
            f[h] = ex2(m_run[mt][h] - base[h]);
            m_run[mt][h] = m;
          }
          if (__any_sync(0xffffffffu, f[0] != 1.f || f[1] != 1.f)) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              l_run[mt][h] *= f[h];
#pragma unroll
              for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int x = 0; x < 2; ++x) { acc[mt][c][0][2 * h + x] *= f[h]; acc[mt][c][1][2 * h + x] *= f[h]; }
            }
          }
#pragma unroll
          for (int nb = 0; nb < 4; ++nb) {
            float2 vs = *reinterpret_cast<const float2*>(sc + QKV_BLOCK + 8 * nb + 2 * rc);
            vs.x *= rs; vs.y *= rs;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float s0 = t[mt][nb][2 * h], s1 = t[mt][nb][2 * h + 1];
              const float p0 = ex2(fmaf(s0, rf[mt][h], -base[h])), p1 = ex2(fmaf(s1, rf[mt][h], -base[h]));
              l_run[mt][h] += p0 + p1;                       // this lane's share; the four lanes of a row are summed at the end
              float w0 = p0 * vs.x, w1 = p1 * vs.y;
              if (!full) {                                   // what a row does not see may have any scale, NaN too
                if (s0 == -CUDART_INF_F) w0 = 0.f;
                if (s1 == -CUDART_INF_F) w1 = 0.f;
              }
              const unsigned hi = pack_f16(w0, w1);
              pa[mt][0][nb >> 1][h + 2 * (nb & 1)] = hi;
              if (NQ == 2) {
                const float2 w = unpack_f16(hi);
                pa[mt][NQ - 1][nb >> 1][h + 2 * (nb & 1)] = pack_f16(w0 - w.x, w1 - w.y);
              }
            }
          }
        }
        // ---- values: register j of a transposed read holds channels 2 n, 2 n + 1 of positions 8 j + 2 rc, + 1 (n = lane / 4)
#pragma unroll
        for (int kc = 0; kc < CH; ++kc) {
          unsigned r[4];
          asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(row_s + QKV_BLOCK * P + ((kc ^ turn) << 4)));
          unsigned b[2][4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (SCHEME == QKV_I8) r[j] ^= 0x80808080u;
            b[0][j] = halves_of<SCHEME, 2>(r[j]);
            b[1][j] = halves_of<SCHEME, 3>(r[j]);
          }
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int half = 0; half < NQ; ++half)
#pragma unroll
              for (int ks = 0; ks < 2; ++ks) {
                mma_f16(acc[mt][kc][0], pa[mt][half][ks], b[0][2 * ks], b[0][2 * ks + 1]);
                mma_f16(acc[mt][kc][1], pa[mt][half][ks], b[1][2 * ks], b[1][2 * ks + 1]);
              }
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
    const float r_inv = pow2(R - 14 + (SCHEME == QKV_E4M3 ? 8 : 0));
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float l = l_run[mt][h];
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if (rc == 0) s_ml[warp * RT + 16 * mt + rg + 8 * h] = make_float2(m_run[mt][h], l);
      }
    __syncthreads();
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = 16 * mt + rg + 8 * h;
        float m = -CUDART_INF_F;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) m = fmaxf(m, s_ml[w * RT + r].x);
        const float f = m_run[mt][h] == -CUDART_INF_F ? 0.f : ex2(m_run[mt][h] - m) * r_inv;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
          for (int x = 0; x < 2; ++x) { acc[mt][c][0][2 * h + x] *= f; acc[mt][c][1][2 * h + x] *= f; }
      }
    constexpr int SUB = 2 / MT;                              // chunks of 16 channels that are exchanged at a time
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
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float (&x)[2][4] = acc[mt][c0 + sub < CH ? c0 + sub : 0];
            *reinterpret_cast<float4*>(s_merge + ((sub * WARPS + warp) * RT + 16 * mt + rg + 8 * h) * 16 + 4 * rc) =
                make_float4(x[0][2 * h], x[1][2 * h], x[0][2 * h + 1], x[1][2 * h + 1]);
          }
      }
      __syncthreads();
      const int c = 16 * (c0 + o_sub) + o_c;
      if (f < du.nf && c < P) {
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
          const float4 y = *reinterpret_cast<const float4*>(s_merge + ((o_sub * WARPS + w) * RT + o_row) * 16 + o_c);
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

template <typename T, int SCHEME, int P, int MT>
int32_t launch(vn_qkv* c, const QkvAttnArgs& a) {
  using C = AttnCfg<T, P, MT>;
  vn_ctx* ctx = c->ctx;
  auto kernel = qkv_attn_kernel<T, SCHEME, P, MT>;
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
  // 32 rows share the conversions of a block where there are more than 16 and registers for their results
  const bool wide = (long long)a.step.T * (a.v.H / a.v.KH) > 16;
#define GO(P, MT) return c->dtype == VN_F32 ? launch<float, SCHEME, P, MT>(c, a) : launch<bf16, SCHEME, P, MT>(c, a)
#define GO2(P) do { if (wide) GO(P, 2); else GO(P, 1); } while (0)
  switch (a.v.P) {
    case 32: GO2(32);
    case 64: GO2(64);
    case 80: GO2(80);
    case 96: GO2(96);
    case 128: GO2(128);
    case 192: GO(192, 1);
    case 256: GO(256, 1);
    default: return vn_fail(c->ctx, VN_ERR_UNSUPPORTED, "pitch %d", a.v.P);
  }
#undef GO2
#undef GO
}

}  // namespace qkv_detail
