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
// all (entry, rows, head) units form one line that is cut into equal shares for the CTAs, whatever the lengths; the parts of a unit that
// several CTAs have are merged, in their order, by a second kernel that has all SMs for it (one CTA that merged a unit's parts by
// itself took 10 to 15 us for 7 parts of 64 rows or 56 parts of 8).
#pragma once
#include "qkv.cuh"

namespace qkv_detail {

using bf16 = __nv_bfloat16;
constexpr int WARPS = 4, THREADS = 32 * WARPS;
constexpr int MIN_SHARE = WARPS;                    // blocks of a CTA at least
constexpr int UNCUT = 8;                            // blocks of a unit that is never cut
constexpr unsigned long long WAIT_CYCLES = 4000000000ull;   // a copy that has not come after about two seconds never will

// RS = 1: the warps share a unit's rows and split its blocks; RS = 4: they split its rows and share its blocks
template <typename T, int P, int NT, int RS>
struct AttnCfg {
  static constexpr int NQ = sizeof(T) == 4 ? 2 : 1;           // halves of a query or weight
  static constexpr int WR = 8 * NT, RT = WR * RS, CH = P / 16, BLOCK = QKV_BLOCK * (2 * P + 8);   // rows of a warp, of a unit
  static constexpr int RINGS = WARPS / RS;
  static constexpr int QP = 2 * P + ((2 * P) % 64 == 0 ? 32 : 0);   // bytes of a staged query row: four rows' 32-byte pieces in 128 bytes of banks
  static constexpr int STAGES = RS > 1 ? 4 : P <= 64 ? 4 : P <= 128 && NT >= 2 && NT * NQ <= 2 ? 3 : 2;
  static constexpr int CTAS = RS > 1 ? (P * NT <= 256 && NT < 4 && NQ == 1 ? 3 : P * NT <= 512 ? 2 : 1) : P > 192 || (P > 128 && NQ * NT > 1) ? 1 : P * NT <= 128 ? 3 : 2;
  static constexpr bool QREG = NT * NQ <= 2 && NT * NQ * P <= (RS > 1 ? 128 : 256);      // query fragments in registers
  static constexpr int SUB = RS > 1 ? 0 : NT >= 4 ? 1 : 2;    // chunks of 16 channels that are merged at a time
  static constexpr int MP = 20;                               // pitch of a merged row: 16 lanes' pairs in different banks
  static constexpr int RING = 0, Q = RING + RINGS * STAGES * BLOCK, MERGE = Q + NQ * RT * QP,
                       MERGE_BYTES = SUB * WARPS * RT * MP * 4 > (THREADS + 8) * 4 ? SUB * WARPS * RT * MP * 4 : (THREADS + 8) * 4, ML = MERGE + MERGE_BYTES,
                       ROWS = ML + (RS > 1 ? 0 : WARPS * RT * 8), RF = ROWS + RT * 16, BARS = RF + RT * 8, SMEM = BARS + RINGS * STAGES * 16,
                       PLAN = MERGE;                          // read before anything is merged
  static_assert(CTAS * RT * P <= QKV_PART, "parts fit their place");
};

struct RowInfo { int t, away; unsigned long long seen; };    // t < 0: no row

__device__ __forceinline__ void mbar_init(unsigned bar, int count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count)); }
__device__ __forceinline__ void mbar_arrive1(unsigned bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
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
__device__ __forceinline__ bool unit_of(const QkvAttnArgs& a, int rts, int z, Unit& u) {
  const int e = rts == 1 ? z : z / rts, rt = rts == 1 ? 0 : z - e * rts, G = a.v.H / a.v.KH;
  u.tiles = 0;
  if (!a.step.entry(a.v, e, &u.slot, &u.r0, &u.n)) return false;
  u.f0 = rt * RT;
  u.nf = u.n * G;
  if (u.f0 >= u.nf) return false;
  const int t0 = rts == 1 ? 0 : u.f0 / G, t1 = rts == 1 ? u.n - 1 : (min(u.f0 + RT, u.nf) - 1) / G;
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

template <typename T, int SCHEME, int P, int NT, int RS>
__global__ void __launch_bounds__(THREADS, (AttnCfg<T, P, NT, RS>::CTAS)) qkv_attn_kernel(QkvAttnArgs a, int rts, bool split) {
  pdl_trigger();
  using C = AttnCfg<T, P, NT, RS>;
  constexpr int RT = C::RT, CH = C::CH, ST = C::STAGES, NQ = C::NQ;
  constexpr bool BIAS = SCHEME == QKV_I8 && NQ == 1;         // keys 1152 too large: taken off the sums instead, at the cost of some bits of them
  extern __shared__ __align__(128) unsigned char smem[];
  const QkvView& v = a.v;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rg = lane >> 2, rc = lane & 3;
  const int G = v.H / v.KH;
  const unsigned s_base = (unsigned)__cvta_generic_to_shared(smem);
  constexpr int RINGS = C::RINGS, WR = C::WR;
  const int kw = RS > 1 ? 0 : warp, row0 = RS > 1 ? warp * WR : 0;            // which of the blocks, which of the rows are the warp's
  unsigned char* ring = smem + C::RING + kw * ST * C::BLOCK;
  const unsigned ring_s = s_base + C::RING + kw * ST * C::BLOCK, bars = s_base + C::BARS + kw * ST * 16;   // a stage is full, is empty
  RowInfo* s_rows = reinterpret_cast<RowInfo*>(smem + C::ROWS);
  float2* s_rf = reinterpret_cast<float2*>(smem + C::RF);    // r of a row, and what its sums begin with
  float2* s_ml = reinterpret_cast<float2*>(smem + C::ML);
  float* s_merge = reinterpret_cast<float*>(smem + C::MERGE);
  int* s_plan = reinterpret_cast<int*>(smem + C::PLAN);

  // ---- the line of blocks (or of units, where they are not cut) and this CTA's share
  const int Z = a.step.n_ent * rts, zc = (Z + THREADS - 1) / THREADS;
  Unit u;
  auto weight = [&]() { return (split ? u.tiles : min(u.tiles, 1)) * v.KH; };
  {
    int sum = 0;
    for (int z = tid * zc; z < min(Z, (tid + 1) * zc); ++z) {
      unit_of<RT>(a, rts, z, u);
      sum += weight();
    }
    if (lane < ST && (RS == 1 || warp == 0)) { mbar_init(bars + 16 * lane, 1); mbar_init(bars + 16 * lane + 8, RS); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    int up = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, up, o);
      if (lane >= o) up += t;
    }
    int* s_tot = s_plan + THREADS + 1;
    if (lane == 31) s_tot[warp] = up;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS - 1; ++w) up += w < warp ? s_tot[w] : 0;
    s_plan[tid + 1] = up;
    if (tid == 0) s_plan[0] = 0;
    __syncthreads();
  }
  const int W = s_plan[THREADS];
  const int share = max((W + (int)gridDim.x - 1) / (int)gridDim.x, split ? MIN_SHARE : 1);
  int at = (int)min((long long)blockIdx.x * share, (long long)W);
  const int end = (int)min((long long)at + share, (long long)W);
  if (tid == 0) a.cuts[blockIdx.x].n = 0;                    // no unit of this CTA goes on in the next, until one does
  if (at >= end) return;
  int z, head, tile;                                         // where the share begins
  {
    int j = 0;
#pragma unroll
    for (int o = THREADS / 2; o > 0; o >>= 1)
      if (s_plan[j + o] <= at) j += o;
    z = j * zc;
    int rem = at - s_plan[j];
    for (;; ++z) {
      unit_of<RT>(a, rts, z, u);
      const int n = weight();
      if (rem < n) break;
      rem -= n;
    }
    head = split ? rem / u.tiles : rem;
    tile = split ? rem - head * u.tiles : 0;
  }

  unsigned it = 0, put = 0;                                  // blocks taken and asked for
  bool dead = false;                                         // a copy did not come: nothing is computed any more
  int page_cur = -1, page_nxt = -1;                          // pages of the warp's next 32 and 64 blocks of a segment
  int seg_a = 0, seg_b = 0;
  auto pages_of = [&](int k0) {
    const int i = seg_a + kw + RINGS * (k0 + lane);
    return i < seg_b ? v.page(u.slot, i * QKV_BLOCK / KV_PAGE) : -1;
  };
  auto came = [&](unsigned bar, unsigned parity) {           // bounded wait
    if (!mbar_try1(bar, parity) && !mbar_wait_long(bar, parity, dead ? 1000000ull : WAIT_CYCLES)) dead = true;
  };
  auto ask = [&](int k, int page) {                          // block k of the warp's in this segment
    if (RS > 1 && warp) return;
    if (lane == 0) {
      const unsigned s = put % ST, bar = bars + 16 * s;
      const int i = seg_a + kw + RINGS * k;
      if (RS > 1 && put >= ST) came(bar + 8, (put / ST - 1) & 1);
      if (page >= 0 && !dead) fetch_block(ring_s + s * C::BLOCK, v.block(page, head, i & 1), C::BLOCK, bar);
      else mbar_arrive1(bar);
    }
    ++put;
  };
  constexpr int AHEAD = RS > 1 ? ST - 1 : ST;                // blocks asked for before their turn; shared ones leave a stage to the slowest warp
  auto begin_segment = [&]() {
    seg_a = u.tile0 + tile;
    seg_b = split ? min(u.tile0 + u.tiles, seg_a + (end - at)) : u.tile0 + u.tiles;
    page_cur = pages_of(0);
    page_nxt = pages_of(32);
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (seg_a + kw + RINGS * k < seg_b) ask(k, __shfl_sync(0xffffffffu, page_cur, k));
  };
  auto stage_queries = [&]() {                               // a warp brings a quarter of the rows, up to 16 asked for at a time
    constexpr int Y = P > 128 ? 2 : 1, PER = RT / WARPS, BATCH = PER < 16 / Y ? PER : 16 / Y;
#pragma unroll 1
    for (int rb = 0; rb < PER; rb += BATCH) {
      float4 x[BATCH][Y];
#pragma unroll
      for (int b = 0; b < BATCH; ++b) {
        const int f = u.f0 + warp * PER + rb + b, t = f / G;
        const bool ok = f < u.nf;
        const T* q = reinterpret_cast<const T*>(a.q) + ((long long)(u.r0 + (ok ? t : 0)) * v.H + head * G + (ok ? f - t * G : 0)) * v.d;
#pragma unroll
        for (int y = 0; y < Y; ++y) {
          const int c = 4 * lane + 128 * y;
          x[b][y] = ok && c < v.d ? load4(q + c) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
      }
      // each reduction for all rows before the next step: a shuffle waits for nothing but the one before it in its own row
      unsigned top[BATCH];
      float up[BATCH], sum[BATCH];
#pragma unroll
      for (int b = 0; b < BATCH; ++b) {
        top[b] = 0;
#pragma unroll
        for (int y = 0; y < Y; ++y)
          top[b] = max(top[b], max(max(__float_as_uint(x[b][y].x) & 0x7fffffffu, __float_as_uint(x[b][y].y) & 0x7fffffffu),
                                   max(__float_as_uint(x[b][y].z) & 0x7fffffffu, __float_as_uint(x[b][y].w) & 0x7fffffffu)));
      }
#pragma unroll
      for (int b = 0; b < BATCH; ++b) top[b] = __reduce_max_sync(0xffffffffu, top[b]);
#pragma unroll
      for (int b = 0; b < BATCH; ++b) {
        top[b] = top[b] >= 0x7f800000u ? 140 : min(max(top[b] >> 23, 27u), 254u);      // a row that is not finite is left as it is
        up[b] = pow2(267 - (int)top[b]);
        sum[b] = 0.f;
#pragma unroll
        for (int y = 0; y < Y; ++y) {
          const int c = 4 * lane + 128 * y;
          if (c >= P) break;
          const float4 w = scaled(x[b][y], up[b]);
          const uint2 h = make_uint2(pack_f16(w.x, w.y), pack_f16(w.z, w.w));
          unsigned char* to = smem + C::Q + (warp * PER + rb + b) * C::QP + 2 * c;
          *reinterpret_cast<uint2*>(to) = h;
          const float2 p0 = unpack_f16(h.x), p1 = unpack_f16(h.y);
          if (BIAS) sum[b] += (p0.x + p0.y) + (p1.x + p1.y);
          if (NQ == 2) *reinterpret_cast<uint2*>(to + RT * C::QP) = make_uint2(pack_f16(w.x - p0.x, w.y - p0.y), pack_f16(w.z - p1.x, w.w - p1.y));
        }
      }
      if (BIAS)
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
#pragma unroll
          for (int b = 0; b < BATCH; ++b) sum[b] += __shfl_xor_sync(0xffffffffu, sum[b], o);
      if (lane == 0)
#pragma unroll
        for (int b = 0; b < BATCH; ++b)
          s_rf[warp * PER + rb + b] = make_float2(fmaxf(a.scale * 1.4426950408889634f * pow2((int)top[b] - 13), 1.17549435e-38f), -1152.f * sum[b]);
    }
  };
  auto describe_rows = [&]() {
    if (tid < RT) {
      RowInfo info = {-1, 0, 0};
      const int f = u.f0 + tid, t = f / G;
      if (f < u.nf) {
        info.t = t;
        info.away = a.tree.away(u.r0 + t, t);
        if (a.tree.seen) info.seen = a.tree.seen[a.tree.per_row ? u.r0 + t : t];
      }
      s_rows[tid] = info;
    }
  };

  begin_segment();
  while (true) {
    describe_rows();
    stage_queries();
    __syncthreads();
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
        const float2 r = s_rf[row0 + 8 * nt + 2 * rc + x];
        rf[nt][x] = r.x;
        first[nt][x] = r.y;
      }
    }
    auto query = [&](int nt, int half, int k, unsigned (&q)[2]) {
      const uint2 x = *reinterpret_cast<const uint2*>(smem + C::Q + half * RT * C::QP + (row0 + 8 * nt + rg) * C::QP + 32 * k + 8 * rc);
      q[0] = x.x; q[1] = x.y;
    };
    if (C::QREG)
#pragma unroll
      for (int k = 0; k < CH; ++k)
#pragma unroll
        for (int j = 0; j < NT * NQ; ++j) query(j / NQ, j % NQ, k, qf[C::QREG ? k : 0][j]);
    int R = 16;                                              // biased exponent of the largest scale of values met
    for (int k = 0, i = seg_a + kw; i < seg_b; ++k, i += RINGS, ++it) {
      if ((k & 31) == 0 && k) { page_cur = page_nxt; page_nxt = pages_of(k + 32); }
      const int page = __shfl_sync(0xffffffffu, page_cur, k & 31);
      const unsigned s = it % ST;
      came(bars + 16 * s, (it / ST) & 1);
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
              const RowInfo row = s_rows[row0 + 8 * nt + 2 * rc + x];
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
        float base[NT][2], f[NT][2];
        bool grew = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int x = 0; x < 2; ++x) base[nt][x] = fmaxf(fmaxf(t[0][nt][x], t[0][nt][2 + x]), fmaxf(t[1][nt][x], t[1][nt][2 + x]));
#pragma unroll
        for (int o = 4; o < 32; o <<= 1)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 2; ++x) base[nt][x] = fmaxf(base[nt][x], __shfl_xor_sync(0xffffffffu, base[nt][x], o));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const float m = fmaxf(m_run[nt][x], base[nt][x] * rf[nt][x]);
            base[nt][x] = m == -CUDART_INF_F ? 0.f : m;      // nothing seen yet: every weight becomes exp2(-inf) = 0
            f[nt][x] = ex2(m_run[nt][x] - base[nt][x]);
            m_run[nt][x] = m;
            grew |= f[nt][x] != 1.f;
          }
        if (__any_sync(0xffffffffu, grew))
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              l_run[nt][x] *= f[nt][x];
#pragma unroll
              for (int c = 0; c < CH; ++c) { acc[c][nt][x] *= f[nt][x]; acc[c][nt][2 + x] *= f[nt][x]; }
            }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float w[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const float s1 = t[j >> 1][nt][2 * (j & 1) + x], p = ex2(fmaf(s1, rf[nt][x], -base[nt][x]));
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
      if (RS > 1 && lane == 0) mbar_arrive1(bars + 16 * s + 8);
      if (i + RINGS * AHEAD < seg_b) {
        const int kn = k + AHEAD;
        ask(kn, __shfl_sync(0xffffffffu, (kn >> 5) == (k >> 5) ? page_cur : page_nxt, kn & 31));
      }
    }
    // ---- the next segment's first blocks are on their way while this one is merged
    const Unit du = u;
    const int d_head = head, done = split ? seg_b - seg_a : 1, u_begin = at - tile;
    const bool whole = !split || done == du.tiles, goes_on = !whole && u_begin + du.tiles > end;
    const bool begun = !whole && tile == 0;                  // this CTA has the unit's first part
    at += done;
    const bool more = at < end;
    if (more) {
      tile = 0;
      if (++head == v.KH) {
        head = 0;
        do { ++z; unit_of<RT>(a, rts, z, u); } while (u.tiles == 0);
      }
      begin_segment();
    }
    const float r_inv = pow2(R - 14);
#pragma unroll
    for (int o = 4; o < 32; o <<= 1)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < 2; ++x) l_run[nt][x] += __shfl_xor_sync(0xffffffffu, l_run[nt][x], o);
    const int part = 2 * (int)blockIdx.x + (begun ? 1 : 0);
    if constexpr (RS > 1) {
      // ---- a warp's rows are its own: straight to memory, 32 bytes of a row (bf16) at a time
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float l = l_run[nt][x];
          const int r = row0 + 8 * nt + 2 * rc + x, f = du.f0 + r;
          if (f >= du.nf) continue;
          const float inv = whole ? (l == 0.f ? 0.f : r_inv / l) : r_inv;    // nothing seen: zero
          T* out = reinterpret_cast<T*>(a.out) + ((long long)(du.r0 + f / G) * v.H + d_head * G + f % G) * v.d + 2 * rg;
          float* part_o = a.part_o + ((long long)part * RT + r) * P + 2 * rg;
#pragma unroll
          for (int c = 0; c < CH; ++c) {
            const float2 y = make_float2(acc[c][nt][x] * inv, acc[c][nt][2 + x] * inv);
            if (!whole) *reinterpret_cast<float2*>(part_o + 16 * c) = y;
            else if (16 * c + 2 * rg < v.d) {
              if constexpr (sizeof(T) == 4) *reinterpret_cast<float2*>(out + 16 * c) = y;
              else *reinterpret_cast<__nv_bfloat162*>(out + 16 * c) = __floats2bfloat162_rn(y.x, y.y);
            }
          }
          if (!whole && rg == 0) a.part_ml[part * RT + r] = make_float2(m_run[nt][x], l);
        }
      __syncthreads();
    } else {
      // ---- the four warps' results of a row
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < 2; ++x)
          if (rg == 0) s_ml[warp * RT + 8 * nt + 2 * rc + x] = make_float2(m_run[nt][x], l_run[nt][x]);
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
    float m_all = -CUDART_INF_F, l_all = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) m_all = fmaxf(m_all, s_ml[w * RT + o_row].x);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float2 x = s_ml[w * RT + o_row];
      l_all += x.y * (x.x == -CUDART_INF_F ? 0.f : ex2(x.x - m_all));       // a sum that is not a number stays one
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
    if (!whole && f < du.nf && tid % 4 == 0 && o_sub == 0) a.part_ml[part * RT + o_row] = make_float2(m_all, l_all);
    }
    if (begun && goes_on && tid == 0)                        // the CTAs that have its blocks: this one and the next ones
      a.cuts[blockIdx.x] = {du.r0, du.f0, du.nf, d_head, (u_begin + du.tiles - 1) / share - (int)blockIdx.x + 1};
    if (!more) break;
  }
}

// Parts of the units that were cut, in the order of their CTAs: a warp per row.  grid (CTAs of the attention, row groups), block 128
template <typename T, int P>
__global__ void __launch_bounds__(THREADS) qkv_merge_kernel(QkvAttnArgs a, int RT) {
  constexpr int Y = P > 128 ? 2 : 1, IN = Y > 1 ? 8 : 16;    // parts asked for at a time
  pdl_wait();
  const QkvCut o = a.cuts[blockIdx.x];
  const int lane = threadIdx.x & 31, rows = min(RT, o.nf - o.f0), G = a.v.H / a.v.KH;
  for (int r = blockIdx.y * WARPS + (threadIdx.x >> 5); o.n > 0 && r < rows; r += gridDim.y * WARPS) {
    auto at = [&](int j) { return (long long)(2 * (blockIdx.x + j) + (j == 0 ? 1 : 0)) * RT + r; };
    float m = -CUDART_INF_F, l = 0.f;
    for (int j = lane; j < o.n; j += 32) m = fmaxf(m, a.part_ml[at(j)].x);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    float4 sum[Y];
#pragma unroll
    for (int y = 0; y < Y; ++y) sum[y] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int j0 = 0; j0 < o.n; j0 += 32) {
      float w = 0.f;
      if (j0 + lane < o.n) {
        const float2 ml = a.part_ml[at(j0 + lane)];
        // nothing seen: no weight; a sum without a maximum is no number
        w = ml.x == -CUDART_INF_F ? (ml.y == 0.f ? 0.f : CUDART_NAN_F) : ex2(ml.x - m);
        l += ml.y * w;
      }
#pragma unroll 1
      for (int j1 = 0; j1 < 32 && j0 + j1 < o.n; j1 += IN) {
        float4 x[IN][Y];
#pragma unroll
        for (int j = 0; j < IN; ++j)
#pragma unroll
          for (int y = 0; y < Y; ++y) {
            const int c = 4 * lane + 128 * y;
            x[j][y] = c < P ? *reinterpret_cast<const float4*>(a.part_o + at(min(j0 + j1 + j, o.n - 1)) * P + c) : make_float4(0.f, 0.f, 0.f, 0.f);
          }
#pragma unroll
        for (int j = 0; j < IN; ++j) {
          const float f = __shfl_sync(0xffffffffu, w, j1 + j);
#pragma unroll
          for (int y = 0; y < Y; ++y)
            sum[y] = make_float4(fmaf(x[j][y].x, f, sum[y].x), fmaf(x[j][y].y, f, sum[y].y), fmaf(x[j][y].z, f, sum[y].z), fmaf(x[j][y].w, f, sum[y].w));
        }
      }
    }
    l = warp_sum(l);
    const int f = o.f0 + r;
    T* out = reinterpret_cast<T*>(a.out) + ((long long)(o.r0 + f / G) * a.v.H + o.head * G + f % G) * a.v.d;
#pragma unroll
    for (int y = 0; y < Y; ++y)
      if (4 * lane + 128 * y < a.v.d) store4(out + 4 * lane + 128 * y, scaled(sum[y], l == 0.f ? 0.f : 1.f / l));
  }
}

template <typename T, int SCHEME, int P, int NT, int RS>
int32_t launch(vn_qkv* c, const QkvAttnArgs& a) {
  using C = AttnCfg<T, P, NT, RS>;
  vn_ctx* ctx = c->ctx;
  auto kernel = qkv_attn_kernel<T, SCHEME, P, NT, RS>;
  static int per_sm[64] = {};
  int& occ = per_sm[ctx->device & 63];
  if (!occ) {
    VN_CUDA(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    int n = 0;
    VN_CUDA(ctx, cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, THREADS, C::SMEM));
    VN_REQUIRE(ctx, n > 0, "qkv_attn_kernel does not fit an SM");
    occ = min(n, C::CTAS);
  }
  const long long rts = ceil_div((long long)a.step.T * (a.v.H / a.v.KH), (long long)C::RT);
  const long long blocks = rts * a.step.n_ent * a.v.KH, tiles = a.v.capacity() / QKV_BLOCK;
  VN_REQUIRE(ctx, rts < (1ll << 31) && blocks < (1ll << 31) / tiles - THREADS, "%d rows over %d positions are too many for one call: bring them in portions", a.step.M, a.v.capacity());
  // units of a few blocks stay whole: cutting them saves less than the merge costs
  const bool split = tiles > UNCUT;
  // no more CTAs than there can be shares
  const unsigned grid = (unsigned)min((long long)occ * ctx->sm_count, split ? ceil_div(blocks * tiles, (long long)MIN_SHARE) : blocks);
  VN_LAUNCH_NAMED(ctx, "qkv_attn_kernel", kernel, grid, THREADS, C::SMEM, a, (int)rts, split);
  if (split) VN_LAUNCH_PDL_LEVEL(ctx, 1, "qkv_merge_kernel", (qkv_merge_kernel<T, P>), dim3(grid, min(C::RT / WARPS, 16)), THREADS, 0, a, C::RT);
  return VN_OK;
}

template <int SCHEME>
int32_t pick(vn_qkv* c, const QkvAttnArgs& a) {
  // as few columns as hold the rows of an entry; from 17 rows on the warps split the rows
  const long long rows = (long long)a.step.T * (a.v.H / a.v.KH);
#define GO(P, NT, RS) return c->dtype == VN_F32 ? launch<float, SCHEME, P, NT, RS>(c, a) : launch<bf16, SCHEME, P, NT, RS>(c, a)
#define GO2(P) do { if (rows <= 8) GO(P, 1, 1); else if (rows <= 16) GO(P, 2, 1); else GO(P, 2, 4); } while (0)
#define GO4(P) do { if (rows <= 8) GO(P, 1, 1); else if (rows <= 16) GO(P, 2, 1); else if (rows <= 64) GO(P, 2, 4); else GO(P, 4, 4); } while (0)
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
