// Attention of a step's rows over the 8-bit cache: the committed positions and the rows that the step has appended.
//
// o = sum_j p_j s_j c_j / sum_j p_j,  p_j = exp2(t_j r - m),  t_j = (q' . k_j) a_j: k_j, c_j codes of keys and values, a_j, s_j their
// scales, q' the query times a power of two that brings its largest channel to [2^13, 2^14), r what undoes that times
// scale * log2(e).  Codes are whole numbers or e4m3, both exact in 16-bit floats, so the products run on the tensor cores
// (mma.sync m16n8k16, fp32 sums) with no rounding of keys and values; queries and weights are rounded to 11 bits for bf16 rows and
// split into two halves of 11 bits for fp32 rows: chosen as a second product for the rest of a weight would double those of the values, for a
// result of 8 bits (bf16: 0.0017 from 64 bits either way) or 2^-22 of a weight (fp32: 2.0e-7 against 1.9e-7).  A weight p_j s_j is taken relative to a power of two R above every s_j that the row has seen so
// far, times 2^15, so that a half holds weights down to 2^-39 of the largest (2^-37 beside rows that see one up to four times as large).  Scales
// are brought to the largest R of the warp's rows; by what a row's own is below that, its weights' exponents are higher (up to 2^BELOW, so
// that their sums are numbers): what a row does not see takes no bits from it.
// 32 x 5 rows behind 1500 positions: 28.9 us, 29.3 with a factor for every weight and row, 27.3 with one R for all rows.
//
// What bounds it is the memory of the codes (few rows) or the mma.sync rate and the conversions (many).  Positions are the rows of the
// products and queries their columns (8 at a time): S = K q^T, O = V^T p^T, with p transposed by movmatrix between.  A warp takes
// blocks of 32 positions for 8 NT rows (tokens x heads of a group) and waits for no other warp.  The blocks of all (entry, rows, head) units
// form one line that is cut into equal shares, whatever the lengths: a share for every warp (RS = 1), or, with more rows than a warp has,
// one for every CTA, whose four warps have rows of their own and share the blocks that come in (RS = 4).  The parts of a unit that
// several shares have are merged, in their order, by a second kernel that has all SMs for it (one CTA that merged a unit's parts by
// itself took 10 to 15 us for 7 parts of 64 rows or 56 parts of 8).
#pragma once
#include "qkv.cuh"

namespace qkv_detail {

using bf16 = __nv_bfloat16;
constexpr int WARPS = 4, THREADS = 32 * WARPS;
constexpr int MIN_SHARE = 4;                        // blocks of a share at least
constexpr int MERGE_WARPS = 8, MANY = 8;           // warps of a merging CTA; parts that one of them takes
constexpr int UNCUT = 8;                            // in caches with room for no more blocks, units are not cut
constexpr int BELOW = 117;                          // a row's R is at most that many powers of two below the largest of its warp
constexpr int MERGE_CTAS = 4;                       // merging CTAs on an SM
// A copy that has not come after about two seconds is taken not to come.  The call is then no good and reported; whoever has met it asks for no more,
// and before its memory goes to somebody else waits once more, LATE_CYCLES, for each copy that it has asked for
constexpr unsigned long long WAIT_CYCLES = 4000000000ull, LATE_CYCLES = 1000000ull;

template <typename T, int P, int NT, int RS>
struct AttnCfg {
  static constexpr int NQ = sizeof(T) == 4 ? 2 : 1;           // halves of a query or weight
  static constexpr int WR = 8 * NT, RT = WR * RS, CH = P / 16, BLOCK = QKV_BLOCK * (2 * P + 8);   // rows of a warp, of a unit
  static constexpr int RINGS = WARPS / RS;
  static constexpr int CTAS = P > 192 ? 1 : NT < 4 && P * NT * NQ <= 256 && P * NT <= 128 ? 3 : P * NT <= 256 && NT < 4 && NQ == 1 && RS > 1 ? 3 : P * NT <= 512 ? 2 : 1;
  static constexpr bool QREG = NT * NQ <= 2 && NT * NQ * P <= (RS > 1 ? 128 : 256);      // query fragments in registers, else a thread's own in shared memory
  static constexpr int STAGES = RS > 1 ? 4 : P <= 64 ? 4 : CTAS == 2 && P * NT <= 256 && QREG ? 3 : 2;
  static constexpr int RING = 0, Q = RING + RINGS * STAGES * BLOCK, BARS = Q + (QREG ? 0 : WARPS * CH * NT * NQ * 256), PLAN = BARS + RINGS * STAGES * 16,
                       SMEM = PLAN + (THREADS + 8) * 8;
  static_assert(CTAS * WARPS * WR * P <= QKV_PART, "parts fit their place");
};

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
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
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
  int tile0, tiles;                          // the tiles of positions that hold them
};

// BLK: positions of a tile
template <int RT, int BLK>
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
  u.tile0 = u.lo / BLK;
  u.tiles = (u.hi + BLK - 1) / BLK - u.tile0;
  if (u.tiles <= 0) { u.tile0 = 0; u.tiles = 1; }            // rows that see nothing still get their zeros
  return true;
}

// The line of tiles of all (entry, rows, head) units (or of the units, where they are not cut) and what of it a worker has: `end` tiles,
// the first of them tile `tile` of unit (z, head).  The line is counted in 64 bits (65 heads of 2^30 positions), a share, from its own first tile
// on, in 32.  False: nothing.  Called by all threads of a CTA; s_plan: THREADS + 8 numbers
struct Share { int z, head, tile, at, end, share; };
__device__ __forceinline__ int quotient(long long x, int y) { return x >> 31 ? (int)(x / y) : (int)x / y; }      // x >= 0, y > 0
template <int RT, int BLK>
__device__ __forceinline__ bool find_share(const QkvAttnArgs& a, int rts, bool split, int least, int worker, int workers, long long* s_plan, Unit& u, Share& s) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, KH = a.v.KH, Z = a.step.n_ent * rts, zc = (Z + THREADS - 1) / THREADS;
  auto weight = [&]() { return (long long)(split ? u.tiles : min(u.tiles, 1)) * KH; };
  long long up = 0;
  if (tid < THREADS) {
    for (int z = tid * zc; z < min(Z, (tid + 1) * zc); ++z) {
      unit_of<RT, BLK>(a, rts, z, u);
      up += weight();
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long t = __shfl_up_sync(0xffffffffu, up, o);
      if (lane >= o) up += t;
    }
    if (lane == 31) s_plan[THREADS + 1 + warp] = up;
  }
  __syncthreads();
  if (tid < THREADS) {
#pragma unroll
    for (int w = 0; w < WARPS - 1; ++w) up += w < warp ? s_plan[THREADS + 1 + w] : 0;
    s_plan[tid + 1] = up;
    if (tid == 0) s_plan[0] = 0;
  }
  __syncthreads();
  const long long W = s_plan[THREADS];
  s.share = max(quotient(W + workers - 1, workers), split ? least : 1);
  const long long from = (long long)worker * s.share;
  if (from >= W) return false;
  s.at = 0;
  s.end = (int)min((long long)s.share, W - from);
  int j = 0;
#pragma unroll
  for (int o = THREADS / 2; o > 0; o >>= 1)
    if (s_plan[j + o] <= from) j += o;
  s.z = j * zc;
  long long rem = from - s_plan[j];
  for (;; ++s.z) {
    unit_of<RT, BLK>(a, rts, s.z, u);
    const long long n = weight();
    if (rem < n) break;
    rem -= n;
  }
  s.head = split ? quotient(rem, u.tiles) : (int)rem;
  s.tile = split ? (int)(rem - (long long)s.head * u.tiles) : 0;
  return true;
}

template <typename T, int SCHEME, int P, int NT, int RS>
__global__ void __launch_bounds__(THREADS, (AttnCfg<T, P, NT, RS>::CTAS)) qkv_attn_kernel(QkvAttnArgs a, int rts, bool split) {
  pdl_trigger();
  using C = AttnCfg<T, P, NT, RS>;
  constexpr int RT = C::RT, CH = C::CH, ST = C::STAGES, NQ = C::NQ, RINGS = C::RINGS, WR = C::WR;
  constexpr bool BIAS = SCHEME == QKV_I8 && NQ == 1;         // keys 1152 too large: taken off the sums instead, at the cost of some bits of them
  extern __shared__ __align__(128) unsigned char smem[];
  const QkvView& v = a.v;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rg = lane >> 2, rc = lane & 3;
  const int G = v.H / v.KH;
  const int ring_no = RS > 1 ? 0 : warp, row0 = RS > 1 ? warp * WR : 0;       // the warp's ring of blocks, its rows in a unit
  const unsigned s_base = (unsigned)__cvta_generic_to_shared(smem);
  unsigned char* ring = smem + C::RING + ring_no * ST * C::BLOCK;
  const unsigned ring_s = s_base + C::RING + ring_no * ST * C::BLOCK, bars = s_base + C::BARS + ring_no * ST * 16;   // a stage is full, is empty
  long long* s_plan = reinterpret_cast<long long*>(smem + C::PLAN);
  if (lane < ST && (RS == 1 || warp == 0)) { mbar_init(bars + 16 * lane, 1); mbar_init(bars + 16 * lane + 8, RS); }
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  pdl_wait();

  const int worker = RS > 1 ? blockIdx.x : blockIdx.x * WARPS + warp, workers = RS > 1 ? gridDim.x : gridDim.x * WARPS;
  Unit u;
  Share sh;
  if (!find_share<RT, QKV_BLOCK>(a, rts, split, MIN_SHARE, worker, workers, s_plan, u, sh)) return;
  int z = sh.z, head = sh.head, tile = sh.tile, at = sh.at;
  const int end = sh.end, share = sh.share;

  unsigned it = 0, put = 0;                                  // blocks taken, and asked for (by the lane that asks)
  bool dead = false;                                         // a copy did not come: nothing is computed any more
  int page_cur = -1, page_nxt = -1;                          // pages of the next 32 and 64 blocks of a segment
  int seg_a = 0, seg_b = 0;
  auto pages_of = [&](int k0) {
    const int i = seg_a + k0 + lane;
    return i < seg_b ? v.page(u.slot, i * QKV_BLOCK / KV_PAGE) : -1;
  };
  auto came = [&](unsigned bar, unsigned parity) {           // bounded wait
    if (!dead && !mbar_try1(bar, parity) && !mbar_wait_long(bar, parity, WAIT_CYCLES)) dead = true;
  };
  auto ask = [&](int k, int page) {                          // block k of this segment
    if (RS > 1 && warp) return;
    if (lane == 0) {
      const unsigned s = put % ST, bar = bars + 16 * s;
      if (RS > 1 && put >= ST) came(bar + 8, (put / ST - 1) & 1);
      if (dead) return;
      if (page >= 0) fetch_block(ring_s + s * C::BLOCK, v.block(page, head, (seg_a + k) & 1), C::BLOCK, bar);
      else mbar_arrive1(bar);
      ++put;
    }
  };
  constexpr int AHEAD = RS > 1 ? ST - 1 : ST;                // blocks asked for before their turn; shared ones leave a stage to the slowest warp
  auto begin_segment = [&]() {
    seg_a = u.tile0 + tile;
    seg_b = split ? min(u.tile0 + u.tiles, seg_a + (end - at)) : u.tile0 + u.tiles;
    page_cur = pages_of(0);
    page_nxt = pages_of(32);
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (seg_a + k < seg_b) ask(k, __shfl_sync(0xffffffffu, page_cur, k));
  };

  begin_segment();
  while (true) {
    // ---- queries: a thread takes channels 16 k + 4 rc .. + 3 of row 8 nt + rg, which is what the product wants of it
    float rf[NT][2], first[NT][2];                           // of rows 8 nt + 2 rc + x: r, and what their sums begin with
    int row_t[NT][2];                                        // their tokens, -1: no row
    unsigned qf[C::QREG ? CH : 1][NT * NQ][2];
    uint2* s_q = reinterpret_cast<uint2*>(smem + C::Q) + warp * CH * NT * NQ * 32 + lane;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int f = u.f0 + row0 + 8 * nt + rg, t = f / G;
      const bool ok = f < u.nf;
      const T* q = reinterpret_cast<const T*>(a.q) + ((long long)(u.r0 + (ok ? t : 0)) * v.H + head * G + (ok ? f - t * G : 0)) * v.d + 4 * rc;
      float4 x[CH];
#pragma unroll
      for (int k = 0; k < CH; ++k) x[k] = ok && 16 * k + 4 * rc < v.d ? load4(q + 16 * k) : make_float4(0.f, 0.f, 0.f, 0.f);
      unsigned top = 0;
#pragma unroll
      for (int k = 0; k < CH; ++k)
        top = max(top, max(max(__float_as_uint(x[k].x) & 0x7fffffffu, __float_as_uint(x[k].y) & 0x7fffffffu),
                           max(__float_as_uint(x[k].z) & 0x7fffffffu, __float_as_uint(x[k].w) & 0x7fffffffu)));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int e = min(max((int)(top >> 23), 27), 254);
      const float up = top >= 0x7f800000u ? CUDART_NAN_F : pow2(267 - e);      // a query that is not finite has no soft-max: NaN for all it sees
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < CH; ++k) {
        const float4 w = scaled(x[k], up);
        const uint2 h = make_uint2(pack_f16(w.x, w.y), pack_f16(w.z, w.w));
        const float2 p0 = unpack_f16(h.x), p1 = unpack_f16(h.y);
        if (BIAS) sum += (p0.x + p0.y) + (p1.x + p1.y);
        const uint2 lo = NQ == 2 ? make_uint2(pack_f16(w.x - p0.x, w.y - p0.y), pack_f16(w.z - p1.x, w.w - p1.y)) : h;
        if (C::QREG) {
          qf[C::QREG ? k : 0][nt * NQ][0] = h.x; qf[C::QREG ? k : 0][nt * NQ][1] = h.y;
          if (NQ == 2) { qf[C::QREG ? k : 0][nt * NQ + NQ - 1][0] = lo.x; qf[C::QREG ? k : 0][nt * NQ + NQ - 1][1] = lo.y; }
        } else {
          s_q[(k * NT * NQ + nt * NQ) * 32] = h;
          if (NQ == 2) s_q[(k * NT * NQ + nt * NQ + NQ - 1) * 32] = lo;
        }
      }
      if (BIAS) {
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      }
      const float r = fmaxf(a.scale * 1.4426950408889634f * pow2(e - 13), 1.17549435e-38f);
#pragma unroll
      for (int x2 = 0; x2 < 2; ++x2) {
        rf[nt][x2] = __shfl_sync(0xffffffffu, r, 4 * (2 * rc + x2));
        first[nt][x2] = BIAS ? -1152.f * __shfl_sync(0xffffffffu, sum, 4 * (2 * rc + x2)) : 0.f;
        row_t[nt][x2] = __shfl_sync(0xffffffffu, ok ? t : -1, 4 * (2 * rc + x2));
      }
    }
    // ---- the blocks of this segment.  A thread's rows are 8 nt + 2 rc + x (x = 0, 1), its positions 8 j + rg of a block
    float acc[CH][NT][4], m_run[NT][2], l_run[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int k = 0; k < CH; ++k)
#pragma unroll
        for (int x = 0; x < 4; ++x) acc[k][nt][x] = 0.f;
#pragma unroll
      for (int x = 0; x < 2; ++x) { m_run[nt][x] = -CUDART_INF_F; l_run[nt][x] = 0.f; }
    }
    int R = 16;                                              // biased exponent of the largest scale of values that a row of the warp has seen
    bool mixed = false;                                      // there are rows whose own is below it
    unsigned R4[(NT + 1) / 2];                               // by how much: four rows in a register
#pragma unroll
    for (int i = 0; i < (NT + 1) / 2; ++i) R4[i] = 0u;
    auto below = [&](int nt, int x) { return (int)((R4[nt / 2] >> (16 * (nt & 1) + 8 * x)) & 255u); };
#pragma unroll 1
    for (int i = seg_a; i < seg_b; ++i, ++it) {
      const int k = i - seg_a;
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
              else { const uint2 y = s_q[(kc * NT * NQ + nt * NQ + half) * 32]; q[0] = y.x; q[1] = y.y; }
              mma_f16(t[0][nt], ka[0], q[0], q[1]);
              mma_f16(t[1][nt], ka[1], q[0], q[1]);
            }
        }
        // ---- scales of the block: where the largest of the values' (numbers only) that some row sees is above R, all rows mostly see one of at least a
        // quarter of it, and take it for theirs; if not, the rows' own are looked up when it is known what they see
        bool odd = mixed;
        {
          const unsigned b = __float_as_uint(sc[QKV_BLOCK + lane]);
          const bool counts = (full || (k0 + lane >= u.lo && k0 + lane < u.hi)) && b < 0x7f800000u;
          const int all = (int)(__reduce_max_sync(0xffffffffu, counts ? b : 0u) >> 23);
          if (all > R && !mixed) {
            odd = !full && !__any_sync(0xffffffffu, counts && (int)(b >> 23) >= all - 2 && k0 + lane >= u.full_lo && k0 + lane < u.full_hi);
            if (!odd) {
              const float f = pow2(127 + R - all);
              R = all;
#pragma unroll
              for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                  for (int x = 0; x < 4; ++x) acc[c][nt][x] *= f;
            }
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
              const int tok = row_t[nt][x], away = tok < 0 || a.window == 0 ? 0 : a.tree.behind(v, u.r0 + tok, tok);
              const unsigned long long seen = a.tree.seen && tok >= 0 ? a.tree.sees(u.r0 + tok, tok, a.window) : 0;
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const int key = k0 + 8 * j + rg, n = key - u.len;
                bool see;
                if (n < 0) see = a.window == 0 || u.len + away - key < a.window;
                else if (a.tree.seen) see = n < u.n && ((seen >> n) & 1);
                else see = n <= tok && (a.window == 0 || tok - n < a.window);
                if (tok < 0 || !see || key >= u.hi) t[j >> 1][nt][2 * (j & 1) + x] = -CUDART_INF_F;
              }
            }
        }
        if (__builtin_expect(odd, 0)) {                      // row by row
          auto raw = [&](int j) { return __float_as_uint(sc[QKV_BLOCK + 8 * j + rg]); };
          unsigned own[(NT + 1) / 2], most = R;
#pragma unroll
          for (int h = 0; h < (NT + 1) / 2; ++h) {
            unsigned seen = 0, valid = 0;                  // bytes, as R4
#pragma unroll
            for (int y = 0; y < 4 && 2 * h + y / 2 < NT; ++y) {
              const int nt = 2 * h + y / 2, x = y & 1;
              unsigned top = 0;
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if (t[j >> 1][nt][2 * (j & 1) + x] != -CUDART_INF_F && raw(j) < 0x7f800000u) top = max(top, raw(j));
              seen |= (top >> 23) << (8 * y);
              if (row_t[nt][x] >= 0) valid |= 255u << (8 * y);
            }
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) seen = __vmaxu4(seen, __shfl_xor_sync(0xffffffffu, seen, o));
            own[h] = __vmaxu4(0x01010101u * (unsigned)R - R4[h], seen) & valid;
            most = max(max(most, max(own[h] & 255u, own[h] >> 24)), max((own[h] >> 8) & 255u, (own[h] >> 16) & 255u));
            own[h] |= ~valid;                              // (rows that are none: 255)
          }
          most = __reduce_max_sync(0xffffffffu, most);
          unsigned any = 0;
#pragma unroll
          for (int h = 0; h < (NT + 1) / 2; ++h) {
            const unsigned to = __vminu4(0x01010101u * most - __vminu4(own[h], 0x01010101u * most), 0x01010101u * BELOW);
#pragma unroll
            for (int y = 0; y < 4 && 2 * h + y / 2 < NT; ++y) {
              const int nt = 2 * h + y / 2, x = y & 1;
              const float f = pow2(127 + R - (int)most + (int)((to >> (8 * y)) & 255u) - (int)((R4[h] >> (8 * y)) & 255u));
#pragma unroll
              for (int c = 0; c < CH; ++c) { acc[c][nt][x] *= f; acc[c][nt][2 + x] *= f; }
            }
            R4[h] = to;
            any |= to;
          }
          R = (int)most;
          mixed = __any_sync(0xffffffffu, any != 0);
          const float rs = pow2(268 - R);
#pragma unroll
          for (int j = 0; j < 4; ++j) vs[j] = sc[QKV_BLOCK + 8 * j + rg] * rs;
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
        if (__builtin_expect(mixed, 0))
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 2; ++x) base[nt][x] -= (float)below(nt, x);
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
        for (int nt = 0; nt < NT; ++nt) {
          float sum[2] = {0.f, 0.f};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float w[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const float s1 = t[j >> 1][nt][2 * (j & 1) + x], p = ex2(fmaf(s1, rf[nt][x], -base[nt][x]));
              sum[x] += p;
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
#pragma unroll
          for (int x = 0; x < 2; ++x) {                      // this lane's share; the eight lanes of a row are summed at the end
            if (__builtin_expect(mixed, 0)) sum[x] *= pow2(127 - below(nt, x));
            l_run[nt][x] += sum[x];
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
      if (i + AHEAD < seg_b) {
        const int kn = k + AHEAD;
        ask(kn, __shfl_sync(0xffffffffu, (kn >> 5) == (k >> 5) ? page_cur : page_nxt, kn & 31));
      }
    }
    // ---- the next segment's first blocks are on their way while this one is written
    const Unit du = u;
    const int d_head = head, done = split ? seg_b - seg_a : 1;
    const bool whole = !split || done == du.tiles, begun = !whole && tile == 0;      // begun: the unit's first part is here
    const int last = worker + (begun ? (at + du.tiles - 1) / share : 0);             // who has its last
    at += done;
    const bool more = at < end;
    if (more) {
      tile = 0;
      if (++head == v.KH) {
        head = 0;
        do { ++z; unit_of<RT, QKV_BLOCK>(a, rts, z, u); } while (u.tiles == 0);
      }
      begin_segment();
    }
    // ---- a warp's rows are its own: straight to memory, 32 bytes of a row (bf16) at a time
    const int part = 2 * worker + (begun ? 1 : 0);
#pragma unroll
    for (int o = 4; o < 32; o <<= 1)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < 2; ++x) l_run[nt][x] += __shfl_xor_sync(0xffffffffu, l_run[nt][x], o);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int r = row0 + 8 * nt + 2 * rc + x, tok = row_t[nt][x];
        const float l = l_run[nt][x];
        if (tok < 0) continue;
        const float r_inv = pow2(R - below(nt, x) - 14);
        const float inv = whole ? (l == 0.f ? 0.f : r_inv / l) : r_inv;      // nothing seen: zero
        T* out = reinterpret_cast<T*>(a.out) + ((long long)(du.r0 + tok) * v.H + d_head * G + (du.f0 + r - tok * G)) * v.d + 2 * rg;
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
    if (begun && lane == 0 && (RS == 1 || warp == 0)) {      // a unit to merge: in any order, each by itself
      const int n = last - worker + 1;
      const bool many = n > MANY;
      const int i = atomicAdd(a.n_cuts + (many ? 1 : 0), 1);
      a.cuts[many ? a.max_cuts - 1 - i : i] = {du.r0, du.f0, du.nf, d_head, worker, n};
    }
    if (!more) break;
  }
  if (dead)
    for (unsigned s = 0; s < min(put, (unsigned)ST); ++s) mbar_wait_long(bars + 16 * s, ((put - 1 - s) / ST) & 1, LATE_CYCLES);
}

// Parts of the units that were cut, in the order of their shares: a warp for a row, or, with many parts, a CTA.  The last CTA empties
// the lists.  The kernel begins while the shares end; it goes through the motions once before it waits for them, so that its
// instructions are there (without that a row took 3 us, most of it fetching them).  That first pass takes a cut of constants, never one from
// the list: what stands there then is an earlier call's, whose shares with other rows lie beyond this call's parts.  Parts are read from L2, as the
// first pass has brought some of them before they were written.  rmax: rows of a unit at most; up: what their results are to be multiplied by
template <typename T, int P>
__global__ void __launch_bounds__(32 * MERGE_WARPS, P > 128 ? MERGE_CTAS - 1 : MERGE_CTAS) qkv_merge_kernel(QkvAttnArgs a, int RT, int rmax, float up) {
  constexpr int Y = P > 128 ? 2 : 1, IN = Y > 1 ? 4 : 8;      // parts asked for at a time
  static_assert(IN <= MANY, "eight warps on a row's parts know the maximum of all of them");
  __shared__ float4 s_sum[MERGE_WARPS][32 * Y];
  __shared__ float s_l[MERGE_WARPS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, G = a.v.H / a.v.KH;
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    int n_few = 1, n_all = 1;
    QkvCut o = {0, 0, rmax, 0, 0, 1};
    if (pass) {
      pdl_wait();
      o = a.cuts[min((blockIdx.x * MERGE_WARPS + warp) / rmax, a.max_cuts - 1)];       // asked for together with the lists' lengths
      n_few = a.n_cuts[0] * rmax;
      n_all = (n_few + MERGE_WARPS - 1) / MERGE_WARPS + a.n_cuts[1] * rmax;
    }
#pragma unroll 1
    for (int item = pass ? blockIdx.x : 0; item < n_all; item += gridDim.x) {
      const int few = item * MERGE_WARPS + warp, x0 = item - (n_few + MERGE_WARPS - 1) / MERGE_WARPS;
      const bool many = x0 >= 0;
      if (!many && few >= n_few) continue;
      if (many) o = a.cuts[a.max_cuts - 1 - x0 / rmax];
      else if (pass && item != blockIdx.x) o = a.cuts[few / rmax];
      const int r = many ? x0 % rmax : few % rmax;
      if (r >= min(RT, o.nf - o.f0)) continue;               // many: the same for all warps
      const int step = many ? MERGE_WARPS : 1, own = many ? warp : 0;        // this warp's parts: own, own + step, ..
      auto at = [&](int j) { return (long long)(2 * (o.first + j) + (j == 0 ? 1 : 0)) * RT + r; };
      float4 sum[Y];
      float m = -CUDART_INF_F, l = 0.f;
#pragma unroll
      for (int y = 0; y < Y; ++y) sum[y] = make_float4(0.f, 0.f, 0.f, 0.f);
      // the maximum of all parts comes first where they do not all come in one go: against a maximum of some of them, the weight of
      // another may be more than 32 bits hold
      if (o.n > IN)
        for (int j0 = lane; j0 < o.n; j0 += 256) {
          float x[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = __ldcg(a.part_ml + at(min(j0 + 32 * e, o.n - 1))).x;
#pragma unroll
          for (int e = 0; e < 8; ++e) m = fmaxf(m, x[e]);
        }
#pragma unroll 1
      for (int j0 = own; j0 < o.n; j0 += IN * step) {
        float4 x[IN][Y];
#pragma unroll
        for (int j = 0; j < IN; ++j)
#pragma unroll
          for (int y = 0; y < Y; ++y) {
            const int c = 4 * lane + 128 * y;
            x[j][y] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (c < P && j0 + j * step < o.n) x[j][y] = __ldcg(reinterpret_cast<const float4*>(a.part_o + at(j0 + j * step) * P + c));
          }
        float2 ml = make_float2(-CUDART_INF_F, 0.f);
        if (lane < IN && j0 + lane * step < o.n) ml = __ldcg(a.part_ml + at(j0 + lane * step));
        if (j0 == own) {
          m = fmaxf(m, ml.x);
#pragma unroll
          for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
        }
        // nothing seen: no weight; a sum without a maximum is no number
        const float w = ml.x == -CUDART_INF_F ? (ml.y == 0.f ? 0.f : CUDART_NAN_F) : ex2(ml.x - m);
        l += ml.y * w;
#pragma unroll
        for (int j = 0; j < IN; ++j) {
          const float f = __shfl_sync(0xffffffffu, w, j);
#pragma unroll
          for (int y = 0; y < Y; ++y)
            sum[y] = make_float4(fmaf(x[j][y].x, f, sum[y].x), fmaf(x[j][y].y, f, sum[y].y), fmaf(x[j][y].z, f, sum[y].z), fmaf(x[j][y].w, f, sum[y].w));
        }
      }
      l = warp_sum(l);
      if (many) {
#pragma unroll
        for (int y = 0; y < Y; ++y) s_sum[warp][lane + 32 * y] = sum[y];
        if (lane == 0) s_l[warp] = l;
        __syncthreads();
        l = 0.f;
#pragma unroll
        for (int y = 0; y < Y; ++y) sum[y] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < MERGE_WARPS; ++w) {
          l += s_l[w];
#pragma unroll
          for (int y = 0; y < Y; ++y) {
            const float4 x = s_sum[w][lane + 32 * y];
            sum[y] = make_float4(sum[y].x + x.x, sum[y].y + x.y, sum[y].z + x.z, sum[y].w + x.w);
          }
        }
        __syncthreads();
      }
      if ((many && warp) || !pass) continue;
      const int f = o.f0 + r;
      T* out = reinterpret_cast<T*>(a.out) + ((long long)(o.r0 + f / G) * a.v.H + o.head * G + f % G) * a.v.d;
#pragma unroll
      for (int y = 0; y < Y; ++y)
        if (4 * lane + 128 * y < a.v.d) store4(out + 4 * lane + 128 * y, scaled(sum[y], l == 0.f ? 0.f : up / l));
    }
  }
  __syncthreads();
  if (threadIdx.x == 0 && atomicAdd(a.n_cuts + 2, 1) == (int)gridDim.x - 1) { a.n_cuts[0] = 0; a.n_cuts[1] = 0; a.n_cuts[2] = 0; }
}

// Row blocks of an entry, and whether units are cut.  They are not where the cache has room for a few tiles only, as cutting them would save
// less than the merge costs; with more room they are, short ones too (the host does not know the lengths)
struct Launch {
  long long rts = 0, units = 0, tiles = 0;
  bool split = false;
  int32_t of(vn_qkv* c, const QkvAttnArgs& a, int RT, int blk, int uncut) {
    rts = ceil_div((long long)a.step.T * (a.v.H / a.v.KH), (long long)RT);
    units = rts * a.step.n_ent * a.v.KH;
    tiles = a.v.capacity() / blk;
    split = tiles > uncut;
    // what the kernels count in 32 bits: rows of an entry, units, tiles of a share and of the unit that it ends in
    VN_REQUIRE(c->ctx, (long long)a.step.T * (a.v.H / a.v.KH) <= (1ll << 30) && units < (1ll << 31) - THREADS && units * tiles / c->ctx->sm_count < (1ll << 30),
               "%d rows over %d positions are too many for one call: bring them in portions", a.step.M, a.v.capacity());
    return VN_OK;
  }
  // shares that there can be
  long long most(int least) const { return split ? ceil_div(units * tiles, (long long)least) : units; }
};

// No more CTAs than there can be rows to merge.  Four on an SM, eight parts of a row asked for at a time, against two and sixteen: 2 x 1000
// rows of a prompt 82 for 90 us in all, their merge 18 for 25.  Few of them with many parts each would all go to the SMs that are free
// first; they ask for memory that lets only two onto an SM (a sequence of 120000 positions: 59 us, 64 with four)
constexpr int MERGE_SPREAD = 76 << 10;
template <typename T, int P>
int32_t merge_ready(vn_qkv* c) {
  VN_CUDA(c->ctx, cudaFuncSetAttribute(qkv_merge_kernel<T, P>, cudaFuncAttributeMaxDynamicSharedMemorySize, MERGE_SPREAD));
  VN_CUDA(c->ctx, cudaFuncSetAttribute(qkv_merge_kernel<T, P>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
  return VN_OK;
}
template <typename T, int P>
int32_t merge(vn_qkv* c, const QkvAttnArgs& a, int RT, long long units, float up = 1.f) {
  const int rmax = (int)min((long long)RT, (long long)a.step.T * (a.v.H / a.v.KH)), sms = c->ctx->sm_count;
  const long long rows = units * rmax;
  VN_LAUNCH_PDL_LEVEL(c->ctx, 1, "qkv_merge_kernel", (qkv_merge_kernel<T, P>), dim3((unsigned)min((long long)sms * MERGE_CTAS, rows)), 32 * MERGE_WARPS, rows <= 2 * sms ? MERGE_SPREAD : 0, a, RT, rmax, up);
  return VN_OK;
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
    // the same division of the SMs' memory for both, so that neither has to wait for another one
    VN_CUDA(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
    if (int32_t st = merge_ready<T, P>(c)) return st;
    occ = min(n, C::CTAS);
  }
  Launch l;
  if (int32_t st = l.of(c, a, C::RT, QKV_BLOCK, UNCUT)) return st;
  const unsigned grid = (unsigned)min((long long)occ * ctx->sm_count, ceil_div(l.most(MIN_SHARE), (long long)C::RINGS));
  VN_LAUNCH_PDL_LEVEL(ctx, 1, "qkv_attn_kernel", kernel, grid, THREADS, C::SMEM, a, (int)l.rts, l.split);
  return l.split ? merge<T, P>(c, a, C::RT, l.units) : VN_OK;
}

template <int SCHEME, int P> int32_t launch_tc(vn_qkv* c, const QkvAttnArgs& a);      // qkv_attn_tc.cuh

template <int SCHEME>
int32_t pick(vn_qkv* c, const QkvAttnArgs& a) {
  // as few columns as hold the rows of an entry; from 17 rows on the warps split the rows
  const long long rows = (long long)a.step.T * (a.v.H / a.v.KH);
  if (c->dtype == VN_BF16 && rows > 16 && (a.v.P == 64 || a.v.P == 128)) return a.v.P == 64 ? launch_tc<SCHEME, 64>(c, a) : launch_tc<SCHEME, 128>(c, a);
#define GO(P, NT, RS) return c->dtype == VN_F32 ? launch<float, SCHEME, P, NT, RS>(c, a) : launch<bf16, SCHEME, P, NT, RS>(c, a)
#define GO2(P) do { if (rows <= 8) GO(P, 1, 1); else if (rows <= 16) GO(P, 2, 1); else GO(P, 2, 4); } while (0)
#define GO4(P) do { if (rows <= 8) GO(P, 1, 1); else if (rows <= 16) GO(P, 2, 1); else if (rows <= 64) GO(P, 2, 4); else GO(P, 4, 4); } while (0)
// (bf16 rows that are many have gone to tcgen05)
#define GOF(P) do { if (rows <= 8) GO(P, 1, 1); else if (rows <= 16) GO(P, 2, 1); else return rows <= 64 ? launch<float, SCHEME, P, 2, 4>(c, a) : launch<float, SCHEME, P, 4, 4>(c, a); } while (0)
  switch (a.v.P) {
    case 32: GO4(32);
    case 64: GOF(64);
    case 80: GO4(80);
    case 96: GO4(96);
    case 128: GOF(128);
    case 192: GO2(192);
    case 256: GO2(256);
    default: return vn_fail(c->ctx, VN_ERR_UNSUPPORTED, "pitch %d", a.v.P);
  }
#undef GOF
#undef GO4
#undef GO2
#undef GO
}

}  // namespace qkv_detail
