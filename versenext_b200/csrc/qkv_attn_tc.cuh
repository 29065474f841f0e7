// Attention over the 8-bit cache for many rows (prompts, trees): 128 rows of a unit on tcgen05.
//
// A CTA has thirteen warps.  Four convert: a page (64 positions) of codes, brought in by one bulk copy, becomes 16-bit floats in shared memory, keys
// and values alike with 128-byte rows of 64 channels and the 128-byte swizzle -- the layout of a K-major operand for the keys
// (S = Q K^T) and of an MN-major one for the values (O += P V).  One warp issues the products.  Eight do the soft-max, two threads for a row, 32
// columns each: S from TMEM, weights back to TMEM as the second product's A operand, results in TMEM (2 x 1000
// rows behind 1500 positions, 16 heads of 128 channels: 74 us; when it was made 73, against 76 with four warps of 64 columns a thread).  S of the next page is computed while the weights of this one are, and two
// CTAs share an SM.
//
// A row's reference maximum is moved only when a page's is more than 2^4 above it, so that the results in TMEM are seldom rescaled; weights
// are at most 2^4 then, and taken relative to R (at least the largest scale of the values that the row sees, with room of up to 2^2) times 2^11: a
// half holds them down to 2^-33 of the largest.  Rows of a warp whose R differ: as in qkv_attn.cuh.
#pragma once
#include "qkv_attn.cuh"

namespace qkv_detail {

constexpr int TC_ROWS = 128, TC_KEYS = KV_PAGE, TC_SOFT = 8, TC_THREADS = 32 * (TC_SOFT + 5), TC_CTAS = 2;      // TC_SOFT warps, four that convert, one that issues
constexpr float TC_PARTS = 16.f;                     // parts are kept that many times smaller: weights may be 2^4 then, and the largest values not
constexpr int TC_MIN_SHARE = 2, TC_UNCUT = 4;       // pages of a share at least; room up to which units are not cut

template <int P>
struct TcCfg {
  static constexpr int PANELS = P / 64, PAGE = 2 * QKV_BLOCK * (2 * P + 8), STAGES = P > 64 ? 2 : 3;
  static constexpr int Q = 0, K = Q + PANELS * TC_ROWS * 128, V = K + PANELS * TC_KEYS * 128, RAW = V + PANELS * TC_KEYS * 128, SCALES = RAW + STAGES * PAGE,
                       WEIGHTS = SCALES + 3 * 2 * TC_KEYS * 4, META = WEIGHTS + TC_SOFT * 32 * 4, FACTORS = META + 64, PAIRS = FACTORS + 2 * TC_ROWS * 4, BARS = PAIRS + 2 * 2 * TC_ROWS * 4, SLOT = BARS + 16 * 8, PLAN = SLOT + 16,
                       SMEM = PLAN + (THREADS + 8) * 8 + 1024;        // the first 1024: the swizzle's alignment
  static constexpr unsigned S_COL = 0, O_COL = 128;          // scores of even and odd pages, whose first half the weights take over; results
  static_assert(P % 64 == 0 && O_COL + P <= 256, "256 columns of TMEM for each of two CTAs");
  static_assert(TC_CTAS * TC_ROWS * P <= QKV_PART, "parts fit their place");
};

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_to_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(unsigned bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// both operands in shared memory
__device__ __forceinline__ void tc_mma_ss(unsigned d, unsigned long long a, unsigned long long b, unsigned idesc, bool add) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((unsigned)add) : "memory");
}
// A in TMEM: two neighbouring k of a row in every column
__device__ __forceinline__ void tc_mma_ts(unsigned d, unsigned a, unsigned long long b, unsigned idesc, bool add) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"((unsigned)add) : "memory");
}
// 128-byte swizzle, groups of eight 128-byte rows 1024 bytes apart; panels: bytes between panels of 64 along M or N (MN-major operands)
__device__ __forceinline__ unsigned long long tc_desc(unsigned addr, unsigned panels) {
  return (unsigned long long)((addr & 0x3ffffu) >> 4) | (unsigned long long)(panels >> 4) << 16 | 64ull << 32 | 1ull << 46 | 2ull << 61;
}
#define QKV_R32(x) "=r"((x)[0]), "=r"((x)[1]), "=r"((x)[2]), "=r"((x)[3]), "=r"((x)[4]), "=r"((x)[5]), "=r"((x)[6]), "=r"((x)[7]), "=r"((x)[8]), "=r"((x)[9]), "=r"((x)[10]), \
  "=r"((x)[11]), "=r"((x)[12]), "=r"((x)[13]), "=r"((x)[14]), "=r"((x)[15]), "=r"((x)[16]), "=r"((x)[17]), "=r"((x)[18]), "=r"((x)[19]), "=r"((x)[20]), "=r"((x)[21]), \
  "=r"((x)[22]), "=r"((x)[23]), "=r"((x)[24]), "=r"((x)[25]), "=r"((x)[26]), "=r"((x)[27]), "=r"((x)[28]), "=r"((x)[29]), "=r"((x)[30]), "=r"((x)[31])
#define QKV_I32(x) "r"((x)[0]), "r"((x)[1]), "r"((x)[2]), "r"((x)[3]), "r"((x)[4]), "r"((x)[5]), "r"((x)[6]), "r"((x)[7]), "r"((x)[8]), "r"((x)[9]), "r"((x)[10]), \
  "r"((x)[11]), "r"((x)[12]), "r"((x)[13]), "r"((x)[14]), "r"((x)[15]), "r"((x)[16]), "r"((x)[17]), "r"((x)[18]), "r"((x)[19]), "r"((x)[20]), "r"((x)[21]), \
  "r"((x)[22]), "r"((x)[23]), "r"((x)[24]), "r"((x)[25]), "r"((x)[26]), "r"((x)[27]), "r"((x)[28]), "r"((x)[29]), "r"((x)[30]), "r"((x)[31])
// 32 columns of the warp's 32 rows
__device__ __forceinline__ void tc_ld(unsigned at, unsigned* x) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
               "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];" : QKV_R32(x) : "r"(at));
}
__device__ __forceinline__ void tc_st(unsigned at, const unsigned* x) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
               "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::QKV_I32(x), "r"(at) : "memory");
}
__device__ __forceinline__ void tc_st16(unsigned at, const unsigned* x) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
               ::"r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(x[4]), "r"(x[5]), "r"(x[6]), "r"(x[7]), "r"(x[8]), "r"(x[9]), "r"(x[10]), "r"(x[11]), "r"(x[12]), "r"(x[13]), "r"(x[14]),
                 "r"(x[15]), "r"(at) : "memory");
}
#undef QKV_R32
#undef QKV_I32
// 32 bytes, a whole sector, of a row
__device__ __forceinline__ void store32(void* p, const unsigned* x) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(x[4]), "r"(x[5]), "r"(x[6]), "r"(x[7]) : "memory");
}
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 16 codes to 16-bit floats in two chunks of a panel's row; none: zeros
template <int SCHEME>
__device__ __forceinline__ void convert16(const unsigned char* from, unsigned char* row, int chunk, int turn, bool none) {
  uint4 u = *reinterpret_cast<const uint4*>(from);
  if (none) u = SCHEME == QKV_I8 ? make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u) : make_uint4(0u, 0u, 0u, 0u);
  uint4 x, y;
  halves_of<SCHEME, false, false>(u.x, x.x, x.y);
  halves_of<SCHEME, false, false>(u.y, x.z, x.w);
  halves_of<SCHEME, false, false>(u.z, y.x, y.y);
  halves_of<SCHEME, false, false>(u.w, y.z, y.w);
  *reinterpret_cast<uint4*>(row + ((chunk ^ turn) << 4)) = x;
  *reinterpret_cast<uint4*>(row + (((chunk + 1) ^ turn) << 4)) = y;
}

template <int SCHEME, int P>
__global__ void __launch_bounds__(TC_THREADS, TC_CTAS) qkv_attn_tc_kernel(QkvAttnArgs a, int rts, bool split) {
  pdl_trigger();
  using C = TcCfg<P>;
  constexpr int ST = C::STAGES, PANELS = C::PANELS, BLOCK = QKV_BLOCK * (2 * P + 8);
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - ((unsigned)__cvta_generic_to_shared(smem_raw) & 1023u)) & 1023u);
  const unsigned s_base = (unsigned)__cvta_generic_to_shared(smem);
  const QkvView& v = a.v;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, G = v.H / v.KH;
  enum { RAW_FULL = 0, K_READY = 4, V_READY, Q_READY, S_FULL, P_FULL = S_FULL + 2, PV_DONE = P_FULL + 2, ALL_DONE = PV_DONE + 2 };         // the last three: of even and odd pages, as their waiters may be a page late
  auto bar = [&](int i) { return s_base + C::BARS + 8 * i; };
  float* s_scales = reinterpret_cast<float*>(smem + C::SCALES);            // [3][keys | values][64]: page t + 1's are written while t - 1's may still be read
  float* s_rf = reinterpret_cast<float*>(smem + C::FACTORS);               // [2][rows] r of a segment's rows
  int* s_meta = reinterpret_cast<int*>(smem + C::META);                    // [3][4]: page there, largest exponent of values' scales of either half
  if (tid == 0) {
    for (int i = 0; i < ST; ++i) mbar_init(bar(RAW_FULL + i), 1);
    for (int i : {(int)K_READY, (int)V_READY, (int)Q_READY}) mbar_init(bar(i), 4);
    for (int i : {(int)P_FULL, (int)P_FULL + 1}) mbar_init(bar(i), TC_SOFT);
    for (int i : {(int)S_FULL, (int)S_FULL + 1, (int)PV_DONE, (int)PV_DONE + 1, (int)ALL_DONE}) mbar_init(bar(i), 1);
  }
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  pdl_wait();
  Unit u;
  Share sh;
  if (!find_share<TC_ROWS, TC_KEYS>(a, rts, split, TC_MIN_SHARE, blockIdx.x, gridDim.x, reinterpret_cast<long long*>(smem + C::PLAN), u, sh)) return;
  unsigned* s_slot = reinterpret_cast<unsigned*>(smem + C::SLOT);
  if (warp == TC_SOFT + 4) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s_base + C::SLOT), "r"(256u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const unsigned tmem = *s_slot;
  bool dead = false;                                         // a wait ran out: the results are no good, but everybody comes to the end
  auto wait = [&](int b, unsigned parity) {
    if (!mbar_try1(bar(b), parity) && !mbar_wait_long(bar(b), parity, dead ? LATE_CYCLES / 16 : WAIT_CYCLES)) { dead = true; v.status[2] = 1; }
  };
  auto wait_scores = [&](unsigned t) { wait(S_FULL + (t & 1), (t >> 1) & 1); };
  auto wait_results = [&](unsigned t) { wait(PV_DONE + (t & 1), (t >> 1) & 1); };
  unsigned n = 0;                                            // pages gone through, the same count for all roles
  int seg_a, seg_n, segs = 0;
  auto begin = [&]() {
    seg_a = u.tile0 + sh.tile;
    seg_n = split ? min(u.tiles - sh.tile, sh.end - sh.at) : u.tiles;
  };
  auto advance = [&]() {                                     // to the next segment; false: none
    sh.at += split ? seg_n : 1;
    if (sh.at >= sh.end) return false;
    sh.tile = 0;
    if (++sh.head == v.KH) {
      sh.head = 0;
      do { ++sh.z; unit_of<TC_ROWS, TC_KEYS>(a, rts, sh.z, u); } while (u.tiles == 0);
    }
    ++segs;
    return true;
  };

  if (warp == TC_SOFT + 4) {
    // ---- products: S of page i + 1 before O of page i
    if (lane == 0) {
      const unsigned idesc_s = 1u << 4 | (unsigned)(TC_KEYS >> 3) << 17 | (unsigned)(TC_ROWS >> 4) << 24;
      const unsigned idesc_o = 1u << 4 | 1u << 16 | (unsigned)(P >> 3) << 17 | (unsigned)(TC_ROWS >> 4) << 24;
      auto scores = [&](unsigned t) {
        wait(K_READY, t & 1);                                // the columns are free: O of page t - 2 was issued before
        tc_fence_after();
#pragma unroll
        for (int p = 0; p < PANELS; ++p) {
          const unsigned long long da = tc_desc(s_base + C::Q + p * TC_ROWS * 128, 16), db = tc_desc(s_base + C::K + p * TC_KEYS * 128, 16);
#pragma unroll
          for (int k = 0; k < 4; ++k) tc_mma_ss(tmem + C::S_COL + 64 * (t & 1), da + 2 * k, db + 2 * k, idesc_s, p || k);
        }
        tc_commit(bar(S_FULL + (t & 1)));
      };
      auto results = [&](unsigned t, bool add) {
        wait(V_READY, t & 1);
        wait(P_FULL + (t & 1), (t >> 1) & 1);
        tc_fence_after();
        const unsigned long long db = tc_desc(s_base + C::V, TC_KEYS * 128);
#pragma unroll
        for (int k = 0; k < TC_KEYS / 16; ++k) tc_mma_ts(tmem + C::O_COL, tmem + C::S_COL + 64 * (t & 1) + 8 * k, db + 128 * k, idesc_o, add || k);
        tc_commit(bar(PV_DONE + (t & 1)));
      };
      do {
        begin();
        wait(Q_READY, segs & 1);
        scores(n);
        for (int i = 1; i < seg_n; ++i) {
          scores(n + i);
          results(n + i - 1, i > 1);
        }
        results(n + seg_n - 1, seg_n > 1);
        n += seg_n;
      } while (advance());
      tc_commit(bar(ALL_DONE));                              // no product is under way when the memory is given back, whatever became of the waits
      if (!mbar_wait_long(bar(ALL_DONE), 0, WAIT_CYCLES)) v.status[2] = 1;
    }
  } else if (warp >= TC_SOFT) {
    // ---- queries and codes to halves: the keys of page i + 1 before the values of page i
    const int ct = tid - 32 * TC_SOFT, cw = warp - TC_SOFT, rg = lane >> 2, rc = lane & 3;
    unsigned asked = 0;                                      // pages asked for in all, by the lane that asks
    do {
      begin();
      // pages of the segment, 32 at a time: lane j has that of page first + j
      int pages = -1, next_pages = -1, first = 0;
      auto pages_of = [&](int i0) { return i0 + lane < seg_n ? v.page(u.slot, seg_a + i0 + lane) : -1; };
      pages = pages_of(0);
      next_pages = pages_of(32);
      auto page = [&](int i) { return __shfl_sync(0xffffffffu, i - first < 32 ? pages : next_pages, (i - first) & 31); };
      auto ask = [&](int i) {                                // by one warp: nobody reads the stage any more
        const int pg = page(i);
        if (lane || dead) return;
        const unsigned s = asked++ % ST;
        if (pg >= 0) fetch_block(s_base + C::RAW + s * C::PAGE, v.block(pg, sh.head, 0), C::PAGE, bar(RAW_FULL + s));
        else mbar_arrive1(bar(RAW_FULL + s));
      };
      if (cw == 0)
        for (int i = 0; i < min(ST, seg_n); ++i) ask(i);
      if (n) wait_scores(n - 1);                      // the queries and keys before these have been multiplied
      // a warp's 32 rows, 16 asked for at a time: four lanes a row, channels 16 k + 4 rc .. + 3 each
#pragma unroll 1
      for (int rb = 0; rb < 32; rb += 16) {
        uint2 x[2][P / 16];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int f = u.f0 + cw * 32 + rb + 8 * h + rg, t = f / G;
          const bool ok = f < u.nf;
          const bf16* q = reinterpret_cast<const bf16*>(a.q) + ((long long)(u.r0 + (ok ? t : 0)) * v.H + sh.head * G + (ok ? f - t * G : 0)) * v.d + 4 * rc;
#pragma unroll
          for (int k = 0; k < P / 16; ++k) x[h][k] = ok && 16 * k + 4 * rc < v.d ? *reinterpret_cast<const uint2*>(q + 16 * k) : make_uint2(0u, 0u);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = cw * 32 + rb + 8 * h + rg;
          unsigned top = 0;                                  // of the magnitudes' upper halves: all of a bf16
#pragma unroll
          for (int k = 0; k < P / 16; ++k) top = __vmaxu2(top, __vmaxu2(x[h][k].x & 0x7fff7fffu, x[h][k].y & 0x7fff7fffu));
          top = max(top >> 16, top & 0xffffu);
          top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
          const int e = min(max((int)(top >> 7), 27), 254);
          const float up = top >= 0x7f80u ? CUDART_NAN_F : pow2(267 - e);                  // a query that is not finite has no soft-max: NaN for all it sees
#pragma unroll
          for (int k = 0; k < P / 16; ++k) {
            auto two = [&](unsigned w) { return pack_f16(__uint_as_float(w << 16) * up, __uint_as_float(w & 0xffff0000u) * up); };
            const int c = 16 * k + 4 * rc;
            *reinterpret_cast<uint2*>(smem + C::Q + (c / 64) * TC_ROWS * 128 + r * 128 + (((c % 64 / 8) ^ (r & 7)) << 4) + (c % 8) * 2) = make_uint2(two(x[h][k].x), two(x[h][k].y));
          }
          if (rc == 0) s_rf[(segs & 1) * TC_ROWS + r] = fmaxf(a.scale * 1.4426950408889634f * pow2(e - 13), 1.17549435e-38f);
        }
      }
      fence_to_async();
      __syncwarp();
      if (lane == 0) mbar_arrive1(bar(Q_READY));
      auto convert = [&](int which, const unsigned char* raw, bool none) {
#pragma unroll
        for (int x = ct; x < TC_KEYS * (P / 16); x += 128) {
          const int r = x / (P / 16), c = x % (P / 16);
          const unsigned char* from = raw + (r / QKV_BLOCK) * BLOCK + (which * QKV_BLOCK + r % QKV_BLOCK) * P + ((c ^ qkv_turn(P / 16, r % QKV_BLOCK)) << 4);
          convert16<SCHEME>(from, smem + (which ? C::V : C::K) + (c / 4) * TC_KEYS * 128 + r * 128, c % 4 * 2, r & 7, none);
        }
        fence_to_async();
        __syncwarp();
        if (lane == 0) mbar_arrive1(bar(which ? V_READY : K_READY));
      };
      bool none = false;
#pragma unroll 1
      for (int i = 0; i <= seg_n; ++i) {
        const unsigned t = n + i;
        const bool none_before = none;
        if (i - first == 32) { first = i; pages = next_pages; next_pages = pages_of(i + 32); }
        if (i < seg_n) {                                     // keys of page i
          none = page(i) < 0;
          const unsigned char* raw = smem + C::RAW + t % ST * C::PAGE;
          if (i) wait_scores(t - 1);
          wait(RAW_FULL + t % ST, (t / ST) & 1);
          // scales, and the largest exponent of those of values that count: 32 positions for each of two warps
          if (ct < TC_KEYS) {
            const float* from = reinterpret_cast<const float*>(raw + (ct / QKV_BLOCK) * BLOCK + 2 * QKV_BLOCK * P) + ct % QKV_BLOCK;
            float* sc = s_scales + t % 3 * 2 * TC_KEYS;
            const int key = (seg_a + i) * TC_KEYS + ct;
            const float vs = none ? 0.f : from[QKV_BLOCK];
            sc[ct] = none ? 0.f : from[0];
            sc[TC_KEYS + ct] = vs;
            const unsigned b = __float_as_uint(vs);
            const bool counts = key >= u.lo && key < u.hi && b < 0x7f800000u;
            const unsigned top = __reduce_max_sync(0xffffffffu, counts ? b : 0u) >> 23;
            const int k0 = (seg_a + i) * TC_KEYS;
            unsigned shared = top;                           // of those that all rows see
            if (k0 < u.full_lo || k0 + TC_KEYS > u.full_hi) shared = __reduce_max_sync(0xffffffffu, counts && key >= u.full_lo && key < u.full_hi ? b : 0u) >> 23;
            if (lane == 0) s_meta[t % 3 * 4 + 1 + ct / 32] = (int)(shared << 8 | top);
            if (ct == 0) {
              s_meta[t % 3 * 4] = !none;
              if (none) v.status[0] = 1;
            }
          }
          convert(0, raw, none);
        }
        if (i) {                                             // values of the page before
          const unsigned t1 = t - 1;
          if (t1) wait_results(t1 - 1);
          convert(1, smem + C::RAW + t1 % ST * C::PAGE, none_before);
          __syncwarp();
          asm volatile("bar.sync 1, 128;" ::: "memory");     // nobody reads the stage any more
          if (cw == 0 && i - 1 + ST < seg_n) ask(i - 1 + ST);
        }
      }
      n += seg_n;
    } while (advance());
    if (dead)
      for (unsigned s = 0; s < min(asked, (unsigned)ST); ++s) mbar_wait_long(bar(RAW_FULL + s), ((asked - 1 - s) / ST) & 1, LATE_CYCLES);
  } else {
    // ---- soft-max: warps w and w + 4 have the two halves of the columns of rows 32 (w mod 4) ..
    const int half = warp >> 2, row = tid & 127;
    const unsigned lanes = tmem + ((unsigned)(warp % 4 * 32) << 16);
    float* s_w = reinterpret_cast<float*>(smem + C::WEIGHTS) + warp * 32;                  // the page's scales of values, relative to R
    float* s_pair = reinterpret_cast<float*>(smem + C::PAIRS);                             // [2][halves][rows], turn about
    unsigned turn = 0;
    auto exchange = [&](float x) {                           // the other half's
      float* p = s_pair + (turn++ & 1) * 2 * TC_ROWS;
      p[half * TC_ROWS + row] = x;
      tc_fence_before();
      __syncwarp();
      asm volatile("bar.sync %0, 64;" ::"r"(2 + warp % 4) : "memory");
      tc_fence_after();
      return p[(half ^ 1) * TC_ROWS + row];
    };
    do {
      begin();
      const int f = u.f0 + row, tok = f < u.nf ? f / G : -1;
      const int away = tok < 0 || a.window == 0 ? 0 : a.tree.behind(v, u.r0 + tok, tok);
      const unsigned long long seen = a.tree.seen && tok >= 0 ? a.tree.sees(u.r0 + tok, tok, a.window) : 0;
      float rf = 0.f, m = -CUDART_INF_F, l = 0.f;
      int R = 16, below = 0;                                 // the largest of the warp's rows, which scales are brought to; what the row's own is below it
      bool mixed = false;                                    // there are such rows
#pragma unroll 1
      for (int i = 0; i < seg_n; ++i) {
        const unsigned t = n + i;
        const float* sc = s_scales + t % 3 * 2 * TC_KEYS + 32 * half;
        const int* meta = s_meta + t % 3 * 4;
        wait_scores(t);                                      // and with them the scales, written before the product was issued
        __syncwarp();
        tc_fence_after();
        if (i == 0) rf = s_rf[(segs & 1) * TC_ROWS + row];
        const unsigned at_s = lanes + C::S_COL + 64 * (t & 1);
        float x[32];
        tc_ld(at_s + 32 * half, reinterpret_cast<unsigned*>(x));
        const int e = max(meta[1] & 255, meta[2] & 255), e_all = max(meta[1], meta[2]) >> 8;         // of the largest scale that some row, that all rows see
        const int k0 = (seg_a + i) * TC_KEYS;
        const bool full = meta[0] && k0 >= u.full_lo && k0 + TC_KEYS <= u.full_hi;
        unsigned see = ~0u;
        if (!full) {                                         // which of the positions the row sees, as bits
          see = 0;
          const int h0 = k0 + 32 * half;
          auto range = [&](int lo, int hi) {                 // positions lo .. hi - 1
            const int p = min(max(lo - h0, 0), 32), q = min(max(hi - h0, 0), 32);
            return p >= q ? 0u : (~0u >> (32 - (q - p))) << p;
          };
          if (tok >= 0 && meta[0]) {
            const int from = a.window > 0 ? max(0, u.len + away - a.window + 1) : 0;
            if (a.tree.seen) {
              const int off = u.len - h0;                    // where the new rows begin
              const unsigned long long rows = u.n >= 64 ? seen : seen & ((1ull << u.n) - 1);
              see = range(from, u.len) | (off >= 32 || off <= -64 ? 0u : off >= 0 ? (unsigned)(rows << off) : (unsigned)(rows >> -off));
            } else {
              see = range(from, u.len + tok + 1);
            }
            see &= range(0, u.hi);
          }
        }
        // where that is above R: for all rows the latter with its room, if that is enough for all, else row by row
        float f_r = 1.f;
        if (e > R && e_all >= e - 2 && !mixed) {
          const int to = min(e_all + 2, 254);
          f_r = pow2(127 + R - to);
          R = to;
        }
        s_w[lane] = sc[TC_KEYS + lane] * pow2(264 - R);
        if (__builtin_expect(e > R || mixed, 0)) {           // the same for both halves
          int e_own = e;
          if (!full) {
            unsigned most = 0;                               // of the scales that the row sees, numbers only
#pragma unroll 1
            for (int c = 0; c < 32; ++c) {
              const unsigned b = __float_as_uint(sc[TC_KEYS + c]);
              if (((see >> c) & 1) && b < 0x7f800000u) most = max(most, b);
            }
            e_own = (int)(max(most, __float_as_uint(exchange(__uint_as_float(most)))) >> 23);
          }
          const int was = R - below, own = e_own > was ? min(e_own + 2, 254) : was;
          R = __reduce_max_sync(0xffffffffu, own);
          below = min(R - own, BELOW);
          f_r = pow2(127 + was - (R - below));
          mixed = __any_sync(0xffffffffu, below != 0);
          __syncwarp();
          s_w[lane] = sc[TC_KEYS + lane] * pow2(264 - R);
        }
        tc_wait_ld();
#pragma unroll
        for (int c = 0; c < 32; c += 4) {
          const float4 k = *reinterpret_cast<const float4*>(sc + c);
          x[c] *= k.x; x[c + 1] *= k.y; x[c + 2] *= k.z; x[c + 3] *= k.w;
        }
        if (!full)
#pragma unroll
          for (int c = 0; c < 32; ++c)
            if (!((see >> c) & 1)) x[c] = -CUDART_INF_F;
        float mx[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
        for (int c = 4; c < 32; ++c) mx[c & 3] = fmaxf(mx[c & 3], x[c]);
        float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        top = fmaxf(top, exchange(top)) * rf;                // both halves come to the same
        float f_m = 1.f;
        if (top > m + 4.f || (m == -CUDART_INF_F && top > m)) {
          f_m = ex2(m - top);                                // from nothing: zero
          m = top;
          l *= f_m;
        }
        float base = m == -CUDART_INF_F ? 0.f : m;           // nothing seen yet: every weight becomes exp2(-inf) = 0
        if (__builtin_expect(mixed, 0)) base -= (float)below;
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
        unsigned pk[16];
        __syncwarp();                                        // s_w
#pragma unroll
        for (int c = 0; c < 32; c += 4) {
          const float4 w = *reinterpret_cast<const float4*>(s_w + c);
          float g[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const float p = ex2(fmaf(x[c + y], rf, -base));
            sum[y] += p;
            g[y] *= p;
            if (!full && x[c + y] == -CUDART_INF_F) g[y] = 0.f;                            // unseen: any scale, NaN too
          }
          pk[c / 2] = pack_f16(g[0], g[1]);
          pk[c / 2 + 1] = pack_f16(g[2], g[3]);
        }
        tc_st16(at_s + 16 * half, pk);                       // over the first half's scores, which that half has read: both have exchanged their maxima
        sum[0] = (sum[0] + sum[1]) + (sum[2] + sum[3]);
        if (__builtin_expect(mixed, 0)) sum[0] *= pow2(127 - below);
        l += sum[0];
        const float f_o = f_m * f_r;
        if (i && __any_sync(0xffffffffu, f_o != 1.f)) {      // the same for both halves
          wait_results(t - 1);
          __syncwarp();
          tc_fence_after();
#pragma unroll 1
          for (int c = half * (P / 2); c < (half + 1) * (P / 2); c += 32) {
            unsigned o[32];
            tc_ld(lanes + C::O_COL + c, o);
            tc_wait_ld();
#pragma unroll
            for (int y = 0; y < 32; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * f_o);
            tc_st(lanes + C::O_COL + c, o);
          }
        }
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive1(bar(P_FULL + (t & 1)));
      }
      n += seg_n;
      // ---- a row's results, half of the channels each
      l += exchange(l);
      wait_results(n - 1);
      __syncwarp();
      tc_fence_after();
      const bool whole = !split || seg_n == u.tiles, begun = !whole && sh.tile == 0;
      const int part = 2 * blockIdx.x + (begun ? 1 : 0);
      const float r_inv = pow2(R - below - 10), inv = whole ? (l == 0.f ? 0.f : r_inv / l) : r_inv * (1.f / TC_PARTS);
      bf16* out = reinterpret_cast<bf16*>(a.out) + ((long long)(u.r0 + max(tok, 0)) * v.H + sh.head * G + (f - max(tok, 0) * G)) * v.d;
      float* part_o = a.part_o + ((long long)part * TC_ROWS + row) * P;
      const bool wide = v.d % 16 == 0 && (reinterpret_cast<unsigned long long>(a.out) & 31) == 0;           // rows begin at whole sectors
#pragma unroll 1
      for (int c = half * (P / 2); c < (half + 1) * (P / 2); c += 32) {
        unsigned o[32];
        __syncwarp();
        tc_ld(lanes + C::O_COL + c, o);
        tc_wait_ld();
        if (tok >= 0) {
#pragma unroll
          for (int y = 0; y < 32; ++y) o[y] = __float_as_uint(l == 0.f ? 0.f : __uint_as_float(o[y]) * inv);     // nothing seen: zero
          if (!whole) {
#pragma unroll
            for (int y = 0; y < 32; y += 8) store32(part_o + c + y, o + y);
          } else {
            unsigned h[16];
#pragma unroll
            for (int y = 0; y < 16; ++y) {
              const __nv_bfloat162 w = __floats2bfloat162_rn(__uint_as_float(o[2 * y]), __uint_as_float(o[2 * y + 1]));
              h[y] = *reinterpret_cast<const unsigned*>(&w);
            }
            if (wide) {
#pragma unroll
              for (int y = 0; y < 32; y += 16)
                if (c + y < v.d) store32(out + c + y, h + y / 2);
            } else {
#pragma unroll
              for (int y = 0; y < 32; y += 8)
                if (c + y < v.d) {
                  *reinterpret_cast<uint2*>(out + c + y) = make_uint2(h[y / 2], h[y / 2 + 1]);
                  *reinterpret_cast<uint2*>(out + c + y + 4) = make_uint2(h[y / 2 + 2], h[y / 2 + 3]);
                }
            }
          }
        }
      }
      if (!whole && tok >= 0 && half == 0) a.part_ml[part * TC_ROWS + row] = make_float2(m, l);
      if (begun && tid == 0) {                               // a unit to merge: in any order, each by itself
        const int cnt = (sh.at + u.tiles - 1) / sh.share + 1;
        const bool many = cnt > MANY;
        const int at = atomicAdd(a.n_cuts + (many ? 1 : 0), 1);
        a.cuts[many ? a.max_cuts - 1 - at : at] = {u.r0, u.f0, u.nf, sh.head, (int)blockIdx.x, cnt};
      }
    } while (advance());
  }
  tc_fence_before();
  __syncthreads();
  __syncwarp();
  if (warp == TC_SOFT + 4) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(256u) : "memory");
}

template <int SCHEME, int P>
int32_t launch_tc(vn_qkv* c, const QkvAttnArgs& a) {
  using C = TcCfg<P>;
  vn_ctx* ctx = c->ctx;
  auto kernel = qkv_attn_tc_kernel<SCHEME, P>;
  static bool ready[64] = {};
  if (!ready[ctx->device & 63]) {
    VN_CUDA(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    VN_CUDA(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
    if (int32_t st = merge_ready<bf16, P>(c)) return st;
    ready[ctx->device & 63] = true;
  }
  Launch l;
  if (int32_t st = l.of(c, a, TC_ROWS, TC_KEYS, TC_UNCUT)) return st;
  const unsigned grid = (unsigned)min((long long)TC_CTAS * ctx->sm_count, l.most(TC_MIN_SHARE));
  VN_LAUNCH_PDL_LEVEL(ctx, 1, "qkv_attn_tc_kernel", kernel, grid, TC_THREADS, C::SMEM, a, (int)l.rts, l.split);
  return l.split ? merge<bf16, P>(c, a, TC_ROWS, l.units, TC_PARTS) : VN_OK;
}

}  // namespace qkv_detail
