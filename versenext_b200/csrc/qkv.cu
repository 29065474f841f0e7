// The paged 8-bit cache's entry points and the kernels that write, read and keep positions; attention is in qkv_attn.cuh.
#include <string.h>

#include <algorithm>
#include <new>

#include "qkv_attn.cuh"

namespace {

using bf16 = __nv_bfloat16;

struct AppendArgs {
  QkvView v;
  QkvStep step;
  QkvTree tree;
  const void* x = nullptr;             // rows [H queries |] KH keys | KH values
  void* q = nullptr;                   // [M, H, d]
  long long ld = 0;
  int off = 0, H = 0;                  // H = 0: the rows hold no queries
  const float *qn = nullptr, *kn = nullptr, *cs = nullptr, *sn = nullptr;
  float eps = 0.f;
  int pairs = 0, interleaved = 0, rope_rows = 0;
  int vec = 0, vec_norm = 0, vec_rope = 0;            // rows, norms' weights, rotation in whole quads
};

template <typename T> __device__ __forceinline__ void put_quad(T* p, float4 v, bool vec) {
  if (vec) { store4(p, v); return; }
  p[0] = from_f<T>(v.x); p[1] = from_f<T>(v.y); p[2] = from_f<T>(v.z); p[3] = from_f<T>(v.w);
}

// x / s to nearest: Markstein's correction (IBM J. Res. Dev. 34, 1990) of the product with 1 / s by its remainder, which is exact while it is
// a normal number; so small heads are made larger by a power of two first
struct Quotient {
  float up, s, r;
  __device__ __forceinline__ explicit Quotient(float scale) : up(scale < 1e-24f ? 1.8446744e19f : 1.f), s(scale * up), r(1.f / s) {}
  __device__ __forceinline__ float of(float x) const {
    const float v = x * up, y = v * r;
    return fmaf(fmaf(-y, s, v), r, y);
  }
};

// four codes of a head, x / scale to nearest even
template <int SCHEME> __device__ __forceinline__ unsigned codes_of(float4 x, const Quotient& q) {
  const float4 y = make_float4(q.of(x.x), q.of(x.y), q.of(x.z), q.of(x.w));
  if (SCHEME == QKV_I8) {
    // |y| is below 127.5: the sum with 1.5 2^23 is rounded to a whole number, whose low byte, plus 128, is the code
    auto c = [](float v) { return __float_as_uint(fminf(fmaxf(v, -127.f), 127.f) + 12582912.f); };
    return __byte_perm(__byte_perm(c(y.x), c(y.y), 0x0040), __byte_perm(c(y.z), c(y.w), 0x0040), 0x5410) ^ 0x80808080u;
  }
  unsigned short lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(y.y), "f"(y.x));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(y.w), "f"(y.z));
  return (unsigned)hi << 16 | lo;
}

// eight neighbouring channels of a row, as they stand in memory; whole: in 16-byte pieces
template <typename T> struct Eight;
template <> struct Eight<float> {
  float v[8];
  __device__ __forceinline__ void load(const float* p, bool whole) {
    if (whole) {
      const float4 x = load4(p), y = load4(p + 4);
      v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w; v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = p[e];
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = v[e];
  }
};
template <> struct Eight<bf16> {
  uint4 u;
  __device__ __forceinline__ void load(const bf16* p, bool whole) {
    if (whole) { u = *reinterpret_cast<const uint4*>(p); return; }
    const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
    u = make_uint4(h[0] | (unsigned)h[1] << 16, h[2] | (unsigned)h[3] << 16, h[4] | (unsigned)h[5] << 16, h[6] | (unsigned)h[7] << 16);
  }
  __device__ __forceinline__ void zero() { u = make_uint4(0u, 0u, 0u, 0u); }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) { x[2 * e] = __uint_as_float(w[e] << 16); x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u); }
  }
};
__device__ __forceinline__ void put_eight(float* p, const float (&x)[8], bool whole) {
  put_quad(p, make_float4(x[0], x[1], x[2], x[3]), whole);
  put_quad(p + 4, make_float4(x[4], x[5], x[6], x[7]), whole);
}
__device__ __forceinline__ void put_eight(bf16* p, const float (&x)[8], bool whole) {
  if (!whole) {
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = __float2bfloat16_rn(x[e]);
    return;
  }
  const __nv_bfloat162 h[4] = {__floats2bfloat162_rn(x[0], x[1]), __floats2bfloat162_rn(x[2], x[3]), __floats2bfloat162_rn(x[4], x[5]), __floats2bfloat162_rn(x[6], x[7])};
  *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(h);
}

// A warp takes `per` tasks of a row, four asked for at a time: a task is 32 / L neighbouring heads, whose lanes hold eight channels each.
// Heads pass through shared memory only for half-split rotation, where a channel meets the one `pairs` further on.  For many
// rows it is bound by instructions (rotation, maxima, quotients: two thirds of the issue slots) and by waits for the row, its entry, length and
// page (a prompt of 8000 rows of 2048 values takes 37 us with events around it, 48 with four channels a lane); for few, by the
// chain entry, length, page, store (the row's values are asked for first).  grid ceil(M ceil(tasks / per) / 8), block 256
template <typename T, int SCHEME, int L>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 4 : 2) qkv_append_kernel(AppendArgs a, int tasks, int per) {
  constexpr int HPW = 32 / L, IN = 4;
  __shared__ __align__(16) float s_head[8][HPW][8 * L];
  const int lane = threadIdx.x & 31, c = lane % L * 8, sub = lane / L, warp = threadIdx.x >> 5;
  const int units = a.H + 2 * a.v.KH, d = a.v.d, P = a.v.P, slices = (tasks + per - 1) / per;
  const unsigned item = blockIdx.x * 8u + warp;
  pdl_wait();
  const int row = (int)(item / (unsigned)slices), first = (int)(item % (unsigned)slices) * per, last = min(tasks, first + per);
  if (row >= a.step.M) return;
  const T* xr = reinterpret_cast<const T*>(a.x) + row * a.ld;
  Eight<T> x[IN];
  auto ask = [&](int task) {
#pragma unroll
    for (int k = 0; k < IN; ++k) {
      const int unit = (task + k) * HPW + sub;
      if (task + k < last && unit < units && c < d) x[k].load(xr + unit * d + c, a.vec); else x[k].zero();
    }
  };
  ask(first);
  int slot, i, n;
  if (!a.step.row(a.v, row, &slot, &i, &n)) return;
  // the length and the offset, at most the capacity: then 32 bits hold the position, and, unsigned, one that there is no room for
  const int len = a.v.len(slot), begin = len + min(a.off, a.v.capacity() - len);
  const unsigned pos = (unsigned)begin + (unsigned)i;
  const int away = a.tree.away(row, i), turn = min(max(begin + min(away, (1 << 30) - 1), 0), a.rope_rows - 1);
  const int page = pos < (unsigned)a.v.capacity() ? a.v.page(slot, pos / KV_PAGE) : -1, at = pos % QKV_BLOCK;
  unsigned char* base = a.v.block(max(page, 0), 0, pos % KV_PAGE / QKV_BLOCK);
  const int to = at * P + (((c >> 4) ^ qkv_turn(P / 16, at)) << 4) + (c & 15), head_bytes = 2 * a.v.block_bytes(), np = a.pairs;
  // what the channels are turned by: half-split, those of the two halves by the same angles
  float cs[8], sn[8];
  const bool turned = c < 2 * np;
  if (np && page >= 0 && turn - begin != away) a.v.status[1] = 1;      // no such angles: those of the nearest position
  if (turned) {
    const float *pc = a.cs + (long long)turn * np, *ps = a.sn + (long long)turn * np;
    if (a.vec_rope && !a.interleaved) {
      const int p = c < np ? c : c - np;
      const float4 u = load4(pc + p), v = load4(pc + p + 4), w = load4(ps + p), y = load4(ps + p + 4);
      cs[0] = u.x; cs[1] = u.y; cs[2] = u.z; cs[3] = u.w; cs[4] = v.x; cs[5] = v.y; cs[6] = v.z; cs[7] = v.w;
      sn[0] = w.x; sn[1] = w.y; sn[2] = w.z; sn[3] = w.w; sn[4] = y.x; sn[5] = y.y; sn[6] = y.z; sn[7] = y.w;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool in = c + e < 2 * np;
        const int p = !in ? 0 : a.interleaved ? (c + e) / 2 : c + e < np ? c + e : c + e - np;
        cs[e] = in ? pc[p] : 1.f;
        sn[e] = in ? ps[p] : 0.f;
      }
    }
    if (!a.interleaved)                                      // the sign that the other half's values enter with
#pragma unroll
      for (int e = 0; e < 8; ++e) sn[e] = c + e < np ? -sn[e] : sn[e];
  }
  float* s = s_head[warp][sub];
#pragma unroll 1
  for (int task = first; task < last; task += IN) {
    if (task != first) ask(task);
#pragma unroll
    for (int k = 0; k < IN; ++k) {
      if (task + k >= last) break;
      const int unit = (task + k) * HPW + sub;
      const bool live = unit < units, is_q = unit < a.H, is_v = unit >= a.H + a.v.KH;
      float v[8];
      x[k].get(v);
      if (a.qn || a.kn) {
        const float* w = is_v || !live ? nullptr : is_q ? a.qn : a.kn;
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(v[e], v[e], ss);
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (w && c < d) {
          const float r = 1.f / sqrtf(ss / (float)d + a.eps);
          Eight<float> g;
          g.load(w + c, a.vec_norm);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = v[e] * r * g.v[e];
        }
      }
      if (np && a.interleaved) {
        if (!is_v && turned)
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            const float y = v[e] * cs[e] - v[e + 1] * sn[e], z = v[e + 1] * cs[e] + v[e] * sn[e];
            v[e] = y; v[e + 1] = z;
          }
      } else if (np && (task + k) * HPW < a.H + a.v.KH) {    // a task with queries or keys
        __syncwarp();
        put_eight(s + c, v, true);
        __syncwarp();
        if (!is_v && turned) {
          float t[8];
          if (a.vec_rope) {
            Eight<float> g;
            g.load(s + (c < np ? c + np : c - np), true);
            g.get(t);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) t[e] = c + e < np ? s[c + e + np] : c + e < 2 * np ? s[c + e - np] : 0.f;
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = v[e] * cs[e] + t[e] * sn[e];
        }
      }
      if (live && is_q && c < d) put_eight(reinterpret_cast<T*>(a.q) + ((long long)row * a.H + unit) * d + c, v, a.vec);
      if ((task + k + 1) * HPW <= a.H) continue;             // queries only
      // ---- a head of the cache
      unsigned top = 0;                                      // magnitudes as bits: what is not finite is above all others
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (!live || is_q) continue;
      if (page < 0) { a.v.status[0] = 1; continue; }
      const bool bad = top >= 0x7f800000u;
      const float scale = fmaxf((top ? __uint_as_float(top) : 1.f) / (SCHEME == QKV_I8 ? 127.f : 448.f), QKV_SCALE_MIN);
      const Quotient by(scale);
      unsigned char* b = base + (long long)(unit - a.H - (is_v ? a.v.KH : 0)) * head_bytes;
      if (c < P) {
        uint2 q = make_uint2(SCHEME == QKV_I8 ? 0x80808080u : 0u, SCHEME == QKV_I8 ? 0x80808080u : 0u);
        if (c < d && !bad) q = make_uint2(codes_of<SCHEME>(make_float4(v[0], v[1], v[2], v[3]), by), codes_of<SCHEME>(make_float4(v[4], v[5], v[6], v[7]), by));
        *reinterpret_cast<uint2*>(b + (is_v ? QKV_BLOCK * P : 0) + to) = q;
      }
      if (c == 0) reinterpret_cast<float*>(b + 2 * QKV_BLOCK * P)[(is_v ? QKV_BLOCK : 0) + at] = bad ? CUDART_NAN_F : scale;
    }
  }
}

// A warp takes RB neighbouring rows of 32 pieces of 16 bytes of results (C channels of a head), keys and values, all asked for before any is
// converted; its first lanes find the rows' blocks (entry, length, page: three loads one after another, which other warps fill).
// Bound by the bytes of codes and results.  grid ceil(ceil(M / RB) slices / 8), block 256
template <typename O, int SCHEME, int RB>
__global__ void __launch_bounds__(256) qkv_read_kernel(QkvView v, QkvStep step, int start, int off, O* __restrict__ k, O* __restrict__ vals, int vec, int slices) {
  constexpr int C = 16 / sizeof(O);
  const unsigned item = blockIdx.x * 8u + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31, per = v.d / C, row0 = (int)(item / (unsigned)slices) * RB, it = (int)(item % (unsigned)slices) * 32 + lane;
  if (row0 >= step.M) return;
  pdl_wait();
  int own_at = -1;                                           // of row row0 + lane: place in its block, -1: no row
  long long own_block = -1;                                  // of head 0, -1: none
  if (lane < RB && row0 + lane < step.M) {
    int slot, i, n;
    if (step.row(v, row0 + lane, &slot, &i, &n)) {
      const long long pos = (start >= 0 ? start : (long long)v.len(slot) + off - (start == -2 ? n : 0)) + i;     // may pass 32 bits where there is no room
      const int page = pos >= 0 && pos < v.capacity() ? v.page(slot, (int)(pos / KV_PAGE)) : -1;
      own_at = page < 0 ? 0 : (int)(pos % QKV_BLOCK);
      if (page < 0) v.status[0] = 1;
      else own_block = ((long long)page * v.KH * 2 + (int)(pos % KV_PAGE) / QKV_BLOCK) * v.block_bytes();
    }
  }
  const int head = it / per, c = it % per * C, CH = v.P / 16, scales = 2 * QKV_BLOCK * v.P;
  const bool reads = it < v.KH * per;
  const unsigned char* pool = v.pool + (long long)head * 2 * v.block_bytes();
  uint2 u[RB][2];
  float sc[RB][2];
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    const long long block = __shfl_sync(0xffffffffu, own_block, r);
    const int at = __shfl_sync(0xffffffffu, own_at, r);
#pragma unroll
    for (int w = 0; w < 2; ++w) { u[r][w] = make_uint2(0u, 0u); sc[r][w] = 0.f; }          // no page: zeros
    if (!reads || block < 0) continue;
    const unsigned char* b = pool + block;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const unsigned char* p = b + (w * QKV_BLOCK + at) * v.P + (((c >> 4) ^ qkv_turn(CH, at)) << 4) + (c & 15);
      if (C == 8) u[r][w] = __ldcs(reinterpret_cast<const uint2*>(p));
      else u[r][w].x = __ldcs(reinterpret_cast<const unsigned*>(p));
      sc[r][w] = reinterpret_cast<const float*>(b + scales)[w * QKV_BLOCK + at];
    }
  }
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    if (__shfl_sync(0xffffffffu, own_at, r) < 0 || !reads) continue;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      O* out = (w ? vals : k) + ((long long)(row0 + r) * v.KH + head) * v.d + c;
      float y[8];
#pragma unroll
      for (int h = 0; h < C / 4; ++h) {
        const unsigned q = h ? u[r][w].y : u[r][w].x;
        float4 x;
        if (SCHEME == QKV_I8) {                              // a byte under the exponent of 2^23, less 2^23 + 128
          const float over = 8388736.f;
          x = make_float4(__uint_as_float(__byte_perm(q, 0x4b000000u, 0x7440)) - over, __uint_as_float(__byte_perm(q, 0x4b000000u, 0x7441)) - over,
                          __uint_as_float(__byte_perm(q, 0x4b000000u, 0x7442)) - over, __uint_as_float(__byte_perm(q, 0x4b000000u, 0x7443)) - over);
        } else {
          unsigned lo, hi;
          asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(lo) : "h"((unsigned short)q));
          asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(hi) : "h"((unsigned short)(q >> 16)));
          const float2 p0 = __half22float2(*reinterpret_cast<const __half2*>(&lo)), p1 = __half22float2(*reinterpret_cast<const __half2*>(&hi));
          x = make_float4(p0.x, p0.y, p1.x, p1.y);
        }
        x = scaled(x, sc[r][w]);
        y[4 * h] = x.x; y[4 * h + 1] = x.y; y[4 * h + 2] = x.z; y[4 * h + 3] = x.w;
      }
      if constexpr (C == 8) put_eight(out, y, vec);
      else put_quad(out, make_float4(y[0], y[1], y[2], y[3]), vec);
    }
  }
}

// A block per (sequence, head): the kept positions are read whole before any is written, so that they may overlap in any
// order; the block that finishes a sequence last moves its length.  grid (KH, sequences)
__global__ void __launch_bounds__(256) qkv_commit_kernel(QkvView v, int n_new, const int* __restrict__ keep, int stride, const int* __restrict__ n_keep,
                                                         int keep_add, int* __restrict__ tickets) {
  __shared__ __align__(16) unsigned char s_codes[QKV_MAX_DRAFT][2][256];
  __shared__ float s_scale[QKV_MAX_DRAFT][2];
  const int head = blockIdx.x, slot = blockIdx.y, tid = threadIdx.x, P = v.P, CH = P / 16;
  pdl_wait();
  const int len = v.len(slot);
  int n = n_keep[slot] + keep_add;
  if (n < 0 || n > n_new || n > v.capacity() - len) {
    if (tid == 0) v.status[1] = 1;
    n = min(max(n, 0), min(n_new, v.capacity() - len));
  }
  auto move = [&](bool in) {
    for (int j = tid / 32; j < n; j += 8) {
      const int from = keep[(long long)slot * stride + j];
      if (from == j) continue;
      if (from < 0 || from >= n_new) { if (tid % 32 == 0) v.status[1] = 1; continue; }
      const int src = len + from, dst = len + j, pos = in ? src : dst;
      const int page_src = src < v.capacity() ? v.page(slot, src / KV_PAGE) : -1, page_dst = v.page(slot, dst / KV_PAGE);
      if (page_src < 0 || page_dst < 0) { if (tid % 32 == 0) v.status[0] = 1; continue; }
      const int page = in ? page_src : page_dst;
      unsigned char* b = v.block(page, head, pos % KV_PAGE / QKV_BLOCK);
      const int at = pos % QKV_BLOCK, t = qkv_turn(CH, at);
      for (int x = tid % 32; x < 2 * CH; x += 32) {
        const int which = x / CH, c = x % CH;
        uint4* g = reinterpret_cast<uint4*>(b + (which * QKV_BLOCK + at) * P + ((c ^ t) << 4));
        uint4* sh = reinterpret_cast<uint4*>(&s_codes[j][which][c << 4]);
        if (in) *sh = *g; else *g = *sh;
      }
      if (tid % 32 < 2) {
        float* g = reinterpret_cast<float*>(b + 2 * QKV_BLOCK * P) + (tid % 32) * QKV_BLOCK + at;
        if (in) s_scale[j][tid % 32] = *g; else *g = s_scale[j][tid % 32];
      }
    }
  };
  if (keep) {
    move(true);
    __syncthreads();
    move(false);
  }
  __syncthreads();
  if (tid == 0) {
    __threadfence();
    if (atomicAdd(&tickets[slot], 1) == (int)gridDim.x - 1) {
      tickets[slot] = 0;
      v.lens[slot] = len + n;
    }
  }
}

__global__ void set_lengths_kernel(QkvView v, const int* __restrict__ from) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  pdl_wait();
  if (i >= v.max_batch) return;
  const int n = from[i];
  if (n < 0 || n > v.capacity()) v.status[1] = 1;
  v.lens[i] = min(max(n, 0), v.capacity());
}

// a wait as the attention kernels', for what never comes
__global__ void qkv_wait_probe_kernel(int* status, unsigned long long limit, long long* waited) {
  __shared__ __align__(8) unsigned long long bar;
  const unsigned b = (unsigned)__cvta_generic_to_shared(&bar);
  qkv_detail::mbar_init(b, 1);
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  const long long t0 = clock64();
  if (!qkv_detail::mbar_try1(b, 0) && !qkv_detail::mbar_wait_long(b, 0, limit)) status[2] = 1;
  *waited = clock64() - t0;
}

// layout of vn_ctx::qkv_parts: two parts for every share (CTA, or warp with a quarter of the rows) that the attention kernel may have
struct Parts { size_t ml, cuts, n_cuts, bytes; int max_cuts; };
Parts parts_of(const vn_ctx* ctx) {
  Parts p;
  p.ml = (size_t)2 * ctx->sm_count * QKV_PART * sizeof(float);
  p.cuts = p.ml + (size_t)2 * ctx->sm_count * QKV_MAX_CTAS * 128 * sizeof(float2);
  p.max_cuts = ctx->sm_count * QKV_MAX_CTAS * 4;
  p.n_cuts = p.cuts + (size_t)p.max_cuts * sizeof(QkvCut);
  p.bytes = p.n_cuts + 3 * sizeof(int);
  return p;
}

bool aligned(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

int32_t step_of(vn_qkv* c, int32_t n_ent, const int32_t* ents, const int32_t* row_ent, int32_t T, int32_t M, QkvStep* s) {
  VN_REQUIRE(c->ctx, n_ent >= 0 && T >= 0 && M >= 0, "negative sizes of a step");
  VN_REQUIRE(c->ctx, (ents == nullptr) == (row_ent == nullptr), "a ragged step has both tables");
  VN_REQUIRE(c->ctx, aligned(ents, 16), "the table of entries is not aligned to 16 bytes");
  VN_REQUIRE(c->ctx, ents || n_ent <= c->v.max_batch, "%d sequences in a cache of %d", n_ent, c->v.max_batch);
  VN_REQUIRE(c->ctx, ents || M == (long long)n_ent * T, "%d rows are not %d entries of %d", M, n_ent, T);
  s->ents = (const int4*)ents; s->row_ent = row_ent;
  s->n_ent = n_ent; s->T = T; s->M = M;
  return VN_OK;
}

#define VN_CHECK_QKV(c)                                                   \
  do {                                                                    \
    if (!(c)) return vn_fail(nullptr, VN_ERR_INVALID, "null cache");      \
    VN_CHECK_CTX((c)->ctx);                                               \
  } while (0)

}  // namespace

extern "C" {

int32_t vn_qkv_create(vn_ctx* ctx, int32_t max_batch, int32_t max_seq, int32_t n_head, int32_t n_kv_head, int32_t head_dim, const char* scheme, int32_t dtype,
                      int32_t pages, vn_qkv** out) {
  VN_CHECK_CTX(ctx);
  VN_REQUIRE(ctx, out && scheme, "null argument");
  *out = nullptr;
  const int kind = !strcmp(scheme, "int8") ? QKV_I8 : !strcmp(scheme, "fp8") ? QKV_E4M3 : -1;
  VN_REQUIRE(ctx, kind >= 0, "unknown scheme '%s' (int8, fp8)", scheme);
  VN_REQUIRE(ctx, dtype == VN_F32 || dtype == VN_BF16, "rows are float32 or bf16");
  VN_REQUIRE(ctx, max_batch > 0 && max_batch <= 65535, "max_batch %d outside 1 .. 65535", max_batch);
  VN_REQUIRE(ctx, max_seq > 0 && max_seq <= (1 << 30), "max_seq %d outside 1 .. 2^30", max_seq);
  VN_REQUIRE(ctx, n_kv_head > 0 && n_head > 0 && n_head % n_kv_head == 0 && n_head <= 65535, "%d query heads over %d key/value heads", n_head, n_kv_head);
  VN_REQUIRE(ctx, head_dim >= 8 && head_dim <= 256 && head_dim % 8 == 0, "head_dim %d: a multiple of 8 up to 256 is needed", head_dim);
  const long long max_pages = ceil_div((long long)max_seq, (long long)KV_PAGE), all = max_pages * max_batch;
  VN_REQUIRE(ctx, pages >= 0 && (pages || all <= (1ll << 30)), "%d pages", pages);
  vn_qkv* c = new (std::nothrow) vn_qkv();
  if (!c) return vn_fail(ctx, VN_ERR_OOM, "out of host memory");
  c->ctx = ctx; c->dtype = dtype;
  QkvView& v = c->v;
  v.max_batch = max_batch; v.max_pages = (int)max_pages; v.n_pages = pages ? pages : (int)all;
  v.H = n_head; v.KH = n_kv_head; v.d = head_dim; v.scheme = kind;
  for (int p : {32, 64, 80, 96, 128, 192, 256})
    if (!v.P && head_dim <= p) v.P = p;
  const size_t pool = (size_t)v.n_pages * v.KH * 2 * v.block_bytes();
  int32_t st = VN_OK;
  auto get = [&](void** p, size_t bytes) {
    cudaError_t e = cudaMalloc(p, bytes);
    if (e == cudaSuccess) e = cudaMemsetAsync(*p, 0, bytes, ctx->stream);
    if (e != cudaSuccess) {
      cudaGetLastError();
      st = vn_fail(ctx, e == cudaErrorMemoryAllocation ? VN_ERR_OOM : VN_ERR_CUDA, "cache of %zu bytes: %s", bytes, cudaGetErrorString(e));
    }
    return e == cudaSuccess;
  };
  if (get((void**)&v.pool, pool) && get((void**)&c->table, (size_t)all * sizeof(int)) && get((void**)&v.lens, (size_t)max_batch * sizeof(int)) &&
      get((void**)&v.status, 3 * sizeof(int)) && get((void**)&c->tickets, (size_t)max_batch * sizeof(int)) &&
      (ctx->qkv_parts || get(&ctx->qkv_parts, parts_of(ctx).bytes))) {
    v.table = c->table;
    std::vector<int> t;
    try { t.resize((size_t)all); } catch (...) { vn_qkv_destroy(c); return vn_fail(ctx, VN_ERR_OOM, "out of host memory"); }
    for (long long i = 0; i < all; ++i) t[i] = pages ? -1 : (int)i;
    cudaError_t e = cudaMemcpyAsync(c->table, t.data(), (size_t)all * sizeof(int), cudaMemcpyHostToDevice, ctx->stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize(ctx->stream);
    if (e != cudaSuccess) st = vn_fail(ctx, VN_ERR_CUDA, "cache set-up: %s", cudaGetErrorString(e));
  }
  if (st != VN_OK) { vn_qkv_destroy(c); return st; }
  *out = c;
  return VN_OK;
}

int32_t vn_qkv_destroy(vn_qkv* c) {
  if (!c) return VN_OK;
  cudaSetDevice(c->ctx->device);
  cudaStreamSynchronize(c->ctx->stream);
  for (void* p : {(void*)c->v.pool, (void*)c->table, (void*)c->v.lens, (void*)c->v.status, (void*)c->tickets})
    if (p) cudaFree(p);
  delete c;
  return VN_OK;
}

int32_t vn_qkv_set_pages(vn_qkv* c, const int32_t* table) {
  VN_CHECK_QKV(c);
  VN_REQUIRE(c->ctx, table, "table is null");
  const size_t n = (size_t)c->v.max_batch * c->v.max_pages;
  for (size_t i = 0; i < n; ++i)
    if (table[i] < -1 || table[i] >= c->v.n_pages) return vn_fail(c->ctx, VN_ERR_INDEX, "page %d outside the pool of %d", table[i], c->v.n_pages);
  VN_CUDA(c->ctx, cudaMemcpyAsync(c->table, table, n * sizeof(int), cudaMemcpyHostToDevice, c->ctx->stream));
  VN_CUDA(c->ctx, cudaStreamSynchronize(c->ctx->stream));
  return VN_OK;
}

int32_t vn_qkv_lengths(vn_qkv* c, int32_t* out) {
  VN_CHECK_QKV(c);
  VN_REQUIRE(c->ctx, out, "out is null");
  VN_CUDA(c->ctx, cudaMemcpyAsync(out, c->v.lens, (size_t)c->v.max_batch * sizeof(int), cudaMemcpyDeviceToHost, c->ctx->stream));
  VN_CUDA(c->ctx, cudaStreamSynchronize(c->ctx->stream));
  return VN_OK;
}

int32_t vn_qkv_set_lengths(vn_qkv* c, const int32_t* lens, int32_t on_device) {
  VN_CHECK_QKV(c);
  VN_REQUIRE(c->ctx, lens, "lens is null");
  if (on_device) {
    VN_LAUNCH_PDL_LEVEL(c->ctx, 1, "set_lengths_kernel", set_lengths_kernel, ceil_div(c->v.max_batch, 256), 256, 0, c->v, lens);
    return VN_OK;
  }
  for (int i = 0; i < c->v.max_batch; ++i)
    if (lens[i] < 0 || lens[i] > c->v.capacity()) return vn_fail(c->ctx, VN_ERR_OVERFLOW, "length %d of sequence %d outside 0 .. %d", lens[i], i, c->v.capacity());
  VN_CUDA(c->ctx, cudaMemcpyAsync(c->v.lens, lens, (size_t)c->v.max_batch * sizeof(int), cudaMemcpyHostToDevice, c->ctx->stream));
  VN_CUDA(c->ctx, cudaStreamSynchronize(c->ctx->stream));
  return VN_OK;
}

int32_t vn_qkv_status(vn_qkv* c, int32_t* no_room, int32_t* bad_index) {
  VN_CHECK_QKV(c);
  int s[3];
  VN_CUDA(c->ctx, cudaMemcpyAsync(s, c->v.status, sizeof s, cudaMemcpyDeviceToHost, c->ctx->stream));
  VN_CUDA(c->ctx, cudaMemsetAsync(c->v.status, 0, sizeof s, c->ctx->stream));
  VN_CUDA(c->ctx, cudaStreamSynchronize(c->ctx->stream));
  if (no_room) *no_room = s[0];
  if (bad_index) *bad_index = s[1];
  if (s[2]) return vn_fail(c->ctx, VN_ERR_TIMEOUT, "a copy from the cache did not arrive");
  if (s[0]) return vn_fail(c->ctx, VN_ERR_OVERFLOW, "a position behind the cache's end, or without a page, was written or read");
  if (s[1]) return vn_fail(c->ctx, VN_ERR_INDEX, "a sequence, row or count outside its range was met");
  return VN_OK;
}

int32_t vn_qkv_probe_wait(vn_qkv* c, uint64_t cycles, int64_t* waited) {
  VN_CHECK_QKV(c);
  VN_REQUIRE(c->ctx, cycles > 0 && cycles <= qkv_detail::WAIT_CYCLES, "a wait of 1 to %llu cycles", qkv_detail::WAIT_CYCLES);
  long long* d = nullptr;
  VN_CUDA(c->ctx, cudaMalloc(&d, sizeof *d));
  qkv_wait_probe_kernel<<<1, 1, 0, c->ctx->stream>>>(c->v.status, cycles, d);
  c->ctx->launches++;
  long long h = 0;
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) e = cudaMemcpyAsync(&h, d, sizeof h, cudaMemcpyDeviceToHost, c->ctx->stream);
  if (e == cudaSuccess) e = cudaStreamSynchronize(c->ctx->stream);
  cudaFree(d);
  VN_CUDA(c->ctx, e);
  if (waited) *waited = h;
  return VN_OK;
}

int32_t vn_qkv_append(vn_qkv* c, const void* rows, int64_t ld, int32_t queries, int32_t n_ent, const int32_t* ents, const int32_t* row_ent, int32_t T, int32_t M,
                      int32_t offset, const int32_t* depth, int32_t depth_per_row, const float* q_norm, const float* k_norm, float eps, const float* cos_,
                      const float* sin_, int32_t rope_rows, int32_t pairs, int32_t interleaved, void* q_out) {
  VN_CHECK_QKV(c);
  AppendArgs a;
  a.v = c->v;
  if (int32_t st = step_of(c, n_ent, ents, row_ent, T, M, &a.step)) return st;
  a.H = queries ? c->v.H : 0;
  const int width = (a.H + 2 * c->v.KH) * c->v.d, es = c->dtype == VN_F32 ? 4 : 2;
  VN_REQUIRE(c->ctx, M == 0 || (rows && (q_out || !queries)), "null rows");
  VN_REQUIRE(c->ctx, ld >= width, "rows of %lld values, %d are needed", (long long)ld, width);
  VN_REQUIRE(c->ctx, aligned(rows, es) && aligned(q_out, es), "rows are not aligned to their values");
  VN_REQUIRE(c->ctx, offset >= 0, "offset %d", offset);
  VN_REQUIRE(c->ctx, pairs >= 0 && 2 * pairs <= c->v.d, "%d rotated pairs in heads of %d", pairs, c->v.d);
  VN_REQUIRE(c->ctx, !pairs || (cos_ && sin_ && rope_rows >= c->v.capacity()), "rotation: tables of %d positions for a cache of %d", rope_rows, c->v.capacity());
  VN_REQUIRE(c->ctx, !depth || T <= QKV_MAX_DRAFT, "a tree of %d rows, at most %d", T, QKV_MAX_DRAFT);
  if (M == 0 || T == 0) return VN_OK;
  a.tree.depth = depth; a.tree.per_row = depth_per_row;
  a.x = rows; a.q = q_out; a.ld = ld; a.off = offset;
  a.qn = q_norm; a.kn = k_norm; a.eps = eps;
  a.cs = cos_; a.sn = sin_; a.pairs = pairs; a.interleaved = interleaved; a.rope_rows = rope_rows;
  a.vec = aligned(rows, 16) && aligned(q_out, 16) && ld * es % 16 == 0;
  a.vec_norm = aligned(q_norm, 16) && aligned(k_norm, 16);
  a.vec_rope = pairs % 8 == 0 && aligned(cos_, 16) && aligned(sin_, 16);
  const int units = a.H + 2 * c->v.KH, L = c->v.P <= 32 ? 4 : c->v.P <= 64 ? 8 : c->v.P <= 128 ? 16 : 32, tasks = ceil_div(units, 32 / L);
  // a warp takes one task where there are few, so that all SMs have some; more, for fewer looks at lengths and angles, where there are many
  int per = 1;
  while (per < tasks && per < 16 && (long long)M * ceil_div(tasks, 2 * per) >= 128ll * c->ctx->sm_count) per *= 2;
  const long long items = (long long)M * ceil_div(tasks, per);
  VN_REQUIRE(c->ctx, items < (1ll << 32), "%d rows are too many for one call", M);
  const unsigned grid = (unsigned)ceil_div(items, 8ll);
#define APPEND(S, L) do { if (es == 4) VN_LAUNCH_PDL_LEVEL(c->ctx, 1, "qkv_append_kernel", (qkv_append_kernel<float, S, L>), grid, 256, 0, a, tasks, per); \
                          else VN_LAUNCH_PDL_LEVEL(c->ctx, 1, "qkv_append_kernel", (qkv_append_kernel<bf16, S, L>), grid, 256, 0, a, tasks, per); } while (0)
#define APPEND_ALL(S) do { if (L == 4) APPEND(S, 4); else if (L == 8) APPEND(S, 8); else if (L == 16) APPEND(S, 16); else APPEND(S, 32); } while (0)
  if (c->v.scheme == QKV_I8) APPEND_ALL(QKV_I8); else APPEND_ALL(QKV_E4M3);
#undef APPEND_ALL
#undef APPEND
  return VN_OK;
}

int32_t vn_qkv_read(vn_qkv* c, int32_t n_ent, const int32_t* ents, const int32_t* row_ent, int32_t T, int32_t M, int32_t start, int32_t offset, int32_t dtype,
                    void* k_out, void* v_out) {
  VN_CHECK_QKV(c);
  QkvStep s;
  if (int32_t st = step_of(c, n_ent, ents, row_ent, T, M, &s)) return st;
  VN_REQUIRE(c->ctx, dtype == VN_F32 || dtype == VN_BF16, "values are read as float32 or bf16");
  VN_REQUIRE(c->ctx, start >= -2 && offset >= 0, "start %d, offset %d", start, offset);
  if (M == 0 || T == 0) return VN_OK;
  VN_REQUIRE(c->ctx, k_out && v_out, "null output");
  const int es = dtype == VN_F32 ? 4 : 2;
  VN_REQUIRE(c->ctx, aligned(k_out, es) && aligned(v_out, es), "outputs are not aligned to their values");
  const int vec = aligned(k_out, 16) && aligned(v_out, 16);
  // rows of a warp: four where there are warps enough for all SMs, else one
  const int slices = ceil_div(c->v.KH * c->v.d * es / 16, 32);
  const bool many = (long long)ceil_div(M, 4) * slices >= 64ll * c->ctx->sm_count;
  const long long items = (long long)ceil_div(M, many ? 4 : 1) * slices;
  VN_REQUIRE(c->ctx, items < (1ll << 32), "%d rows are too many for one call", M);
  const unsigned grid = (unsigned)ceil_div(items, 8ll);
#define READ2(O, S, RB) VN_LAUNCH_PDL_LEVEL(c->ctx, 1, "qkv_read_kernel", (qkv_read_kernel<O, S, RB>), grid, 256, 0, c->v, s, start, offset, (O*)k_out, (O*)v_out, vec, slices)
#define READ(O, S) do { if (many) READ2(O, S, 4); else READ2(O, S, 1); } while (0)
  if (c->v.scheme == QKV_I8) { if (es == 4) READ(float, QKV_I8); else READ(bf16, QKV_I8); }
  else { if (es == 4) READ(float, QKV_E4M3); else READ(bf16, QKV_E4M3); }
#undef READ
#undef READ2
  return VN_OK;
}

int32_t vn_qkv_commit(vn_qkv* c, int32_t n_new, const int32_t* keep_idx, int32_t stride, const int32_t* n_keep, int32_t keep_add) {
  VN_CHECK_QKV(c);
  VN_REQUIRE(c->ctx, n_keep, "n_keep is null");
  VN_REQUIRE(c->ctx, n_new >= 0, "n_new %d", n_new);
  VN_REQUIRE(c->ctx, !keep_idx || (n_new <= QKV_MAX_DRAFT && stride >= 0), "rows are picked from at most %d, not %d", QKV_MAX_DRAFT, n_new);
  VN_LAUNCH_PDL_LEVEL(c->ctx, 1, "qkv_commit_kernel", qkv_commit_kernel, dim3(keep_idx ? c->v.KH : 1, c->v.max_batch), 256, 0, c->v, n_new, keep_idx, stride, n_keep, keep_add, c->tickets);
  return VN_OK;
}

int32_t vn_qkv_attention(vn_qkv* c, const void* q, int32_t n_ent, const int32_t* ents, const int32_t* row_ent, int32_t T, int32_t M, const uint64_t* seen,
                         const int32_t* depth, int32_t tree_per_row, int32_t window, float scale, void* out) {
  VN_CHECK_QKV(c);
  QkvAttnArgs a;
  a.v = c->v;
  if (int32_t st = step_of(c, n_ent, ents, row_ent, T, M, &a.step)) return st;
  VN_REQUIRE(c->ctx, (seen == nullptr) == (depth == nullptr), "a tree has both tables");
  VN_REQUIRE(c->ctx, !seen || T <= QKV_MAX_DRAFT, "a tree of %d rows, at most %d", T, QKV_MAX_DRAFT);
  VN_REQUIRE(c->ctx, window >= 0, "window %d", window);
  VN_REQUIRE(c->ctx, isfinite(scale) && scale > 0.f, "a scale above zero is needed");
  if (M == 0 || T == 0 || n_ent == 0) return VN_OK;          // no entries: rows of nobody stay as they were
  VN_REQUIRE(c->ctx, q && out, "null rows");
  const int es = c->dtype == VN_F32 ? 4 : 2;
  VN_REQUIRE(c->ctx, aligned(q, 4 * es) && aligned(out, 4 * es), "rows are not aligned to four values");
  a.tree.seen = (const unsigned long long*)seen; a.tree.depth = depth; a.tree.per_row = tree_per_row;
  a.q = q; a.out = out; a.window = window; a.scale = scale;
  const Parts p = parts_of(c->ctx);
  a.part_o = (float*)c->ctx->qkv_parts;
  a.part_ml = (float2*)((char*)c->ctx->qkv_parts + p.ml);
  a.cuts = (QkvCut*)((char*)c->ctx->qkv_parts + p.cuts);
  a.n_cuts = (int*)((char*)c->ctx->qkv_parts + p.n_cuts);
  a.max_cuts = p.max_cuts;
  return c->v.scheme == QKV_I8 ? qkv_attention_i8(c, a) : qkv_attention_e4m3(c, a);
}

}  // extern "C"
