// The paged 8-bit cache's entry points and the kernels that write, read and keep positions; attention is in qkv_attn.cuh.
#include <string.h>

#include <new>

#include "qkv.cuh"

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

template <typename T> __device__ __forceinline__ float4 quad_of(const T* p, bool vec) {
  if (vec) return load4(p);
  return make_float4(to_f<T>(p[0]), to_f<T>(p[1]), to_f<T>(p[2]), to_f<T>(p[3]));
}
template <typename T> __device__ __forceinline__ void put_quad(T* p, float4 v, bool vec) {
  if (vec) { store4(p, v); return; }
  p[0] = from_f<T>(v.x); p[1] = from_f<T>(v.y); p[2] = from_f<T>(v.z); p[3] = from_f<T>(v.w);
}

__device__ __forceinline__ unsigned char code_of(float y, int scheme) {
  if (scheme == QKV_I8) return (unsigned char)(max(-127, min(127, __float2int_rn(y))) + 128);
  unsigned short r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.f), "f"(y));
  return (unsigned char)r;
}

__device__ __forceinline__ float4 quad_at(const float* p, bool vec) { return vec ? load4(p) : make_float4(p[0], p[1], p[2], p[3]); }

// A warp takes `per` tasks of a row, four asked for at a time: a task is 32 / L neighbouring heads, whose L lanes hold Y quads of channels
// each (lane, lane + 32).  Heads pass through shared memory only for half-split rotation, where a quad meets the one pairs further on.
// What bounds it: the rows' bytes for many rows; for few, the chain entry, length, page, store (the row's values are asked for first).
// grid ceil(M ceil(tasks / per) / 8), block 256
template <typename T, int L, int Y>
__global__ void __launch_bounds__(256) qkv_append_kernel(AppendArgs a, int tasks, int per) {
  constexpr int HPW = 32 / L, IN = Y > 1 ? 2 : 4;
  __shared__ __align__(16) float s_head[8][HPW][4 * L * Y];
  const int lane = threadIdx.x & 31, l = lane % L, sub = lane / L, warp = threadIdx.x >> 5;
  const int units = a.H + 2 * a.v.KH, d = a.v.d, P = a.v.P, slices = (tasks + per - 1) / per;
  const unsigned item = blockIdx.x * 8u + warp;
  pdl_wait();
  const int row = (int)(item / (unsigned)slices), first = (int)(item % (unsigned)slices) * per, last = min(tasks, first + per);
  if (row >= a.step.M) return;
  const T* xr = reinterpret_cast<const T*>(a.x) + row * a.ld;
  float4 x[IN][Y];
  auto ask = [&](int task) {
#pragma unroll
    for (int k = 0; k < IN; ++k)
#pragma unroll
      for (int y = 0; y < Y; ++y) {
        const int unit = (task + k) * HPW + sub, c = 4 * l + 128 * y;
        x[k][y] = task + k < last && unit < units && c < d ? quad_of(xr + (long long)unit * d + c, a.vec) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
  };
  ask(first);
  int slot, i, n;
  if (!a.step.row(a.v, row, &slot, &i, &n)) return;
  const int len = a.v.len(slot), pos = len + a.off + i;
  const int turn = min(max(len + a.off + a.tree.away(row, i), 0), a.rope_rows - 1);
  const int page = pos >= 0 && pos < a.v.capacity() ? a.v.page(slot, pos / KV_PAGE) : -1, at = pos % QKV_BLOCK;
  // what a quad is turned by: half-split, quads of the two halves by the same angles
  float4 cs[Y], sn[Y];
  bool turned[Y];
#pragma unroll
  for (int y = 0; y < Y; ++y) {
    const int c = 4 * l + 128 * y, np = a.pairs;
    turned[y] = np && c < 2 * np;
    cs[y] = make_float4(1.f, 1.f, 1.f, 1.f);
    sn[y] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (!turned[y]) continue;
    const float *pc = a.cs + (long long)turn * np, *ps = a.sn + (long long)turn * np;
    if (a.interleaved) {
      const bool two = c + 2 < 2 * np;
      cs[y].x = cs[y].y = pc[c / 2]; sn[y].x = sn[y].y = ps[c / 2];
      if (two) { cs[y].z = cs[y].w = pc[c / 2 + 1]; sn[y].z = sn[y].w = ps[c / 2 + 1]; }
    } else if (a.vec_rope) {
      cs[y] = load4(pc + (c < np ? c : c - np)); sn[y] = load4(ps + (c < np ? c : c - np));
    } else {
      auto angle = [&](int e, float& u, float& w) {
        if (c + e < 2 * np) { const int p = c + e < np ? c + e : c + e - np; u = pc[p]; w = ps[p]; }
      };
      angle(0, cs[y].x, sn[y].x); angle(1, cs[y].y, sn[y].y); angle(2, cs[y].z, sn[y].z); angle(3, cs[y].w, sn[y].w);
    }
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
      float4 v[Y];
#pragma unroll
      for (int y = 0; y < Y; ++y) v[y] = x[k][y];
      const float* w = is_v || !live ? nullptr : is_q ? a.qn : a.kn;
      if (__any_sync(0xffffffffu, w != nullptr)) {           // a warp's heads may be of two kinds
        float ss = 0.f;
#pragma unroll
        for (int y = 0; y < Y; ++y) ss += v[y].x * v[y].x + v[y].y * v[y].y + v[y].z * v[y].z + v[y].w * v[y].w;
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (w) {
          const float r = sqrtf(ss / (float)d + a.eps);
#pragma unroll
          for (int y = 0; y < Y; ++y) {
            const int c = 4 * l + 128 * y;
            if (c >= d) break;
            const float4 g = quad_at(w + c, a.vec_norm);
            v[y] = make_float4(v[y].x / r * g.x, v[y].y / r * g.y, v[y].z / r * g.z, v[y].w / r * g.w);
          }
        }
      }
      if (a.pairs && a.interleaved) {
        if (!is_v)
#pragma unroll
          for (int y = 0; y < Y; ++y)
            v[y] = make_float4(v[y].x * cs[y].x - v[y].y * sn[y].x, v[y].y * cs[y].x + v[y].x * sn[y].x, v[y].z * cs[y].z - v[y].w * sn[y].z, v[y].w * cs[y].z + v[y].z * sn[y].z);
      } else if (a.pairs) {
        __syncwarp();
#pragma unroll
        for (int y = 0; y < Y; ++y) *reinterpret_cast<float4*>(s + 4 * l + 128 * y) = v[y];
        __syncwarp();
#pragma unroll
        for (int y = 0; y < Y; ++y) {
          const int c = 4 * l + 128 * y, np = a.pairs;
          if (is_v || !turned[y]) continue;
          // the other half's values, with the sign that they enter with
          auto other = [&](int e) { return c + e < np ? -s[c + e + np] : c + e < 2 * np ? s[c + e - np] : 0.f; };
          float4 t;
          if (a.vec_rope) {
            t = *reinterpret_cast<const float4*>(s + (c < np ? c + np : c - np));
            if (c < np) t = make_float4(-t.x, -t.y, -t.z, -t.w);
          } else {
            t = make_float4(other(0), other(1), other(2), other(3));
          }
          v[y] = make_float4(v[y].x * cs[y].x + t.x * sn[y].x, v[y].y * cs[y].y + t.y * sn[y].y, v[y].z * cs[y].z + t.z * sn[y].z, v[y].w * cs[y].w + t.w * sn[y].w);
        }
      }
      if (live && is_q) {
        T* o = reinterpret_cast<T*>(a.q) + ((long long)row * a.H + unit) * d;
#pragma unroll
        for (int y = 0; y < Y; ++y)
          if (4 * l + 128 * y < d) put_quad(o + 4 * l + 128 * y, v[y], a.vec);
      }
      if (__all_sync(0xffffffffu, !live || is_q)) continue;
      // ---- a head of the cache
      unsigned top = 0;                                      // magnitudes as bits: what is not finite is above all others
#pragma unroll
      for (int y = 0; y < Y; ++y)
        top = max(top, max(max(__float_as_uint(v[y].x) & 0x7fffffffu, __float_as_uint(v[y].y) & 0x7fffffffu),
                           max(__float_as_uint(v[y].z) & 0x7fffffffu, __float_as_uint(v[y].w) & 0x7fffffffu)));
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (!live || is_q) continue;
      if (page < 0) { if (l == 0) a.v.status[0] = 1; continue; }
      const bool bad = top >= 0x7f800000u;
      const float scale = fmaxf((top ? __uint_as_float(top) : 1.f) / (a.v.scheme == QKV_I8 ? 127.f : 448.f), QKV_SCALE_MIN);
      const int head = unit - a.H - (is_v ? a.v.KH : 0), t = qkv_turn(P / 16, at);
      unsigned char* b = a.v.block(page, head, pos % KV_PAGE / QKV_BLOCK);
      unsigned char* codes = b + (is_v ? QKV_BLOCK * P : 0) + at * P;
#pragma unroll
      for (int y = 0; y < Y; ++y) {
        const int c = 4 * l + 128 * y;
        if (c >= P) break;
        const unsigned char none = a.v.scheme == QKV_I8 ? 128 : 0;
        uchar4 q = make_uchar4(none, none, none, none);
        if (c < d && !bad) q = make_uchar4(code_of(v[y].x / scale, a.v.scheme), code_of(v[y].y / scale, a.v.scheme), code_of(v[y].z / scale, a.v.scheme), code_of(v[y].w / scale, a.v.scheme));
        *reinterpret_cast<uchar4*>(codes + (((c >> 4) ^ t) << 4) + (c & 15)) = q;
      }
      if (l == 0) reinterpret_cast<float*>(b + 2 * QKV_BLOCK * P)[(is_v ? QKV_BLOCK : 0) + at] = bad ? CUDART_NAN_F : scale;
    }
  }
}

// A thread takes 16 bytes of results (C channels of a head) of RB neighbouring rows, all asked for before any is converted; the rows'
// blocks are found by the first threads.  Bound by the bytes of codes and results.
// grid (ceil(M / RB), ceil(KH d / C / 256), 2), block 256
template <typename O, int SCHEME, int RB>
__global__ void __launch_bounds__(256) qkv_read_kernel(QkvView v, QkvStep step, int start, int off, O* __restrict__ k, O* __restrict__ vals, int vec) {
  constexpr int C = 16 / sizeof(O);
  __shared__ long long s_block[RB];                          // of head 0, -1: none
  __shared__ int s_at[RB];                                   // place in the block, -1: no row
  const int row0 = blockIdx.x * RB, per = v.d / C, it = blockIdx.y * 256 + threadIdx.x;
  pdl_wait();
  if (threadIdx.x < RB) {
    const int row = row0 + threadIdx.x;
    int slot, i, n, at = -1;
    long long block = -1;
    if (row < step.M && step.row(v, row, &slot, &i, &n)) {
      const int pos = (start >= 0 ? start : v.len(slot) + off - (start == -2 ? n : 0)) + i;
      const int page = pos >= 0 && pos < v.capacity() ? v.page(slot, pos / KV_PAGE) : -1;
      at = page < 0 ? 0 : pos % QKV_BLOCK;
      if (page < 0) v.status[0] = 1;
      else block = ((long long)page * v.KH * 2 + pos % KV_PAGE / QKV_BLOCK) * v.block_bytes();
    }
    s_block[threadIdx.x] = block;
    s_at[threadIdx.x] = at;
  }
  __syncthreads();
  if (it >= v.KH * per) return;
  const int head = it / per, c = it % per * C;
  const unsigned char* pool = v.pool + (long long)head * 2 * v.block_bytes();
  uint2 u[RB];
  float sc[RB];
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    const long long block = s_block[r];
    const int at = s_at[r];
    u[r] = make_uint2(SCHEME == QKV_I8 ? 0x80808080u : 0u, SCHEME == QKV_I8 ? 0x80808080u : 0u);
    sc[r] = 0.f;
    if (block < 0) continue;
    const unsigned char* b = pool + block;
    const unsigned char* p = b + (blockIdx.z * QKV_BLOCK + at) * v.P + (((c >> 4) ^ qkv_turn(v.P / 16, at)) << 4) + (c & 15);
    if (C == 8) u[r] = *reinterpret_cast<const uint2*>(p);
    else u[r].x = *reinterpret_cast<const unsigned*>(p);
    sc[r] = reinterpret_cast<const float*>(b + 2 * QKV_BLOCK * v.P)[blockIdx.z * QKV_BLOCK + at];
  }
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    if (s_at[r] < 0) continue;
    O* o = (blockIdx.z ? vals : k) + ((long long)(row0 + r) * v.KH + head) * v.d + c;
    float4 y[2];
#pragma unroll
    for (int h = 0; h < C / 4; ++h) {
      const unsigned w = h ? u[r].y : u[r].x;
      float4 x;
      if (SCHEME == QKV_I8) {                                // a byte under the exponent of 2^23, less 2^23 + 128
        const float off8 = 8388736.f;
        x = make_float4(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440)) - off8, __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7441)) - off8,
                        __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7442)) - off8, __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7443)) - off8);
      } else {
        unsigned lo, hi;
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(lo) : "h"((unsigned short)w));
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(hi) : "h"((unsigned short)(w >> 16)));
        const float2 p0 = __half22float2(*reinterpret_cast<const __half2*>(&lo)), p1 = __half22float2(*reinterpret_cast<const __half2*>(&hi));
        x = make_float4(p0.x, p0.y, p1.x, p1.y);
      }
      y[h] = scaled(x, sc[r]);
    }
    if (C == 8 && vec) {                                     // 16 bytes in one piece
      const __nv_bfloat162 p[4] = {__floats2bfloat162_rn(y[0].x, y[0].y), __floats2bfloat162_rn(y[0].z, y[0].w), __floats2bfloat162_rn(y[1].x, y[1].y), __floats2bfloat162_rn(y[1].z, y[1].w)};
      *reinterpret_cast<uint4*>(o) = *reinterpret_cast<const uint4*>(p);
    } else {
#pragma unroll
      for (int h = 0; h < C / 4; ++h) put_quad(o + 4 * h, y[h], vec);
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
  if (n < 0 || n > n_new || len + n > v.capacity()) {
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

__global__ void set_lengths_kernel(int* __restrict__ lens, const int* __restrict__ from, int n) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  pdl_wait();
  if (i < n) lens[i] = from[i];
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
    VN_LAUNCH_PDL_LEVEL(c->ctx, 1, "set_lengths_kernel", set_lengths_kernel, ceil_div(c->v.max_batch, 256), 256, 0, c->v.lens, lens, c->v.max_batch);
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
  a.vec = aligned(rows, 4 * es) && aligned(q_out, 4 * es) && ld % 4 == 0;
  a.vec_norm = aligned(q_norm, 16) && aligned(k_norm, 16);
  a.vec_rope = pairs % 4 == 0 && aligned(cos_, 16) && aligned(sin_, 16);
  const int units = a.H + 2 * c->v.KH, L = c->v.P <= 32 ? 8 : c->v.P <= 64 ? 16 : 32, tasks = ceil_div(units, 32 / L);
  // a warp takes one task where there are few, so that all SMs have some; more, for fewer looks at lengths and angles, where there are many
  int per = 1;
  while (per < tasks && per < 16 && (long long)M * ceil_div(tasks, 2 * per) >= 128ll * c->ctx->sm_count) per *= 2;
  const long long items = (long long)M * ceil_div(tasks, per);
  VN_REQUIRE(c->ctx, items < (1ll << 32), "%d rows are too many for one call", M);
  const unsigned grid = (unsigned)ceil_div(items, 8ll);
#define APPEND(L, Y) do { if (es == 4) VN_LAUNCH_PDL_LEVEL(c->ctx, 1, "qkv_append_kernel", (qkv_append_kernel<float, L, Y>), grid, 256, 0, a, tasks, per); \
                          else VN_LAUNCH_PDL_LEVEL(c->ctx, 1, "qkv_append_kernel", (qkv_append_kernel<bf16, L, Y>), grid, 256, 0, a, tasks, per); } while (0)
  if (L == 8) APPEND(8, 1); else if (L == 16) APPEND(16, 1); else if (c->v.P <= 128) APPEND(32, 1); else APPEND(32, 2);
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
  // rows of a CTA: more of them in flight for each thread where there are CTAs enough
  const int y = ceil_div(c->v.KH * c->v.d * es / 16, 256);
  const bool many = (long long)ceil_div(M, 8) * y >= 4ll * c->ctx->sm_count;
  VN_REQUIRE(c->ctx, y <= 65535, "%d heads of %d", c->v.KH, c->v.d);
  const dim3 grid(ceil_div(M, many ? 8 : 2), y, 2);
#define READ2(O, S, RB) VN_LAUNCH_PDL_LEVEL(c->ctx, 1, "qkv_read_kernel", (qkv_read_kernel<O, S, RB>), grid, 256, 0, c->v, s, start, offset, (O*)k_out, (O*)v_out, vec)
#define READ(O, S) do { if (many) READ2(O, S, 8); else READ2(O, S, 2); } while (0)
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
  if (M == 0 || T == 0) return VN_OK;
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
