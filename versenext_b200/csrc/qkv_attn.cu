// Attention of a step's rows over the 8-bit cache: the committed positions and the rows that the step has appended.
#include "qkv.cuh"

namespace {

using bf16 = __nv_bfloat16;

// One warp per (row, head), a lane per four channels of two quads.  grid ceil(M H / 8)
template <typename T, int SCHEME>
__global__ void __launch_bounds__(256) qkv_attn_kernel(QkvAttnArgs a) {
  const QkvView& v = a.v;
  const int lane = threadIdx.x & 31;
  const long long task = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (task / v.H >= a.step.M) return;
  const int h = (int)(task % v.H), row = (int)(task / v.H);
  int slot, i, n;
  if (!a.step.row(v, row, &slot, &i, &n)) return;
  const int len = v.len(slot), at = len + a.tree.away(row, i), d = v.d, P = v.P, g = h / (v.H / v.KH);
  const unsigned long long seen = a.tree.seen ? a.tree.seen[a.tree.per_row ? row : i] : 0;
  const T* q = reinterpret_cast<const T*>(a.q) + ((long long)row * v.H + h) * d;
  float4 x[2], acc[2];
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    const int c = 4 * lane + 128 * y;
    x[y] = c < d ? load4(q + c) : make_float4(0.f, 0.f, 0.f, 0.f);
    acc[y] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  float m = -CUDART_INF_F, l = 0.f;
  const int end = min(len + (a.tree.seen ? n : i + 1), v.capacity());
  for (int p = a.window > 0 ? min(max(0, at - a.window + 1), len) : 0; p < end; ++p) {
    if (p >= len) {
      const int j = p - len;
      if (a.tree.seen ? !((seen >> j) & 1) : a.window > 0 && i - j >= a.window) continue;
    }
    const int page = v.page(slot, p / KV_PAGE);
    if (page < 0) { if (lane == 0) v.status[0] = 1; continue; }
    const unsigned char* b = v.block(page, g, p % KV_PAGE / QKV_BLOCK);
    const int r = p % QKV_BLOCK, t = qkv_turn(P / 16, r);
    const float* sc = reinterpret_cast<const float*>(b + 2 * QKV_BLOCK * P);
    float s = 0.f;
    float4 vv[2];
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const int c = 4 * lane + 128 * y;
      if (c >= d) { vv[y] = make_float4(0.f, 0.f, 0.f, 0.f); continue; }
      const int o = (((c >> 4) ^ t) << 4) + (c & 15);
      const uchar4 k = *reinterpret_cast<const uchar4*>(b + r * P + o), w = *reinterpret_cast<const uchar4*>(b + (QKV_BLOCK + r) * P + o);
      s += x[y].x * qkv_value<SCHEME>(k.x) + x[y].y * qkv_value<SCHEME>(k.y) + x[y].z * qkv_value<SCHEME>(k.z) + x[y].w * qkv_value<SCHEME>(k.w);
      vv[y] = make_float4(qkv_value<SCHEME>(w.x), qkv_value<SCHEME>(w.y), qkv_value<SCHEME>(w.z), qkv_value<SCHEME>(w.w));
    }
    s = warp_sum(s) * sc[r] * a.scale;
    const float m2 = fmaxf(m, s), base = m2 == -CUDART_INF_F ? 0.f : m2, f = expf(m - base), e = expf(s - base), ev = e * sc[QKV_BLOCK + r];
    l = l * f + e;
#pragma unroll
    for (int y = 0; y < 2; ++y)
      acc[y] = make_float4(fmaf(acc[y].x, f, ev * vv[y].x), fmaf(acc[y].y, f, ev * vv[y].y), fmaf(acc[y].z, f, ev * vv[y].z), fmaf(acc[y].w, f, ev * vv[y].w));
    m = m2;
  }
  T* o = reinterpret_cast<T*>(a.out) + ((long long)row * v.H + h) * d;
  const float inv = l == 0.f ? 0.f : 1.f / l;             // nothing seen: zero
#pragma unroll
  for (int y = 0; y < 2; ++y)
    if (4 * lane + 128 * y < d) store4(o + 4 * lane + 128 * y, scaled(acc[y], inv));
}

}  // namespace

int32_t qkv_attention(vn_qkv* c, const QkvAttnArgs& a) {
  const unsigned grid = (unsigned)ceil_div((long long)a.v.H * a.step.M, 8ll);
#define AT(T, S) VN_LAUNCH_NAMED(c->ctx, "qkv_attn_kernel", (qkv_attn_kernel<T, S>), grid, 256, 0, a)
  if (a.v.scheme == QKV_I8) { if (c->dtype == VN_F32) AT(float, QKV_I8); else AT(bf16, QKV_I8); }
  else { if (c->dtype == VN_F32) AT(float, QKV_E4M3); else AT(bf16, QKV_E4M3); }
#undef AT
  return VN_OK;
}
