// A paged cache of keys and values in 8 bits (vn_qkv): layout, rows of a step, and codes.
//
// A block holds 32 positions of one key/value head: [32][P] codes of the keys, [32][P] of the values, 32 fp32 scales of the
// keys, 32 of the values (P = padded head size); it is one piece of memory, so that a reader brings it in with one copy.  A
// page is 64 positions = two blocks per head: block((page KH + head) 2 + half).  A head at a position is scale * code, with
// scale = max |x| / 127 (int8) or / 448 (e4m3), at least 2^-126; where it holds a value that is not finite its scale is NaN and its codes are 0.
// int8 codes stand with 128 added.  Within a block the 16-byte chunks of a position's codes are permuted by its number (chunk c stands at c ^ turn), so that the
// eight positions of a matrix that ldmatrix reads lie in different shared memory banks.
#pragma once
#include "rows.cuh"
#include <cuda_fp16.h>
#include <math_constants.h>

enum { QKV_I8 = 0, QKV_E4M3 = 1 };
constexpr int QKV_BLOCK = 32;                       // positions of a block
constexpr float QKV_SCALE_MIN = 1.17549435e-38f;
constexpr int QKV_MAX_DRAFT = 64;                   // rows of a tree, rows that commit may pick from

struct QkvView {
  unsigned char* pool = nullptr;
  const int* table = nullptr;                       // [max_batch][max_pages] page of a sequence's positions 64 i .., -1: none
  int* lens = nullptr;                              // [max_batch] committed positions
  int* status = nullptr;                            // [3] a position without a page was wanted; a bad slot, row or length was met; a copy did not arrive
  int max_batch = 0, max_pages = 0, n_pages = 0, H = 0, KH = 0, d = 0, P = 0, scheme = 0;
  __host__ __device__ __forceinline__ int capacity() const { return max_pages * KV_PAGE; }
  __host__ __device__ __forceinline__ int block_bytes() const { return QKV_BLOCK * (2 * P + 8); }
  // committed positions of a sequence; a length that a program wrote wrongly is met here
  __device__ __forceinline__ int len(int slot) const { return min(max(lens[slot], 0), capacity()); }
  // page of a position's sequence, or -1
  __device__ __forceinline__ int page(int slot, int i) const {
    const int p = table[(long long)slot * max_pages + i];
    return p >= 0 && p < n_pages ? p : -1;
  }
  __device__ __forceinline__ unsigned char* block(int page, int head, int half) const {
    return pool + (((long long)page * KH + head) * 2 + half) * block_bytes();
  }
};

// what a position's chunk number is permuted with, for rows of n chunks: eight neighbouring positions fill 128 bytes
__host__ __device__ constexpr int qkv_turn(int n, int pos) {
  return n % 8 == 0 ? pos & 7 : n % 4 == 0 ? (pos >> 1) & 3 : n % 2 == 0 ? (pos >> 2) & 1 : 0;
}

// Rows of a step: entry e brings cnt rows, from row r0 on, for sequence slot.  ents null: entry e = sequence e with T rows.
struct QkvStep {
  const int4* ents = nullptr;                       // [n_ent] slot, first row, rows, 0
  const int* row_ent = nullptr;                     // [M] entry of a row, -1: a row that belongs to none
  int n_ent = 0, T = 0, M = 0;                      // T: rows of an entry at most
  // false: the entry has nothing that may be touched
  __device__ __forceinline__ bool entry(const QkvView& v, int e, int* slot, int* r0, int* n) const {
    if (!ents) { *slot = e; *r0 = e * T; *n = T; return true; }
    const int4 x = ents[e];
    *slot = x.x; *r0 = x.y; *n = x.z;
    if (x.x < 0 || x.x >= v.max_batch || x.y < 0 || x.z < 0 || x.z > T || x.y > M - x.z) { v.status[1] = 1; return false; }
    return true;
  }
  // entry of a row and its place there; false: none
  __device__ __forceinline__ bool row(const QkvView& v, int r, int* slot, int* i, int* n) const {
    int e, r0;
    if (!ents) e = r / T;
    else {
      e = row_ent[r];
      if (e < 0) return false;
      if (e >= n_ent) { v.status[1] = 1; return false; }
    }
    if (!entry(v, e, slot, &r0, n)) return false;
    *i = r - r0;
    if (*i < 0 || *i >= *n) { v.status[1] = 1; return false; }
    return true;
  }
};

// A tree: which new rows a row sees (bit j: row j of its entry) and how many tokens stand between it and the committed ones.
// Null: row i sees rows 0 .. i and is i tokens away.
struct QkvTree {
  const unsigned long long* seen = nullptr;
  const int* depth = nullptr;
  int per_row = 0;                                  // the tables go by the row of the step, else by its place in its entry
  __device__ __forceinline__ int away(int row, int i) const { return depth ? depth[per_row ? row : i] : i; }
  // as attention takes it, whose windows rely on a path of at most QKV_MAX_DRAFT rows
  __device__ __forceinline__ int behind(const QkvView& v, int row, int i) const {
    const int n = away(row, i);
    if (!depth || (n >= 0 && n < QKV_MAX_DRAFT)) return n;
    v.status[1] = 1;
    return n < 0 ? 0 : QKV_MAX_DRAFT - 1;
  }
  // rows that a row sees through a window: of a path, parents before children, the last ones
  __device__ __forceinline__ unsigned long long sees(int row, int i, int window) const {
    unsigned long long s = seen[per_row ? row : i];
    if (window > 0)
      for (int n = __popcll(s); n > window; --n) s &= s - 1;
    return s;
  }
};

struct vn_qkv {
  vn_ctx* ctx = nullptr;
  QkvView v;
  int dtype = VN_BF16;
  int* table = nullptr;
  int* tickets = nullptr;                           // zero between kernels
};

// a unit whose blocks several shares have, the first of them `first`: rows f0 .. of nf (tokens x heads of the group) from row r0 on; n parts
struct QkvCut { int r0, f0, nf, head, first, n; };

struct QkvAttnArgs {
  QkvView v;
  QkvStep step;
  QkvTree tree;
  const void* q = nullptr;                          // [M, H, d]
  void* out = nullptr;
  int window = 0;
  float scale = 1.f;
  float* part_o = nullptr;                          // [2 shares][rows of a unit][P] results of a share's first and last unit
  float2* part_ml = nullptr;
  QkvCut* cuts = nullptr;                           // [max_cuts] units to merge: with few parts from the front, with many from the back
  int* n_cuts = nullptr;                            // [3] how many of each, and CTAs that are done with them; zero between calls
  int max_cuts = 0;
};
constexpr int QKV_MAX_CTAS = 3;                     // of the attention kernel on an SM
constexpr int QKV_PART = 2 * 128 * 128;             // values of parts: CTAs on an SM x rows x padded head size, at most
int32_t qkv_attention_i8(vn_qkv* c, const QkvAttnArgs& a);
int32_t qkv_attention_e4m3(vn_qkv* c, const QkvAttnArgs& a);
