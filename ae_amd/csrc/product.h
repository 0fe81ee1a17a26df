// Matrix products with an epilogue, dense or grouped: what their kernels share.
//
// Every product here is C[r][c] = sum_k Q[r][k] P[c][k], with "row operand" Q (r: rows of the
// output) and "column operand" P (c: its columns). An operand is either contiguous along the
// contraction k (element (r, k) at r * ld + k) or strided along it (at k * ld + r):
//
//   forward           z  = x W^T    Q = x, contiguous     P = W, contiguous     k: input columns
//   input gradient    dx = dz W     Q = dz, contiguous    P = W, strided        k: weight rows
//   weight gradient   dW = dz^T x   Q = dz, strided       P = x, strided        k: rows of x
//
// Grouped products take their groups from row bounds on the device: the first two along the output
// rows (each group its own P), the third along the contraction (each group its own output).
//
// MFMA fragments: P is the instruction's A operand and Q its B operand, so that a lane holds four
// consecutive output columns of one output row: row (lane % 16), columns 4 (lane / 16) .. + 3 of a
// 16 x 16 tile.
#pragma once

#include "expert_items.h"

namespace smx {

enum Activation : int { kActNone = 0, kActRelu, kActGelu, kActGeluTanh, kActSilu, kActSwiglu };

constexpr int kPThreads = 256;
constexpr int kPWaves = kPThreads / kWave;
constexpr int kPStep = 128;          // bytes of contraction per row and step
constexpr int kPRowBlock = 4;        // row tiles that run side by side over the column tiles
constexpr uint32_t kPOutside = 0x80000000u;  // a buffer offset past every buffer: loads give zeros
constexpr int64_t kPMaxPitch = (int64_t{1} << 23) - 1;  // bytes: 256 rows stay below kPOutside

struct ProductArgs {
  const char* p;
  const char* q;
  int64_t p_ld, q_ld;       // elements
  int64_t p_group;          // elements from one group's P (forward, dx) to the next
  int rows, cols;           // of the product; grouped along the rows: of all groups
  int depth;                // contraction length; grouped along it: of all groups
  const int64_t* offsets;   // [groups + 1] row bounds, or null: one group of everything
  const int64_t* slots;     // [groups] index of the group's P (and bias), or null
  int64_t weights;          // number of P's that slots may name
  int groups;
  int gated;                // columns are gate columns, then as many up columns
  // epilogue
  char* out;                // rounded result
  int64_t out_ld, out_group;
  const char* bias;
  int64_t bias_ld;
  const char* res;
  int64_t res_ld;
  float* z;                 // product + bias, or null
  int64_t z_ld;
  float* part;              // splits > 1: partial sums [splits][rows][cols]
  int splits, split_steps;  // contraction splits, steps of kPStep bytes in each
  int act;
  int out_cols;             // columns of out: cols, or half of them where gated
  int vec;                  // 4 consecutive outputs are one aligned store in every array
  int item_blocks;          // workgroups of the product; those behind fill rows of no group
  int fill_blocks;
};

// ---------------------------------------------------------------------------------------
// Groups
// ---------------------------------------------------------------------------------------

// Row bounds of group g, inside [0, total] and in order whatever the caller's bounds hold.
__device__ __forceinline__ void group_bounds(const ProductArgs& a, int g, int total, int& lo, int& n) {
  if (a.offsets == nullptr) {
    lo = 0;
    n = total;
    return;
  }
  const int64_t b0 = a.offsets[g], b1 = a.offsets[g + 1];
  const int64_t c0 = min(max(b0, int64_t{0}), static_cast<int64_t>(total));
  const int64_t c1 = min(max(b1, c0), static_cast<int64_t>(total));
  lo = static_cast<int>(c0);
  n = static_cast<int>(c1 - c0);
}

// The group's P, or -1: a slot outside the pool holds no weights, and its rows are of no group.
__device__ __forceinline__ int64_t group_weight(const ProductArgs& a, int g) {
  if (a.slots == nullptr) return g;
  const int64_t s = a.slots[g];
  return s >= 0 && s < a.weights ? s : -1;
}

// A workgroup's tile of the output.
struct ProductItem {
  int g;          // group
  int64_t w;      // its P
  int row;        // first output row (in out)
  int m;          // rows of the tile that exist
  int ct;         // column tile
  int split;
  int k0, depth;  // contraction: first index (grouped along it), length
};

// Item of workgroup b among `total` ones. Consecutive workgroups go to the 8 XCDs in turn, each with an L2 of its
// own: XCD x takes the x-th eighth of the items, so that neighbours in the item order share it.
__device__ __forceinline__ int xcd_item(int b, int total) {
  const int x = b & 7, i = b >> 3;
  const int per = total >> 3, extra = total & 7;
  if (i >= per + (x < extra ? 1 : 0)) return -1;
  return x * per + min(x, extra) + i;
}

// Row tile, column tile and split of item `id`: blocks of kPRowBlock row tiles, over all column tiles before
// the next block; the splits outermost.
__device__ __forceinline__ void item_order(int id, int rt, int ct, int& r, int& c, int& split) {
  split = id / (rt * ct);
  id -= split * rt * ct;
  const int blk = id / (kPRowBlock * ct);
  id -= blk * kPRowBlock * ct;
  const int size = min(kPRowBlock, rt - blk * kPRowBlock);
  c = id / size;
  r = blk * kPRowBlock + id - c * size;
}

// The item of workgroup b of a product whose groups lie along its rows, on tiles of bm rows; false past the last.
// Every wave of the workgroup finds it by itself: a lane per group, row tiles counted by a scan.
__device__ __forceinline__ bool find_row_item(const ProductArgs& a, int b, int bm, int col_tiles, ProductItem& it) {
  it.k0 = 0;
  it.depth = a.depth;
  if (a.offsets == nullptr) {
    const int rt = (a.rows + bm - 1) / bm;
    const int id = xcd_item(b, rt * col_tiles * a.splits);
    if (id < 0) return false;
    int r;
    item_order(id, rt, col_tiles, r, it.ct, it.split);
    it.g = 0;
    it.w = 0;
    it.row = r * bm;
    it.m = min(bm, a.rows - it.row);
    return true;
  }
  const int lane = lane_id();
  int rt = 0, lo = 0, n = 0, incl = 0;
  auto scan = [&](int base) {
    const int g = base + lane;
    lo = n = 0;
    if (g < a.groups) {
      group_bounds(a, g, a.rows, lo, n);
      if (a.slots != nullptr && group_weight(a, g) < 0) n = 0;
    }
    incl = wave_incl_scan((n + bm - 1) / bm);
  };
  for (int base = 0; base < a.groups; base += kWave) {
    scan(base);
    rt += last_lane(incl);
  }
  const int id = xcd_item(b, rt * col_tiles * a.splits);
  if (id < 0) return false;
  int r;
  item_order(id, rt, col_tiles, r, it.ct, it.split);
  int before = 0;
  for (int base = 0; base < a.groups; base += kWave) {
    if (a.groups > kWave) scan(base);
    const int here = last_lane(incl);
    if (r < before + here) {
      const int l = __ffsll(static_cast<unsigned long long>(ballot(before + incl > r))) - 1;
      const int first = before + __builtin_amdgcn_readlane(incl, l) - (__builtin_amdgcn_readlane(n, l) + bm - 1) / bm;
      it.g = base + l;
      it.row = __builtin_amdgcn_readlane(lo, l) + (r - first) * bm;
      it.m = min(bm, __builtin_amdgcn_readlane(n, l) - (r - first) * bm);
      it.w = uniform64(group_weight(a, it.g));
      return it.w >= 0;
    }
    before += here;
  }
  return false;
}

// The same of a product whose groups lie along its contraction.
__device__ __forceinline__ bool find_depth_item(const ProductArgs& a, int b, int bm, int col_tiles, ProductItem& it) {
  const int rt = (a.rows + bm - 1) / bm;
  const int per = rt * col_tiles * a.splits;
  int id = xcd_item(b, per * a.groups);
  if (id < 0) return false;
  it.g = id / per;
  it.w = it.g;
  int r;
  item_order(id - it.g * per, rt, col_tiles, r, it.ct, it.split);
  it.row = r * bm;
  it.m = min(bm, a.rows - it.row);
  group_bounds(a, it.g, a.depth, it.k0, it.depth);
  it.k0 = uniform(it.k0);
  it.depth = uniform(it.depth);
  return true;
}

// ---------------------------------------------------------------------------------------
// Epilogue
// ---------------------------------------------------------------------------------------

__device__ __forceinline__ float sigmoid_f32(float z) { return 1.0f / (1.0f + expf(-z)); }
// Normal distribution function by the complementary error function: relative accuracy in the left tail.
__device__ __forceinline__ float normal_cdf(float z) { return 0.5f * erfcf(z * -0.70710678f); }
// gelu's tanh form is z * sigmoid(2 u), u = sqrt(2 / pi) (z + 0.044715 z^3).
__device__ __forceinline__ float gelu_tanh_2u(float z) { return 1.59576912f * fmaf(0.044715f * z * z, z, z); }

__device__ __forceinline__ float activate(int act, float z) {
  switch (act) {
    case kActRelu: return z < 0.0f ? 0.0f : z;
    case kActGelu: return z * normal_cdf(z);
    case kActGeluTanh: return z * sigmoid_f32(gelu_tanh_2u(z));
    case kActSilu: return z * sigmoid_f32(z);
    default: return z;
  }
}

// d act / dz. The slope terms vanish faster than any power of z grows: 0 where they underflow, also at infinity.
__device__ __forceinline__ float activate_grad(int act, float z) {
  switch (act) {
    case kActRelu: return z > 0.0f ? 1.0f : (z != z ? z : 0.0f);
    case kActGelu: {
      const float e = expf(-0.5f * z * z);
      return e == 0.0f ? normal_cdf(z) : fmaf(z, 0.398942280f * e, normal_cdf(z));
    }
    case kActGeluTanh: {
      const float s = sigmoid_f32(gelu_tanh_2u(z)), t = s * (1.0f - s);
      return t == 0.0f ? s : fmaf(z * t, 1.59576912f * fmaf(3.0f * 0.044715f * z, z, 1.0f), s);
    }
    case kActSilu: {
      const float s = sigmoid_f32(z), t = s * (1.0f - s);
      return t == 0.0f ? s : fmaf(z, t, s);
    }
    default: return 1.0f;
  }
}

// Four consecutive elements of an array of T (DT), those from column `n` on left alone.
template <int DT>
__device__ __forceinline__ f32x4 load4(const char* base, int64_t at, int left, bool vec) {
  using S = typename Elem<DT>::S;
  const S* s = reinterpret_cast<const S*>(base) + at;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  if (vec) {
    if constexpr (DT == kF32) {
      v = *reinterpret_cast<const f32x4*>(s);
    } else {
      const u32x2 b = *reinterpret_cast<const u32x2*>(s);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = Elem<DT>::to_f32(static_cast<uint16_t>(b[e >> 1] >> (16 * (e & 1))));
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < left) v[e] = Elem<DT>::to_f32(s[e]);
  }
  return v;
}

template <int DT>
__device__ __forceinline__ void store4(char* base, int64_t at, int left, bool vec, const f32x4& v) {
  using S = typename Elem<DT>::S;
  S* s = reinterpret_cast<S*>(base) + at;
  if (vec) {
    if constexpr (DT == kF32) {
      *reinterpret_cast<f32x4*>(s) = v;
    } else {
      u32x2 b;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        b[h] = static_cast<uint32_t>(Elem<DT>::from_f32(v[2 * h])) |
               static_cast<uint32_t>(Elem<DT>::from_f32(v[2 * h + 1])) << 16;
      *reinterpret_cast<u32x2*>(s) = b;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < left) s[e] = Elem<DT>::from_f32(v[e]);
  }
}

// The bias of a column group of four (gated: of gate and up columns), and the residual of a row's.
template <int DT>
__device__ __forceinline__ f32x4 bias4(const ProductArgs& a, const ProductItem& it, int col, int left) {
  if (a.bias == nullptr || left <= 0) return f32x4{0.f, 0.f, 0.f, 0.f};
  return load4<DT>(a.bias, it.w * a.bias_ld + col, left, a.vec);
}
template <int DT>
__device__ __forceinline__ f32x4 res4(const ProductArgs& a, int64_t row, int col, int left) {
  if (a.res == nullptr || left <= 0) return f32x4{0.f, 0.f, 0.f, 0.f};
  return load4<DT>(a.res, row * a.res_ld + col, left, a.vec);
}

// Output columns col .. col + 3 of one row: product + bias -> z, activation, residual, one rounding. `left` of them
// exist.
template <int DT>
__device__ __forceinline__ void finish4(const ProductArgs& a, const ProductItem& it, int64_t row, int col, int left,
                                        f32x4 v, const f32x4& bias, const f32x4& res) {
  if (left <= 0) return;
  if (a.bias != nullptr) v += bias;
  if (a.z != nullptr) store4<kF32>(reinterpret_cast<char*>(a.z), row * a.z_ld + col, left, a.vec, v);
  if (a.act != kActNone) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = activate(a.act, v[e]);
  }
  if (a.res != nullptr) v += res;
  store4<DT>(a.out, it.g * a.out_group + row * a.out_ld + col, left, a.vec, v);
}

// The same of a gated product: gate and up columns of outputs col .. col + 3.
template <int DT>
__device__ __forceinline__ void finish4_gated(const ProductArgs& a, int64_t row, int col, int left, f32x4 gate, f32x4 up,
                                              const f32x4& gate_bias, const f32x4& up_bias, const f32x4& res) {
  if (left <= 0) return;
  if (a.bias != nullptr) {
    gate += gate_bias;
    up += up_bias;
  }
  if (a.z != nullptr) {
    store4<kF32>(reinterpret_cast<char*>(a.z), row * a.z_ld + col, left, a.vec, gate);
    store4<kF32>(reinterpret_cast<char*>(a.z), row * a.z_ld + a.out_cols + col, left, a.vec, up);
  }
  f32x4 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = activate(kActSilu, gate[e]) * up[e];
  if (a.res != nullptr) v += res;
  store4<DT>(a.out, row * a.out_ld + col, left, a.vec, v);
}

// Rows of no group (before the first, behind the last, of a group without weights): the residual's row, or zeros.
template <int DT>
__device__ __forceinline__ void fill_rows(const ProductArgs& a, int fb) {
  using S = typename Elem<DT>::S;
  if (a.offsets == nullptr) return;
  const int64_t total = a.rows;
  const int64_t lo = min(max(a.offsets[0], int64_t{0}), total);
  const int64_t hi = min(max(a.offsets[a.groups], lo), total);
  auto row = [&](int64_t r) {
    S* dst = reinterpret_cast<S*>(a.out) + r * a.out_ld;
    const S* src = reinterpret_cast<const S*>(a.res) + r * a.res_ld;
    for (int c = threadIdx.x; c < a.out_cols; c += kPThreads) dst[c] = a.res != nullptr ? src[c] : S{};
  };
  for (int64_t i = fb; i < lo + total - hi; i += a.fill_blocks) row(i < lo ? i : hi + i - lo);
  if (a.slots == nullptr) return;
  for (int g = 0; g < a.groups; ++g) {
    if (group_weight(a, g) >= 0) continue;
    int r0, n;
    group_bounds(a, g, a.rows, r0, n);
    for (int i = fb; i < n; i += a.fill_blocks) row(static_cast<int64_t>(r0) + i);
  }
}

// Launchers. Sizes and alignments that a kernel assumes are checked by the plan (products.hip) that chooses it.
struct TileShape {
  int bm, bn;   // output rows and columns of a workgroup (product columns: gated outputs take two)
  bool staged;  // operands go through registers: any alignment. Otherwise straight into LDS (whole 16-byte slots)
};
hipError_t launch_product_tile(int dtype, bool p_strided, bool q_strided, bool depth_groups, const TileShape& t,
                               const ProductArgs& a, hipStream_t s);


// 256 x 256 tiles, 16-bit types, sizes and pitches in whole 16-byte slots.
hipError_t launch_product_wide(int dtype, bool p_strided, bool q_strided, bool depth_groups, const ProductArgs& a,
                               hipStream_t s);

}  // namespace smx
