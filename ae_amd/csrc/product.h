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

#include <type_traits>

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
  int rows, cols;           // of the product; grouped along the rows: of all groups. A strided P may be padded: cols
                            // counts its columns, out_cols those of the result
  int q_cols;               // columns of a strided Q, at least rows
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
  int stream;               // results are stored past the caches
  int vec;                  // 4 consecutive outputs are one aligned store in every array
  int item_blocks;          // workgroups of the product; those behind fill rows of no group
  int fill_blocks;
};

// ---------------------------------------------------------------------------------------
// Groups
// ---------------------------------------------------------------------------------------

// The maps as constant memory (no kernel writes them): where the group is the same for the wave, a scalar load.
typedef const __attribute__((address_space(4))) int64_t* ConstMap;

// Row bounds of group g, inside [0, total] and in order whatever the caller's bounds hold.
__device__ __forceinline__ void group_bounds(const ProductArgs& a, int g, int total, int& lo, int& n) {
  if (a.offsets == nullptr) {
    lo = 0;
    n = total;
    return;
  }
  const ConstMap offsets = (ConstMap)(a.offsets);
  const int64_t b0 = offsets[g], b1 = offsets[g + 1];
  const int64_t c0 = min(max(b0, int64_t{0}), static_cast<int64_t>(total));
  const int64_t c1 = min(max(b1, c0), static_cast<int64_t>(total));
  lo = static_cast<int>(c0);
  n = static_cast<int>(c1 - c0);
}

// The group's P, or -1: a slot outside the pool holds no weights, and its rows are of no group.
__device__ __forceinline__ int64_t group_weight(const ProductArgs& a, int g) {
  if (a.slots == nullptr) return g;
  const int64_t s = ((ConstMap)(a.slots))[g];
  return s >= 0 && s < a.weights ? s : -1;
}

// fp32 sums run in chains of kFold steps (256 products; 288 where three stages are walked), whose results are added up: a
// single chain of thousands of products would lose a bit or two more than blocked sums do.
constexpr int kFold = 8;
template <int NI, int NJ>
__device__ __forceinline__ void fold(f32x4 (&total)[NI][NJ], f32x4 (&acc)[NI][NJ]) {
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      total[i][j] += acc[i][j];
      acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
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
  int rt = 0, lo = 0, n = 0, incl = 0, w = 0;
  auto scan = [&](int base) {
    const int g = base + lane;
    lo = n = 0;
    if (g < a.groups) {
      w = static_cast<int>(group_weight(a, g));  // (the host checks that there are fewer than 2^31)
      group_bounds(a, g, a.rows, lo, n);
      if (w < 0) n = 0;
    }
    incl = wave_incl_scan((n + bm - 1) / bm);
  };
  // (as many tiles as the grid was made for, whatever the caller's bounds hold: bounds that decrease name rows twice)
  const int most = a.rows / bm + min(a.groups, a.rows);
  for (int base = 0; base < a.groups; base += kWave) {
    scan(base);
    rt = min(rt + last_lane(incl), most);
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
      it.w = __builtin_amdgcn_readlane(w, l);
      return true;
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

// fp32 results: the library's exponential and complementary error function and IEEE quotients (an ulp or two).
// 16-bit results (step 2^-8 or 2^-11): the hardware's exponential and reciprocal, and the normal distribution function in
// the tail as exp(-z^2 / 2) times a polynomial in t = 1 / (1 + 0.36 |z|), fitted here to the least relative error
// over |z| <= 14 (1.2e-6 in fp32, the tail's own relative accuracy kept): 5 to 17 operations instead of 25 to 60 per
// value, which one wave per SIMD does not hide (256 x 256 tiles, 8192 x 4096 -> 14336: gelu_tanh cost 206 us
// of 1062, gelu 280 of 1136).
constexpr float kLog2e = 1.44269504f;
constexpr float kTanh0 = 1.59576912f, kTanh1 = 0.0713548163f;  // gelu's tanh form: z * sigmoid(z (kTanh0 + kTanh1 z^2))

template <bool EXACT>
__device__ __forceinline__ float sigmoid_f32(float z) {
  if constexpr (EXACT) return 1.0f / (1.0f + expf(-z));
  else return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -kLog2e));
}
// exp(-z^2 / 2).
template <bool EXACT>
__device__ __forceinline__ float bell_f32(float z) {
  if constexpr (EXACT) return expf(-0.5f * z * z);
  else return __builtin_amdgcn_exp2f(z * z * (-0.5f * kLog2e));
}
// Normal distribution function of -|z|, bell = exp(-z^2 / 2).
template <bool EXACT>
__device__ __forceinline__ float normal_tail(float z, float bell) {
  if constexpr (EXACT) {
    return 0.5f * erfcf(fabsf(z) * 0.70710678f);
  } else {
    const float t = __builtin_amdgcn_rcpf(fmaf(0.36f, fabsf(z), 1.0f));
    float p = 0.0470067784f;
    p = fmaf(p, t, -0.179588974f);
    p = fmaf(p, t, 0.180709541f);
    p = fmaf(p, t, 0.0267180651f);
    p = fmaf(p, t, 0.139659077f);
    p = fmaf(p, t, 0.141782865f);
    p = fmaf(p, t, 0.143712372f);
    return p * t * bell;
  }
}
template <bool EXACT>
__device__ __forceinline__ float normal_cdf(float z, float bell) {
  const float c = normal_tail<EXACT>(z, bell);
  return z > 0.0f ? 1.0f - c : c;
}

template <bool EXACT>
__device__ __forceinline__ float activate(int act, float z) {
  switch (act) {
    case kActRelu: return z < 0.0f ? 0.0f : z;
    case kActGelu: return z * normal_cdf<EXACT>(z, bell_f32<EXACT>(z));
    case kActGeluTanh: return z * sigmoid_f32<EXACT>(z * fmaf(kTanh1 * z, z, kTanh0));
    case kActSilu: return z * sigmoid_f32<EXACT>(z);
    default: return z;
  }
}

// The activation of N groups of four (one branch for all of them: the operations of different values overlap).
template <bool EXACT, int N>
__device__ __forceinline__ void activate_all(int act, f32x4 (&v)[N]) {
  auto each = [&](auto code) {
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[n][e] = activate<EXACT>(decltype(code)::value, v[n][e]);
  };
  switch (act) {
    case kActRelu: each(std::integral_constant<int, kActRelu>{}); break;
    case kActGelu: each(std::integral_constant<int, kActGelu>{}); break;
    case kActGeluTanh: each(std::integral_constant<int, kActGeluTanh>{}); break;
    case kActSilu: each(std::integral_constant<int, kActSilu>{}); break;
    default: break;
  }
}

// d act / dz of a smooth activation. The slope terms vanish faster than any power of z grows: 0 where they underflow, also
// at infinity.
template <bool EXACT>
__device__ __forceinline__ float activate_grad(int act, float z) {
  switch (act) {
    case kActGelu: {
      const float e = bell_f32<EXACT>(z), c = normal_cdf<EXACT>(z, e);
      return e == 0.0f ? c : fmaf(z, 0.398942280f * e, c);
    }
    case kActGeluTanh: {
      const float s = sigmoid_f32<EXACT>(z * fmaf(kTanh1 * z, z, kTanh0)), t = s * (1.0f - s);
      return t == 0.0f ? s : fmaf(z * t, fmaf(3.0f * kTanh1 * z, z, kTanh0), s);
    }
    case kActSilu: {
      const float s = sigmoid_f32<EXACT>(z), t = s * (1.0f - s);
      return t == 0.0f ? s : fmaf(z, t, s);
    }
    default: return 1.0f;
  }
}

// d times d act / dz, of N groups of four.
template <bool EXACT, int N>
__device__ __forceinline__ void activate_grad_all(int act, const f32x4 (&z)[N], f32x4 (&d)[N]) {
  auto each = [&](auto code) {
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // relu selects: a closed one passes nothing on, infinities and NaN neither
        if constexpr (decltype(code)::value == kActRelu) d[n][e] = z[n][e] > 0.0f ? d[n][e] : (z[n][e] != z[n][e] ? z[n][e] : 0.0f);
        else d[n][e] *= activate_grad<EXACT>(decltype(code)::value, z[n][e]);
      }
  };
  switch (act) {
    case kActRelu: each(std::integral_constant<int, kActRelu>{}); break;
    case kActGelu: each(std::integral_constant<int, kActGelu>{}); break;
    case kActGeluTanh: each(std::integral_constant<int, kActGeluTanh>{}); break;
    case kActSilu: each(std::integral_constant<int, kActSilu>{}); break;
    default: break;
  }
}

// A 16-byte slot of T's of an operand in memory, of any alignment: `have` of its elements exist, the others are 0.
template <int DT>
__device__ __forceinline__ u32x4 load_slot(const typename Elem<DT>::S* at, int have) {
  using S = typename Elem<DT>::S;
  constexpr int kEps = 16 / sizeof(S);
  u32x4 r = {0, 0, 0, 0};
  if (have >= kEps) {
    __builtin_memcpy(&r, at, 16);
  } else if (have > 0) {
    S e[kEps];
#pragma unroll
    for (int i = 0; i < kEps; ++i) e[i] = i < have ? at[i] : S{};
    __builtin_memcpy(&r, e, 16);
  }
  return r;
}

// Four consecutive elements of an array of T (DT), of which `left` exist: one access where all four do (`vec`: an aligned
// one).
template <int DT>
__device__ __forceinline__ f32x4 load4(const char* base, int64_t at, int left, bool vec) {
  using S = typename Elem<DT>::S;
  const S* s = reinterpret_cast<const S*>(base) + at;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  auto widen = [&](const u32x2& b) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = Elem<DT>::to_f32(static_cast<typename Elem<DT>::S>(b[e >> 1] >> (16 * (e & 1))));
  };
  if constexpr (DT == kF32) {
    if (vec) v = *reinterpret_cast<const f32x4*>(s);
    else if (left >= 4) __builtin_memcpy(&v, s, 16);
  } else {
    u32x2 b;
    if (vec) {
      widen(*reinterpret_cast<const u32x2*>(s));
    } else if (left >= 4) {
      __builtin_memcpy(&b, s, 8);
      widen(b);
    }
  }
  if (!vec && left < 4) {
#pragma unroll
    for (int e = 0; e < 3; ++e)
      if (e < left) v[e] = Elem<DT>::to_f32(s[e]);
  }
  return v;
}

// Four values rounded to T, as they lie in memory.
template <int DT>
__device__ __forceinline__ auto pack4(const f32x4& v) {
  typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
  typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
  if constexpr (DT == kF32) return v;
  else if constexpr (DT == kBF16) return __builtin_bit_cast(u32x2, __builtin_convertvector(v, bf16x4));
  else return __builtin_bit_cast(u32x2, __builtin_convertvector(v, f16x4));
}

// stream: past the caches.
template <int DT>
__device__ __forceinline__ void store4(char* base, int64_t at, int left, bool vec, const f32x4& v, bool stream = false) {
  using S = typename Elem<DT>::S;
  S* s = reinterpret_cast<S*>(base) + at;
  const auto b = pack4<DT>(v);
  using B = std::remove_const_t<decltype(b)>;
  if (vec && stream) {
    __builtin_nontemporal_store(b, reinterpret_cast<B*>(s));
  } else if (vec) {
    *reinterpret_cast<B*>(s) = b;
  } else if (left >= 4) {
    __builtin_memcpy(s, &b, sizeof b);
  } else {
#pragma unroll
    for (int e = 0; e < 3; ++e)
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

// N rows' output columns col .. col + 3 (of row[n]; `left` of the columns exist, where in[n]): product + bias -> z,
// activation, residual, one rounding.
template <int DT, int N>
__device__ __forceinline__ void finish_rows(const ProductArgs& a, const ProductItem& it, const int64_t (&row)[N],
                                            const bool (&in)[N], int col, int left, f32x4 (&v)[N], const f32x4& bias,
                                            const f32x4 (&res)[N]) {
  if (left <= 0) return;
  if (a.bias != nullptr) {
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] += bias;
  }
  if (a.z != nullptr) {
#pragma unroll
    for (int n = 0; n < N; ++n)
      if (in[n]) store4<kF32>(reinterpret_cast<char*>(a.z), row[n] * a.z_ld + col, left, a.vec, v[n], a.stream);
  }
  activate_all<DT == kF32>(a.act, v);
  if (a.res != nullptr) {
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] += res[n];
  }
#pragma unroll
  for (int n = 0; n < N; ++n)
    if (in[n]) store4<DT>(a.out, it.g * a.out_group + row[n] * a.out_ld + col, left, a.vec, v[n], a.stream);
}

// The same of a gated product: gate and up columns of outputs col .. col + 3.
template <int DT, int N>
__device__ __forceinline__ void finish_rows_gated(const ProductArgs& a, const int64_t (&row)[N], const bool (&in)[N],
                                                  int col, int left, f32x4 (&gate)[N], f32x4 (&up)[N],
                                                  const f32x4& gate_bias, const f32x4& up_bias, const f32x4 (&res)[N]) {
  if (left <= 0) return;
  if (a.bias != nullptr) {
#pragma unroll
    for (int n = 0; n < N; ++n) gate[n] += gate_bias, up[n] += up_bias;
  }
  if (a.z != nullptr) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if (!in[n]) continue;
      store4<kF32>(reinterpret_cast<char*>(a.z), row[n] * a.z_ld + col, left, a.vec, gate[n], a.stream);
      store4<kF32>(reinterpret_cast<char*>(a.z), row[n] * a.z_ld + a.out_cols + col, left, a.vec, up[n], a.stream);
    }
  }
  activate_all<DT == kF32>(kActSilu, gate);
#pragma unroll
  for (int n = 0; n < N; ++n) {
    gate[n] *= up[n];
    if (a.res != nullptr) gate[n] += res[n];
    if (in[n]) store4<DT>(a.out, row[n] * a.out_ld + col, left, a.vec, gate[n], a.stream);
  }
}

// One row of either kind.
template <int DT>
__device__ __forceinline__ void finish4(const ProductArgs& a, const ProductItem& it, int64_t row, int col, int left,
                                        const f32x4& v, const f32x4& up, const f32x4& bias, const f32x4& up_bias,
                                        const f32x4& res) {
  const int64_t rows[1] = {row};
  const bool in[1] = {true};
  const f32x4 r[1] = {res};
  f32x4 x[1] = {v}, u[1] = {up};
  if (a.gated) finish_rows_gated<DT, 1>(a, rows, in, col, left, x, u, bias, up_bias, r);
  else finish_rows<DT, 1>(a, it, rows, in, col, left, x, bias, r);
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
  int bm, bn;  // output rows and columns of a workgroup (product columns: gated outputs take two)
  // The kernel: operands through registers (any alignment) or straight into LDS (whole 16-byte slots)
  enum Form { kStaged, kCopied, kWide, kRows, kRowsStaged, kShallow } form;
};
// kStaged: 64 x 64. kCopied: 128 x 128, 64 x 64, and not grouped along the contraction 64 x 128, 32 x 128.
hipError_t launch_product_tile(int dtype, bool p_strided, bool q_strided, bool depth_groups, const TileShape& t,
                               const ProductArgs& a, hipStream_t s);
// kShallow: 128 x 128, grouped along the contraction, no splits.
hipError_t launch_product_shallow(int dtype, const ProductArgs& a, hipStream_t s);
// kWide: 16-bit types, 256 x 256.
hipError_t launch_product_wide(int dtype, bool p_strided, bool q_strided, bool depth_groups, const ProductArgs& a,
                               hipStream_t s);
// Forward, no splits. kRows: 16 x 16 (not gated), 16 x 32, 32 x 32, 64 x 64. kRowsStaged: 16 x 32, 32 x 32.
hipError_t launch_product_rows(int dtype, const TileShape& t, const ProductArgs& a, hipStream_t s);

}  // namespace smx
