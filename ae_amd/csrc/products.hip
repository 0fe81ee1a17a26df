// Matrix products with an epilogue: the C entry points, the choice of kernels, and the elementwise kernels (gradient
// of the activation with the bias gradient's column sums, joining of contraction splits).
#include "../../include/specmoe_mi355x.h"
#include "../../include/specmoe_mi355x_products.h"
#include <algorithm>
#include <cmath>

#include "product.h"

namespace smx {

constexpr int kGradRows = 64;   // rows of a workgroup of the activation gradient
constexpr int kGradCols = 256;  // its output columns: 64 lanes of 4, the 4 waves take rows in turn
constexpr int kJoinRows = 4;    // rows of a workgroup that joins splits, one per wave

// dz = dy * act'(z), rounded into dz (unless null), and its fp32 column sums over the workgroup's rows.
struct ActGradArgs {
  ProductArgs p;          // groups; rows; cols = columns of z; out_cols; gated; act
  const char* dy;
  int64_t dy_ld;
  const float* z;         // null where act is the identity
  int64_t z_ld;
  char* dz;
  int64_t dz_ld;
  float* sums;            // [max_tiles][cols], or null
  int max_tiles;
};

template <int DT>
__global__ __launch_bounds__(kPThreads) void act_grad_kernel(ActGradArgs a) {
  const int col_tiles = (a.p.out_cols + kGradCols - 1) / kGradCols;
  ProductItem it;
  if (!find_row_item(a.p, static_cast<int>(blockIdx.x), kGradRows, col_tiles, it)) return;
  __shared__ f32x4 lds[2][kPWaves][kWave];
  const int lane = lane_id(), wave = wave_id();
  const int col = it.ct * kGradCols + 4 * lane;
  const int left = a.p.out_cols - col;
  const bool vec = a.p.vec;
  f32x4 sum[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
  if (left > 0) {
    for (int r = wave; r < it.m; r += kPWaves) {
      const int64_t row = it.row + r;
      const f32x4 dy = load4<DT>(a.dy, row * a.dy_ld + col, left, vec);
      if (a.p.gated) {
        const char* z = reinterpret_cast<const char*>(a.z);
        const f32x4 g = load4<kF32>(z, row * a.z_ld + col, left, vec);
        const f32x4 u = load4<kF32>(z, row * a.z_ld + a.p.out_cols + col, left, vec);
        f32x4 dg, du;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          dg[e] = dy[e] * u[e] * activate_grad(kActSilu, g[e]);
          du[e] = dy[e] * activate(kActSilu, g[e]);
        }
        store4<DT>(a.dz, row * a.dz_ld + col, left, vec, dg);
        store4<DT>(a.dz, row * a.dz_ld + a.p.out_cols + col, left, vec, du);
        sum[0] += dg;
        sum[1] += du;
      } else {
        f32x4 d = dy;
        if (a.z != nullptr) {
          const f32x4 z = load4<kF32>(reinterpret_cast<const char*>(a.z), row * a.z_ld + col, left, vec);
#pragma unroll
          for (int e = 0; e < 4; ++e) d[e] *= activate_grad(a.p.act, z[e]);
        }
        if (a.dz != nullptr) store4<DT>(a.dz, row * a.dz_ld + col, left, vec, d);
        sum[0] += d;
      }
    }
  }
  if (a.sums == nullptr) return;
  // the row tile's own place: row tiles of the groups before it, and of its group before it
  int tile = 0;
  if (a.p.offsets == nullptr) {
    tile = it.row / kGradRows;
  } else {
    for (int base = 0; base <= it.g; base += kWave) {
      int lo = 0, n = 0;
      if (base + lane <= it.g) group_bounds(a.p, base + lane, a.p.rows, lo, n);
      if (base + lane == it.g) n = it.row - lo;  // whole tiles
      tile += last_lane(wave_incl_scan((n + kGradRows - 1) / kGradRows));
    }
  }
  lds[0][wave][lane] = sum[0];
  lds[1][wave][lane] = sum[1];
  __syncthreads();
  // (tiles past max_tiles: row bounds that decrease)
  if (wave >= (a.p.gated ? 2 : 1) || left <= 0 || tile >= a.max_tiles) return;
  f32x4 v = lds[wave][0][lane];
#pragma unroll
  for (int w = 1; w < kPWaves; ++w) v += lds[wave][w][lane];
  store4<kF32>(reinterpret_cast<char*>(a.sums), static_cast<int64_t>(tile) * a.p.cols + wave * a.p.out_cols + col, left,
               false, v);
}

// Bias gradient: the group's row tiles' sums, added in order.
template <int DT>
__global__ __launch_bounds__(kPThreads) void bias_grad_kernel(ProductArgs p, const float* sums, int max_tiles, char* grad) {
  using S = typename Elem<DT>::S;
  const int cb = (p.cols + kWave - 1) / kWave;
  const int g = static_cast<int>(blockIdx.x) / cb;
  const int lane = lane_id(), wave = wave_id();
  const int col = (static_cast<int>(blockIdx.x) - g * cb) * kWave + lane;
  int first = 0, count = 0;
  for (int base = 0; base <= g; base += kWave) {
    int lo = 0, n = 0;
    if (base + lane <= g) group_bounds(p, base + lane, p.rows, lo, n);
    const int t = (n + kGradRows - 1) / kGradRows;
    if (base + kWave > g) count = __builtin_amdgcn_readlane(t, g - base);
    first += last_lane(wave_incl_scan(t));
  }
  first -= count;
  count = min(count, max_tiles - first);
  __shared__ float lds[kPWaves][kWave];
  float v = 0.0f;
  if (col < p.cols)
    for (int t = wave; t < count; t += kPWaves) v += sums[static_cast<int64_t>(first + t) * p.cols + col];
  lds[wave][lane] = v;
  __syncthreads();
  if (wave > 0 || col >= p.cols) return;
  for (int w = 1; w < kPWaves; ++w) v += lds[w][lane];
  reinterpret_cast<S*>(grad)[static_cast<int64_t>(g) * p.cols + col] = Elem<DT>::from_f32(v);
}

// Joins the contraction splits: one row per wave, 256 output columns.
template <int DT>
__global__ __launch_bounds__(kPThreads) void join_kernel(ProductArgs a, int splits) {
  const int b = static_cast<int>(blockIdx.x);
  if (b >= a.item_blocks) {
    fill_rows<DT>(a, b - a.item_blocks);
    return;
  }
  ProductItem it;
  const int col_tiles = (a.out_cols + kGradCols - 1) / kGradCols;
  if (!find_row_item(a, b, kJoinRows, col_tiles, it)) return;
  const int r = wave_id();
  const int col = it.ct * kGradCols + 4 * lane_id();
  const int left = a.out_cols - col;
  if (r >= it.m || left <= 0) return;
  const int64_t row = it.row + r;
  const bool vec = a.cols % 4 == 0 && a.out_cols % 4 == 0;
  const char* part = reinterpret_cast<const char*>(a.part);
  f32x4 v = {0.f, 0.f, 0.f, 0.f}, u = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < splits; ++s) {
    const int64_t at = (static_cast<int64_t>(s) * a.rows + row) * a.cols + col;
    v += load4<kF32>(part, at, left, vec);
    if (a.gated) u += load4<kF32>(part, at + a.out_cols, left, vec);
  }
  const f32x4 bias = bias4<DT>(a, it, col, left), res = res4<DT>(a, row, col, left);
  if (a.gated) finish4_gated<DT>(a, row, col, left, v, u, bias, bias4<DT>(a, it, a.out_cols + col, left), res);
  else finish4<DT>(a, it, row, col, left, v, bias, res);
}

namespace {

constexpr int64_t kMaxSize = int64_t{1} << 30;
constexpr int kFillBlocks = 64;

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }
bool aligned(const void* p, int64_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
bool valid_dtype(int dt) { return dt == kF32 || dt == kF16 || dt == kBF16; }

enum Kind { kForward, kInputGrad, kWeightGrad };

// How a product runs.
struct ProductPlan {
  TileShape tile{64, 64, true};
  int splits = 1, split_steps = 0;
  int64_t part_bytes = 0;
};

// Tiles of the copied kernels with the time of one contraction step (us, 128 bytes of it) when 1, 2, .. workgroups run
// on a CU, as many as fit (bf16, 4096 x 4096 weight, 1 to 8192 rows).
struct TileCost {
  int bm, bn, fit;
  float step[4];
};
constexpr TileCost kTileCosts[] = {
    {256, 256, 1, {1.6f, 0.f, 0.f, 0.f}},
    {128, 128, 2, {0.70f, 1.06f, 0.f, 0.f}},
    {64, 128, 3, {0.46f, 0.66f, 0.97f, 0.f}},
    {32, 128, 4, {0.38f, 0.50f, 0.75f, 0.96f}},
};
constexpr int kCUs = 256;

// slots: both operands consist of whole 16-byte slots (see launch_product_*).
ProductPlan plan_product(Kind kind, int dtype, int64_t rows, int64_t cols, int64_t depth, int64_t groups, bool gated,
                         bool slots) {
  ProductPlan p;
  if (!slots || rows == 0) return p;
  const bool depth_groups = kind == kWeightGrad;
  const double mean_depth = depth_groups ? static_cast<double>(depth) / groups : static_cast<double>(depth);
  const double steps = std::max(1.0, mean_depth / (kPStep / dtype_bytes(dtype)));
  double best = 0;
  for (const TileCost& t : kTileCosts) {
    if (t.bm == 256 && dtype == kF32) continue;
    if (kind == kWeightGrad && t.bm < 128) continue;
    // row tiles: of every group with rows, half a tile more than its rows fill
    double row_tiles = static_cast<double>(cdiv(rows, t.bm));
    if (!depth_groups && groups > 1) {
      const double active = static_cast<double>(std::min(groups, rows));
      row_tiles = std::max(active, static_cast<double>(rows) / t.bm + active / 2);
    }
    const double tiles = row_tiles * static_cast<double>(cdiv(cols, t.bn)) * (depth_groups ? groups : 1);
    for (int splits = 1; splits <= 16; splits *= 2) {
      if (splits > 1 && (t.bm == 256 || (depth_groups && groups > 1) || splits * 4 > steps)) break;
      double per_cu = std::ceil(tiles * splits / kCUs), time = 0;
      const double len = steps / splits + 6;  // and the ends of a tile
      time += std::floor(per_cu / t.fit) * t.step[t.fit - 1] * len;
      const int rest = static_cast<int>(per_cu) % t.fit;
      if (rest > 0) time += t.step[rest - 1] * len;
      if (splits > 1) time += 5.0 + 8.0 * splits * rows * cols / 4e6;  // the joining launch, partial sums out and in
      if (best == 0 || time < best) {
        best = time;
        p.tile = TileShape{t.bm, t.bn, false};
        const int64_t all = cdiv(depth, kPStep / dtype_bytes(dtype));
        p.split_steps = static_cast<int>(cdiv(all, splits));
        p.splits = splits == 1 ? 1 : static_cast<int>(cdiv(all, p.split_steps));
        p.part_bytes = p.splits > 1 ? p.splits * rows * cols * 4 : 0;
      }
    }
  }
  return p;
}

// Row tiles of at most: every group may end in a part of a tile.
int64_t max_row_tiles(int64_t rows, int64_t groups, int bm) {
  return groups <= 1 ? cdiv(rows, bm) : rows / bm + std::min(groups, rows);
}

int run_product(Kind kind, int dtype, const ProductPlan& plan, ProductArgs& a, bool fill, hipStream_t s) {
  const int64_t ct = a.gated ? cdiv(a.out_cols, plan.tile.bn / 2) : cdiv(a.cols, plan.tile.bn);
  const bool depth_groups = kind == kWeightGrad;
  int64_t items = depth_groups ? cdiv(a.rows, plan.tile.bm) * ct * a.groups : max_row_tiles(a.rows, a.groups, plan.tile.bm) * ct;
  items *= plan.splits;
  const int fills = fill && a.offsets != nullptr ? kFillBlocks : 0;
  if (items + fills > INT32_MAX) return SMX_ERR_UNSUPPORTED;
  if (items + fills == 0) return SMX_OK;
  a.splits = plan.splits;
  a.split_steps = plan.split_steps;
  a.item_blocks = static_cast<int>(items);
  a.fill_blocks = plan.splits > 1 ? 0 : fills;
  hipError_t err = plan.tile.bm == 256
                       ? launch_product_wide(dtype, kind != kForward, kind == kWeightGrad, depth_groups, a, s)
                       : launch_product_tile(dtype, kind != kForward, kind == kWeightGrad, depth_groups, plan.tile, a, s);
  if (err != hipSuccess || plan.splits == 1) return static_cast<int>(err);
  const int splits = a.splits;
  a.splits = 1;
  const int64_t joins = max_row_tiles(a.rows, a.groups, kJoinRows) * cdiv(a.out_cols, kGradCols);
  if (joins + fills > INT32_MAX) return SMX_ERR_UNSUPPORTED;
  a.item_blocks = static_cast<int>(joins);
  a.fill_blocks = fills;
  const unsigned blocks = static_cast<unsigned>(joins + fills);
  switch (dtype) {
    case kF32: join_kernel<kF32><<<blocks, kPThreads, 0, s>>>(a, splits); break;
    case kF16: join_kernel<kF16><<<blocks, kPThreads, 0, s>>>(a, splits); break;
    default: join_kernel<kBF16><<<blocks, kPThreads, 0, s>>>(a, splits); break;
  }
  return static_cast<int>(hipGetLastError());
}

// Sizes of a call, checked.
struct Sizes {
  int64_t rows, K, N, Nw, G;  // G: groups, at least 1
  bool grouped;
  int dtype, act;
  int64_t es;
};

int check_sizes(int64_t rows, int64_t K, int64_t N, int64_t G, int act, int dtype, Sizes& z) {
  if (rows < 0 || K <= 0 || N <= 0 || G < 0 || act < SMX_ACT_NONE || act > SMX_ACT_SWIGLU || !valid_dtype(dtype))
    return SMX_ERR_INVALID_ARG;
  if (rows > kMaxSize || K > kMaxSize || N > kMaxSize / 2 || G > kMaxSize) return SMX_ERR_UNSUPPORTED;
  z = Sizes{rows, K, N, act == SMX_ACT_SWIGLU ? 2 * N : N, std::max<int64_t>(G, 1), G > 0, dtype, act, dtype_bytes(dtype)};
  return SMX_OK;
}

int check_pitch(int64_t stride, int64_t len, int64_t es) {
  if (stride < len) return SMX_ERR_INVALID_ARG;
  return stride * es > kPMaxPitch ? SMX_ERR_UNSUPPORTED : SMX_OK;
}

struct GradLayout {
  ProductPlan dx, dw;
  int64_t dz = 0, dz_ld = 0, sums = 0, part = 0, total = 0;
};

// Whole 16-byte slots: the base and the pitch, and the length of whatever lies side by side.
bool whole_slots(const void* base, int64_t pitch, int64_t length, int64_t es) {
  return aligned(base, 16) && pitch * es % 16 == 0 && length * es % 16 == 0;
}

GradLayout grad_layout(const Sizes& z, bool dx_slots, bool dw_slots) {
  GradLayout l;
  l.dx = plan_product(kInputGrad, z.dtype, z.rows, z.K, z.Nw, z.G, false, dx_slots);
  l.dw = plan_product(kWeightGrad, z.dtype, z.Nw, z.K, z.rows, z.G, false, dw_slots);
  l.dz_ld = cdiv(z.Nw, 16 / z.es) * (16 / z.es);
  int64_t at = 0;
  if (z.act != SMX_ACT_NONE) at += align256(z.rows * l.dz_ld * z.es);
  l.sums = at;
  at += align256(max_row_tiles(z.rows, z.G, kGradRows) * z.Nw * 4);
  l.part = at;
  at += align256(std::max(l.dx.part_bytes, l.dw.part_bytes));
  l.total = at;
  return l;
}

struct Groups {
  const int64_t* offsets = nullptr;
  const int64_t* slots = nullptr;
  int64_t stride = 0, weights = 1;
};

int check_groups(const Sizes& z, const Groups& g) {
  if (!z.grouped) return SMX_OK;
  if (!g.offsets || g.weights <= 0 || g.stride < 0) return SMX_ERR_INVALID_ARG;
  if (!g.slots && g.weights != z.G) return SMX_ERR_INVALID_ARG;
  if (!aligned(g.offsets, 8) || !aligned(g.slots, 8)) return SMX_ERR_MISALIGNED;
  return SMX_OK;
}

ProductArgs group_args(const Sizes& z, const Groups& g) {
  ProductArgs a{};
  a.rows = static_cast<int>(z.rows);
  a.offsets = g.offsets;
  a.slots = g.slots;
  a.weights = g.weights;
  a.groups = static_cast<int>(z.G);
  a.splits = 1;
  return a;
}

int forward(const Sizes& z, const void* x, int64_t x_stride, const void* weight, int64_t weight_stride, const Groups& g,
            const void* bias, const void* residual, int64_t residual_stride, bool fill, void* y, int64_t y_stride,
            float* preact, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_groups(z, g);
  if (rc == SMX_OK) rc = check_pitch(weight_stride, z.K, z.es);
  if (rc == SMX_OK) rc = check_pitch(x_stride, z.K, z.es);
  if (rc == SMX_OK) rc = check_pitch(y_stride, z.N, z.es);
  if (rc == SMX_OK && residual) rc = check_pitch(residual_stride, z.N, z.es);
  if (rc != SMX_OK) return rc;
  if (z.Nw * weight_stride * z.es >= int64_t{kPOutside}) return SMX_ERR_UNSUPPORTED;
  if (z.rows == 0) return SMX_OK;
  if (!x || !weight || !y) return SMX_ERR_INVALID_ARG;
  if (!aligned(x, z.es) || !aligned(weight, z.es) || !aligned(y, z.es) || !aligned(bias, z.es) ||
      !aligned(residual, z.es) || !aligned(preact, 4))
    return SMX_ERR_MISALIGNED;
  const bool slots = whole_slots(x, x_stride, z.K, z.es) && whole_slots(weight, weight_stride, z.K, z.es) &&
                     g.stride * z.es % 16 == 0;
  const ProductPlan plan = plan_product(kForward, z.dtype, z.rows, z.Nw, z.K, z.G, z.Nw != z.N, slots);
  if (plan.part_bytes > 0) {
    if (!workspace || workspace_bytes < static_cast<size_t>(plan.part_bytes)) return SMX_ERR_WORKSPACE;
    if (!aligned(workspace, 16)) return SMX_ERR_MISALIGNED;
  }
  ProductArgs a = group_args(z, g);
  a.q = static_cast<const char*>(x);
  a.q_ld = x_stride;
  a.p = static_cast<const char*>(weight);
  a.p_ld = weight_stride;
  a.p_group = g.stride;
  a.cols = static_cast<int>(z.Nw);
  a.depth = static_cast<int>(z.K);
  a.gated = z.Nw != z.N;
  a.out = static_cast<char*>(y);
  a.out_ld = y_stride;
  a.bias = static_cast<const char*>(bias);
  a.bias_ld = z.Nw;
  a.res = static_cast<const char*>(residual);
  a.res_ld = residual_stride;
  a.z = preact;
  a.z_ld = z.Nw;
  a.part = static_cast<float*>(workspace);
  a.act = a.gated ? kActNone : z.act;
  a.out_cols = static_cast<int>(z.N);
  const int64_t v = 4 * z.es;
  a.vec = z.N % 4 == 0 && y_stride % 4 == 0 && aligned(y, v) && aligned(bias, v) && aligned(preact, 16) &&
          (!residual || (residual_stride % 4 == 0 && aligned(residual, v)));
  return run_product(kForward, z.dtype, plan, a, fill, static_cast<hipStream_t>(stream));
}

int gradients(const Sizes& z, const void* dy, int64_t dy_stride, const float* preact, const void* x, int64_t x_stride,
              const void* weight, int64_t weight_stride, const Groups& g, void* grad_x, void* grad_weight,
              void* grad_bias, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_groups(z, g);
  if (rc == SMX_OK) rc = check_pitch(weight_stride, z.K, z.es);
  if (rc == SMX_OK) rc = check_pitch(x_stride, z.K, z.es);
  if (rc == SMX_OK) rc = check_pitch(dy_stride, z.N, z.es);
  if (rc != SMX_OK) return rc;
  if (g.slots && (grad_weight || grad_bias)) return SMX_ERR_INVALID_ARG;
  // dz is dy itself, or rows of whole slots in the workspace
  const bool own_dz = z.act != SMX_ACT_NONE;
  const bool dz_slots = z.Nw * z.es % 16 == 0 && (own_dz || whole_slots(dy, dy_stride, z.N, z.es));
  const bool dx_slots = dz_slots && whole_slots(weight, weight_stride, z.K, z.es) && g.stride * z.es % 16 == 0;
  const bool dw_slots = dz_slots && whole_slots(x, x_stride, z.K, z.es);
  const GradLayout l = grad_layout(z, dx_slots, dw_slots);
  if (l.dz_ld * z.es > kPMaxPitch || z.K * z.es > kPMaxPitch) return SMX_ERR_UNSUPPORTED;
  if (z.rows > 0) {
    if (!dy || (grad_weight && !x) || (grad_x && !weight) || (z.act != SMX_ACT_NONE && !preact)) return SMX_ERR_INVALID_ARG;
    if (!aligned(dy, z.es) || !aligned(x, z.es) || !aligned(weight, z.es) || !aligned(preact, 4)) return SMX_ERR_MISALIGNED;
    if (l.total > 0 && (!workspace || workspace_bytes < static_cast<size_t>(l.total))) return SMX_ERR_WORKSPACE;
  }
  if (!aligned(grad_x, z.es) || !aligned(grad_weight, z.es) || !aligned(grad_bias, z.es) || !aligned(workspace, 16))
    return SMX_ERR_MISALIGNED;
  hipStream_t s = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  const void* dz = dy;
  int64_t dz_ld = dy_stride;
  ActGradArgs ag{};
  ag.p = group_args(z, g);
  ag.p.cols = static_cast<int>(z.Nw);
  ag.p.out_cols = static_cast<int>(z.N);
  ag.p.gated = z.Nw != z.N;
  ag.p.act = z.act;
  ag.max_tiles = static_cast<int>(max_row_tiles(z.rows, z.G, kGradRows));
  if (z.rows > 0 && (z.act != SMX_ACT_NONE || grad_bias)) {
    ag.dy = static_cast<const char*>(dy);
    ag.dy_ld = dy_stride;
    ag.p.vec = z.N % 4 == 0 && dy_stride % 4 == 0 && aligned(dy, 4 * z.es);
    if (z.act != SMX_ACT_NONE) {
      ag.z = preact;
      ag.z_ld = z.Nw;
      ag.dz = ws + l.dz;
      ag.dz_ld = l.dz_ld;
      ag.p.vec = ag.p.vec && aligned(preact, 16);
      dz = ag.dz;
      dz_ld = l.dz_ld;
    }
    if (grad_bias) ag.sums = reinterpret_cast<float*>(ws + l.sums);
    const int64_t blocks = max_row_tiles(z.rows, z.G, kGradRows) * cdiv(z.N, kGradCols);
    if (blocks > INT32_MAX) return SMX_ERR_UNSUPPORTED;
    const unsigned n = static_cast<unsigned>(blocks);
    switch (z.dtype) {
      case kF32: act_grad_kernel<kF32><<<n, kPThreads, 0, s>>>(ag); break;
      case kF16: act_grad_kernel<kF16><<<n, kPThreads, 0, s>>>(ag); break;
      default: act_grad_kernel<kBF16><<<n, kPThreads, 0, s>>>(ag); break;
    }
    hipError_t err = hipGetLastError();
    if (err != hipSuccess) return static_cast<int>(err);
  }
  if (grad_bias) {
    const int64_t blocks = z.G * cdiv(z.Nw, kWave);
    if (blocks > INT32_MAX) return SMX_ERR_UNSUPPORTED;
    const unsigned n = static_cast<unsigned>(blocks);
    const float* sums = reinterpret_cast<const float*>(ws + l.sums);
    char* out = static_cast<char*>(grad_bias);
    switch (z.dtype) {
      case kF32: bias_grad_kernel<kF32><<<n, kPThreads, 0, s>>>(ag.p, sums, ag.max_tiles, out); break;
      case kF16: bias_grad_kernel<kF16><<<n, kPThreads, 0, s>>>(ag.p, sums, ag.max_tiles, out); break;
      default: bias_grad_kernel<kBF16><<<n, kPThreads, 0, s>>>(ag.p, sums, ag.max_tiles, out); break;
    }
    hipError_t err = hipGetLastError();
    if (err != hipSuccess) return static_cast<int>(err);
  }
  if (grad_x && z.rows > 0) {
    ProductArgs a = group_args(z, g);
    a.q = static_cast<const char*>(dz);
    a.q_ld = dz_ld;
    a.p = static_cast<const char*>(weight);
    a.p_ld = weight_stride;
    a.p_group = g.stride;
    a.cols = a.out_cols = static_cast<int>(z.K);
    a.depth = static_cast<int>(z.Nw);
    a.out = static_cast<char*>(grad_x);
    a.out_ld = z.K;
    a.part = reinterpret_cast<float*>(ws + l.part);
    a.vec = z.K % 4 == 0 && aligned(grad_x, 4 * z.es);
    rc = run_product(kInputGrad, z.dtype, l.dx, a, true, s);
    if (rc != SMX_OK) return rc;
  }
  if (grad_weight) {
    ProductArgs a = group_args(z, g);
    a.q = static_cast<const char*>(dz);
    a.q_ld = dz_ld;
    a.p = static_cast<const char*>(x);
    a.p_ld = x_stride;
    a.rows = static_cast<int>(z.Nw);
    a.cols = a.out_cols = static_cast<int>(z.K);
    a.depth = static_cast<int>(z.rows);
    a.out = static_cast<char*>(grad_weight);
    a.out_ld = z.K;
    a.out_group = z.Nw * z.K;
    a.part = reinterpret_cast<float*>(ws + l.part);
    a.vec = z.K % 4 == 0 && aligned(grad_weight, 4 * z.es);
    rc = run_product(kWeightGrad, z.dtype, l.dw, a, false, s);
  }
  return rc;
}

}  // namespace
}  // namespace smx

using namespace smx;

extern "C" {

size_t smx_linear_workspace_size(int64_t rows, int64_t K, int64_t N, int64_t G, int activation, int dtype) {
  Sizes z;
  if (check_sizes(rows, K, N, G, activation, dtype, z) != SMX_OK) return 0;
  // whatever the alignment
  return static_cast<size_t>(std::max(plan_product(kForward, dtype, rows, z.Nw, K, z.G, z.Nw != N, true).part_bytes,
                                      plan_product(kForward, dtype, rows, z.Nw, K, z.G, z.Nw != N, false).part_bytes));
}

int smx_linear(const void* x, int64_t x_stride, int dtype, int64_t rows, int64_t K, const void* weight,
               int64_t weight_stride, int64_t N, const void* bias, int activation, const void* residual,
               int64_t residual_stride, void* y, int64_t y_stride, float* preact, void* workspace,
               size_t workspace_bytes, void* stream) {
  Sizes z;
  const int rc = check_sizes(rows, K, N, 0, activation, dtype, z);
  if (rc != SMX_OK) return rc;
  return forward(z, x, x_stride, weight, weight_stride, Groups{}, bias, residual, residual_stride, false, y, y_stride,
                 preact, workspace, workspace_bytes, stream);
}

int smx_grouped_linear(const void* x, int64_t x_stride, int dtype, int64_t rows, int64_t K, const void* weight,
                       int64_t weight_stride, int64_t group_stride, int64_t num_weights, int64_t N, const void* bias,
                       int activation, const void* residual, int64_t residual_stride, const int64_t* group_offsets,
                       int64_t G, const int64_t* weight_slots, int fill_rest, void* y, int64_t y_stride, float* preact,
                       void* workspace, size_t workspace_bytes, void* stream) {
  Sizes z;
  const int rc = G <= 0 ? static_cast<int>(SMX_ERR_INVALID_ARG) : check_sizes(rows, K, N, G, activation, dtype, z);
  if (rc != SMX_OK) return rc;
  return forward(z, x, x_stride, weight, weight_stride, Groups{group_offsets, weight_slots, group_stride, num_weights},
                 bias, residual, residual_stride, fill_rest != 0, y, y_stride, preact, workspace, workspace_bytes, stream);
}

size_t smx_linear_grad_workspace_size(int64_t rows, int64_t K, int64_t N, int64_t G, int activation, int dtype) {
  Sizes z;
  if (check_sizes(rows, K, N, G, activation, dtype, z) != SMX_OK) return 0;
  return static_cast<size_t>(std::max(grad_layout(z, true, true).total, grad_layout(z, false, false).total));
}

int smx_linear_grad(const void* dy, int64_t dy_stride, const float* preact, const void* x, int64_t x_stride, int dtype,
                    int64_t rows, int64_t K, const void* weight, int64_t weight_stride, int64_t N, int activation,
                    void* grad_x, void* grad_weight, void* grad_bias, void* workspace, size_t workspace_bytes,
                    void* stream) {
  Sizes z;
  const int rc = check_sizes(rows, K, N, 0, activation, dtype, z);
  if (rc != SMX_OK) return rc;
  return gradients(z, dy, dy_stride, preact, x, x_stride, weight, weight_stride, Groups{}, grad_x, grad_weight,
                   grad_bias, workspace, workspace_bytes, stream);
}

int smx_grouped_linear_grad(const void* dy, int64_t dy_stride, const float* preact, const void* x, int64_t x_stride,
                            int dtype, int64_t rows, int64_t K, const void* weight, int64_t weight_stride,
                            int64_t group_stride, int64_t num_weights, int64_t N, int activation,
                            const int64_t* group_offsets, int64_t G, const int64_t* weight_slots, void* grad_x,
                            void* grad_weight, void* grad_bias, void* workspace, size_t workspace_bytes, void* stream) {
  Sizes z;
  const int rc = G <= 0 ? static_cast<int>(SMX_ERR_INVALID_ARG) : check_sizes(rows, K, N, G, activation, dtype, z);
  if (rc != SMX_OK) return rc;
  return gradients(z, dy, dy_stride, preact, x, x_stride, weight, weight_stride,
                   Groups{group_offsets, weight_slots, group_stride, num_weights}, grad_x, grad_weight, grad_bias,
                   workspace, workspace_bytes, stream);
}

}  // extern "C"
