// Matrix products with an epilogue: the C entry points, the choice of kernels, and the elementwise kernels (gradient
// of the activation with the bias gradient's column sums, joining of contraction splits).
#include "../../include/specmoe_mi355x.h"
#include "../../include/specmoe_mi355x_products.h"
#include <algorithm>
#include <cmath>

#include "product.h"

namespace smx {

constexpr int kGradRows = 16;   // rows of a workgroup of the activation gradient, four per wave: all loaded at once
constexpr int kSumWaves = 16;   // waves of a workgroup of the bias gradient
constexpr int kGradCols = 256;  // its output columns: 64 lanes of 4
constexpr int kJoinRows = 4;    // rows of a workgroup that joins splits, one per wave

// dz = dy * act'(z), rounded into dz (unless null), and its fp32 column sums over the workgroup's rows.
// The rounding is that of an operand of the matrix instructions: the gradients of x and of the weight then err by that and by
// their own, 2.35e-3 relative in bf16 (1.66e-3 if only the results were rounded; 4096 rows, 2048 -> 5632 with gelu) and 2.9e-4
// in fp16 (2.1e-4). Carrying what the rounding leaves as a second operand would double the two products (205 of 367 us
// there are theirs).
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
    constexpr int kN = kGradRows / kPWaves;
    f32x4 d[kN], z[kN], u[kN];
    bool in[kN];
    int64_t row[kN];
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      in[n] = wave + n * kPWaves < it.m;
      row[n] = static_cast<int64_t>(it.row) + wave + n * kPWaves;
      d[n] = in[n] ? load4<DT>(a.dy, row[n] * a.dy_ld + col, left, vec) : f32x4{};
      const char* zp = reinterpret_cast<const char*>(a.z);
      z[n] = in[n] && a.z != nullptr ? load4<kF32>(zp, row[n] * a.z_ld + col, left, vec) : f32x4{};
      u[n] = in[n] && a.p.gated ? load4<kF32>(zp, row[n] * a.z_ld + a.p.out_cols + col, left, vec) : f32x4{};
    }
    if (a.p.gated) {
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        f32x4 du;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          du[e] = d[n][e] * activate<DT == kF32>(kActSilu, z[n][e]);
          d[n][e] *= u[n][e] * activate_grad<DT == kF32>(kActSilu, z[n][e]);
        }
        if (in[n]) store4<DT>(a.dz, row[n] * a.dz_ld + a.p.out_cols + col, left, vec, du);
        if (in[n]) sum[1] += du;
      }
    } else if (a.z != nullptr) {
      activate_grad_all<DT == kF32>(a.p.act, z, d);
    }
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      if (in[n] && a.dz != nullptr) store4<DT>(a.dz, row[n] * a.dz_ld + col, left, vec, d[n]);
      if (in[n]) sum[0] += d[n];
    }
  }
  // the columns that round dz's rows up to whole slots: zeros, as a contraction takes them along
  if (a.dz != nullptr && it.ct == col_tiles - 1 && lane < a.dz_ld - a.p.cols) {
    for (int r = wave; r < it.m; r += kPWaves)
      reinterpret_cast<typename Elem<DT>::S*>(a.dz)[(static_cast<int64_t>(it.row) + r) * a.dz_ld + a.p.cols + lane] = 0;
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
__global__ __launch_bounds__(kSumWaves* kWave) void bias_grad_kernel(ProductArgs p, const float* sums, int max_tiles, char* grad) {
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
  __shared__ float lds[kSumWaves][kWave];
  float v = 0.0f;
  if (col < p.cols) {
#pragma unroll 4
    for (int t = wave; t < count; t += kSumWaves) v += sums[static_cast<int64_t>(first + t) * p.cols + col];
  }
  lds[wave][lane] = v;
  __syncthreads();
  if (wave > 0 || col >= p.cols) return;
  for (int w = 1; w < kSumWaves; ++w) v += lds[w][lane];
  reinterpret_cast<S*>(grad)[static_cast<int64_t>(g) * p.cols + col] = Elem<DT>::from_f32(v);
}

// Copies rows of `len` elements, `per` of them in each of the groups, into rows of whole 16-byte slots, with zeros behind.
template <int DT>
__global__ __launch_bounds__(kPThreads) void pad_kernel(const char* src, int64_t ld, int64_t group, int64_t per, int len,
                                                        char* dst, int slots, int64_t rows) {
  using S = typename Elem<DT>::S;
  constexpr int kEps = 16 / sizeof(S);
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kPWaves + wave_id();
  if (row >= rows) return;
  const int64_t g = row / per;
  const S* from = reinterpret_cast<const S*>(src) + g * group + (row - g * per) * ld;
  u32x4* to = reinterpret_cast<u32x4*>(dst) + row * slots;
  for (int s = lane_id(); s < slots; s += kWave) to[s] = load_slot<DT>(from + s * kEps, len - s * kEps);
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
  finish4<DT>(a, it, row, col, left, v, u, bias, a.gated ? bias4<DT>(a, it, a.out_cols + col, left) : f32x4{}, res);
}

namespace {

constexpr int64_t kMaxSize = int64_t{1} << 30;
constexpr int64_t kMaxWeight = int64_t{1} << 40;  // bytes
constexpr int kFillBlocks = 64;
constexpr int64_t kL2Bytes = int64_t{32} << 20;

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }
bool aligned(const void* p, int64_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
bool whole_lines(const void* base, int64_t pitch) { return aligned(base, 128) && pitch % 128 == 0; }
bool valid_dtype(int dt) { return dt == kF32 || dt == kF16 || dt == kBF16; }

enum Kind { kForward, kInputGrad, kWeightGrad };

// How a product runs.
struct ProductPlan {
  TileShape tile{64, 64, TileShape::kStaged};
  int splits = 1, split_steps = 0;
  int64_t part_bytes = 0;
  double time = 0;  // estimate, us
};

// The tiles, with the time of a call in us that n workgroups per CU take: 2.5 + end * n + steps * (first + each * n), a
// step being 128 bytes of the contraction. Fitted to measured calls (bf16: 1 to 8192 rows, 4096 and 696 -> 4096 and
// 1200, weight gradients of 1 to 100 groups of 3 to 800 rows, unaligned 1 to 3000 rows of 1999 -> 1333); the fit is
// within about 20 % of what was measured, and where two tiles come closer than that either will do. Both sides of some
// choices (us): 32 rows, 4096 -> 4096, 16 x 32 rows 11.4, 32 x 128 copied 33; 128 rows 28 and 64 x 64 rows 23; 512 rows
// 64 x 64 rows 38.5, 64 x 128 copied 36; 2048 rows 128 x 128 73, wide 97; 4096 rows 129 and 117. 64 x 64 copied against
// the tile without it: weight gradients of 1000 rows, 1024 -> 1024 in bf16, 8.4 and 14.2, of 777 rows, 1024 -> 2816 in
// fp32 48 and 63, forward 200 rows, 2048 -> 6000 16.5 and 21.1, but of 4096 rows, 2048 -> 5632 165 and 100. Wide
// against 128 x 128 at 176 to 192 wide tiles, a part of the CUs: input gradient of 3000 rows, 4096 -> 14336 290 and 354, of
// 6000 rows, 2048 -> 5632 124 and 145; at 128 tiles (2000 rows, 4096 -> 4096) 86 and 71. Rows tiles on a part of the CUs
// against the tile that their times on all of them would choose: 3 rows, 5424 -> 1376 6.7 and 11.7 (splits of 32 x 128),
// 92 rows, 3792 -> 392 in fp32 11.1 and 15.5.
struct TileCost {
  TileShape t;
  float end, first, each;
  float each32;    // fp32 (of the same bytes: half the elements, at a 16th of the matrix rate); 0: not for fp32
  float depth_end; // end of a product grouped along its contraction; 0: not for them
  float few = 0, few32 = 0;  // a step of at most a workgroup per CU, where it is its reads' latency (both types)
};
using Tile = TileShape;
constexpr TileCost kTileCosts[] = {
    {{16, 16, Tile::kRows}, 0.3f, 0.085f, 0.052f, 0.06f, 0.f, 0.05f, 0.072f},
    {{16, 32, Tile::kRows}, 0.5f, 0.06f, 0.08f, 0.092f, 0.f, 0.075f, 0.095f},
    {{32, 32, Tile::kRows}, 0.8f, 0.065f, 0.085f, 0.17f, 0.f, 0.088f, 0.16f},
    {{64, 64, Tile::kRows}, 2.0f, 0.03f, 0.24f, 0.68f, 0.f},
    {{64, 64, Tile::kCopied}, 1.0f, 0.10f, 0.20f, 0.50f, 1.2f},
    {{32, 128, Tile::kCopied}, 0.7f, 0.20f, 0.22f, 0.52f, 0.f}, {{64, 128, Tile::kCopied}, 1.0f, 0.20f, 0.30f, 1.0f, 0.f},
    {{128, 128, Tile::kCopied}, 3.0f, 0.20f, 0.43f, 1.95f, 4.5f}, {{128, 128, Tile::kShallow}, 1.4f, 0.2f, 0.55f, 2.3f, 1.4f},
    {{256, 256, Tile::kWide}, 10.f, 0.0f, 1.54f, 0.f, 16.f},
    // any alignment
    {{16, 32, Tile::kRowsStaged}, 0.5f, 0.10f, 0.12f, 0.13f, 0.f}, {{32, 32, Tile::kRowsStaged}, 0.5f, 0.10f, 0.20f, 0.20f, 0.f},
    {{64, 64, Tile::kStaged}, 1.5f, 0.18f, 0.33f, 0.9f, 1.5f},
};
constexpr int kCUs = 256;

// slots: both operands consist of whole 16-byte slots (see launch_product_*).
ProductPlan plan_product(Kind kind, int dtype, int64_t rows, int64_t cols, int64_t depth, int64_t groups, bool gated,
                         bool slots) {
  ProductPlan p;
  if (rows == 0) return p;
  const bool depth_groups = kind == kWeightGrad;
  const int64_t all = cdiv(depth, kPStep / dtype_bytes(dtype));
  const double mean = depth_groups ? static_cast<double>(depth) / groups : static_cast<double>(depth);
  const double steps = std::max(1.0, mean / (kPStep / dtype_bytes(dtype)));
  for (const TileCost& c : kTileCosts) {
    const TileShape& t = c.t;
    const bool by_rows = t.form == Tile::kRows || t.form == Tile::kRowsStaged;
    if ((t.form == Tile::kStaged || t.form == Tile::kRowsStaged) == slots) continue;
    if (by_rows && (kind != kForward || (gated && t.bn < 32))) continue;
    if (t.form == Tile::kShallow && !depth_groups) continue;
    const float end = depth_groups ? c.depth_end : c.end, each = dtype == kF32 ? c.each32 : c.each;
    if (end == 0 || each == 0) continue;
    // row tiles: of every group with rows, half a tile more than its rows fill
    double row_tiles = static_cast<double>(cdiv(rows, t.bm));
    if (!depth_groups && groups > 1) {
      const double active = static_cast<double>(std::min(groups, rows));
      row_tiles = std::max(active, static_cast<double>(rows) / t.bm + active / 2);
    }
    const double tiles = row_tiles * static_cast<double>(cdiv(cols, t.bn)) * (depth_groups ? groups : 1);
    // (splits: not of rows tiles, whose waves split the contraction already, and of groups along it only of a single one)
    const bool may_split = !by_rows && t.form != Tile::kShallow && !(depth_groups && groups > 1);
    for (int splits = 1; splits <= 16 && (splits == 1 || (may_split && splits * 4 <= steps)); splits *= 2) {
      // workgroups per CU: of the small tiles and of 128 x 128 in 16 bits several run on a CU at once
      const double share = tiles * splits / kCUs;
      double n = std::max(1.0, share);
      if (!by_rows || t.bm == 64) n = t.bm == 128 && dtype != kF32 ? std::ceil(2 * n) / 2 : std::ceil(n);
      // a last round of wide tiles on a part of the CUs leaves them more of the power and of the L2s
      const double last = share - std::floor(share);
      const double work = t.form == Tile::kWide && last > 0 ? std::floor(share) + 0.65 + 0.35 * last * last : n;
      double step = c.first + each * work;
      if (c.few != 0) {
        if (share <= 1) step = dtype == kF32 ? c.few32 : c.few;
        else if (dtype == kF32) step = c.first + each * std::ceil(share);  // bound by the matrix rate
        else if (share < 2) step = c.few + (share - 1) * (c.first + 2 * each - c.few);
      }
      double time = 2.5 + end * n + steps / splits * step;
      if (splits > 1) time += 5.0 + 8.0 * splits * rows * cols / 4e6;  // the joining launch; partial sums out and in
      if (p.time != 0 && time >= p.time) continue;
      p.time = time;
      p.tile = t;
      p.split_steps = static_cast<int>(cdiv(cdiv(all, splits), 2) * 2);  // in pairs
      p.splits = splits == 1 ? 1 : static_cast<int>(cdiv(all, p.split_steps));
      p.part_bytes = p.splits > 1 ? p.splits * rows * cols * 4 : 0;
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
  // Results that the L2s (8 of 4 MB) cannot hold are stored past them, where they would only displace the operands that
  // the tiles share: 8192 x 4096 -> 14336 with gelu_tanh 844 -> 782 us, 12282 rows in 64 groups 2048 -> 2 x 1408 with
  // its pre-activations 281 -> 272. Smaller ones stay for the next operator to read, and so do those whose rows are no
  // whole 128-byte lines, which would go to memory in parts: weight gradients of 4 groups of 48 rows, 5208 -> 9184 254 past
  // the caches and 129 through them, 2000 rows, 64 -> 20008 with pre-activations 126 and 48.
  const int64_t result = (a.out_group != 0 ? a.groups : 1) * static_cast<int64_t>(a.rows) *
                         (a.out_cols * int64_t{dtype_bytes(dtype)} + (a.z != nullptr ? a.cols * int64_t{4} : 0));
  a.stream = result > kL2Bytes && whole_lines(a.out, a.out_ld * dtype_bytes(dtype)) &&
             (a.z == nullptr || whole_lines(a.z, a.z_ld * int64_t{4}));
  a.item_blocks = static_cast<int>(items);
  a.fill_blocks = plan.splits > 1 ? 0 : fills;
  const bool ps = kind != kForward, qs = kind == kWeightGrad;
  hipError_t err;
  switch (plan.tile.form) {
    case TileShape::kRows:
    case TileShape::kRowsStaged:
      err = launch_product_rows(dtype, plan.tile, a, s);
      break;
    case TileShape::kShallow: err = launch_product_shallow(dtype, a, s); break;
    case TileShape::kWide: err = launch_product_wide(dtype, ps, qs, depth_groups, a, s); break;
    default: err = launch_product_tile(dtype, ps, qs, depth_groups, plan.tile, a, s);
  }
  if (err != hipSuccess || plan.splits == 1) return static_cast<int>(err);
  const int splits = a.splits;
  a.splits = 1;
  // Groups along the contraction (a single one where it is split): its bounds are of the operands' rows, and the partial
  // sums cover every row of the result.
  if (depth_groups) a.offsets = nullptr;
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

// Whole 16-byte slots: the base and the pitch, and the length of whatever lies side by side.
bool whole_slots(const void* base, int64_t pitch, int64_t length, int64_t es) {
  return aligned(base, 16) && pitch * es % 16 == 0 && length * es % 16 == 0;
}
int64_t whole(int64_t length, int64_t es) { return cdiv(length * es, 16) * 16 / es; }

// Operands whose rows are no whole slots may be copied into the workspace first, where they are: where the product gains
// by it well over what the copies take (2 us each and their bytes at 4 TB/s). A training step of 7174 rows of 2677 ->
// 2112 in fp32: 2825 us without the copies, 2128 with; a forward product of 3000 rows of 1999 -> 1333 in bf16 50 and 59,
// which the factor keeps without them.
constexpr double kPadGain = 0.8;
double copy_time(int64_t elems, int64_t es) { return 2.0 + 2.0 * elems * es / 4e6; }

struct Layout {
  ProductPlan plan;
  bool pad = false;
  int64_t x = 0, w = 0, part = 0, total = 0;  // offsets of the copies and the partial sums; bytes in all
};

Layout forward_layout(const Sizes& z, bool slots, bool may_pad) {
  Layout l;
  l.plan = plan_product(kForward, z.dtype, z.rows, z.Nw, z.K, z.G, z.Nw != z.N, slots);
  const int64_t k = whole(z.K, z.es);
  if (!slots && may_pad && k != z.K && z.G * z.Nw <= kMaxSize && z.Nw * k * z.es < int64_t{kPOutside}) {
    const ProductPlan fast = plan_product(kForward, z.dtype, z.rows, z.Nw, k, z.G, z.Nw != z.N, true);
    if (fast.time + copy_time(z.rows * k, z.es) + copy_time(z.G * z.Nw * k, z.es) < kPadGain * l.plan.time) {
      l.plan = fast;
      l.pad = true;
      l.w = align256(z.rows * k * z.es);
      l.part = l.w + align256(z.G * z.Nw * k * z.es);
    }
  }
  l.total = l.part + align256(l.plan.part_bytes);
  return l;
}

struct GradLayout {
  ProductPlan dx, dw;
  bool pad_w = false, pad_x = false;
  int64_t dz = 0, dz_ld = 0, sums = 0, copy = 0, part = 0, total = 0;
};

// w_slots, x_slots: the weight's and x's rows are whole slots; dz's always are.
GradLayout grad_layout(const Sizes& z, bool w_slots, bool x_slots, bool may_pad) {
  GradLayout l;
  l.dx = plan_product(kInputGrad, z.dtype, z.rows, z.K, z.Nw, z.G, false, w_slots);
  l.dw = plan_product(kWeightGrad, z.dtype, z.Nw, z.K, z.rows, z.G, false, x_slots);
  const int64_t k = whole(z.K, z.es);
  int64_t copy = 0;
  if (may_pad && k != z.K && z.rows > 0 && z.G * z.Nw <= kMaxSize) {
    ProductPlan fast = plan_product(kInputGrad, z.dtype, z.rows, k, z.Nw, z.G, false, true);
    if (!w_slots && fast.time + copy_time(z.G * z.Nw * k, z.es) < kPadGain * l.dx.time) {
      l.dx = fast;
      l.pad_w = true;
      copy = z.G * z.Nw * k * z.es;
    }
    fast = plan_product(kWeightGrad, z.dtype, z.Nw, k, z.rows, z.G, false, true);
    if (!x_slots && fast.time + copy_time(z.rows * k, z.es) < kPadGain * l.dw.time) {
      l.dw = fast;
      l.pad_x = true;
      copy = std::max(copy, z.rows * k * z.es);
    }
  }
  l.dz_ld = whole(z.Nw, z.es);
  l.sums = align256(z.rows * l.dz_ld * z.es);
  l.copy = l.sums + align256(max_row_tiles(z.rows, z.G, kGradRows) * z.Nw * 4);
  l.part = l.copy + align256(copy);
  l.total = l.part + align256(std::max(l.dx.part_bytes, l.dw.part_bytes));
  return l;
}

// Rows (per group: `per`) of len elements into rows of whole slots.
hipError_t launch_pad(int dtype, const void* src, int64_t ld, int64_t group, int64_t groups, int64_t per, int64_t len,
                      char* dst, hipStream_t s) {
  const int64_t rows = groups * per;
  const unsigned blocks = static_cast<unsigned>(cdiv(rows, kPWaves));
  const int slots = static_cast<int>(cdiv(len * dtype_bytes(dtype), 16)), n = static_cast<int>(len);
  const char* p = static_cast<const char*>(src);
  switch (dtype) {
    case kF32: pad_kernel<kF32><<<blocks, kPThreads, 0, s>>>(p, ld, group, per, n, dst, slots, rows); break;
    case kF16: pad_kernel<kF16><<<blocks, kPThreads, 0, s>>>(p, ld, group, per, n, dst, slots, rows); break;
    default: pad_kernel<kBF16><<<blocks, kPThreads, 0, s>>>(p, ld, group, per, n, dst, slots, rows); break;
  }
  return hipGetLastError();
}

struct Groups {
  const int64_t* offsets = nullptr;
  const int64_t* slots = nullptr;
  int64_t stride = 0, weights = 1;
};

int check_groups(const Sizes& z, const Groups& g) {
  if (!z.grouped) return SMX_OK;
  if (!g.offsets || g.weights <= 0 || g.stride < 0) return SMX_ERR_INVALID_ARG;
  if (g.weights > kMaxSize) return SMX_ERR_UNSUPPORTED;
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
  // (gate and up rows are reached from one base with 32-bit offsets; beyond any memory, a product of sizes gone wrong)
  const int64_t extent = z.Nw * weight_stride * z.es;
  if (extent >= (z.Nw != z.N ? int64_t{kPOutside} : kMaxWeight)) return SMX_ERR_UNSUPPORTED;
  if (z.rows == 0) return SMX_OK;
  if (!x || !weight || !y) return SMX_ERR_INVALID_ARG;
  if (!aligned(x, z.es) || !aligned(weight, z.es) || !aligned(y, z.es) || !aligned(bias, z.es) ||
      !aligned(residual, z.es) || !aligned(preact, 4))
    return SMX_ERR_MISALIGNED;
  const bool slots = whole_slots(x, x_stride, z.K, z.es) && whole_slots(weight, weight_stride, z.K, z.es) &&
                     g.stride * z.es % 16 == 0;
  const Layout l = forward_layout(z, slots, g.slots == nullptr);
  if (l.total > 0) {
    if (!workspace || workspace_bytes < static_cast<size_t>(l.total)) return SMX_ERR_WORKSPACE;
    if (!aligned(workspace, 16)) return SMX_ERR_MISALIGNED;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  ProductArgs a = group_args(z, g);
  a.q = static_cast<const char*>(x);
  a.q_ld = x_stride;
  a.p = static_cast<const char*>(weight);
  a.p_ld = weight_stride;
  a.p_group = g.stride;
  int64_t depth = z.K;
  if (l.pad) {
    depth = whole(z.K, z.es);
    hipError_t err = launch_pad(z.dtype, x, x_stride, 0, 1, z.rows, z.K, ws + l.x, s);
    if (err == hipSuccess) err = launch_pad(z.dtype, weight, weight_stride, g.stride, z.G, z.Nw, z.K, ws + l.w, s);
    if (err != hipSuccess) return static_cast<int>(err);
    a.q = ws + l.x;
    a.p = ws + l.w;
    a.q_ld = a.p_ld = depth;
    a.p_group = z.Nw * depth;
  }
  a.cols = static_cast<int>(z.Nw);
  a.depth = static_cast<int>(depth);
  a.gated = z.Nw != z.N;
  a.out = static_cast<char*>(y);
  a.out_ld = y_stride;
  a.bias = static_cast<const char*>(bias);
  a.bias_ld = z.Nw;
  a.res = static_cast<const char*>(residual);
  a.res_ld = residual_stride;
  a.z = preact;
  a.z_ld = z.Nw;
  a.part = reinterpret_cast<float*>(ws + l.part);
  a.act = a.gated ? kActNone : z.act;
  a.out_cols = static_cast<int>(z.N);
  const int64_t v = 4 * z.es;
  a.vec = z.N % 4 == 0 && y_stride % 4 == 0 && aligned(y, v) && aligned(bias, v) && aligned(preact, 16) &&
          (!residual || (residual_stride % 4 == 0 && aligned(residual, v)));
  return run_product(kForward, z.dtype, l.plan, a, fill, s);
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
  // dz is dy itself where that is all right, or rows of whole slots in the workspace
  const bool own_dz = z.act != SMX_ACT_NONE || !whole_slots(dy, dy_stride, z.N, z.es);
  const GradLayout l = grad_layout(z, whole_slots(weight, weight_stride, z.K, z.es) && g.stride * z.es % 16 == 0,
                                   whole_slots(x, x_stride, z.K, z.es), g.slots == nullptr);
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
  if (z.rows > 0 && (own_dz || grad_bias)) {
    ag.dy = static_cast<const char*>(dy);
    ag.dy_ld = dy_stride;
    ag.p.vec = z.N % 4 == 0 && dy_stride % 4 == 0 && aligned(dy, 4 * z.es);
    if (own_dz) {
      ag.dz = ws + l.dz;
      ag.dz_ld = l.dz_ld;
      dz = ag.dz;
      dz_ld = l.dz_ld;
    }
    if (z.act != SMX_ACT_NONE) {
      ag.z = preact;
      ag.z_ld = z.Nw;
      ag.p.vec = ag.p.vec && aligned(preact, 16);
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
      case kF32: bias_grad_kernel<kF32><<<n, kSumWaves * kWave, 0, s>>>(ag.p, sums, ag.max_tiles, out); break;
      case kF16: bias_grad_kernel<kF16><<<n, kSumWaves * kWave, 0, s>>>(ag.p, sums, ag.max_tiles, out); break;
      default: bias_grad_kernel<kBF16><<<n, kSumWaves * kWave, 0, s>>>(ag.p, sums, ag.max_tiles, out); break;
    }
    hipError_t err = hipGetLastError();
    if (err != hipSuccess) return static_cast<int>(err);
  }
  const int64_t padded = whole(z.K, z.es);
  if (grad_x && z.rows > 0) {
    ProductArgs a = group_args(z, g);
    a.q = static_cast<const char*>(dz);
    a.q_ld = dz_ld;
    a.p = static_cast<const char*>(weight);
    a.p_ld = weight_stride;
    a.p_group = g.stride;
    a.cols = a.out_cols = static_cast<int>(z.K);
    if (l.pad_w) {
      hipError_t err = launch_pad(z.dtype, weight, weight_stride, g.stride, z.G, z.Nw, z.K, ws + l.copy, s);
      if (err != hipSuccess) return static_cast<int>(err);
      a.p = ws + l.copy;
      a.p_ld = padded;
      a.p_group = z.Nw * padded;
      a.cols = static_cast<int>(padded);
    }
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
    a.q_cols = static_cast<int>(own_dz ? l.dz_ld : z.Nw);
    a.p = static_cast<const char*>(x);
    a.p_ld = x_stride;
    a.rows = static_cast<int>(z.Nw);
    a.cols = a.out_cols = static_cast<int>(z.K);
    if (l.pad_x) {
      hipError_t err = launch_pad(z.dtype, x, x_stride, 0, 1, z.rows, z.K, ws + l.copy, s);
      if (err != hipSuccess) return static_cast<int>(err);
      a.p = ws + l.copy;
      a.p_ld = padded;
      a.cols = static_cast<int>(padded);
    }
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
  // whatever the alignment, with and without a slot map
  int64_t n = 0;
  for (const bool slots : {true, false})
    for (const bool may_pad : {true, false}) n = std::max(n, forward_layout(z, slots, may_pad).total);
  return static_cast<size_t>(n);
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
  int64_t n = 0;
  for (const bool w : {true, false})
    for (const bool x : {true, false})
      for (const bool may_pad : {true, false}) n = std::max(n, grad_layout(z, w, x, may_pad).total);
  return static_cast<size_t>(n);
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
