// Layer norm and RMS norm with a residual, forward and backward.
//
//   norm_kernel        s = x + residual, y = (s - mean) rstd w + b: a row stays in the registers of its threads, so that the mean,
//                      the mean square of the differences from it, and the result are three passes over registers and one over
//                      memory. Bound by memory: 16384 rows of 4096 in bf16 with a residual 86-87 us (537 MB, 6.2 TB/s; a
//                      copy of 2 GiB runs at 4.9), 131072 rows of 128 12 us (5.4 TB/s), one row of 2048 2.1 us.
//   norm_grad_kernel   dx, and the workgroup's partial sums of dw and db over the rows that it walks over. Bound by memory: the
//                      same rows 109-111 us (537 MB and 8 MB of partial sums, 4.9-5.0 TB/s); 131072 rows of 128 19 us (5.3).
//   norm_fold_kernel   the partial sums added up, in a fixed order: 4-5 us, of which two are the launch.
//
// Threads of a row: 16 to 1024, so that a thread has one 16-byte chunk of most widths; a workgroup of 256 holds several short
// rows, each in lanes of one wave. Two chunks a thread at 4096 columns instead: backward 98 -> 113 us. Workgroups walk over rows
// and load the next one while they sum: as many as the chip holds forward, half of that backward, where each leaves partial
// sums (a quarter: 98 -> 135 us; as many as forward: 105). Loads or stores past the caches gain 1-4 % at 16384 rows and lose
// 15-20 % at 2048, where what was just written is read from there.
//
// Rows that are no whole chunks go by chunks at any alignment: 60000 rows of 1001 in bf16 forward 45 -> 39 us, backward 109 -> 94
// against elements one by one (the last chunk's elements one by one: 121), in fp32 the same; 15000 rows of 4097, where half of
// a row's threads have one element, 135 -> 130.
#include <algorithm>

#include "blocks.h"

namespace smx {
namespace {

constexpr int kMaxNorm = 16384;     // columns
constexpr int kSmallBlock = 256;    // threads of a workgroup that holds several rows
constexpr int kFoldThreads = 1024;  // of a workgroup that adds up the partial weight gradients
constexpr int kFoldCols = 32;       // its columns

struct NormArgs {
  const char* x;         // forward: x; backward: s
  const char* residual;  // forward: residual; backward: gradient of the sum
  const char* dy;
  int64_t x_ld, residual_ld, dy_ld;
  int64_t rows;
  int H;
  const void* weight;
  const void* bias;
  bool wide;             // the weights are fp32 and x is not
  float eps;
  char* y;               // forward: y; backward: gradient of x
  char* sum;
  float* stats;
  float* part;           // backward: [2][blocks][H] partial sums, or null
};

template <int TPR> constexpr int block_threads() { return TPR < kSmallBlock ? kSmallBlock : TPR; }

template <int DT, int TPR, int NV, bool kVec, bool kRms>
__global__ __launch_bounds__(block_threads<TPR>()) void norm_kernel(NormArgs a) {
  constexpr int kN = Chunk<DT>::kN, kRows = block_threads<TPR>() / TPR;
  using S = typename Elem<DT>::S;
  using Sum = RowSum<TPR, 1>;
  __shared__ typename Sum::Lds lds;
  int turn = 0;
  const RowWalk<DT, TPR, kVec> walk{a.H, static_cast<int>(threadIdx.x) % TPR};
  const int sub = threadIdx.x / TPR;
  float w[NV][kN], b[NV][kN];
#pragma unroll
  for (int c = 0; c < NV; ++c) {
    walk.params(a.weight, a.wide, 1.0f, c, w[c]);
    walk.params(a.bias, a.wide, 0.0f, c, b[c]);
  }
  const float inv = 1.0f / static_cast<float>(a.H);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
  Chunk<DT> xr[NV], rr[NV];
  auto fetch = [&](int64_t row) {
    const S* x = reinterpret_cast<const S*>(a.x) + row * a.x_ld;
#pragma unroll
    for (int c = 0; c < NV; ++c) xr[c] = walk.load(x, c);
    if (a.residual != nullptr) {
      const S* r = reinterpret_cast<const S*>(a.residual) + row * a.residual_ld;
#pragma unroll
      for (int c = 0; c < NV; ++c) rr[c] = walk.load(r, c);
    }
  };
  auto clamped = [&](int64_t row) { return row < a.rows ? row : a.rows - 1; };
  int64_t row0 = static_cast<int64_t>(blockIdx.x) * kRows;
  if (row0 < a.rows) fetch(clamped(row0 + sub));
  for (; row0 < a.rows; row0 += step) {
    const int64_t row = row0 + sub;
    const bool live = row < a.rows;
    float h[NV][kN];
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      if (a.residual != nullptr) {
        Chunk<DT> s;
#pragma unroll
        for (int j = 0; j < kN; ++j) s.e[j] = round_to<DT>(xr[c].get(j) + rr[c].get(j));
        if (live) walk.store(reinterpret_cast<S*>(a.sum) + row * a.H, c, s);
        xr[c] = s;
      }
#pragma unroll
      for (int j = 0; j < kN; ++j) h[c][j] = xr[c].get(j);
    }
    if (row0 + step < a.rows) fetch(clamped(row + step));  // on its way while this row is summed
    float mean = 0.0f;
    if constexpr (!kRms) {
      float s[1] = {0.0f};
#pragma unroll
      for (int c = 0; c < NV; ++c)
#pragma unroll
        for (int j = 0; j < kN; ++j) s[0] += kVec || walk.in(c, j) ? h[c][j] : 0.0f;
      Sum::all(s, lds, turn);
      mean = s[0] * inv;
    }
    float q[1] = {0.0f};
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int j = 0; j < kN; ++j) {
        if constexpr (!kRms) h[c][j] -= mean;
        q[0] += (kVec && kRms) || walk.in(c, j) ? h[c][j] * h[c][j] : 0.0f;  // (behind the end: zeros, or less the mean)
      }
    Sum::all(q, lds, turn);
    const float rstd = rsqrtf(q[0] * inv + a.eps);
    if (live) {
      if (a.stats != nullptr && walk.tid == 0) {
        if constexpr (kRms) {
          a.stats[row] = rstd;
        } else {
          a.stats[2 * row] = mean;
          a.stats[2 * row + 1] = rstd;
        }
      }
      S* y = reinterpret_cast<S*>(a.y) + row * a.H;
#pragma unroll
      for (int c = 0; c < NV; ++c) {
        Chunk<DT> o;
#pragma unroll
        for (int j = 0; j < kN; ++j) o.e[j] = round_to<DT>(h[c][j] * rstd * w[c][j] + b[c][j]);
        walk.store(y, c, o);
      }
    }
  }
}

// Between the sums and the results the rows' elements stay as they were loaded. The widest rows (a workgroup of 1024 threads a
// CU, so 128 registers) leave the weight in LDS and load a row when they come to it: with both in registers the kernel spilled
// (2048 rows of 16384 in bf16 with a residual 107 -> 68 us, 1024 in fp32 160 -> 89).
template <int DT, int TPR, int NV, bool kVec, bool kRms>
__global__ __launch_bounds__(block_threads<TPR>()) void norm_grad_kernel(NormArgs a) {
  constexpr int kN = Chunk<DT>::kN, kRows = block_threads<TPR>() / TPR;
  constexpr bool kLdsWeight = TPR == 1024 && NV > 1, kAhead = !kLdsWeight;
  using S = typename Elem<DT>::S;
  using Sum = RowSum<TPR, kRms ? 1 : 2>;
  union Shared {
    typename Sum::Lds sum;
    float fold[kRows > 1 ? kRows : 1][kRows > 1 ? TPR * NV * kN : 1];
  };
  __shared__ Shared lds;
  __shared__ f32x4 weights[kLdsWeight ? NV * kN / 4 : 1][kLdsWeight ? TPR : 1];
  int turn = 0;
  const RowWalk<DT, TPR, kVec> walk{a.H, static_cast<int>(threadIdx.x) % TPR};
  const int sub = threadIdx.x / TPR;
  float w[kLdsWeight ? 1 : NV][kN], dw[NV][kN] = {}, db[NV][kN] = {};
#pragma unroll
  for (int c = 0; c < NV; ++c) {
    walk.params(a.weight, a.wide, 1.0f, c, w[kLdsWeight ? 0 : c]);
    if constexpr (kLdsWeight) {  // (each thread reads its own)
#pragma unroll
      for (int j = 0; j < kN; j += 4) weights[(c * kN + j) / 4][threadIdx.x] = f32x4{w[0][j], w[0][j + 1], w[0][j + 2], w[0][j + 3]};
    }
  }
  auto weight_of = [&](int c, float (&v)[kN]) {
#pragma unroll
    for (int j = 0; j < kN; ++j) {
      if constexpr (kLdsWeight) v[j] = weights[(c * kN + j) / 4][threadIdx.x][j % 4];
      else v[j] = w[c][j];
    }
  };
  const float inv = 1.0f / static_cast<float>(a.H);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
  Chunk<DT> xr[NV], gr[NV], sr[NV];
  float mean_next = 0.0f, rstd_next = 0.0f;
  auto fetch = [&](int64_t row) {
    const S* x = reinterpret_cast<const S*>(a.x) + row * a.x_ld;
    const S* g = reinterpret_cast<const S*>(a.dy) + row * a.dy_ld;
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      xr[c] = walk.load(x, c);
      gr[c] = walk.load(g, c);
    }
    if (a.residual != nullptr) {
      const S* r = reinterpret_cast<const S*>(a.residual) + row * a.residual_ld;
#pragma unroll
      for (int c = 0; c < NV; ++c) sr[c] = walk.load(r, c);
    }
    mean_next = kRms ? 0.0f : a.stats[2 * row];
    rstd_next = kRms ? a.stats[row] : a.stats[2 * row + 1];
  };
  auto clamped = [&](int64_t row) { return row < a.rows ? row : a.rows - 1; };
  int64_t row0 = static_cast<int64_t>(blockIdx.x) * kRows;
  if (kAhead && row0 < a.rows) fetch(clamped(row0 + sub));
  for (; row0 < a.rows; row0 += step) {
    const int64_t row = row0 + sub;
    const bool live = row < a.rows;
    if (!kAhead) fetch(clamped(row));
    const float mean = mean_next, rstd = rstd_next;
    Chunk<DT> x[NV], g[NV], add[NV];
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      x[c] = xr[c];
      g[c] = gr[c];
      if (a.residual != nullptr) add[c] = sr[c];
    }
    if (kAhead && row0 + step < a.rows) fetch(clamped(row + step));  // on its way while this row is summed
    auto n_of = [&](int c, int j) { return (x[c].get(j) - mean) * rstd; };
    float s[kRms ? 1 : 2] = {};
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      float wc[kN];
      weight_of(c, wc);
#pragma unroll
      for (int j = 0; j < kN; ++j) {
        const float n = n_of(c, j), dy = g[c].get(j), gw = dy * wc[j];
        if (live) {  // (nobody reads the sums of elements that are another chunk's or behind the end)
          dw[c][j] += dy * n;
          if constexpr (!kRms) db[c][j] += dy;
        }
        const bool mine = walk.in(c, j);  // (a mean behind the end could leave 0 * inf)
        s[0] += mine ? gw * n : 0.0f;
        if constexpr (!kRms) s[1] += mine ? gw : 0.0f;
      }
    }
    Sum::all(s, lds.sum, turn);
    if (live && a.y != nullptr) {
      const float c2 = s[0] * inv, c1 = kRms ? 0.0f : s[kRms ? 0 : 1] * inv;
      S* dx = reinterpret_cast<S*>(a.y) + row * a.H;
#pragma unroll
      for (int c = 0; c < NV; ++c) {
        float wc[kN];
        weight_of(c, wc);
        Chunk<DT> o;
#pragma unroll
        for (int j = 0; j < kN; ++j) {
          float v = g[c].get(j) * wc[j] - n_of(c, j) * c2;
          if constexpr (!kRms) v -= c1;
          v *= rstd;
          if (a.residual != nullptr) v += add[c].get(j);
          o.e[j] = round_to<DT>(v);
        }
        walk.store(dx, c, o);
      }
    }
  }
  if (a.part == nullptr) return;
  // the workgroup's column sums, its rows' threads added up in their order
#pragma unroll
  for (int which = 0; which < (kRms ? 1 : 2); ++which) {
    float (&v)[NV][kN] = which == 0 ? dw : db;
    float* out = a.part + (static_cast<int64_t>(which) * gridDim.x + blockIdx.x) * a.H;
    if constexpr (kRows > 1) {
      __syncthreads();
#pragma unroll
      for (int c = 0; c < NV; ++c)
#pragma unroll
        for (int j = 0; j < kN; ++j)
          if (walk.in(c, j)) lds.fold[sub][walk.col(c, j)] = v[c][j];
      __syncthreads();
      for (int col = threadIdx.x; col < a.H; col += block_threads<TPR>()) {
        float t = lds.fold[0][col];
        for (int r = 1; r < kRows; ++r) t += lds.fold[r][col];
        out[col] = t;
      }
    } else {
#pragma unroll
      for (int c = 0; c < NV; ++c)
#pragma unroll
        for (int j = 0; j < kN; ++j) {
          if (walk.in(c, j)) out[walk.col(c, j)] = v[c][j];
        }
    }
  }
}

// Column sums of part [2][parts][H] into the gradients of the weight (plane 0) and the bias (plane 1): a workgroup takes
// kFoldCols columns, its threads of a column a share of the parts each.
template <int DT>
__global__ __launch_bounds__(kFoldThreads) void norm_fold_kernel(const float* part, int parts, int H, char* grad_weight, char* grad_bias) {
  constexpr int kShares = kFoldThreads / kFoldCols;
  __shared__ float lds[kShares][kFoldCols];
  const int lane = static_cast<int>(threadIdx.x) % kFoldCols, share = static_cast<int>(threadIdx.x) / kFoldCols;
  const int col = static_cast<int>(blockIdx.x) * kFoldCols + lane;
  char* out = blockIdx.y == 0 ? grad_weight : grad_bias;
  if (out == nullptr) return;
  const float* p = part + static_cast<int64_t>(blockIdx.y) * parts * H;
  float t = 0.0f;
  if (col < H) {
#pragma unroll 16
    for (int i = share; i < parts; i += kShares) t += p[static_cast<int64_t>(i) * H + col];
  }
  lds[share][lane] = t;
  __syncthreads();
  if (share != 0 || col >= H) return;
#pragma unroll
  for (int w = 1; w < kShares; ++w) t += lds[w][lane];
  reinterpret_cast<typename Elem<DT>::S*>(out)[col] = round_to<DT>(t);
}

// ---- host ----------------------------------------------------------------------------------------

struct NormShape { int tpr, nv; };

// Threads of a row and 16-byte chunks of a thread.
NormShape shape_of(int64_t H, int dtype) {
  const int64_t chunks = (H * dtype_bytes(dtype) + 15) / 16;
  if (chunks <= 16) return {16, 1};
  if (chunks <= 32) return {32, 1};
  if (chunks <= 64) return {64, 1};
  if (chunks <= 128) return {64, 2};
  if (chunks <= 256) return {256, 1};
  if (chunks <= 512) return {512, 1};
  if (chunks <= 1024) return {1024, 1};
  if (chunks <= 2048) return {1024, 2};
  return {1024, 4};
}

int64_t rows_at_once(const NormShape& s) { return s.tpr < kSmallBlock ? kSmallBlock / s.tpr : 1; }

// Workgroups of the forward pass: as many as the chip holds at once, walking over the rows.
int64_t forward_blocks(const NormShape& s, int64_t rows) {
  const int64_t threads = std::max(s.tpr, kSmallBlock);
  return std::min((rows + rows_at_once(s) - 1) / rows_at_once(s), int64_t{256} * 2048 / threads);
}

// Of the backward pass: fewer, since each leaves its partial weight gradients.
int64_t grad_blocks(const NormShape& s, int64_t rows) {
  const int64_t threads = std::max(s.tpr, kSmallBlock);
  return std::min((rows + 4 * rows_at_once(s) - 1) / (4 * rows_at_once(s)), int64_t{256} * 1024 / threads);
}

int check_norm(int kind, int64_t rows, int64_t H, int dtype) {
  if ((kind != SMX_NORM_LAYER && kind != SMX_NORM_RMS) || rows < 0 || H <= 0 || !known_dtype(dtype)) return SMX_ERR_INVALID_ARG;
  if (H > kMaxNorm || rows > (int64_t{1} << 40)) return SMX_ERR_UNSUPPORTED;
  return SMX_OK;
}

template <bool kGrad, int DT, int TPR, int NV, bool kVec>
void launch(const NormArgs& a, bool rms, unsigned blocks, hipStream_t s) {
  constexpr int threads = block_threads<TPR>();
  if constexpr (kGrad) {
    if (rms) norm_grad_kernel<DT, TPR, NV, kVec, true><<<blocks, threads, 0, s>>>(a);
    else norm_grad_kernel<DT, TPR, NV, kVec, false><<<blocks, threads, 0, s>>>(a);
  } else {
    if (rms) norm_kernel<DT, TPR, NV, kVec, true><<<blocks, threads, 0, s>>>(a);
    else norm_kernel<DT, TPR, NV, kVec, false><<<blocks, threads, 0, s>>>(a);
  }
}

template <bool kGrad, int DT, bool kVec>
void launch_shape(const NormShape& f, const NormArgs& a, bool rms, unsigned blocks, hipStream_t s) {
  switch (f.tpr) {
    case 16: return launch<kGrad, DT, 16, 1, kVec>(a, rms, blocks, s);
    case 32: return launch<kGrad, DT, 32, 1, kVec>(a, rms, blocks, s);
    case 64:
      if (f.nv == 1) return launch<kGrad, DT, 64, 1, kVec>(a, rms, blocks, s);
      return launch<kGrad, DT, 64, 2, kVec>(a, rms, blocks, s);
    case 256: return launch<kGrad, DT, 256, 1, kVec>(a, rms, blocks, s);
    case 512: return launch<kGrad, DT, 512, 1, kVec>(a, rms, blocks, s);
    default:
      if (f.nv == 1) return launch<kGrad, DT, 1024, 1, kVec>(a, rms, blocks, s);
      if (f.nv == 2) return launch<kGrad, DT, 1024, 2, kVec>(a, rms, blocks, s);
      if constexpr (DT == kF32) return launch<kGrad, DT, 1024, 4, kVec>(a, rms, blocks, s);
  }
}

template <bool kGrad>
hipError_t launch_norm(int dtype, bool vec, const NormShape& f, const NormArgs& a, bool rms, int64_t blocks, hipStream_t s) {
  const unsigned n = static_cast<unsigned>(blocks);
  switch (dtype) {
    case kF32:
      vec ? launch_shape<kGrad, kF32, true>(f, a, rms, n, s) : launch_shape<kGrad, kF32, false>(f, a, rms, n, s);
      break;
    case kF16:
      vec ? launch_shape<kGrad, kF16, true>(f, a, rms, n, s) : launch_shape<kGrad, kF16, false>(f, a, rms, n, s);
      break;
    default:
      vec ? launch_shape<kGrad, kBF16, true>(f, a, rms, n, s) : launch_shape<kGrad, kBF16, false>(f, a, rms, n, s);
      break;
  }
  return hipGetLastError();
}

}  // namespace
}  // namespace smx

using namespace smx;

extern "C" {

int smx_norm(int kind, const void* x, int64_t x_stride, const void* residual, int64_t residual_stride, int dtype,
             int64_t rows, int64_t H, const void* weight, const void* bias, int weight_dtype, float eps, void* y,
             void* sum, float* stats, void* stream) {
  const int rc = check_norm(kind, rows, H, dtype);
  if (rc != SMX_OK) return rc;
  const bool any = weight != nullptr || bias != nullptr;
  if (x_stride < H || (residual && residual_stride < H) || !(eps >= 0.0f) || (any && weight_dtype != dtype && weight_dtype != kF32))
    return SMX_ERR_INVALID_ARG;
  if (rows == 0) return SMX_OK;
  if (!x || !y || (residual == nullptr) != (sum == nullptr)) return SMX_ERR_INVALID_ARG;
  const int64_t es = dtype_bytes(dtype), ws = dtype_bytes(weight_dtype);
  if (!aligned_to(x, es) || !aligned_to(residual, es) || !aligned_to(y, es) || !aligned_to(sum, es) ||
      (any && (!aligned_to(weight, ws) || !aligned_to(bias, ws))) || !aligned_to(stats, 4))
    return SMX_ERR_MISALIGNED;
  const bool vec = whole_chunks(x, x_stride, es) && whole_chunks(y, H, es) && (!residual || (whole_chunks(residual, residual_stride, es) && whole_chunks(sum, H, es))) &&
                   aligned_to(weight, 16) && aligned_to(bias, 16);
  NormArgs a{};
  a.x = static_cast<const char*>(x);
  a.x_ld = x_stride;
  a.residual = static_cast<const char*>(residual);
  a.residual_ld = residual_stride;
  a.rows = rows;
  a.H = static_cast<int>(H);
  a.weight = weight;
  a.bias = bias;
  a.wide = any && weight_dtype != dtype;
  a.eps = eps;
  a.y = static_cast<char*>(y);
  a.sum = static_cast<char*>(sum);
  a.stats = stats;
  const NormShape f = shape_of(H, dtype);
  return static_cast<int>(launch_norm<false>(dtype, vec, f, a, kind == SMX_NORM_RMS, forward_blocks(f, rows), static_cast<hipStream_t>(stream)));
}

size_t smx_norm_grad_workspace_size(int kind, int64_t rows, int64_t H, int dtype) {
  if (check_norm(kind, rows, H, dtype) != SMX_OK) return 0;
  return static_cast<size_t>(grad_blocks(shape_of(H, dtype), rows) * H * 4 * (kind == SMX_NORM_RMS ? 1 : 2));
}

int smx_norm_grad(int kind, const void* grad_y, int64_t grad_y_stride, const void* grad_sum, int64_t grad_sum_stride,
                  const void* s, int64_t s_stride, int dtype, int64_t rows, int64_t H, const void* weight,
                  int weight_dtype, const float* stats, void* grad_x, void* grad_weight, void* grad_bias, void* workspace,
                  size_t workspace_bytes, void* stream) {
  const int rc = check_norm(kind, rows, H, dtype);
  if (rc != SMX_OK) return rc;
  const bool rms = kind == SMX_NORM_RMS, sums = grad_weight || grad_bias;
  if (grad_y_stride < H || s_stride < H || (grad_sum && grad_sum_stride < H) || (rms && grad_bias) ||
      ((weight || sums) && weight_dtype != dtype && weight_dtype != kF32))
    return SMX_ERR_INVALID_ARG;
  const int64_t es = dtype_bytes(dtype), ws = dtype_bytes(weight_dtype);
  if (rows > 0 && (!grad_y || !s || !stats)) return SMX_ERR_INVALID_ARG;
  if (!aligned_to(grad_y, es) || !aligned_to(grad_sum, es) || !aligned_to(s, es) || !aligned_to(grad_x, es) || !aligned_to(stats, 4) ||
      ((weight || sums) && (!aligned_to(weight, ws) || !aligned_to(grad_weight, ws) || !aligned_to(grad_bias, ws))))
    return SMX_ERR_MISALIGNED;
  const NormShape f = shape_of(H, dtype);
  const int64_t blocks = grad_blocks(f, rows);
  if (sums && rows > 0) {
    if (!workspace || workspace_bytes < smx_norm_grad_workspace_size(kind, rows, H, dtype)) return SMX_ERR_WORKSPACE;
    if (!aligned_to(workspace, 16)) return SMX_ERR_MISALIGNED;
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (rows > 0 && (grad_x || sums)) {
    NormArgs a{};
    a.x = static_cast<const char*>(s);
    a.x_ld = s_stride;
    a.dy = static_cast<const char*>(grad_y);
    a.dy_ld = grad_y_stride;
    a.residual = grad_x ? static_cast<const char*>(grad_sum) : nullptr;
    a.residual_ld = grad_sum_stride;
    a.rows = rows;
    a.H = static_cast<int>(H);
    a.weight = weight;
    a.wide = weight && weight_dtype != dtype;
    a.y = static_cast<char*>(grad_x);
    a.stats = const_cast<float*>(stats);
    a.part = sums ? static_cast<float*>(workspace) : nullptr;
    const bool vec = whole_chunks(s, s_stride, es) && whole_chunks(grad_y, grad_y_stride, es) && whole_chunks(grad_x, H, es) &&
                     (!a.residual || whole_chunks(grad_sum, grad_sum_stride, es)) && aligned_to(weight, 16);
    const hipError_t err = launch_norm<true>(dtype, vec, f, a, rms, blocks, st);
    if (err != hipSuccess) return static_cast<int>(err);
  }
  if (sums) {
    const dim3 grid(static_cast<unsigned>((H + kFoldCols - 1) / kFoldCols), grad_bias ? 2 : 1);
    const float* part = static_cast<const float*>(workspace);
    const int parts = rows > 0 ? static_cast<int>(blocks) : 0, n = static_cast<int>(H);
    char* gw = static_cast<char*>(grad_weight);
    char* gb = static_cast<char*>(grad_bias);
    switch (weight_dtype) {
      case kF32: norm_fold_kernel<kF32><<<grid, kFoldThreads, 0, st>>>(part, parts, n, gw, gb); break;
      case kF16: norm_fold_kernel<kF16><<<grid, kFoldThreads, 0, st>>>(part, parts, n, gw, gb); break;
      default: norm_fold_kernel<kBF16><<<grid, kFoldThreads, 0, st>>>(part, parts, n, gw, gb); break;
    }
    return static_cast<int>(hipGetLastError());
  }
  return SMX_OK;
}

}  // extern "C"
