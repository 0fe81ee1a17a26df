// Rows to the experts and back: a token's row to its picks' places, and the weighted sum of the rows at its places, with
// gradients. All walk over tokens, so that what belongs to a token once (its row, the gradient of its sum) is moved once, and
// what belongs to a pick once. Bound by memory (a copy of 2 GiB runs at 4.9 TB/s):
//
//   spread_kernel        8192 tokens, 2 picks, 4096 columns in bf16: 33-39 us (201 MB, 5.1-6 TB/s)
//   combine_kernel       the same back: 34 us (5.9 TB/s); 8191 tokens, 6 picks, 2048 columns with a residual: 45-52 us (268 MB)
//   combine_grad_kernel  the latter's gradients: 86-96 us (436 MB, 4.6-5.1 TB/s)
//
// The picks' rows are read past the caches: nothing reads them again soon, and what the call writes then stays there for the
// next (combine 55 -> 45 us at 8191 tokens). Results are not stored past them: a dispatch alone would gain (39 -> 30 us), but
// its reader loses that and more (dispatch and combine of what it wrote, 6 picks of 2048 columns: 8192 tokens 74 -> 82 us,
// 4096 38 -> 42). Rows that are no whole chunks go by chunks at any alignment: 10000 tokens, 4 picks, 1001 columns in bf16 combine
// 40 -> 25 us, its gradient 48 -> 42-47, in fp32 36 -> 38 and 76 -> 62, against elements one by one.
#include <algorithm>

#include "blocks.h"

namespace smx {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxPicks = 16;
constexpr int64_t kMaxCols = int64_t{1} << 24;
constexpr int64_t kGridX = int64_t{1} << 22;  // workgroups along x (HIP takes less than 2^32 threads there); the rest goes along z

struct MoveArgs {
  const char* x;         // one row a token: x, or the gradient of the sum
  const char* rows;      // the picks' rows
  const int32_t* places;
  const float* weights;  // null: 1
  const char* residual;
  int64_t x_ld, rows_ld, residual_ld;
  int64_t T, picks;      // picks: T k
  int H, k;
  int shift;             // log2 of the threads of a token's columns
  char* y;               // dense: one row a token, or the picks' rows
  float* grad_weights;
};

// One thread's chunk of a row, from element `first` on; it lies at `col` (see Chunk).
template <int DT, bool kVec> struct Part {
  static constexpr int kN = Chunk<DT>::kN;
  using S = typename Elem<DT>::S;
  int first, col, H;

  __device__ __forceinline__ Part(int first, int H) : first(first), col(kVec || H < kN ? first : min(first, H - kN)), H(H) {}
  __device__ __forceinline__ bool any() const { return first < H; }
  __device__ __forceinline__ bool in(int j) const { return kVec || (col + j >= first && col + j < H); }

  // kOnce: nothing else reads it soon, so it takes no room in the caches (measured above).
  template <bool kOnce = false> __device__ __forceinline__ Chunk<DT> load(const char* base, int64_t row, int64_t ld) const {
    const S* p = reinterpret_cast<const S*>(base) + row * ld + col;
    if constexpr (kVec) {
      const u32x4* q = reinterpret_cast<const u32x4*>(p);
      return __builtin_bit_cast(Chunk<DT>, kOnce ? __builtin_nontemporal_load(q) : *q);
    } else {
      if (H < kN) return load_short<DT>(p, H - col);
      const auto* q = reinterpret_cast<const typename Loose<DT>::V*>(p);
      return __builtin_bit_cast(Chunk<DT>, static_cast<u32x4>(kOnce ? __builtin_nontemporal_load(q) : *q));
    }
  }
  __device__ __forceinline__ void store(char* base, int64_t row, const Chunk<DT>& r) const {
    S* p = reinterpret_cast<S*>(base) + row * H + col;
    if constexpr (kVec) *reinterpret_cast<u32x4*>(p) = __builtin_bit_cast(u32x4, r);
    else if (H < kN) store_short<DT>(p, H - col, r);
    else *reinterpret_cast<typename Loose<DT>::V*>(p) = __builtin_bit_cast(u32x4, r);
  }
};

__device__ __forceinline__ int64_t block_of() { return static_cast<int64_t>(blockIdx.z) * gridDim.x + blockIdx.x; }

// The token of a thread, and its chunk of the columns.
__device__ __forceinline__ int64_t token_of(const MoveArgs& a) {
  return block_of() * (kThreads >> a.shift) + (threadIdx.x >> a.shift);
}
template <int DT, bool kVec> __device__ __forceinline__ Part<DT, kVec> part_of(const MoveArgs& a) {
  const int width = 1 << a.shift, lane = static_cast<int>(threadIdx.x) & (width - 1);
  return Part<DT, kVec>((static_cast<int>(blockIdx.y) * width + lane) * Chunk<DT>::kN, a.H);
}

// y[t] = residual[t] + sum_j weights[t, j] rows[places[t, j]]. The loads of four picks are on their way at once (of eight: 61
// us for 55, with more registers).
template <int DT, bool kVec>
__global__ __launch_bounds__(kThreads) void combine_kernel(MoveArgs a) {
  constexpr int kN = Chunk<DT>::kN, kBatch = 4;
  const int64_t t = token_of(a);
  const Part<DT, kVec> part = part_of<DT, kVec>(a);
  if (t >= a.T || !part.any()) return;
  float sum[kN] = {};
  const int32_t* at = a.places + t * a.k;
  for (int j0 = 0; j0 < a.k; j0 += kBatch) {
    int32_t p[kBatch];
    float w[kBatch];
    Chunk<DT> r[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) p[i] = j0 + i < a.k ? at[j0 + i] : -1;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (p[i] >= a.picks) p[i] = -1;
      w[i] = p[i] >= 0 && a.weights != nullptr ? a.weights[t * a.k + j0 + i] : 1.0f;
      r[i] = Chunk<DT>{};
      if (p[i] >= 0) r[i] = part.template load<true>(a.rows, p[i], a.rows_ld);
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (p[i] < 0) continue;
#pragma unroll
      for (int j = 0; j < kN; ++j) sum[j] += w[i] * r[i].get(j);
    }
  }
  Chunk<DT> o;
  if (a.residual != nullptr) {
    const Chunk<DT> r = part.load(a.residual, t, a.residual_ld);
#pragma unroll
    for (int j = 0; j < kN; ++j) o.e[j] = round_to<DT>(sum[j] + r.get(j));
  } else {
#pragma unroll
    for (int j = 0; j < kN; ++j) o.e[j] = round_to<DT>(sum[j]);
  }
  part.store(a.y, t, o);
}

// y[places[t, j]] = weights[t, j] x[t], zeros for picks of nobody.
template <int DT, bool kVec>
__global__ __launch_bounds__(kThreads) void spread_kernel(MoveArgs a) {
  constexpr int kN = Chunk<DT>::kN;
  const int64_t t = token_of(a);
  const Part<DT, kVec> part = part_of<DT, kVec>(a);
  if (t >= a.T || !part.any()) return;
  const Chunk<DT> x = part.load(a.x, t, a.x_ld);
  const int32_t* at = a.places + t * a.k;
  for (int j = 0; j < a.k; ++j) {
    const int32_t p = at[j], q = p < 0 ? ~p : p;
    if (q >= a.picks) continue;
    Chunk<DT> o{};
    if (p >= 0) {
      if (a.weights != nullptr) {
        const float w = a.weights[t * a.k + j];
#pragma unroll
        for (int i = 0; i < kN; ++i) o.e[i] = round_to<DT>(w * x.get(i));
      } else {
        o = x;
      }
    }
    part.store(a.y, q, o);
  }
}

// The same with the products <rows[places[t, j]], x[t]>: TPR threads walk over a token's columns, and add up in the end. A
// wave has one token, so that its places, weights and row addresses are scalars (as vectors they left room for three waves a
// SIMD: 106 -> 96 us).
template <int TPR> constexpr int grad_threads() { return TPR == kWave ? kThreads : TPR; }

template <int DT, bool kVec, int TPR, int K>
__global__ __launch_bounds__(grad_threads<TPR>()) void combine_grad_kernel(MoveArgs a) {
  constexpr int kN = Chunk<DT>::kN;
  using Sum = RowSum<TPR, K>;
  __shared__ typename Sum::Lds lds;
  int turn = 0;
  const int64_t t = TPR == kWave ? block_of() * (kThreads / kWave) + wave_id() : block_of();
  const int tid = static_cast<int>(threadIdx.x) % TPR;
  if (t >= a.T) return;  // (whole waves; with TPR > kWave there is a workgroup a token)
  int p[K];
  float w[K], dot[K];
#pragma unroll
  for (int j = 0; j < K; ++j) {
    p[j] = j < a.k ? __builtin_amdgcn_readfirstlane(a.places[t * a.k + j]) : INT32_MAX;
    w[j] = 1.0f;
    if (a.weights != nullptr && j < a.k)
      w[j] = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(a.weights[t * a.k + j])));
    dot[j] = 0.0f;
  }
  const int picks = static_cast<int>(a.picks);
  for (int first = 0; first < a.H; first += TPR * kN) {
    const Part<DT, kVec> part(first + tid * kN, a.H);
    if (!part.any()) break;
    const Chunk<DT> x = part.load(a.x, t, a.x_ld);
    Chunk<DT> r[K];
#pragma unroll
    for (int j = 0; j < K; ++j) {
      r[j] = Chunk<DT>{};
      if (p[j] >= 0 && p[j] < picks) r[j] = part.template load<true>(a.rows, p[j], a.rows_ld);
    }
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const int q = p[j] < 0 ? ~p[j] : p[j];
      if (q >= picks) continue;
      Chunk<DT> o{};
      if (p[j] >= 0) {
#pragma unroll
        for (int i = 0; i < kN; ++i) {
          dot[j] += part.in(i) ? r[j].get(i) * x.get(i) : 0.0f;
          o.e[i] = round_to<DT>(w[j] * x.get(i));
        }
      }
      if (a.y != nullptr) part.store(a.y, q, o);
    }
  }
  Sum::all(dot, lds, turn);
  if (tid == 0) {
#pragma unroll
    for (int j = 0; j < K; ++j)
      if (j < a.k) a.grad_weights[t * a.k + j] = dot[j];
  }
}

// ---- host ----------------------------------------------------------------------------------------

int check_move(int64_t T, int64_t H, int64_t k, int dtype) {
  if (T < 0 || H <= 0 || k <= 0 || !known_dtype(dtype)) return SMX_ERR_INVALID_ARG;
  if (H > kMaxCols || k > kMaxPicks || T > INT32_MAX / k) return SMX_ERR_UNSUPPORTED;
  return SMX_OK;
}

MoveArgs move_args(int64_t T, int64_t H, int64_t k, const int32_t* places) {
  MoveArgs a{};
  a.T = T;
  a.picks = T * k;
  a.H = static_cast<int>(H);
  a.k = static_cast<int>(k);
  a.places = places;
  return a;
}

// `blocks` workgroups of a part of the columns.
dim3 grid_of(int64_t blocks, int64_t parts) {
  return dim3(static_cast<unsigned>(std::min(blocks, kGridX)), static_cast<unsigned>(parts), static_cast<unsigned>((blocks + kGridX - 1) / kGridX));
}

template <typename Kernel>
hipError_t launch_parts(Kernel kernel, MoveArgs& a, int64_t es, hipStream_t s) {
  const int64_t chunks = (a.H * es + 15) / 16;
  a.shift = 0;
  while (a.shift < 8 && (int64_t{1} << a.shift) < chunks) ++a.shift;
  const int64_t tokens = kThreads >> a.shift, width = int64_t{1} << a.shift;
  kernel<<<grid_of((a.T + tokens - 1) / tokens, (chunks + width - 1) / width), kThreads, 0, s>>>(a);
  return hipGetLastError();
}

hipError_t launch_combine(int dtype, bool vec, MoveArgs& a, hipStream_t s) {
  switch (dtype) {
    case kF32: return launch_parts(vec ? combine_kernel<kF32, true> : combine_kernel<kF32, false>, a, 4, s);
    case kF16: return launch_parts(vec ? combine_kernel<kF16, true> : combine_kernel<kF16, false>, a, 2, s);
    default: return launch_parts(vec ? combine_kernel<kBF16, true> : combine_kernel<kBF16, false>, a, 2, s);
  }
}

hipError_t launch_spread(int dtype, bool vec, MoveArgs& a, hipStream_t s) {
  switch (dtype) {
    case kF32: return launch_parts(vec ? spread_kernel<kF32, true> : spread_kernel<kF32, false>, a, 4, s);
    case kF16: return launch_parts(vec ? spread_kernel<kF16, true> : spread_kernel<kF16, false>, a, 2, s);
    default: return launch_parts(vec ? spread_kernel<kBF16, true> : spread_kernel<kBF16, false>, a, 2, s);
  }
}

template <int DT, bool kVec, int TPR>
hipError_t launch_grad_picks(const MoveArgs& a, hipStream_t s) {
  constexpr int threads = grad_threads<TPR>(), tokens = threads / TPR;
  const dim3 n = grid_of((a.T + tokens - 1) / tokens, 1);
  if (a.k <= 2) combine_grad_kernel<DT, kVec, TPR, 2><<<n, threads, 0, s>>>(a);
  else if (a.k <= 4) combine_grad_kernel<DT, kVec, TPR, 4><<<n, threads, 0, s>>>(a);
  else if (a.k <= 8) combine_grad_kernel<DT, kVec, TPR, 8><<<n, threads, 0, s>>>(a);
  else combine_grad_kernel<DT, kVec, TPR, 16><<<n, threads, 0, s>>>(a);
  return hipGetLastError();
}

template <int DT, bool kVec>
hipError_t launch_grad_shape(const MoveArgs& a, hipStream_t s) {
  // As many threads as a row has chunks, up to 256: 8192 tokens, 6 picks, 512 columns 23 us with 64 threads and 31 with 128;
  // 1024 columns 48 and 47 (256: 61); 2048 columns 111, 110 and 96 (512: 133).
  const int64_t chunks = (a.H * dtype_bytes(DT) + 15) / 16;
  if (chunks <= 64) return launch_grad_picks<DT, kVec, 64>(a, s);
  if (chunks <= 128) return launch_grad_picks<DT, kVec, 128>(a, s);
  return launch_grad_picks<DT, kVec, 256>(a, s);
}

template <int DT>
hipError_t launch_grad(bool vec, const MoveArgs& a, hipStream_t s) {
  return vec ? launch_grad_shape<DT, true>(a, s) : launch_grad_shape<DT, false>(a, s);
}

}  // namespace
}  // namespace smx

using namespace smx;

extern "C" {

int smx_dispatch_rows(const void* x, int64_t x_stride, int dtype, int64_t T, int64_t H, const int32_t* places, int64_t k,
                      void* rows, void* stream) {
  const int rc = check_move(T, H, k, dtype);
  if (rc != SMX_OK) return rc;
  if (x_stride < H) return SMX_ERR_INVALID_ARG;
  if (T == 0) return SMX_OK;
  if (!x || !places || !rows) return SMX_ERR_INVALID_ARG;
  const int64_t es = dtype_bytes(dtype);
  if (!aligned_to(x, es) || !aligned_to(rows, es) || !aligned_to(places, 4)) return SMX_ERR_MISALIGNED;
  MoveArgs a = move_args(T, H, k, places);
  a.x = static_cast<const char*>(x);
  a.x_ld = x_stride;
  a.y = static_cast<char*>(rows);
  return static_cast<int>(launch_spread(dtype, whole_chunks(x, x_stride, es) && whole_chunks(rows, H, es), a, static_cast<hipStream_t>(stream)));
}

int smx_combine_rows(const void* rows, int64_t rows_stride, int dtype, int64_t T, int64_t H, const int32_t* places,
                     int64_t k, const float* weights, const void* residual, int64_t residual_stride, void* y,
                     void* stream) {
  const int rc = check_move(T, H, k, dtype);
  if (rc != SMX_OK) return rc;
  if (rows_stride < H || (residual && residual_stride < H)) return SMX_ERR_INVALID_ARG;
  if (T == 0) return SMX_OK;
  if (!rows || !places || !y) return SMX_ERR_INVALID_ARG;
  const int64_t es = dtype_bytes(dtype);
  if (!aligned_to(rows, es) || !aligned_to(residual, es) || !aligned_to(y, es) || !aligned_to(places, 4) || !aligned_to(weights, 4))
    return SMX_ERR_MISALIGNED;
  MoveArgs a = move_args(T, H, k, places);
  a.rows = static_cast<const char*>(rows);
  a.rows_ld = rows_stride;
  a.weights = weights;
  a.residual = static_cast<const char*>(residual);
  a.residual_ld = residual_stride;
  a.y = static_cast<char*>(y);
  const bool vec = whole_chunks(rows, rows_stride, es) && whole_chunks(y, H, es) && (!residual || whole_chunks(residual, residual_stride, es));
  return static_cast<int>(launch_combine(dtype, vec, a, static_cast<hipStream_t>(stream)));
}

int smx_combine_rows_grad(const void* grad_y, int64_t grad_y_stride, const void* rows, int64_t rows_stride, int dtype,
                          int64_t T, int64_t H, const int32_t* places, int64_t k, const float* weights, void* grad_rows,
                          float* grad_weights, void* stream) {
  const int rc = check_move(T, H, k, dtype);
  if (rc != SMX_OK) return rc;
  if (grad_y_stride < H || (grad_weights && rows_stride < H)) return SMX_ERR_INVALID_ARG;
  if (T == 0 || (!grad_rows && !grad_weights)) return SMX_OK;
  if (!grad_y || !places || (grad_weights && !rows)) return SMX_ERR_INVALID_ARG;
  const int64_t es = dtype_bytes(dtype);
  if (!aligned_to(grad_y, es) || !aligned_to(rows, es) || !aligned_to(grad_rows, es) || !aligned_to(places, 4) || !aligned_to(weights, 4) ||
      !aligned_to(grad_weights, 4))
    return SMX_ERR_MISALIGNED;
  MoveArgs a = move_args(T, H, k, places);
  a.x = static_cast<const char*>(grad_y);
  a.x_ld = grad_y_stride;
  a.weights = weights;
  a.y = static_cast<char*>(grad_rows);
  const bool vec = whole_chunks(grad_y, grad_y_stride, es) && whole_chunks(grad_rows, H, es);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (!grad_weights) return static_cast<int>(launch_spread(dtype, vec, a, s));
  a.rows = static_cast<const char*>(rows);
  a.rows_ld = rows_stride;
  a.grad_weights = grad_weights;
  const bool all = vec && whole_chunks(rows, rows_stride, es);
  switch (dtype) {
    case kF32: return static_cast<int>(launch_grad<kF32>(all, a, s));
    case kF16: return static_cast<int>(launch_grad<kF16>(all, a, s));
    default: return static_cast<int>(launch_grad<kBF16>(all, a, s));
  }
}

}  // extern "C"
