// What the kernels around the products share: 16-byte chunks of a row's elements, sums over the threads of a row.
#pragma once

#include "../../include/specmoe_mi355x.h"
#include "../../include/specmoe_mi355x_blocks.h"
#include "topk_device.h"

namespace smx {

// Elements of one 16-byte load. kVec below: rows are whole chunks, 16-byte aligned. Otherwise a chunk is only aligned as its
// elements are (global loads and stores take any alignment), and the last one of a row ends with the row: its first elements
// are the one's before it too, which counts them; both write the same there. (Rows shorter than a chunk: element by element.)
template <int DT> struct Chunk {
  using S = typename Elem<DT>::S;
  static constexpr int kN = 16 / sizeof(S);
  S e[kN];
  __device__ __forceinline__ float get(int j) const { return Elem<DT>::to_f32(e[j]); }
};

// 16 bytes at an element's alignment.
typedef uint32_t u32x4_at2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4_at4 __attribute__((ext_vector_type(4), aligned(4)));
template <int DT> struct Loose { using V = u32x4_at2; };
template <> struct Loose<kF32> { using V = u32x4_at4; };

// Round to nearest even (v_cvt_pk_bf16_f32); NaN stays NaN.
template <int DT> __device__ __forceinline__ typename Elem<DT>::S round_to(float f) { return Elem<DT>::from_f32(f); }
template <> __device__ __forceinline__ uint16_t round_to<kBF16>(float f) {
  return __builtin_bit_cast(uint16_t, static_cast<__bf16>(f));
}

// Elements at p, of which only the first `rest` are there.
template <int DT> __device__ __forceinline__ Chunk<DT> load_short(const typename Elem<DT>::S* p, int rest) {
  Chunk<DT> r{};
#pragma unroll
  for (int j = 0; j < Chunk<DT>::kN; ++j)
    if (j < rest) r.e[j] = p[j];
  return r;
}
template <int DT> __device__ __forceinline__ void store_short(typename Elem<DT>::S* p, int rest, const Chunk<DT>& r) {
#pragma unroll
  for (int j = 0; j < Chunk<DT>::kN; ++j)
    if (j < rest) p[j] = r.e[j];
}

// Chunk c of the TPR threads' walk over a row of H elements: elements (c TPR + tid) N .. + N - 1.
template <int DT, int TPR, bool kVec> struct RowWalk {
  static constexpr int kN = Chunk<DT>::kN;
  using S = typename Elem<DT>::S;
  int H, tid;

  __device__ __forceinline__ int first(int c) const { return (c * TPR + tid) * kN; }
  __device__ __forceinline__ int at(int c) const { return kVec || H < kN ? first(c) : min(first(c), H - kN); }
  __device__ __forceinline__ bool any(int c) const { return first(c) < H; }
  __device__ __forceinline__ int col(int c, int j) const { return at(c) + j; }
  // Whether the element is in the row, and this chunk's.
  __device__ __forceinline__ bool in(int c, int j) const {
    return kVec ? any(c) : any(c) && col(c, j) >= first(c) && col(c, j) < H;
  }

  // Chunks behind the row's end are zeros.
  __device__ __forceinline__ Chunk<DT> load(const S* row, int c) const {
    Chunk<DT> r{};
    if constexpr (kVec) {
      if (any(c)) r = __builtin_bit_cast(Chunk<DT>, *reinterpret_cast<const u32x4*>(row + at(c)));
    } else if (H < kN) {
      if (any(c)) r = load_short<DT>(row + at(c), H - at(c));
    } else {
      if (any(c)) r = __builtin_bit_cast(Chunk<DT>, static_cast<u32x4>(*reinterpret_cast<const typename Loose<DT>::V*>(row + at(c))));
    }
    return r;
  }

  __device__ __forceinline__ void store(S* row, int c, const Chunk<DT>& r) const {
    if (!any(c)) return;
    if constexpr (kVec) *reinterpret_cast<u32x4*>(row + at(c)) = __builtin_bit_cast(u32x4, r);
    else if (H < kN) store_short<DT>(row + at(c), H - at(c), r);
    else *reinterpret_cast<typename Loose<DT>::V*>(row + at(c)) = __builtin_bit_cast(u32x4, r);
  }

  // A vector of parameters of the row's type or fp32, `rest` where there is none.
  __device__ __forceinline__ void params(const void* p, bool wide, float rest, int c, float (&w)[kN]) const {
    if (p == nullptr) {
#pragma unroll
      for (int j = 0; j < kN; ++j) w[j] = rest;
    } else if (DT != kF32 && wide) {
      const float* q = static_cast<const float*>(p);
      if constexpr (kVec) {
#pragma unroll
        for (int j = 0; j < kN; j += 4) {
          f32x4 v = {0.f, 0.f, 0.f, 0.f};
          if (any(c)) v = *reinterpret_cast<const f32x4*>(q + at(c) + j);
#pragma unroll
          for (int i = 0; i < 4; ++i) w[j + i] = v[i];
        }
      } else {
#pragma unroll
        for (int j = 0; j < kN; ++j) w[j] = any(c) && col(c, j) < H ? q[col(c, j)] : 0.0f;
      }
    } else {
      const Chunk<DT> r = load(static_cast<const S*>(p), c);
#pragma unroll
      for (int j = 0; j < kN; ++j) w[j] = r.get(j);
    }
  }
};

// Sums of n values over the TPR threads of a row; every thread gets them. Within a wave by lane exchange, over the
// waves of a workgroup (which then holds one row) through LDS, in the order of the waves. Two sets of slots in turn:
// a set is written again only behind the other's barrier, so one barrier a call is enough.
template <int TPR, int N> struct RowSum {
  static constexpr int kWaves = TPR > kWave ? TPR / kWave : 1;
  struct Lds { float v[2][N][kWaves]; };

  __device__ static __forceinline__ void all(float (&v)[N], Lds& lds, int& turn) {
#pragma unroll
    for (int n = 0; n < N; ++n)
      v[n] = group_reduce<(TPR < kWave ? TPR : kWave)>(v[n], [](float a, float b) { return a + b; });
    if constexpr (TPR > kWave) {
      turn ^= 1;
      if (lane_id() == 0) {
#pragma unroll
        for (int n = 0; n < N; ++n) lds.v[turn][n][wave_id()] = v[n];
      }
      __syncthreads();
#pragma unroll
      for (int n = 0; n < N; ++n) {
        v[n] = lds.v[turn][n][0];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) v[n] += lds.v[turn][n][w];
      }
    }
  }
};

inline bool aligned_to(const void* p, int64_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
inline bool known_dtype(int dt) { return dt == kF32 || dt == kF16 || dt == kBF16; }
// Rows of whole chunks: the base and the pitch (the length is the caller's to check).
inline bool whole_chunks(const void* p, int64_t pitch, int64_t es) { return aligned_to(p, 16) && pitch * es % 16 == 0; }

}  // namespace smx
