// What the kernels around the products share: 16-byte chunks of a row's elements, sums over the threads of a row.
#pragma once

#include "../../include/specmoe_mi355x.h"
#include "../../include/specmoe_mi355x_blocks.h"
#include "topk_device.h"

namespace smx {

// Elements of one 16-byte load. Where rows are not whole chunks, a chunk's elements lie apart instead and are loaded
// one by one (kVec false below).
template <int DT> struct Chunk {
  using S = typename Elem<DT>::S;
  static constexpr int kN = 16 / sizeof(S);
  S e[kN];
  __device__ __forceinline__ float get(int j) const { return Elem<DT>::to_f32(e[j]); }
};

// Round to nearest even (v_cvt_pk_bf16_f32); NaN stays NaN.
template <int DT> __device__ __forceinline__ typename Elem<DT>::S round_to(float f) { return Elem<DT>::from_f32(f); }
template <> __device__ __forceinline__ uint16_t round_to<kBF16>(float f) {
  return __builtin_bit_cast(uint16_t, static_cast<__bf16>(f));
}

// Chunk c of the TPR threads' walk over a row of H elements: elements (c TPR + tid) N .. + N - 1, or one by one
// (c N + j) TPR + tid, so that neighbouring threads touch neighbouring elements either way.
template <int DT, int TPR, bool kVec> struct RowWalk {
  static constexpr int kN = Chunk<DT>::kN;
  using S = typename Elem<DT>::S;
  int H, tid;

  __device__ __forceinline__ int col(int c, int j) const {
    return kVec ? (c * TPR + tid) * kN + j : (c * kN + j) * TPR + tid;
  }
  __device__ __forceinline__ bool in(int c, int j) const { return col(c, kVec ? 0 : j) < H; }

  // Elements behind the row's end are zeros.
  __device__ __forceinline__ Chunk<DT> load(const S* row, int c) const {
    Chunk<DT> r;
    if constexpr (kVec) {
      u32x4 v = {0u, 0u, 0u, 0u};
      if (in(c, 0)) v = *reinterpret_cast<const u32x4*>(row + col(c, 0));
      r = __builtin_bit_cast(Chunk<DT>, v);
    } else {
#pragma unroll
      for (int j = 0; j < kN; ++j) r.e[j] = in(c, j) ? row[col(c, j)] : S{};
    }
    return r;
  }

  __device__ __forceinline__ void store(S* row, int c, const Chunk<DT>& r) const {
    if constexpr (kVec) {
      if (in(c, 0)) *reinterpret_cast<u32x4*>(row + col(c, 0)) = __builtin_bit_cast(u32x4, r);
    } else {
#pragma unroll
      for (int j = 0; j < kN; ++j)
        if (in(c, j)) row[col(c, j)] = r.e[j];
    }
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
          if (in(c, 0)) v = *reinterpret_cast<const f32x4*>(q + col(c, j));
#pragma unroll
          for (int i = 0; i < 4; ++i) w[j + i] = v[i];
        }
      } else {
#pragma unroll
        for (int j = 0; j < kN; ++j) w[j] = in(c, j) ? q[col(c, j)] : 0.0f;
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
