// Tiled matrix products: one output tile per workgroup of 4 waves, any size, stride, alignment and type.
//
// A step takes 128 bytes of the contraction (64 16-bit or 32 fp32 elements) of both operands through LDS:
// an operand contiguous along the contraction as rows of 8 16-byte slots, a strided one as contraction rows of
// R elements. The slots of a row are permuted (an exclusive-or with the row) so that fragment reads have no bank
// conflicts; a strided 16-bit operand's fragments come through the transposing LDS read.
//
// Two ways in: `staged` loads registers and writes LDS behind them, for operands of any alignment (16-byte loads
// that need not be aligned, element loads at the edges); otherwise the operands are copied straight into LDS.
#include "product.h"

namespace smx {

typedef short i16x4 __attribute__((ext_vector_type(4)));

// LDS stage of R rows (or columns) of an operand over one step.
template <int DT, int R, bool ST>
struct Stage {
  using S = typename Elem<DT>::S;
  static constexpr int kEs = sizeof(S);
  static constexpr int kEps = 16 / kEs;                    // elements per slot
  static constexpr int kDepth = kPStep / kEs;              // contraction elements per step
  static constexpr int kSlots = R * 8;                     // 16-byte slots
  static constexpr int kRowSlots = ST ? R / kEps : 8;      // slots per LDS row
  static constexpr int kLoads = kSlots / kPThreads;        // 16-byte loads per thread and step

  // Slot s of LDS row y stands at slot perm(y, s). It is its own inverse.
  static __device__ __forceinline__ int perm(int y, int s) {
    if constexpr (!ST) return s ^ (y & 7);
    else if constexpr (DT == kF32) return s ^ (((y >> 2) & 3) * 4 & (kRowSlots - 1));
    else return s ^ ((((y & 3) | ((y >> 1) & 4)) * 2) & (kRowSlots - 1));
  }

  // The lane's part of the fragment of 16 rows from `row`, half u of the step: elements of row
  // row + lane % 16, contraction indices (4 u + lane / 16) kEps ..; tile rows are multiples of 16.
  static __device__ __forceinline__ u32x4 frag(const u32x4* st, int row, int u) {
    const int lane = lane_id(), r = lane & 15, g = lane >> 4;
    if constexpr (!ST) {
      return st[(row + r) * 8 + perm(r, 4 * u + g)];
    } else if constexpr (DT == kF32) {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(st);
      u32x4 v;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = 16 * u + 4 * g + j;
        v[j] = w[(k * kRowSlots + perm(k, (row + r) >> 2)) * 4 + (r & 3)];
      }
      return v;
    } else {
      // Transposing read of 8 bytes per lane: the 16 lanes of a group address four rows of 16
      // elements (lane r: row r / 4, elements 4 (r % 4) ..); lane r receives element r of each.
      u32x2 h[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int k = 32 * u + 8 * g + 4 * j + (r >> 2);
        const char* at = reinterpret_cast<const char*>(st + k * kRowSlots + perm(k, (row >> 3) + ((r & 3) >> 1))) + 8 * (r & 1);
        h[j] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) i16x4*)(at)));
      }
      return u32x4{h[0][0], h[0][1], h[1][0], h[1][1]};
    }
  }
};

// Where an operand's step comes from, staged through registers.
template <int DT, int R, bool ST>
struct StagedLoad {
  using G = Stage<DT, R, ST>;
  using S = typename G::S;
  const S* base;   // first element at contraction index 0
  int64_t ld;
  int n;           // contiguous: rows that exist; strided: columns
  int depth;       // contraction length
  u32x4 v[G::kLoads];

  // Element `e` of a slot lies at `at[e]`; the first `have` of the kEps exist.
  static __device__ __forceinline__ u32x4 load_slot(const S* at, int have) {
    u32x4 r = {0, 0, 0, 0};
    if (have >= G::kEps) {
      __builtin_memcpy(&r, at, 16);
    } else if (have > 0) {
      S e[G::kEps];
#pragma unroll
      for (int i = 0; i < G::kEps; ++i) e[i] = i < have ? at[i] : S{};
      __builtin_memcpy(&r, e, 16);
    }
    return r;
  }

  template <typename RowAt>
  __device__ __forceinline__ void load(int k0, RowAt&& row_at) {
#pragma unroll
    for (int j = 0; j < G::kLoads; ++j) {
      const int i = threadIdx.x + kPThreads * j;
      const int y = i / G::kRowSlots, s = i % G::kRowSlots;
      if constexpr (!ST) {
        const int k = k0 + s * G::kEps;
        v[j] = y < n ? load_slot(base + row_at(y) * ld + k, depth - k) : u32x4{0, 0, 0, 0};
      } else {
        const int k = k0 + y;
        v[j] = k < depth ? load_slot(base + k * ld + s * G::kEps, n - s * G::kEps) : u32x4{0, 0, 0, 0};
      }
    }
  }
  __device__ __forceinline__ void store(u32x4* st) const {
#pragma unroll
    for (int j = 0; j < G::kLoads; ++j) {
      const int i = threadIdx.x + kPThreads * j;
      const int y = i / G::kRowSlots, s = i % G::kRowSlots;
      st[y * G::kRowSlots + G::perm(y, s)] = v[j];
    }
  }
};

// Waves of a tile: 2 x 2, but side by side over the columns of a tile of few rows. A wave's column tiles come in pairs
// (gated products need gate and up in one wave).
template <int BM, int BN>
struct Waves {
  static constexpr int kRowWaves = BM >= 128 || BN < 128 ? 2 : 1;
  static constexpr int kColWaves = kPWaves / kRowWaves;
  static constexpr int kNI = BN / kColWaves / 16;  // 16-column tiles of a wave
  static constexpr int kNJ = BM / kRowWaves / 16;  // 16-row tiles
  static_assert(kNI >= 2 && kNI % 2 == 0 && kNJ >= 1, "column tiles in pairs");
};

// Row of P that column q of a tile stands for, relative to the tile's first. Gated: 16 gate columns, then the
// matching 16 up columns (out_cols further), and so on.
__device__ __forceinline__ int64_t p_row(const ProductArgs& a, int q) {
  return a.gated ? ((q >> 5) << 4) + (q & 15) + ((q >> 4) & 1) * static_cast<int64_t>(a.out_cols) : q;
}

// Epilogue of a wave's accumulators; c0: first product column of the tile (gated: twice its first output column).
template <int DT, int NI, int NJ>
__device__ __forceinline__ void finish_tile(const ProductArgs& a, const ProductItem& it, int c0, int wrow, int wcol,
                                            const f32x4 (&acc)[NI][NJ]) {
  const int lane = lane_id();
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int r = wrow + j * 16 + (lane & 15);
    if (r >= it.m) continue;
    const int64_t row = it.row + r;
    if (a.splits > 1) {
      float* dst = a.part + (static_cast<int64_t>(it.split) * a.rows + row) * a.cols;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int q = wcol + i * 16 + 4 * (lane >> 4);
        const int col = (a.gated ? c0 / 2 : c0) + static_cast<int>(p_row(a, q));
        const int end = a.gated && !((q >> 4) & 1) ? a.out_cols : a.cols;
        if (col < end) store4<kF32>(reinterpret_cast<char*>(dst), col, end - col, a.cols % 4 == 0 && a.out_cols % 4 == 0, acc[i][j]);
      }
    } else if (a.gated) {
      if constexpr (NI % 2 == 0) {
#pragma unroll
        for (int i = 0; i < NI; i += 2)
          finish4_gated<DT>(a, it, row, (c0 + wcol) / 2 + i * 8 + 4 * (lane >> 4), acc[i][j], acc[i + 1][j]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NI; ++i) finish4<DT>(a, it, row, c0 + wcol + i * 16 + 4 * (lane >> 4), acc[i][j]);
    }
  }
}

template <int DT, int BM, int BN, bool PS, bool QS, bool DG>
__global__ __launch_bounds__(kPThreads) void product_staged_kernel(ProductArgs a) {
  using GP = Stage<DT, BN, PS>;
  using GQ = Stage<DT, BM, QS>;
  using W = Waves<BM, BN>;
  using S = typename GP::S;
  const int b = static_cast<int>(blockIdx.x);
  if (b >= a.item_blocks) {
    fill_rows<DT>(a, b - a.item_blocks);
    return;
  }
  ProductItem it;
  const int col_tiles = (a.gated ? (a.out_cols + BN / 2 - 1) / (BN / 2) : (a.cols + BN - 1) / BN);
  if (!(DG ? find_depth_item(a, b, BM, col_tiles, it) : find_row_item(a, b, BM, col_tiles, it))) return;
  __shared__ u32x4 sp[GP::kSlots], sq[GQ::kSlots];

  const int c0 = it.ct * BN;
  const int cfirst = a.gated ? c0 / 2 : c0;
  const S* pb = reinterpret_cast<const S*>(a.p) + (DG ? 0 : it.w * a.p_group);
  const S* qb = reinterpret_cast<const S*>(a.q);
  StagedLoad<DT, BN, PS> lp;
  StagedLoad<DT, BM, QS> lq;
  lp.ld = a.p_ld;
  lq.ld = a.q_ld;
  lp.depth = lq.depth = it.depth;
  if constexpr (PS) pb += static_cast<int64_t>(it.k0) * a.p_ld + cfirst;
  else pb += cfirst * a.p_ld;
  if constexpr (QS) qb += static_cast<int64_t>(it.k0) * a.q_ld + it.row;
  else qb += static_cast<int64_t>(it.row) * a.q_ld;
  lp.base = pb;
  lq.base = qb;
  lp.n = PS ? a.cols - c0 : BN;
  lq.n = it.m;
  // columns past the last: the last one again (not stored)
  const int last = a.out_cols - 1 - cfirst;
  auto p_at = [&](int q) -> int64_t {
    if (a.gated) return min(((q >> 5) << 4) + (q & 15), last) + ((q >> 4) & 1) * static_cast<int64_t>(a.out_cols);
    return min(q, last);
  };
  auto q_at = [](int q) -> int64_t { return q; };

  const int steps = (it.depth + GP::kDepth - 1) / GP::kDepth;
  const int s0 = it.split * a.split_steps;
  const int s1 = a.splits > 1 ? min(steps, s0 + a.split_steps) : steps;
  const int wave = wave_id();
  const int wrow = (wave / W::kColWaves) * W::kNJ * 16, wcol = (wave % W::kColWaves) * W::kNI * 16;
  f32x4 acc[W::kNI][W::kNJ];
#pragma unroll
  for (int i = 0; i < W::kNI; ++i)
#pragma unroll
    for (int j = 0; j < W::kNJ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (s0 < s1) {
    lp.load(s0 * GP::kDepth, p_at);
    lq.load(s0 * GP::kDepth, q_at);
  }
  for (int s = s0; s < s1; ++s) {
    __syncthreads();
    lp.store(sp);
    lq.store(sq);
    __syncthreads();
    if (s + 1 < s1) {
      lp.load((s + 1) * GP::kDepth, p_at);
      lq.load((s + 1) * GP::kDepth, q_at);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      u32x4 fp[W::kNI], fq[W::kNJ];
#pragma unroll
      for (int i = 0; i < W::kNI; ++i) fp[i] = GP::frag(sp, wcol + i * 16, u);
#pragma unroll
      for (int j = 0; j < W::kNJ; ++j) fq[j] = GQ::frag(sq, wrow + j * 16, u);
#pragma unroll
      for (int i = 0; i < W::kNI; ++i)
#pragma unroll
        for (int j = 0; j < W::kNJ; ++j) acc[i][j] = Elem<DT>::mfma(fp[i], fq[j], acc[i][j]);
    }
  }
  finish_tile<DT>(a, it, c0, wrow, wcol, acc);
}

template <int DT, int BM, int BN>
static hipError_t staged_launch(bool ps, bool qs, bool dg, const ProductArgs& a, hipStream_t s) {
  const unsigned blocks = static_cast<unsigned>(a.item_blocks + a.fill_blocks);
  if (!ps && !qs && !dg) product_staged_kernel<DT, BM, BN, false, false, false><<<blocks, kPThreads, 0, s>>>(a);
  else if (ps && !qs && !dg) product_staged_kernel<DT, BM, BN, true, false, false><<<blocks, kPThreads, 0, s>>>(a);
  else if (ps && qs && dg) product_staged_kernel<DT, BM, BN, true, true, true><<<blocks, kPThreads, 0, s>>>(a);
  else return hipErrorInvalidValue;
  return hipGetLastError();
}

template <int DT>
static hipError_t tile_launch(bool ps, bool qs, bool dg, const TileShape& t, const ProductArgs& a, hipStream_t s) {
  if (t.staged && t.bm == 64 && t.bn == 64) return staged_launch<DT, 64, 64>(ps, qs, dg, a, s);
  if (t.staged && t.bm == 128 && t.bn == 128) return staged_launch<DT, 128, 128>(ps, qs, dg, a, s);
  return hipErrorInvalidValue;
}

hipError_t launch_product_tile(int dtype, bool p_strided, bool q_strided, bool depth_groups, const TileShape& t,
                               const ProductArgs& a, hipStream_t s) {
  switch (dtype) {
    case kF32: return tile_launch<kF32>(p_strided, q_strided, depth_groups, t, a, s);
    case kF16: return tile_launch<kF16>(p_strided, q_strided, depth_groups, t, a, s);
    case kBF16: return tile_launch<kBF16>(p_strided, q_strided, depth_groups, t, a, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace smx
