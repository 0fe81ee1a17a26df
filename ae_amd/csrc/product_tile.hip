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
      const int k = 8 * g + (r >> 2);
      const char* base = reinterpret_cast<const char*>(st) + (k * kRowSlots + perm(k, (row >> 3) + ((r & 3) >> 1))) * 16 + 8 * (r & 1);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const char* at = base + (32 * u + 4 * j) * kRowSlots * 16;
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

  template <typename RowAt>
  __device__ __forceinline__ void load(int k0, RowAt&& row_at) {
#pragma unroll
    for (int j = 0; j < G::kLoads; ++j) {
      const int i = threadIdx.x + kPThreads * j;
      const int y = i / G::kRowSlots, s = i % G::kRowSlots;
      if constexpr (!ST) {
        const int k = k0 + s * G::kEps;
        v[j] = y < n ? load_slot<DT>(base + row_at(y) * ld + k, depth - k) : u32x4{0, 0, 0, 0};
      } else {
        const int k = k0 + y;
        v[j] = k < depth ? load_slot<DT>(base + k * ld + s * G::kEps, n - s * G::kEps) : u32x4{0, 0, 0, 0};
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

// Epilogue of a wave's accumulators: through its part of LDS, CJ row tiles at a time, as rows of 4 NI 16-byte slots
// (slot s of row r at s ^ r, modulo the row: no bank conflicts), from which a lane takes four columns (gated: the gate
// and up columns of four outputs) of some rows. The bias then stays in registers, stores cover whole row pieces, and
// the activation's code stands once.
// c0: first product column of the tile (gated: 16 gate columns, the matching 16 up columns, and so on: twice the
// first output column). wrow, wcol: the wave's place in the tile.
template <int DT, int NI, int NJ, int CJ>
__device__ __forceinline__ void finish_wave(const ProductArgs& a, const ProductItem& it, int c0, int wrow, int wcol,
                                            u32x4* lds, const f32x4 (&acc)[NI][NJ]) {
  constexpr int kS = 4 * NI;  // slots of a row
  static_assert(NJ % CJ == 0, "whole chunks");
  f32x4* st = reinterpret_cast<f32x4*>(lds);
  const int lane = lane_id();
  // lanes side by side along a row: one per output column quad
  const int quads = a.gated ? kS / 2 : kS;
  const int c = lane & (quads - 1), rr = lane / quads, rows = kWave / quads;
  const int s0 = a.gated ? (c >> 2) * 8 + (c & 3) : c;
  const int col = a.gated ? (c0 + wcol) / 2 + 4 * c : c0 + wcol + 4 * c;
  const int left = a.out_cols - col;
  const bool part = a.splits > 1;
  const f32x4 bias0 = part ? f32x4{} : bias4<DT>(a, it, col, left);
  const f32x4 bias1 = part || !a.gated ? f32x4{} : bias4<DT>(a, it, a.out_cols + col, left);
#pragma unroll
  for (int j0 = 0; j0 < NJ; j0 += CJ) {
#pragma unroll
    for (int j = 0; j < CJ; ++j)
#pragma unroll
      for (int i = 0; i < NI; ++i)
        st[(j * 16 + (lane & 15)) * kS + ((4 * i + (lane >> 4)) ^ (lane & (kS - 1) & 15))] = acc[i][j0 + j];
    constexpr int kBatch = 4;  // rows of a lane that are finished together
    for (int y0 = rr; y0 < CJ * 16; y0 += kBatch * rows) {
      int64_t row[kBatch];
      bool in[kBatch];
      f32x4 v[kBatch], u[kBatch], res[kBatch];
#pragma unroll
      for (int n = 0; n < kBatch; ++n) {
        const int y = y0 + n * rows, r = wrow + j0 * 16 + y;
        in[n] = y < CJ * 16 && r < it.m && left > 0;
        row[n] = static_cast<int64_t>(it.row) + r;
        const int yy = y < CJ * 16 ? y : 0;
        v[n] = st[yy * kS + (s0 ^ (yy & (kS - 1) & 15))];
        u[n] = a.gated ? st[yy * kS + ((s0 + 4) ^ (yy & (kS - 1) & 15))] : f32x4{};
        res[n] = res4<DT>(a, row[n], col, in[n] && !part ? left : 0);
      }
      if (part) {
        const bool vec = a.cols % 4 == 0 && a.out_cols % 4 == 0;
#pragma unroll
        for (int n = 0; n < kBatch; ++n) {
          if (!in[n]) continue;
          const int64_t at = (static_cast<int64_t>(it.split) * a.rows + row[n]) * a.cols + col;
          store4<kF32>(reinterpret_cast<char*>(a.part), at, left, vec, v[n]);
          if (a.gated) store4<kF32>(reinterpret_cast<char*>(a.part), at + a.out_cols, left, vec, u[n]);
        }
      } else if (a.gated) {
        finish_rows_gated<DT>(a, row, in, col, left, v, u, bias0, bias1, res);
      } else {
        finish_rows<DT>(a, it, row, in, col, left, v, bias0, res);
      }
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
  f32x4 acc[W::kNI][W::kNJ] = {}, total[W::kNI][W::kNJ] = {};
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
    if (DT == kF32 && (s - s0) % kFold == kFold - 1) fold(total, acc);
  }
  if constexpr (DT == kF32) {
    fold(total, acc);
    fold(acc, total);
  }
  __syncthreads();
  u32x4* mine = (wave < 2 ? sp : sq) + (wave & 1) * (GP::kSlots / 2);
  static_assert(GP::kSlots == GQ::kSlots, "a square tile");
  constexpr int kChunk = GP::kSlots / 2 / (W::kNI * 64);
  finish_wave<DT, W::kNI, W::kNJ, kChunk < W::kNJ ? kChunk : W::kNJ>(a, it, c0, wrow, wcol, mine, acc);
}

// Copies of one operand's steps straight into LDS: copy j of wave w fills stage slots 64 (4 j + w) .. in lane order.
template <int DT, int R, bool ST>
struct TileCopy {
  using G = Stage<DT, R, ST>;
  const char* base;
  int64_t step_bytes;
  uint32_t off[G::kLoads];
  int k[G::kLoads];  // the lane's first contraction element within a step
  // at(y): byte offset of the operand's row y (contiguous); last: byte offset of its last whole slot (strided)
  template <typename At>
  __device__ __forceinline__ void init(int wave, int64_t pitch, At&& at, int last) {
    step_bytes = ST ? G::kDepth * pitch : kPStep;
#pragma unroll
    for (int j = 0; j < G::kLoads; ++j) {
      const int p = 64 * (kPWaves * j + wave) + lane_id();
      const int y = p / G::kRowSlots, s = G::perm(y, p % G::kRowSlots);
      k[j] = ST ? y : s * G::kEps;
      off[j] = ST ? static_cast<uint32_t>(y * pitch) + min(s * 16, last) : at(y) + s * 16;
    }
  }
  // Elements of the step from contraction index `left` on are left out (zeros); left <= 0: nothing is read.
  __device__ __forceinline__ void copy(u32x4* st, int wave, int step, int left) const {
    const auto r = make_rsrc(base + step * step_bytes, left > 0 ? kPOutside : 0u);
#pragma unroll
    for (int j = 0; j < G::kLoads; ++j) {
      const uint32_t o = k[j] < left ? off[j] : kPOutside;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          r, (__attribute__((address_space(3))) void*)(st + (j * kPWaves + wave) * kWave), 16, o, 0, 0, 0);
    }
  }
};

__device__ __forceinline__ void bare_barrier() {  // without a memory fence, which would wait for the copies
  asm volatile("s_barrier" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// The same tile with the operands copied straight into LDS, two stages: while one step is multiplied the next one's
// copies are under way, and the other workgroup of the CU covers the waits.
template <int DT, int BM, int BN, bool PS, bool QS, bool DG>
__global__ __launch_bounds__(kPThreads, 2) void product_copied_kernel(ProductArgs a) {
  using GP = Stage<DT, BN, PS>;
  using GQ = Stage<DT, BM, QS>;
  using W = Waves<BM, BN>;
  constexpr int64_t kEs = GP::kEs;
  const int b = static_cast<int>(blockIdx.x);
  if (b >= a.item_blocks) {
    fill_rows<DT>(a, b - a.item_blocks);
    return;
  }
  ProductItem it;
  const int col_tiles = (a.gated ? (a.out_cols + BN / 2 - 1) / (BN / 2) : (a.cols + BN - 1) / BN);
  if (!(DG ? find_depth_item(a, b, BM, col_tiles, it) : find_row_item(a, b, BM, col_tiles, it))) return;
  __shared__ u32x4 p0[GP::kSlots], p1[GP::kSlots], q0[GQ::kSlots], q1[GQ::kSlots];

  const int c0 = it.ct * BN;
  const int cfirst = a.gated ? c0 / 2 : c0;
  const int wave = wave_id();
  const int64_t p_pitch = a.p_ld * kEs, q_pitch = a.q_ld * kEs;
  TileCopy<DT, BN, PS> cp;
  TileCopy<DT, BM, QS> cq;
  cp.base = a.p + (DG ? int64_t{0} : it.w * a.p_group * kEs) + (PS ? it.k0 * p_pitch + cfirst * kEs : cfirst * p_pitch);
  cq.base = a.q + (QS ? it.k0 * q_pitch + it.row * kEs : it.row * q_pitch);
  const int plast = a.out_cols - 1 - cfirst;  // columns past the last: the last one again (not stored)
  cp.init(wave, p_pitch, [&](int q) -> uint32_t {
    const int64_t row = a.gated ? min(((q >> 5) << 4) + (q & 15), plast) + ((q >> 4) & 1) * static_cast<int64_t>(a.out_cols)
                                : static_cast<int64_t>(min(q, plast));
    return static_cast<uint32_t>(row * p_pitch);
  }, static_cast<int>((a.cols - cfirst) * kEs) - 16);
  cq.init(wave, q_pitch, [&](int q) -> uint32_t { return static_cast<uint32_t>(min(q, it.m - 1) * q_pitch); },
          static_cast<int>((a.q_cols - it.row) * kEs) - 16);

  const int steps = (it.depth + GP::kDepth - 1) / GP::kDepth;
  const int s0 = it.split * a.split_steps;
  const int s1 = a.splits > 1 ? min(steps, s0 + a.split_steps) : steps;
  const int wrow = (wave / W::kColWaves) * W::kNJ * 16, wcol = (wave % W::kColWaves) * W::kNI * 16;
  f32x4 acc[W::kNI][W::kNJ] = {}, total[W::kNI][W::kNJ] = {};
  constexpr int kCopies = GP::kLoads + GQ::kLoads;
  auto copy = [&](u32x4* sp, u32x4* sq, int s) {
    const int left = s < s1 ? it.depth - s * GP::kDepth : 0;
    cp.copy(sp, wave, s, left);
    cq.copy(sq, wave, s, left);
    __builtin_amdgcn_sched_barrier(0);
  };
  // one step, with the copies of the step after the next behind it; or one of the last two, without them
  auto step = [&](u32x4* sp, u32x4* sq, int s, auto more) {
    // this step's copies have landed, the next one's may be under way
    if constexpr (decltype(more)::value) __builtin_amdgcn_s_waitcnt(vmcnt_imm(kCopies));
    else __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
    bare_barrier();
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
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (decltype(more)::value) {
      bare_barrier();  // every wave has read the stage (its fragments are in registers: the MFMAs are issued)
      copy(sp, sq, s + 2);
    }
  };
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
  __builtin_amdgcn_sched_barrier(0);
  const std::true_type more{};
  const std::false_type last{};
  if (s0 < s1) {
    copy(p0, q0, s0);
    copy(p1, q1, s0 + 1);
    int s = s0;
    for (; s + 2 < s1; s += 2) {
      step(p0, q0, s, more);
      step(p1, q1, s + 1, more);
      if (DT == kF32 && (s - s0) % kFold == kFold - 2) fold(total, acc);
    }
    // (a step past the end multiplies zeros: a branch inside the loop costs waits for all copies)
    step(p0, q0, s, last);
    step(p1, q1, s + 1, last);
  }
  if constexpr (DT == kF32) {
    fold(total, acc);
    fold(acc, total);
  }
  __syncthreads();
  u32x4* mine = wave == 0 ? p0 : wave == 1 ? p1 : wave == 2 ? q0 : q1;
  constexpr int kSmall = GP::kSlots < GQ::kSlots ? GP::kSlots : GQ::kSlots;
  constexpr int kChunk = kSmall / (W::kNI * 64);
  static_assert(kChunk >= 1, "a row tile of the wave fits its LDS");
  finish_wave<DT, W::kNI, W::kNJ, kChunk < W::kNJ ? kChunk : W::kNJ>(a, it, c0, wrow, wcol, mine, acc);
}

template <int DT, int BM, int BN>
static hipError_t copied_launch(bool ps, bool qs, bool dg, const ProductArgs& a, hipStream_t s) {
  const unsigned blocks = static_cast<unsigned>(a.item_blocks + a.fill_blocks);
  // whole 16-byte slots: the contraction of a contiguous operand, the columns (rows) of a strided one
  constexpr int n = 16 / dtype_bytes(DT);
  if (a.p_ld % n != 0 || a.q_ld % n != 0 || a.p_group % n != 0) return hipErrorInvalidValue;
  // (beside a strided P a contiguous Q may end inside a slot, with zeros up to the slot's end)
  if (!ps && a.depth % n != 0) return hipErrorInvalidValue;
  if ((ps && a.cols % n != 0) || (qs && (a.q_cols % n != 0 || a.q_cols < a.rows))) return hipErrorInvalidValue;
  if (dg) {
    if constexpr (BM == BN) {
      if (!ps || !qs) return hipErrorInvalidValue;
      product_copied_kernel<DT, BM, BN, true, true, true><<<blocks, kPThreads, 0, s>>>(a);
    } else return hipErrorInvalidValue;
  } else {
    if (qs) return hipErrorInvalidValue;
    if (ps) product_copied_kernel<DT, BM, BN, true, false, false><<<blocks, kPThreads, 0, s>>>(a);
    else product_copied_kernel<DT, BM, BN, false, false, false><<<blocks, kPThreads, 0, s>>>(a);
  }
  return hipGetLastError();
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

// TileCopy of a strided operand in few registers: a wave's copies lie kRows contraction rows apart, and rows twice as
// far apart share their slot permutation.
template <int DT, int R>
struct StridedCopy {
  using G = Stage<DT, R, true>;
  static constexpr int kRows = kPThreads / G::kRowSlots;
  const char* base;
  int64_t step_bytes;
  uint32_t copy_bytes;
  uint32_t off[2];  // copies of even and odd j
  int k;            // the lane's contraction row within a step, copy 0
  __device__ __forceinline__ void init(int wave, int64_t pitch, int last) {
    step_bytes = G::kDepth * pitch;
    copy_bytes = static_cast<uint32_t>(kRows * pitch);
    k = (wave * kWave + lane_id()) / G::kRowSlots;
#pragma unroll
    for (int o = 0; o < 2; ++o)
      off[o] = static_cast<uint32_t>(k * pitch) + min(G::perm(k + kRows * o, lane_id() % G::kRowSlots) * 16, last);
  }
  __device__ __forceinline__ void copy(u32x4* st, int wave, int step, int left) const {
    const auto r = make_rsrc(base + step * step_bytes, left > 0 ? kPOutside : 0u);
#pragma unroll
    for (int j = 0; j < G::kLoads; ++j) {
      const uint32_t o = k + kRows * j < left ? off[j & 1] : kPOutside;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          r, (__attribute__((address_space(3))) void*)(st + (j * kPWaves + wave) * kWave), 16, o, j * copy_bytes, 0, 0);
    }
  }
};

// Weight gradients of groups of few rows: 128 x 128 tiles whose contraction is a few steps, so that a tile is a chain of
// latencies (bounds, copies, stores) and the results' bytes bound the whole. One stage of 32 KB, so that four workgroups
// share a CU; each walks over tiles, and sends the next tile's first copies out before it stores the last one's sums. Those
// go out as buffer stores whose lanes outside the result are turned off by their offset: always the same number of
// them, so that the barrier in front of the next tile waits for its copies (older than the stores) and not for the stores
// (behind it the compiler waits for these too, before it reads what the copies brought). 16-bit sums pass
// through the stage first, so that a store writes whole lines (8 rows of 128 bytes): halves of lines, 64 bytes of each of
// 16 rows, cost 474 us past the caches and 423 through them where this takes 351.
// Large results go past the caches (ProductArgs::stream): their bytes would drive the tiles' operands out of L2.
// 64 groups of 192 rows on average, 2816 x 2048 (738 MB of results, 142 GFLOP), behind another operator's traffic: 351 us
// (2.1 TB/s of results; 379 through the caches), repeated alone 249; 16 rows a group 162 (4.6 TB/s) and 209. 256 x 256 tiles
// 472 and 350 alone, 128 x 128 tiles in two stages 454 and 305.
__device__ __forceinline__ void store_slot(__amdgpu_buffer_rsrc_t r, const u32x4& v, uint32_t off, bool stream) {
  if (stream) __builtin_amdgcn_raw_buffer_store_b128(v, r, off, 0, kNonTemporal);
  else __builtin_amdgcn_raw_buffer_store_b128(v, r, off, 0, 0);
}

// SLOTS: the results' rows are whole 16-byte slots too.
template <int DT, bool SLOTS>
__global__ __launch_bounds__(kPThreads, 4) void product_shallow_kernel(ProductArgs a) {
  constexpr int kTile = 128;
  using G = Stage<DT, kTile, true>;
  using W = Waves<kTile, kTile>;
  constexpr int64_t kEs = G::kEs;
  constexpr int kStores = DT == kF32 ? W::kNI * W::kNJ : W::kNJ * 2;  // per wave and tile
  const int col_tiles = (a.cols + kTile - 1) / kTile;
  const int lane = lane_id(), wave = wave_id(), r = lane & 15, g = lane >> 4;
  const int wrow = (wave / W::kColWaves) * W::kNJ * 16, wcol = (wave % W::kColWaves) * W::kNI * 16;
  const int64_t p_pitch = a.p_ld * kEs, q_pitch = a.q_ld * kEs;
  __shared__ u32x4 sp[G::kSlots], sq[G::kSlots];
  StridedCopy<DT, kTile> cp, cq;
  ProductItem it;
  int b = static_cast<int>(blockIdx.x);
  if (!find_depth_item(a, b, kTile, col_tiles, it)) return;
  auto copy = [&](const ProductItem& t, int s) {
    const int left = t.depth - s * G::kDepth;  // of an empty group: no reads, zeros
    cp.copy(sp, wave, s, left);
    cq.copy(sq, wave, s, left);
    __builtin_amdgcn_sched_barrier(0);
  };
  auto first = [&](const ProductItem& t) {
    const int c0 = t.ct * kTile;
    cp.base = a.p + t.k0 * p_pitch + c0 * kEs;
    cq.base = a.q + t.k0 * q_pitch + t.row * kEs;
    cp.init(wave, p_pitch, static_cast<int>((a.cols - c0) * kEs) - 16);
    cq.init(wave, q_pitch, static_cast<int>((a.q_cols - t.row) * kEs) - 16);
    copy(t, 0);
  };
  first(it);
  bool stores = false;  // the last tile's are under way, behind this tile's first copies
  for (;;) {
    const int steps = max(1, (it.depth + G::kDepth - 1) / G::kDepth);
    f32x4 acc[W::kNI][W::kNJ] = {};
    // fp32 chains (see fold): four workgroups per CU leave no registers for a second set of sums, so those of a group of
    // more than one chain wait in the result's own place: `more`: on top of what is there; `leave`: left there. A single
    // group of 12737 rows (of 64, 256 x 256) then takes 1083 us where one chain took 953, 16384 rows in groups of 512
    // (512 x 1024) 146 and 145; groups of at most 256 rows have no such chain.
    auto fold_out = [&](bool more, auto leave) {
      int ln = lane;
      asm volatile("" : "+v"(ln));
      char* base = a.out + (it.g * a.out_group + it.row * a.out_ld) * kEs;
      const auto from = make_rsrc(base, more ? kPOutside : 0u);  // (an empty buffer: zeros)
      const auto to = make_rsrc(base, kPOutside);
#pragma unroll
      for (int j = 0; j < W::kNJ; ++j) {
        const int row = wrow + j * 16 + (ln & 15);
        const int64_t at = row * a.out_ld + it.ct * kTile + wcol + 4 * (ln >> 4);
        const int left = row < it.m ? a.out_cols - (it.ct * kTile + wcol + 4 * (ln >> 4)) : 0;
        if constexpr (SLOTS) {
          uint32_t off[W::kNI];
          f32x4 sum[W::kNI];
#pragma unroll
          for (int i = 0; i < W::kNI; ++i) {
            off[i] = left > 16 * i ? static_cast<uint32_t>((at + 16 * i) * kEs) : kPOutside;
            sum[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(from, off[i], 0, 0));
          }
#pragma unroll
          for (int i = 0; i < W::kNI; ++i) {
            acc[i][j] += sum[i];
            if constexpr (decltype(leave)::value) store_slot(to, __builtin_bit_cast(u32x4, acc[i][j]), off[i], false);
          }
          __builtin_amdgcn_sched_barrier(0);
        } else {
#pragma unroll
          for (int i = 0; i < W::kNI; ++i) {
            if (left <= 16 * i) continue;
            if (more) acc[i][j] += load4<DT>(base, at + 16 * i, left - 16 * i, false);
            if constexpr (decltype(leave)::value) store4<DT>(base, at + 16 * i, left - 16 * i, false, acc[i][j]);
          }
        }
      }
      if constexpr (decltype(leave)::value) {
#pragma unroll
        for (int i = 0; i < W::kNI; ++i)
#pragma unroll
          for (int j = 0; j < W::kNJ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
    };
    for (int s = 0; s < steps; ++s) {
      if (s == 0 && stores) __builtin_amdgcn_s_waitcnt(vmcnt_imm(kStores));
      else __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
      bare_barrier();
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        u32x4 fp[W::kNI], fq[W::kNJ];
#pragma unroll
        for (int i = 0; i < W::kNI; ++i) fp[i] = G::frag(sp, wcol + i * 16, u);
#pragma unroll
        for (int j = 0; j < W::kNJ; ++j) fq[j] = G::frag(sq, wrow + j * 16, u);
#pragma unroll
        for (int i = 0; i < W::kNI; ++i)
#pragma unroll
          for (int j = 0; j < W::kNJ; ++j) acc[i][j] = Elem<DT>::mfma(fp[i], fq[j], acc[i][j]);
        __builtin_amdgcn_sched_barrier(0);
      }
      bare_barrier();  // every wave has read the stage
      if (s + 1 < steps) copy(it, s + 1);
      if (DT == kF32 && s % kFold == kFold - 1 && s + 1 < steps) fold_out(s >= kFold, std::true_type{});
    }
    if (DT == kF32 && steps > kFold) fold_out(true, std::false_type{});
    const ProductItem done = it;
    const int c0 = done.ct * kTile + wcol;
    char* base = a.out + (done.g * a.out_group + done.row * a.out_ld) * kEs;
    // 16-bit sums, rounded, through the wave's quarter of the stage: rows of 64 columns (128 bytes), slots permuted
    constexpr int kRowsOf = 8;  // rows that one store covers, 8 lanes each
    constexpr int kPacked = DT == kF32 ? 1 : W::kNJ * 16 / kRowsOf;
    u32x4 packed[kPacked];
    int ln = lane;  // (opaque: its addresses would otherwise be kept in registers through the whole walk)
    asm volatile("" : "+v"(ln));
    if constexpr (!SLOTS) {  // at once
#pragma unroll
      for (int j = 0; j < W::kNJ; ++j) {
        const int row = wrow + j * 16 + (ln & 15);
        if (row >= done.m) continue;
#pragma unroll
        for (int i = 0; i < W::kNI; ++i) {
          const int col = c0 + i * 16 + 4 * (ln >> 4), left = a.out_cols - col;
          if (left > 0) store4<DT>(base, row * a.out_ld + col, left, false, acc[i][j]);
        }
      }
    } else if constexpr (DT != kF32) {
      u32x2* half = reinterpret_cast<u32x2*>((wave < 2 ? sp : sq) + (wave & 1) * (G::kSlots / 2));
#pragma unroll
      for (int j = 0; j < W::kNJ; ++j)
#pragma unroll
        for (int i = 0; i < W::kNI; ++i)
          half[((j * 16 + (ln & 15)) * 8 + ((2 * i + (ln >> 5)) ^ (ln & 7))) * 2 + ((ln >> 4) & 1)] = pack4<DT>(acc[i][j]);
      const u32x4* full = reinterpret_cast<const u32x4*>(half);
#pragma unroll
      for (int t = 0; t < kPacked; ++t) packed[t] = full[(t * 8 + (ln >> 3)) * 8 + ((ln & 7) ^ (ln >> 3))];
      __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt 0
      bare_barrier();                      // the next tile's copies may come
    }
    b += static_cast<int>(gridDim.x);
    const bool more = b < a.item_blocks && find_depth_item(a, b, kTile, col_tiles, it);
    if (more) first(it);
    if constexpr (SLOTS) {
      const auto rs = make_rsrc(base, kPOutside);
      auto put = [&](auto stream) {
        if constexpr (DT == kF32) {
#pragma unroll
          for (int j = 0; j < W::kNJ; ++j) {
            const int row = wrow + j * 16 + (ln & 15);
#pragma unroll
            for (int i = 0; i < W::kNI; ++i) {
              const int col = c0 + i * 16 + 4 * (ln >> 4);
              uint32_t off = row < done.m && col < a.out_cols ? static_cast<uint32_t>((row * a.out_ld + col) * kEs) : kPOutside;
              asm volatile("" : "+v"(off));  // (one store for both cases, not one in each: they are counted)
              store_slot(rs, __builtin_bit_cast(u32x4, acc[i][j]), off, decltype(stream)::value);
            }
          }
        } else {
          const int col = c0 + 8 * (ln & 7);
          const uint32_t at = static_cast<uint32_t>(((wrow + (ln >> 3)) * a.out_ld + col) * kEs);
          const int left = col < a.out_cols ? done.m - wrow - (ln >> 3) : 0;
#pragma unroll
          for (int t = 0; t < kPacked; ++t)
            store_slot(rs, packed[t], t * kRowsOf < left ? at + static_cast<uint32_t>(t * kRowsOf * a.out_ld * kEs) : kPOutside,
                       decltype(stream)::value);
        }
      };
      if (a.stream) put(std::true_type{});
      else put(std::false_type{});
    }
    if (!more) return;
    stores = SLOTS;
  }
}

template <int DT>
static hipError_t shallow_launch(const ProductArgs& a, hipStream_t s) {
  constexpr int n = 16 / dtype_bytes(DT);
  if (a.p_ld % n != 0 || a.q_ld % n != 0 || a.splits != 1 || a.cols % n != 0 || a.q_cols % n != 0 || a.q_cols < a.rows)
    return hipErrorInvalidValue;
  // as many workgroups as run at once; a multiple of 8, which keeps a workgroup's tiles on its XCD
  const unsigned blocks = static_cast<unsigned>(a.item_blocks < 1024 ? a.item_blocks : 1024);
  const bool slots = a.out_cols % n == 0 && a.out_ld % n == 0 && reinterpret_cast<uintptr_t>(a.out) % 16 == 0;
  if (slots) product_shallow_kernel<DT, true><<<blocks, kPThreads, 0, s>>>(a);
  else product_shallow_kernel<DT, false><<<blocks, kPThreads, 0, s>>>(a);
  return hipGetLastError();
}

hipError_t launch_product_shallow(int dtype, const ProductArgs& a, hipStream_t s) {
  switch (dtype) {
    case kF32: return shallow_launch<kF32>(a, s);
    case kF16: return shallow_launch<kF16>(a, s);
    case kBF16: return shallow_launch<kBF16>(a, s);
    default: return hipErrorInvalidValue;
  }
}

template <int DT>
static hipError_t tile_launch(bool ps, bool qs, bool dg, const TileShape& t, const ProductArgs& a, hipStream_t s) {
  if (t.form == TileShape::kStaged && t.bm == 64 && t.bn == 64) return staged_launch<DT, 64, 64>(ps, qs, dg, a, s);
  if (t.form == TileShape::kCopied && t.bm == 64 && t.bn == 64) return copied_launch<DT, 64, 64>(ps, qs, dg, a, s);
  if (t.form != TileShape::kCopied || t.bn != 128) return hipErrorInvalidValue;
  if (t.bm == 128) return copied_launch<DT, 128, 128>(ps, qs, dg, a, s);
  if (t.bm == 64) return copied_launch<DT, 64, 128>(ps, qs, dg, a, s);
  if (t.bm == 32) return copied_launch<DT, 32, 128>(ps, qs, dg, a, s);
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
