// Wide tiled matrix products (16-bit types): 256 x 256 output tiles, one workgroup of 4 waves per CU, a 128 x 128
// quarter per wave with its accumulators in 256 AGPRs. The walk is that of wide.hip, whose notes say why it has this
// shape (energy per multiply-add: fewest LDS bytes; operands copied straight into LDS in two stages, fragments of
// one half step read while the other half's products run, one barrier per step). Here:
//
//  - an operand may be strided along the contraction (both gradients). Its stage holds 64 contraction rows of
//    256 elements, copied in 512-byte pieces, and its fragments come through the transposing LDS read: two
//    instructions of 8 bytes per lane instead of one of 16, the same bytes and no bank conflicts;
//  - any contraction length: the steps go in pairs, and the walk begins with the last pair, whose copies
//    past the end are turned off lane by lane (a buffer offset outside the buffer reads nothing and leaves zeros).
//    Every other pair is whole, so the loop has no masks;
//  - copies that run ahead of the walk's end are turned off by an empty buffer: no reads.
#include <utility>

#include "product.h"

namespace smx {

constexpr int kWDepth = 64;  // contraction elements per step

// A tile of BM x BN outputs: every wave owns BM / 2 rows and BN / 2 columns.
template <int BM, int BN>
struct WideTile {
  static constexpr int kCols = BN / 32;         // 16-column tiles of a wave
  static constexpr int kRows = BM / 32;         // its 16-row tiles at most
  static constexpr int kPStage = BN * 8, kQStage = BM * 8;          // 16-byte slots
  static constexpr int kPCopies = BN / 32, kQCopies = BM / 32;      // per wave and step
};

typedef short s16x4 __attribute__((ext_vector_type(4)));

template <int DT>
__device__ __forceinline__ void wmfma(f32x4& acc, const u32x4& a, const u32x4& b) {
  if constexpr (DT == kBF16) asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(a), "v"(b));
  else asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(acc) : "v"(a), "v"(b));
}

// Copies of one operand's steps into LDS, R rows (columns) of it. Copy j of wave w fills stage slots 64 (4 j + w) ..:
// of a contiguous operand rows 32 j + 8 w + lane / 8, of a strided one the next 512 / R contraction rows.
template <int R, bool ST>
struct WideCopy;

template <int R>
struct WideCopy<R, false> {
  const char* base;      // the tile's first row
  uint32_t off[R / 32];  // row and slot of the lane
  int k;                 // the lane's first contraction element within a step
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t at(int64_t step, bool on) const {
    return make_rsrc(base + step * kPStep, on ? kPOutside : 0u);
  }
  template <int J, bool MASKED>
  __device__ __forceinline__ void copy(__amdgpu_buffer_rsrc_t r, u32x4* st, int wave, int left) const {
    const uint32_t o = !MASKED || k < left ? off[J] : kPOutside;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(st + (J * kPWaves + wave) * kWave),
                                             16, o, 0, 0, 0);
  }
};

template <int R>
struct WideCopy<R, true> {
  static constexpr int kRowSlots = R / 8;                         // slots of a contraction row
  static constexpr int kCopyRows = kPWaves * kWave / kRowSlots;   // contraction rows of the waves' j-th copies
  const char* base;    // contraction row 0, the tile's first column
  int64_t step_bytes;
  uint32_t off[2];     // contraction row and slot of the lane, copies of even and odd j
  uint32_t copy_bytes; // bytes of kCopyRows contraction rows
  int k;               // the lane's contraction row within a step, copy 0
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t at(int64_t step, bool on) const {
    return make_rsrc(base + step * step_bytes, on ? kPOutside : 0u);
  }
  template <int J, bool MASKED>
  __device__ __forceinline__ void copy(__amdgpu_buffer_rsrc_t r, u32x4* st, int wave, int left) const {
    const uint32_t o = !MASKED || k + kCopyRows * J < left ? off[J & 1] : kPOutside;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(st + (J * kPWaves + wave) * kWave),
                                             16, o, J * copy_bytes, 0, 0);
  }
};

// Slot permutation of contraction row k of a strided stage (see product_tile.hip); rows 16 apart share it.
__device__ __forceinline__ int strided_perm(int k) { return ((k & 3) | ((k >> 1) & 4)) * 2; }

// Tile q of a wave in a stage, as its first row: columns (P) in two blocks of R / 4, one in each half of the stage
// (gated tiles have gate columns in the first half and up columns in the other); rows (Q) interleaved between the
// two row groups, so that an item of few rows has few tiles in each.
template <int R, bool P>
__device__ __forceinline__ constexpr int wide_tile_row(int q) {
  constexpr int kHalf = R / 64;  // tiles of a block
  return P ? (q < kHalf ? 0 : R / 2) + (q % kHalf) * 16 : q * 32;
}

// Fragment reads of one operand from LDS: the lane's byte offsets in a stage.
template <int R, bool ST, bool P>
struct WideRead {
  int at[ST ? 4 : 2];  // strided: tiles q & 3; contiguous: halves
  __device__ __forceinline__ void init(int group) {
    const int lane = lane_id(), r = lane & 15, g = lane >> 4;
    const int row = group * (P ? R / 4 : 16);
    if constexpr (ST) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int slot = ((row + wide_tile_row<R, P>(q)) >> 3) + ((r & 3) >> 1);
        const int k = 8 * g + (r >> 2);
        at[q] = (k * (R / 8) + (slot ^ strided_perm(k))) * 16 + 8 * (r & 1);
      }
    } else {
#pragma unroll
      for (int u = 0; u < 2; ++u) at[u] = ((row + r) * 8 + ((4 * u + g) ^ (r & 7))) * 16;
    }
  }
  template <int U, int Q>
  __device__ __forceinline__ u32x4 frag(const u32x4* st) const {
    const char* s = reinterpret_cast<const char*>(st);
    if constexpr (ST) {
      static_assert(R == 128 || R == 256, "16 or 32 slots: the permutation's 8 pairs");
      // (R = 256) tiles q and q + 4 lie 128 rows (16 slots) apart, a slot bit that the permutation leaves alone
      const char* p = s + at[Q & 3] + (Q >> 2) * 256 + U * 32 * R * 2;
      const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) s16x4*)(p)));
      const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) s16x4*)(p + 4 * R * 2)));
      return u32x4{lo[0], lo[1], hi[0], hi[1]};
    } else {
      return *reinterpret_cast<const u32x4*>(s + at[U] + wide_tile_row<R, P>(Q) * 128);
    }
  }
};

template <int CT, int NT>
struct WideFragments {
  u32x4 a[CT], b[NT];
};

__device__ constexpr int spread_over(int n, int count, int places) {
  const int v = (n * count + places - 1) / places;
  return v < count ? v : count;
}

// The MFMAs of one half from `cur`; between them the next half's fragments are read (`read`: fragment by number), and
// kCopies copies go out, evenly spread.
template <int DT, int CT, int NT, int kCopies, typename R, typename F, int... Ns>
__device__ __forceinline__ void wide_half(const WideFragments<CT, NT>& cur, R&& read, f32x4 (&acc)[CT][NT], F&& copy,
                                          std::integer_sequence<int, Ns...>) {
  constexpr int kM = CT * NT, kR = CT + NT, kRs = kM * 3 / 4;
  auto place = [&](auto nc) {
    constexpr int n = decltype(nc)::value;
    constexpr int r0 = spread_over(n, kR, kRs), r1 = spread_over(n + 1, kR, kRs);
    if constexpr (r0 < r1) read(std::integral_constant<int, r0>{});
    if constexpr (r0 + 1 < r1) read(std::integral_constant<int, r0 + 1>{});
    static_assert(r1 - r0 <= 2, "at most two fragments per MFMA");
    constexpr int d0 = spread_over(n, kCopies, kM), d1 = spread_over(n + 1, kCopies, kM);
    static_assert(d1 - d0 <= 1, "at most one copy per MFMA");
    if constexpr (d0 < d1) copy(std::integral_constant<int, d0>{});
    wmfma<DT>(acc[n % CT][n / CT], cur.a[n % CT], cur.b[n / CT]);
    __builtin_amdgcn_sched_barrier(0);
  };
  (place(std::integral_constant<int, Ns>{}), ...);
}

constexpr int wide_wait_imm(int n) { return (n & 15) | (7 << 4) | ((n >> 4) << 14); }  // vmcnt n, lgkmcnt 0

__device__ __forceinline__ void wide_sync() {  // without a memory fence, which would wait for later steps' copies
  asm volatile("s_barrier" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

template <int BM, int BN, bool PS, bool QS>
struct WideProduct {
  using T = WideTile<BM, BN>;
  WideCopy<BN, PS> p;
  WideCopy<BM, QS> q;
  WideRead<BN, PS, true> rp;
  WideRead<BM, QS, false> rq;
  int wave;
  int pairs;   // pairs of steps
  int depth;   // contraction elements
  int rot;     // where the walk over the whole pairs begins
  // Pair that the walk's c-th one is.
  __device__ __forceinline__ int pair(int c) const {
    if (c == 0) return pairs - 1;
    const int v = c - 1 + rot;
    return v >= pairs - 1 ? v - (pairs - 1) : v;
  }
};

// Fragment number F of half U: the row operand's first (each MFMA column of a half needs one of them).
template <int NT, int U, typename W>
struct WideReader {
  const W& w;
  const u32x4 *sp, *sq;
  WideFragments<W::T::kCols, NT>& f;
  template <int F>
  __device__ __forceinline__ void operator()(std::integral_constant<int, F>) const {
    if constexpr (F < NT) f.b[F] = w.rq.template frag<U, F>(sq);
    else f.a[F - NT] = w.rp.template frag<U, F - NT>(sp);
  }
};

// One step from stage (sp, sq), the next one's being (np, nq). `step`: the step whose copies go out into (sp, sq).
template <int DT, int NT, int KQ, typename W>
__device__ __forceinline__ void wide_step(const W& w, u32x4* sp, u32x4* sq, const u32x4* np, const u32x4* nq, int step,
                                          bool on, WideFragments<W::T::kCols, NT>& f0,
                                          WideFragments<W::T::kCols, NT>& f1, f32x4 (&acc)[W::T::kCols][NT]) {
  constexpr int CT = W::T::kCols, KP = W::T::kPCopies;
  constexpr auto kSeq = std::make_integer_sequence<int, CT * NT>{};
  wide_half<DT, CT, NT, 0>(f0, WideReader<NT, 1, W>{w, sp, sq, f1}, acc, [](auto) {}, kSeq);
  __builtin_amdgcn_s_waitcnt(wide_wait_imm(0));
  wide_sync();
  const auto bp = w.p.at(step, on), bq = w.q.at(step, on);
  wide_half<DT, CT, NT, KP + KQ>(f1, WideReader<NT, 0, W>{w, np, nq, f0}, acc, [&](auto jc) {
    constexpr int j = decltype(jc)::value;
    if constexpr (j < KP) w.p.template copy<j, false>(bp, sp, w.wave, 0);
    else w.q.template copy<j - KP, false>(bq, sq, w.wave, 0);
  }, kSeq);
}

template <typename W, int... Js>
__device__ __forceinline__ void wide_first(const W& w, u32x4* sp, u32x4* sq, int step, std::integer_sequence<int, Js...>) {
  constexpr int KP = W::T::kPCopies;
  const auto bp = w.p.at(step, true), bq = w.q.at(step, true);
  const int left = w.depth - step * kWDepth;
  auto one = [&](auto jc) {
    constexpr int j = decltype(jc)::value;
    if constexpr (j < KP) w.p.template copy<j, true>(bp, sp, w.wave, left);
    else w.q.template copy<j - KP, true>(bq, sq, w.wave, left);
  };
  (one(std::integral_constant<int, Js>{}), ...);
}

template <int NT, typename W, int... Fs>
__device__ __forceinline__ void wide_read_all(const W& w, const u32x4* sp, const u32x4* sq,
                                              WideFragments<W::T::kCols, NT>& f, std::integer_sequence<int, Fs...>) {
  WideReader<NT, 0, W> r{w, sp, sq, f};
  (r(std::integral_constant<int, Fs>{}), ...);
}

// acc += the product over all pairs. NT: row tiles per wave; KQ: copies of the row operand per wave and step (a strided
// one always copies whole contraction rows).
template <int DT, int NT, bool QS, typename W>
__device__ __forceinline__ void wide_product(const W& w, u32x4* p0, u32x4* q0, u32x4* p1, u32x4* q1,
                                             f32x4 (&acc)[W::T::kCols][NT]) {
  constexpr int KQ = QS ? W::T::kQCopies : NT;
  constexpr auto kCopies = std::make_integer_sequence<int, W::T::kPCopies + KQ>{};
  WideFragments<W::T::kCols, NT> f0, f1;
  const int first = 2 * w.pair(0);
  wide_first(w, p0, q0, first, kCopies);
  __builtin_amdgcn_sched_barrier(0);
  wide_first(w, p1, q1, first + 1, kCopies);
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(wide_wait_imm(W::T::kPCopies + KQ));
  wide_sync();
  wide_read_all<NT>(w, p0, q0, f0, std::make_integer_sequence<int, W::T::kCols + NT>{});
  __builtin_amdgcn_sched_barrier(0);
  for (int c = 1; c <= w.pairs; ++c) {
    const bool on = c < w.pairs;
    const int next = on ? 2 * w.pair(c) : 0;
    asm volatile("s_nop 1");
    __builtin_amdgcn_sched_barrier(0);
    wide_step<DT, NT, KQ>(w, p0, q0, p1, q1, next, on, f0, f1, acc);
    wide_step<DT, NT, KQ>(w, p1, q1, p0, q0, next + 1, on, f0, f1, acc);
    asm volatile("s_nop 15");
    __builtin_amdgcn_sched_barrier(0);
  }
}

// The epilogue of a wave's part. Its accumulators go through LDS, as many rows at a time as its 1 / 4 of the stages
// holds: as rows of 4 CT 16-byte slots (slot s of row r at s ^ (r % 16): no bank conflicts either way). A lane then takes
// four columns of each of the part's two column blocks, for some of the rows: the bias stays in registers, stores
// cover 64 or 128 contiguous bytes, and the loop body stands once in the code (unrolled over the 64 accumulator tiles
// with an activation in each, the compiler kept the accumulators in scratch memory).
template <int DT, int BM, int BN, int NT>
__device__ __forceinline__ void wide_finish(const ProductArgs& a, const ProductItem& it, int wave, u32x4* lds,
                                            const f32x4 (&acc)[WideTile<BM, BN>::kCols][NT]) {
  using T = WideTile<BM, BN>;
  constexpr int CT = T::kCols, kS = 4 * CT, kMask = kS < 16 ? kS - 1 : 15;
  constexpr int kQuads = kS / 2, kLaneRows = kWave / kQuads;
  constexpr int kRegion = T::kPStage < T::kQStage ? T::kPStage : T::kQStage;  // slots
  constexpr int kGroup = kRegion / (16 * kS) < NT ? kRegion / (16 * kS) : NT;
  static_assert(kGroup >= 1, "a row tile fits");
  constexpr int kBatch = 16 * kGroup / kLaneRows < 4 ? 16 * kGroup / kLaneRows : 4;  // rows of a lane finished together
  const int lane = lane_id();
  const int wr = wave >> 1, wt = wave & 1;
  f32x4* st = reinterpret_cast<f32x4*>(lds);
  const int c = lane % kQuads, rr = lane / kQuads;
  const int col0 = it.ct * (a.gated ? BN / 2 : BN) + wr * (BN / 4) + 4 * c;
  const int col1 = a.gated ? a.out_cols + col0 : col0 + BN / 2;
  const int left0 = a.out_cols - col0, left1 = a.gated ? left0 : a.out_cols - col1;
  const bool part = a.splits > 1;
  const f32x4 bias0 = part ? f32x4{} : bias4<DT>(a, it, col0, left0);
  const f32x4 bias1 = part ? f32x4{} : bias4<DT>(a, it, col1, left1);
#pragma unroll
  for (int j0 = 0; j0 < NT; j0 += kGroup) {
    const int tiles = NT - j0 < kGroup ? NT - j0 : kGroup;
#pragma unroll
    for (int j = 0; j < kGroup; ++j) {
      if (j >= tiles) break;
      const int r = j * 16 + (lane & 15);
#pragma unroll
      for (int i = 0; i < CT; ++i) st[r * kS + ((4 * i + (lane >> 4)) ^ (lane & kMask))] = acc[i][j0 + j];
    }
#pragma unroll 1
    for (int b = 0; b < tiles * 16; b += kLaneRows * kBatch) {
      f32x4 v0[kBatch], v1[kBatch], res0[kBatch], res1[kBatch];
      int64_t row[kBatch];
      bool in[kBatch];
#pragma unroll
      for (int q = 0; q < kBatch; ++q) {
        const int y = b + kLaneRows * q + rr;                                  // row in LDS
        const int r = (wt + 2 * (j0 + (y >> 4))) * 16 + (y & 15);              // row in the tile: the groups alternate
        v0[q] = st[y * kS + (c ^ (y & kMask))];
        v1[q] = st[y * kS + ((c + kQuads) ^ (y & kMask))];
        in[q] = r < it.m;
        row[q] = static_cast<int64_t>(it.row) + r;
        res0[q] = res4<DT>(a, row[q], col0, in[q] && !part ? left0 : 0);
        res1[q] = res4<DT>(a, row[q], col1, in[q] && !part && !a.gated ? left1 : 0);
      }
      if (part) {
        const bool vec = a.cols % 4 == 0 && a.out_cols % 4 == 0;
#pragma unroll
        for (int q = 0; q < kBatch; ++q) {
          if (!in[q]) continue;
          const int64_t at = (static_cast<int64_t>(it.split) * a.rows + row[q]) * a.cols;
          if (left0 > 0) store4<kF32>(reinterpret_cast<char*>(a.part), at + col0, left0, vec, v0[q]);
          if (left1 > 0) store4<kF32>(reinterpret_cast<char*>(a.part), at + col1, left1, vec, v1[q]);
        }
      } else if (a.gated) {
        finish_rows_gated<DT>(a, row, in, col0, left0, v0, v1, bias0, bias1, res0);
      } else {
        finish_rows<DT>(a, it, row, in, col0, left0, v0, bias0, res0);
        finish_rows<DT>(a, it, row, in, col1, left1, v1, bias1, res1);
      }
    }
  }
}

template <int DT, int BM, int BN, int NT, bool PS, bool QS>
__device__ __forceinline__ void wide_item(const ProductArgs& a, const ProductItem& it,
                                          const WideProduct<BM, BN, PS, QS>& w, u32x4* p0, u32x4* q0, u32x4* p1,
                                          u32x4* q1) {
  constexpr int CT = WideTile<BM, BN>::kCols;
  f32x4 acc[CT][NT];
#pragma unroll
  for (int i = 0; i < CT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (w.pairs > 0) wide_product<DT, NT, QS>(w, p0, q0, p1, q1, acc);
  // the copies sent ahead of the walk's end still write zeros into the stages, and other waves may still read them
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
  __syncthreads();
  u32x4* mine = w.wave == 0 ? p0 : w.wave == 1 ? p1 : w.wave == 2 ? q0 : q1;
  wide_finish<DT, BM, BN, NT>(a, it, w.wave, mine, acc);
}

template <int DT, int BM, int BN, bool PS, bool QS, bool DG>
__global__ __launch_bounds__(kPThreads, 1) void product_wide_kernel(ProductArgs a) {
  using T = WideTile<BM, BN>;
  const int b = static_cast<int>(blockIdx.x);
  if (b >= a.item_blocks) {
    fill_rows<DT>(a, b - a.item_blocks);
    return;
  }
  ProductItem it;
  const int tile_cols = a.gated ? BN / 2 : BN;
  const int col_tiles = (a.out_cols + tile_cols - 1) / tile_cols;
  if (!(DG ? find_depth_item(a, b, BM, col_tiles, it) : find_row_item(a, b, BM, col_tiles, it))) return;
  __shared__ u32x4 p0[T::kPStage], p1[T::kPStage], q0[T::kQStage], q1[T::kQStage];
  const int lane = lane_id();
  WideProduct<BM, BN, PS, QS> w;
  w.wave = wave_id();
  w.depth = it.depth;
  if (a.splits > 1) {  // a split's part: whole pairs of steps but for the last split's
    const int from = it.split * a.split_steps * kWDepth;
    it.k0 += from;
    w.depth = max(min(it.depth - from, a.split_steps * kWDepth), 0);
  }
  w.pairs = (w.depth + 2 * kWDepth - 1) / (2 * kWDepth);
  w.rot = w.pairs > 1 ? (it.ct & 7) * (w.pairs - 1) / 8 : 0;
  w.rp.init(w.wave >> 1);
  w.rq.init(w.wave & 1);
  const int cfirst = it.ct * tile_cols;
  const int64_t p_pitch = a.p_ld * 2, q_pitch = a.q_ld * 2;
  w.p.base = a.p + (DG ? int64_t{0} : it.w * a.p_group * 2);
  if constexpr (PS) {
    using C = WideCopy<BN, true>;
    w.p.base += it.k0 * p_pitch + static_cast<int64_t>(cfirst) * 2;
    w.p.step_bytes = kWDepth * p_pitch;
    w.p.copy_bytes = static_cast<uint32_t>(C::kCopyRows * p_pitch);
    w.p.k = (w.wave * kWave + lane) / C::kRowSlots;
#pragma unroll
    for (int o = 0; o < 2; ++o) {  // columns past the last (a multiple of 8): the last slot again
      const int slot = (lane % C::kRowSlots) ^ strided_perm(w.p.k + C::kCopyRows * o);
      w.p.off[o] = static_cast<uint32_t>(w.p.k * p_pitch) + min(slot * 8, a.cols - 8 - cfirst) * 2;
    }
  } else {
    w.p.base += cfirst * p_pitch + it.k0 * 2;
    const int slot = (lane & 7) ^ (lane >> 3);
    w.p.k = slot * 8;
    const int last = a.out_cols - 1 - cfirst;  // rows past the last: the last one again
#pragma unroll
    for (int j = 0; j < T::kPCopies; ++j) {
      const int q = j * 32 + w.wave * 8;
      const int64_t row = a.gated ? min((q & (BN / 2 - 1)) + (lane >> 3), last) + (q >= BN / 2 ? a.out_cols : 0)
                                  : min(q + (lane >> 3), last);
      w.p.off[j] = static_cast<uint32_t>(row * p_pitch) + slot * 16;
    }
  }
  w.q.base = a.q;
  if constexpr (QS) {
    using C = WideCopy<BM, true>;
    w.q.base += it.k0 * q_pitch + static_cast<int64_t>(it.row) * 2;
    w.q.step_bytes = kWDepth * q_pitch;
    w.q.copy_bytes = static_cast<uint32_t>(C::kCopyRows * q_pitch);
    w.q.k = (w.wave * kWave + lane) / C::kRowSlots;
#pragma unroll
    for (int o = 0; o < 2; ++o) {
      const int slot = (lane % C::kRowSlots) ^ strided_perm(w.q.k + C::kCopyRows * o);
      w.q.off[o] = static_cast<uint32_t>(w.q.k * q_pitch) + min(slot * 8, a.q_cols - 8 - it.row) * 2;
    }
  } else {
    w.q.base += it.row * q_pitch + it.k0 * 2;
    const int slot = (lane & 7) ^ (lane >> 3);
    w.q.k = slot * 8;
#pragma unroll
    for (int j = 0; j < T::kQCopies; ++j)
      w.q.off[j] = static_cast<uint32_t>(min(j * 32 + w.wave * 8 + (lane >> 3), it.m - 1) * q_pitch) + slot * 16;
  }
  if constexpr (QS) {
    wide_item<DT, BM, BN, T::kRows, PS, QS>(a, it, w, p0, q0, p1, q1);
  } else {  // items of few rows: only the row tiles that they have
    static_assert(BM == 256, "2, 4, 6 or 8 row tiles per wave");
    switch ((it.m + 63) / 64) {
      case 1: wide_item<DT, BM, BN, 2, PS, QS>(a, it, w, p0, q0, p1, q1); break;
      case 2: wide_item<DT, BM, BN, 4, PS, QS>(a, it, w, p0, q0, p1, q1); break;
      case 3: wide_item<DT, BM, BN, 6, PS, QS>(a, it, w, p0, q0, p1, q1); break;
      default: wide_item<DT, BM, BN, 8, PS, QS>(a, it, w, p0, q0, p1, q1); break;
    }
  }
}

template <int DT, int BM, int BN>
static hipError_t wide_launch(bool ps, bool qs, bool dg, const ProductArgs& a, hipStream_t s) {
  const unsigned blocks = static_cast<unsigned>(a.item_blocks + a.fill_blocks);
  if (!ps && !qs && !dg) product_wide_kernel<DT, BM, BN, false, false, false><<<blocks, kPThreads, 0, s>>>(a);
  else if (ps && !qs && !dg) product_wide_kernel<DT, BM, BN, true, false, false><<<blocks, kPThreads, 0, s>>>(a);
  else if (ps && qs && dg) product_wide_kernel<DT, BM, BN, true, true, true><<<blocks, kPThreads, 0, s>>>(a);
  else return hipErrorInvalidValue;
  return hipGetLastError();
}

hipError_t launch_product_wide(int dtype, bool p_strided, bool q_strided, bool depth_groups, const ProductArgs& a,
                               hipStream_t s) {
  // whole 16-byte slots: the contraction of a contiguous operand, the columns (rows) of a strided one
  if (a.p_ld % 8 != 0 || a.q_ld % 8 != 0 || a.p_group % 8 != 0) return hipErrorInvalidValue;
  // (beside a strided P a contiguous Q may end inside a slot, with zeros up to the slot's end)
  if (!p_strided && a.depth % 8 != 0) return hipErrorInvalidValue;
  if ((p_strided && a.cols % 8 != 0) || (q_strided && (a.q_cols % 8 != 0 || a.q_cols < a.rows))) return hipErrorInvalidValue;
  if (a.splits > 1 && a.split_steps % 2 != 0) return hipErrorInvalidValue;
  switch (dtype) {
    case kF16: return wide_launch<kF16, 256, 256>(p_strided, q_strided, depth_groups, a, s);
    case kBF16: return wide_launch<kBF16, 256, 256>(p_strided, q_strided, depth_groups, a, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace smx
