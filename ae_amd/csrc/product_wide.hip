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

constexpr int kWRows = 256;                    // rows and columns of the tile
constexpr int kWDepth = 64;                    // contraction elements per step
constexpr int kWTiles = 8;                     // 16-column tiles of a wave; 16-row tiles at most
constexpr int kWDma = kWRows * 8 / kPThreads;  // copies per wave, operand and step
constexpr int kWStage = kWRows * 8;            // 16-byte slots of a stage

typedef short s16x4 __attribute__((ext_vector_type(4)));

template <int DT>
__device__ __forceinline__ void wmfma(f32x4& acc, const u32x4& a, const u32x4& b) {
  if constexpr (DT == kBF16) asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(a), "v"(b));
  else asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(acc) : "v"(a), "v"(b));
}

// Copies of one operand's steps into LDS. Copy j of wave w fills stage slots 64 (4 j + w) ..: of a contiguous operand
// rows 32 j + 8 w + lane / 8, of a strided one contraction rows 8 j + 2 w + lane / 32.
template <bool ST>
struct WideCopy;

template <>
struct WideCopy<false> {
  const char* base;      // the tile's first row
  uint32_t off[kWDma];   // row and slot of the lane
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

template <>
struct WideCopy<true> {
  const char* base;    // contraction row 0, the tile's first column
  int64_t step_bytes;
  uint32_t off[2];     // contraction row and slot of the lane, copies of even and odd j
  uint32_t row8;       // bytes of 8 contraction rows
  int k;               // the lane's contraction row within a step, copy 0
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t at(int64_t step, bool on) const {
    return make_rsrc(base + step * step_bytes, on ? kPOutside : 0u);
  }
  template <int J, bool MASKED>
  __device__ __forceinline__ void copy(__amdgpu_buffer_rsrc_t r, u32x4* st, int wave, int left) const {
    const uint32_t o = !MASKED || k + 8 * J < left ? off[J & 1] : kPOutside;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(st + (J * kPWaves + wave) * kWave),
                                             16, o, J * row8, 0, 0);
  }
};

// Slot permutations of a stage (see product_tile.hip): of row r, and of contraction row k.
__device__ __forceinline__ int strided_perm(int k) { return ((k & 3) | ((k >> 1) & 4)) * 2; }

// Tile q of a wave in a stage, as its first row: columns (P) in two blocks of 64, at 64 wr and 128 + 64 wr (gated
// tiles have gate columns in the first 128 and up columns in the rest); rows (Q) interleaved between the two
// row groups, so that an item of few rows has few tiles in each.
template <bool P>
__device__ __forceinline__ constexpr int wide_tile_row(int q) {
  return P ? (q < 4 ? 0 : 128) + (q & 3) * 16 : q * 32;
}

// Fragment reads of one operand from LDS: the lane's byte offsets in a stage.
template <bool ST, bool P>
struct WideRead {
  int at[ST ? 4 : 2];  // strided: tiles q & 3; contiguous: halves
  __device__ __forceinline__ void init(int group) {
    const int lane = lane_id(), r = lane & 15, g = lane >> 4;
    const int row = group * (P ? 64 : 16);
    if constexpr (ST) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int slot = ((row + wide_tile_row<P>(q)) >> 3) + ((r & 3) >> 1);
        const int k = 8 * g + (r >> 2);
        at[q] = (k * 32 + (slot ^ strided_perm(k))) * 16 + 8 * (r & 1);
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
      // tiles q and q + 4 lie 128 rows (16 slots) apart, a slot bit that the permutation leaves alone
      const char* p = s + at[Q & 3] + (Q >> 2) * 256 + U * 32 * 512;
      const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) s16x4*)(p)));
      const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) s16x4*)(p + 4 * 512)));
      return u32x4{lo[0], lo[1], hi[0], hi[1]};
    } else {
      return *reinterpret_cast<const u32x4*>(s + at[U] + wide_tile_row<P>(Q) * 128);
    }
  }
};

template <int NT>
struct WideFragments {
  u32x4 a[kWTiles], b[NT];
};

__device__ constexpr int spread_over(int n, int count, int places) {
  const int v = (n * count + places - 1) / places;
  return v < count ? v : count;
}

// The MFMAs of one half from `cur`; between them the next half's fragments are read into `nxt` (`read`: fragment
// by number), and kCopies copies go out, evenly spread.
template <int DT, int NT, int kCopies, typename R, typename F, int... Ns>
__device__ __forceinline__ void wide_half(const WideFragments<NT>& cur, R&& read, f32x4 (&acc)[kWTiles][NT], F&& copy,
                                          std::integer_sequence<int, Ns...>) {
  constexpr int kM = kWTiles * NT, kR = kWTiles + NT, kRs = kM * 3 / 4;
  auto place = [&](auto nc) {
    constexpr int n = decltype(nc)::value;
    constexpr int r0 = spread_over(n, kR, kRs), r1 = spread_over(n + 1, kR, kRs);
    if constexpr (r0 < r1) read(std::integral_constant<int, r0>{});
    if constexpr (r0 + 1 < r1) read(std::integral_constant<int, r0 + 1>{});
    static_assert(r1 - r0 <= 2, "at most two fragments per MFMA");
    constexpr int d0 = spread_over(n, kCopies, kM), d1 = spread_over(n + 1, kCopies, kM);
    static_assert(d1 - d0 <= 1, "at most one copy per MFMA");
    if constexpr (d0 < d1) copy(std::integral_constant<int, d0>{});
    wmfma<DT>(acc[n % kWTiles][n / kWTiles], cur.a[n % kWTiles], cur.b[n / kWTiles]);
    __builtin_amdgcn_sched_barrier(0);
  };
  (place(std::integral_constant<int, Ns>{}), ...);
}

constexpr int wide_wait_imm(int n) { return (n & 15) | (7 << 4) | ((n >> 4) << 14); }  // vmcnt n, lgkmcnt 0

__device__ __forceinline__ void wide_sync() {  // without a memory fence, which would wait for later steps' copies
  asm volatile("s_barrier" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

template <bool PS, bool QS>
struct WideProduct {
  WideCopy<PS> p;
  WideCopy<QS> q;
  WideRead<PS, true> rp;
  WideRead<QS, false> rq;
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
template <int DT, int NT, bool PS, bool QS, int U>
struct WideReader {
  const WideProduct<PS, QS>& w;
  const u32x4 *sp, *sq;
  WideFragments<NT>& f;
  template <int F>
  __device__ __forceinline__ void operator()(std::integral_constant<int, F>) const {
    if constexpr (F < NT) f.b[F] = w.rq.template frag<U, F>(sq);
    else f.a[F - NT] = w.rp.template frag<U, F - NT>(sp);
  }
};

// One step from stage (sp, sq), the next one's being (np, nq). `step`: the step whose copies go out into (sp, sq).
template <int DT, int NT, int KQ, bool PS, bool QS>
__device__ __forceinline__ void wide_step(const WideProduct<PS, QS>& w, u32x4* sp, u32x4* sq, const u32x4* np,
                                          const u32x4* nq, int step, bool on, WideFragments<NT>& f0,
                                          WideFragments<NT>& f1, f32x4 (&acc)[kWTiles][NT]) {
  constexpr auto kSeq = std::make_integer_sequence<int, kWTiles * NT>{};
  wide_half<DT, NT, 0>(f0, WideReader<DT, NT, PS, QS, 1>{w, sp, sq, f1}, acc, [](auto) {}, kSeq);
  __builtin_amdgcn_s_waitcnt(wide_wait_imm(0));
  wide_sync();
  const auto bp = w.p.at(step, on), bq = w.q.at(step, on);
  wide_half<DT, NT, kWDma + KQ>(f1, WideReader<DT, NT, PS, QS, 0>{w, np, nq, f0}, acc, [&](auto jc) {
    constexpr int j = decltype(jc)::value;
    if constexpr (j < kWDma) w.p.template copy<j, false>(bp, sp, w.wave, 0);
    else w.q.template copy<j - kWDma, false>(bq, sq, w.wave, 0);
  }, kSeq);
}

template <int KQ, bool PS, bool QS, int... Js>
__device__ __forceinline__ void wide_first(const WideProduct<PS, QS>& w, u32x4* sp, u32x4* sq, int step,
                                           std::integer_sequence<int, Js...>) {
  const auto bp = w.p.at(step, true), bq = w.q.at(step, true);
  const int left = w.depth - step * kWDepth;
  auto one = [&](auto jc) {
    constexpr int j = decltype(jc)::value;
    if constexpr (j < kWDma) w.p.template copy<j, true>(bp, sp, w.wave, left);
    else w.q.template copy<j - kWDma, true>(bq, sq, w.wave, left);
  };
  (one(std::integral_constant<int, Js>{}), ...);
}

template <int NT, bool PS, bool QS, int U, int... Fs>
__device__ __forceinline__ void wide_read_all(const WideProduct<PS, QS>& w, const u32x4* sp, const u32x4* sq,
                                              WideFragments<NT>& f, std::integer_sequence<int, Fs...>) {
  WideReader<kBF16, NT, PS, QS, U> r{w, sp, sq, f};
  (r(std::integral_constant<int, Fs>{}), ...);
}

// acc += the product over all pairs. NT: row tiles per wave; KQ: copies of the row operand per wave and step (a strided
// one always copies whole contraction rows).
template <int DT, int NT, bool PS, bool QS>
__device__ __forceinline__ void wide_product(const WideProduct<PS, QS>& w, u32x4* p0, u32x4* q0, u32x4* p1, u32x4* q1,
                                             f32x4 (&acc)[kWTiles][NT]) {
  constexpr int KQ = QS ? kWDma : NT;
  constexpr auto kCopies = std::make_integer_sequence<int, kWDma + KQ>{};
  WideFragments<NT> f0, f1;
  const int first = 2 * w.pair(0);
  wide_first<KQ>(w, p0, q0, first, kCopies);
  __builtin_amdgcn_sched_barrier(0);
  wide_first<KQ>(w, p1, q1, first + 1, kCopies);
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(wide_wait_imm(kWDma + KQ));
  wide_sync();
  wide_read_all<NT, PS, QS, 0>(w, p0, q0, f0, std::make_integer_sequence<int, kWTiles + NT>{});
  __builtin_amdgcn_sched_barrier(0);
  for (int c = 1; c <= w.pairs; ++c) {
    const bool on = c < w.pairs;
    const int next = on ? 2 * w.pair(c) : 0;
    asm volatile("s_nop 1");
    __builtin_amdgcn_sched_barrier(0);
    wide_step<DT, NT, KQ, PS, QS>(w, p0, q0, p1, q1, next, on, f0, f1, acc);
    wide_step<DT, NT, KQ, PS, QS>(w, p1, q1, p0, q0, next + 1, on, f0, f1, acc);
    asm volatile("s_nop 15");
    __builtin_amdgcn_sched_barrier(0);
  }
}

// The epilogue of a wave's quarter. Its accumulators go through LDS, 64 rows at a time, into the wave's own 32 KB: as
// rows of 32 16-byte slots (slot s of row r at s ^ (r % 16): no bank conflicts either way). A lane then takes four
// columns of each of the quarter's two column blocks, for every fourth row: the bias stays in registers, 16 lanes
// write 128 contiguous bytes, and the loop body stands once in the code (unrolled over the 64 accumulator tiles
// with an activation in each, the compiler kept the accumulators in scratch memory).
template <int DT, int NT>
__device__ __forceinline__ void wide_finish(const ProductArgs& a, const ProductItem& it, int wave, u32x4* lds,
                                            const f32x4 (&acc)[kWTiles][NT]) {
  constexpr int kBatch = 4;  // rows of a lane whose residuals are loaded together
  const int lane = lane_id();
  const int wr = wave >> 1, wt = wave & 1;
  f32x4* st = reinterpret_cast<f32x4*>(lds);
  const int c = lane & 15, rr = lane >> 4;
  const int col0 = it.ct * (a.gated ? kWRows / 2 : kWRows) + wr * 64 + 4 * c;
  const int col1 = a.gated ? a.out_cols + col0 : col0 + kWRows / 2;
  const int left0 = a.out_cols - col0, left1 = a.gated ? left0 : a.out_cols - col1;
  const f32x4 bias0 = bias4<DT>(a, it, col0, left0), bias1 = bias4<DT>(a, it, col1, left1);
#pragma unroll
  for (int j0 = 0; j0 < NT; j0 += 4) {
    constexpr int kGroup = NT < 4 ? NT : 4;
    const int tiles = NT - j0 < kGroup ? NT - j0 : kGroup;
#pragma unroll
    for (int j = 0; j < kGroup; ++j) {
      if (j >= tiles) break;
      const int r = j * 16 + (lane & 15);
#pragma unroll
      for (int i = 0; i < kWTiles; ++i) st[r * 32 + ((4 * i + rr) ^ (lane & 15))] = acc[i][j0 + j];
    }
#pragma unroll 1
    for (int b = 0; b < tiles * 16; b += 4 * kBatch) {
      // tile row of the b-th row of the wave's 64: row tiles of the two row groups alternate
      const int r0 = (wt + 2 * (j0 + (b >> 4))) * 16;
      f32x4 v0[kBatch], v1[kBatch], res0[kBatch], res1[kBatch];
#pragma unroll
      for (int q = 0; q < kBatch; ++q) {
        const int y = 4 * q + rr;
        v0[q] = st[(b + y) * 32 + (c ^ (y & 15))];
        v1[q] = st[(b + y) * 32 + ((c + 16) ^ (y & 15))];
        const bool in = r0 + y < it.m;
        res0[q] = res4<DT>(a, static_cast<int64_t>(it.row) + r0 + y, col0, in ? left0 : 0);
        if (!a.gated) res1[q] = res4<DT>(a, static_cast<int64_t>(it.row) + r0 + y, col1, in ? left1 : 0);
      }
#pragma unroll
      for (int q = 0; q < kBatch; ++q) {
        const int y = r0 + 4 * q + rr;
        if (y >= it.m) continue;
        const int64_t row = static_cast<int64_t>(it.row) + y;
        if (a.gated) {
          finish4_gated<DT>(a, row, col0, left0, v0[q], v1[q], bias0, bias1, res0[q]);
        } else {
          finish4<DT>(a, it, row, col0, left0, v0[q], bias0, res0[q]);
          finish4<DT>(a, it, row, col1, left1, v1[q], bias1, res1[q]);
        }
      }
    }
  }
}

template <int DT, int NT, bool PS, bool QS>
__device__ __forceinline__ void wide_item(const ProductArgs& a, const ProductItem& it, const WideProduct<PS, QS>& w,
                                          u32x4* p0, u32x4* q0, u32x4* p1, u32x4* q1) {
  f32x4 acc[kWTiles][NT];
#pragma unroll
  for (int i = 0; i < kWTiles; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (w.pairs > 0) wide_product<DT, NT, PS, QS>(w, p0, q0, p1, q1, acc);
  // the copies sent ahead of the walk's end still write zeros into the stages, and other waves may still read them
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
  __syncthreads();
  u32x4* mine = w.wave == 0 ? p0 : w.wave == 1 ? p1 : w.wave == 2 ? q0 : q1;
  wide_finish<DT, NT>(a, it, w.wave, mine, acc);
}

template <int DT, bool PS, bool QS, bool DG>
__global__ __launch_bounds__(kPThreads, 1) void product_wide_kernel(ProductArgs a) {
  const int b = static_cast<int>(blockIdx.x);
  if (b >= a.item_blocks) {
    fill_rows<DT>(a, b - a.item_blocks);
    return;
  }
  ProductItem it;
  const int tile_cols = a.gated ? kWRows / 2 : kWRows;
  const int col_tiles = (a.out_cols + tile_cols - 1) / tile_cols;
  if (!(DG ? find_depth_item(a, b, kWRows, col_tiles, it) : find_row_item(a, b, kWRows, col_tiles, it))) return;
  __shared__ u32x4 p0[kWStage], p1[kWStage], q0[kWStage], q1[kWStage];
  const int lane = lane_id();
  WideProduct<PS, QS> w;
  w.wave = wave_id();
  w.depth = it.depth;
  w.pairs = (it.depth + 2 * kWDepth - 1) / (2 * kWDepth);
  w.rot = w.pairs > 1 ? (it.ct & 7) * (w.pairs - 1) / 8 : 0;
  w.rp.init(w.wave >> 1);
  w.rq.init(w.wave & 1);
  const int cfirst = it.ct * tile_cols;
  const int64_t p_pitch = a.p_ld * 2, q_pitch = a.q_ld * 2;
  w.p.base = a.p + (DG ? int64_t{0} : it.w * a.p_group * 2);
  if constexpr (PS) {
    w.p.base += it.k0 * p_pitch + static_cast<int64_t>(cfirst) * 2;
    w.p.step_bytes = kWDepth * p_pitch;
    w.p.row8 = static_cast<uint32_t>(8 * p_pitch);
    w.p.k = 2 * w.wave + (lane >> 5);
#pragma unroll
    for (int o = 0; o < 2; ++o) {  // columns past the last (a multiple of 8): the last slot again
      const int slot = (lane & 31) ^ strided_perm(w.p.k + 8 * o);
      w.p.off[o] = static_cast<uint32_t>(w.p.k * p_pitch) + min(slot * 8, a.cols - 8 - cfirst) * 2;
    }
  } else {
    w.p.base += cfirst * p_pitch;
    const int slot = (lane & 7) ^ (lane >> 3);
    w.p.k = slot * 8;
    const int last = a.out_cols - 8 - cfirst;  // rows past the last: its block of 8 again
#pragma unroll
    for (int j = 0; j < kWDma; ++j) {
      const int q = j * 32 + w.wave * 8;
      const int64_t row = a.gated ? min(q & 127, last) + (q >= 128 ? a.out_cols : 0) : min(q, last);
      w.p.off[j] = static_cast<uint32_t>((row + (lane >> 3)) * p_pitch) + slot * 16;
    }
  }
  w.q.base = a.q;
  if constexpr (QS) {
    w.q.base += it.k0 * q_pitch + static_cast<int64_t>(it.row) * 2;
    w.q.step_bytes = kWDepth * q_pitch;
    w.q.row8 = static_cast<uint32_t>(8 * q_pitch);
    w.q.k = 2 * w.wave + (lane >> 5);
#pragma unroll
    for (int o = 0; o < 2; ++o) {
      const int slot = (lane & 31) ^ strided_perm(w.q.k + 8 * o);
      w.q.off[o] = static_cast<uint32_t>(w.q.k * q_pitch) + min(slot * 8, a.rows - 8 - it.row) * 2;
    }
  } else {
    w.q.base += it.row * q_pitch;
    const int slot = (lane & 7) ^ (lane >> 3);
    w.q.k = slot * 8;
#pragma unroll
    for (int j = 0; j < kWDma; ++j)
      w.q.off[j] = static_cast<uint32_t>(min(j * 32 + w.wave * 8 + (lane >> 3), it.m - 1) * q_pitch) + slot * 16;
  }
  if constexpr (QS) {
    wide_item<DT, 8, PS, QS>(a, it, w, p0, q0, p1, q1);
  } else {
    switch ((it.m + 63) / 64) {
      case 1: wide_item<DT, 2, PS, QS>(a, it, w, p0, q0, p1, q1); break;
      case 2: wide_item<DT, 4, PS, QS>(a, it, w, p0, q0, p1, q1); break;
      case 3: wide_item<DT, 6, PS, QS>(a, it, w, p0, q0, p1, q1); break;
      default: wide_item<DT, 8, PS, QS>(a, it, w, p0, q0, p1, q1); break;
    }
  }
}

template <int DT>
static hipError_t wide_launch(bool ps, bool qs, bool dg, const ProductArgs& a, hipStream_t s) {
  const unsigned blocks = static_cast<unsigned>(a.item_blocks + a.fill_blocks);
  if (!ps && !qs && !dg) product_wide_kernel<DT, false, false, false><<<blocks, kPThreads, 0, s>>>(a);
  else if (ps && !qs && !dg) product_wide_kernel<DT, true, false, false><<<blocks, kPThreads, 0, s>>>(a);
  else if (ps && qs && dg) product_wide_kernel<DT, true, true, true><<<blocks, kPThreads, 0, s>>>(a);
  else return hipErrorInvalidValue;
  return hipGetLastError();
}

hipError_t launch_product_wide(int dtype, bool p_strided, bool q_strided, bool depth_groups, const ProductArgs& a,
                               hipStream_t s) {
  // whole 16-byte slots: the contraction of a contiguous operand, the columns of a strided one
  const bool rows8 = !q_strided || a.rows % 8 == 0;
  const bool cols8 = a.cols % 8 == 0 && a.out_cols % 8 == 0;
  const bool depth8 = (p_strided && q_strided) || a.depth % 8 == 0 ;
  if (!rows8 || !cols8 || !depth8 || a.p_ld % 8 != 0 || a.q_ld % 8 != 0 || a.p_group % 8 != 0 || a.splits != 1)
    return hipErrorInvalidValue;
  switch (dtype) {
    case kF16: return wide_launch<kF16>(p_strided, q_strided, depth_groups, a, s);
    case kBF16: return wide_launch<kBF16>(p_strided, q_strided, depth_groups, a, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace smx
