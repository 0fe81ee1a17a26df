// Matrix products of few rows (decode, verify and short calls): every wave works by itself.
//
// A workgroup of 4 waves owns 16 NP rows of the weight (gated: half of them gate rows, half the matching up rows) and
// 16 NJ rows of x. The waves split the contraction: wave w takes the steps w, w + 4, .. of 128 bytes, copies both
// operands' step straight into a ring of NS stages of its own in LDS (NS - 1 steps in flight), and adds its sums to
// the others' through LDS at the end. So there are no barriers in the walk, no partial sums in memory and no second
// launch, and small outputs already give many waves. (Fragments loaded straight into registers, 16 rows at 64 bytes
// each, reach 3.7 TB/s of weights: a load's quarter wave then touches 16 cache lines, a copy's two.)
#include "product.h"

namespace smx {

template <int NP, int NJ, int NS>
struct RowsTile {
  static constexpr int kP = NP * 16, kQ = NJ * 16;        // rows of the operands
  static constexpr int kSlots = (kP + kQ) * 8;            // 16-byte slots of a wave's stage: P rows, then Q rows
  static constexpr int kCopies = (kP + kQ) / 8;           // per step, 8 rows each
};

// 16 bytes per lane from `off` into the 64 slots at `st`, in lane order.
__device__ __forceinline__ void copy_rows8(__amdgpu_buffer_rsrc_t r, u32x4* st, uint32_t off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)st, 16, off, 0, 0, 0);
}

// The sums of the four waves, each of which has `SLOTS` 16-byte slots of each of s0 and s1: accumulator tiles in lane
// order, half of them in each; then a wave finishes every fourth unit: a tile, or gated a gate tile and its up tile.
template <int DT, int NP, int NJ, int SLOTS>
__device__ __forceinline__ void rows_finish(const ProductArgs& a, const ProductItem& it, int c0, int wave, u32x4* s0,
                                            u32x4* s1, const f32x4 (&acc)[NP][NJ]) {
  const int lane = lane_id(), r = lane & 15, g = lane >> 4;
  constexpr int kTiles = NP * NJ;
  constexpr int kHalf = (kTiles + 1) / 2;
  static_assert(kHalf * kWave <= SLOTS, "the tiles fit");
  f32x4* r0 = reinterpret_cast<f32x4*>(s0);
  f32x4* r1 = reinterpret_cast<f32x4*>(s1);
#pragma unroll
  for (int i = 0; i < NP; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int t = i * NJ + j;
      (t < kHalf ? r0 : r1)[wave * SLOTS + (t % kHalf) * kWave + lane] = acc[i][j];
    }
  __syncthreads();
  auto sum = [&](int t) {
    const f32x4* p = (t < kHalf ? r0 : r1) + (t < kHalf ? t : t - kHalf) * kWave + lane;
    f32x4 v = p[0];
#pragma unroll
    for (int w = 1; w < kPWaves; ++w) v += p[w * SLOTS];
    return v;
  };
  const int units = a.gated ? kTiles / 2 : kTiles;
  for (int t = wave; t < units; t += kPWaves) {
    const int i = t / NJ, row = (t - i * NJ) * 16 + r;
    const int col = c0 + i * 16 + 4 * g;
    const int left = row < it.m ? a.out_cols - col : 0;
    if (left <= 0) continue;
    const f32x4 bias0 = bias4<DT>(a, it, col, left);
    const f32x4 bias1 = a.gated ? bias4<DT>(a, it, a.out_cols + col, left) : f32x4{};
    const f32x4 res = res4<DT>(a, static_cast<int64_t>(it.row) + row, col, left);
    finish4<DT>(a, it, static_cast<int64_t>(it.row) + row, col, left, sum(t), a.gated ? sum(t + kTiles / 2) : f32x4{},
                bias0, bias1, res);
  }
}

template <int DT, int NP, int NJ, int NS>
__global__ __launch_bounds__(kPThreads) void product_rows_kernel(ProductArgs a) {
  using T = RowsTile<NP, NJ, NS>;
  constexpr int64_t kEs = sizeof(typename Elem<DT>::S);
  constexpr int kDepth = kPStep / kEs;
  static_assert(NS >= 2 && NS <= 4, "stages");
  const int b = static_cast<int>(blockIdx.x);
  if (b >= a.item_blocks) {
    fill_rows<DT>(a, b - a.item_blocks);
    return;
  }
  ProductItem it;
  const int width = a.gated ? T::kP / 2 : T::kP;  // output columns
  const int col_tiles = (a.out_cols + width - 1) / width;
  if (!find_row_item(a, b, T::kQ, col_tiles, it)) return;
  __shared__ u32x4 s0[kPWaves * T::kSlots], s1[kPWaves * T::kSlots], s2[NS > 2 ? kPWaves * T::kSlots : 1],
      s3[NS > 3 ? kPWaves * T::kSlots : 1];
  const int lane = lane_id(), wave = wave_id(), r = lane & 15, g = lane >> 4;
  const int c0 = it.ct * width;

  // copy n of a step: rows 8 n + lane / 8 of the stage, slot (lane % 8) ^ (lane / 8)
  const int64_t p_pitch = a.p_ld * kEs, q_pitch = a.q_ld * kEs;
  const char* pb = a.p + it.w * a.p_group * kEs + c0 * p_pitch;
  const char* qb = a.q + it.row * q_pitch;
  const int last = a.out_cols - 1 - c0;  // rows past the last: the last one again (not stored)
  const int slot = (lane & 7) ^ (lane >> 3);
  uint32_t off[T::kCopies];
#pragma unroll
  for (int n = 0; n < T::kCopies; ++n) {
    const int y = n * 8 + (lane >> 3);
    if (n < T::kP / 8) {
      const int64_t row = a.gated ? min(y & (T::kP / 2 - 1), last) + (y >= T::kP / 2 ? static_cast<int64_t>(a.out_cols) : 0)
                                  : static_cast<int64_t>(min(y, last));
      off[n] = static_cast<uint32_t>(row * p_pitch) + slot * 16;
    } else {
      off[n] = static_cast<uint32_t>(min(y - T::kP, it.m - 1) * q_pitch) + slot * 16;
    }
  }
  const int k = slot * (16 / static_cast<int>(kEs));  // the lane's first contraction element within a step
  const int steps = (it.depth + kDepth - 1) / kDepth;
  // Neighbouring workgroups begin at different places: the row pitches are multiples of 2 KB, so that at one step the
  // rows of all of them lie on a few memory channels.
  const int rot = static_cast<int>(static_cast<int64_t>(it.ct & 15) * steps / 16);
  auto copy = [&](u32x4* st, int c) {
    int step = c + rot;
    step -= step >= steps ? steps : 0;
    const uint32_t size = c < steps ? kPOutside : 0u;  // past the end: an empty buffer, zeros
    const int left = it.depth - step * kDepth;
    const auto rp = make_rsrc(pb + static_cast<int64_t>(step) * kPStep, size);
    const auto rq = make_rsrc(qb + static_cast<int64_t>(step) * kPStep, size);
    u32x4* mine = st + wave * T::kSlots;
#pragma unroll
    for (int n = 0; n < T::kCopies; ++n) {
      const uint32_t o = k < left ? off[n] : kPOutside;
      if (n < T::kP / 8) copy_rows8(rp, mine + n * kWave, o);
      else copy_rows8(rq, mine + n * kWave, o);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  f32x4 acc[NP][NJ] = {}, total[NP][NJ] = {};
  int chain = 0;  // steps since the last fold
  auto folds = [&](int n) {
    if (DT == kF32 && (chain += n) >= kFold) {
      fold(total, acc);
      chain = 0;
    }
  };
  // one step from `st`; the copies of the step NS later follow into it
  auto step = [&](u32x4* st, int c) {
    __builtin_amdgcn_s_waitcnt(vmcnt_imm((NS - 1) * T::kCopies));
    __builtin_amdgcn_sched_barrier(0);
    const u32x4* mine = st + wave * T::kSlots;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      u32x4 fp[NP], fq[NJ];
#pragma unroll
      for (int i = 0; i < NP; ++i) fp[i] = mine[(i * 16 + r) * 8 + ((4 * u + g) ^ (r & 7))];
#pragma unroll
      for (int j = 0; j < NJ; ++j) fq[j] = mine[(T::kP + j * 16 + r) * 8 + ((4 * u + g) ^ (r & 7))];
#pragma unroll
      for (int i = 0; i < NP; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[i][j] = Elem<DT>::mfma(fp[i], fq[j], acc[i][j]);
    }
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt 0: the stage is read
    __builtin_amdgcn_sched_barrier(0);
    copy(st, c + NS * kPWaves);
  };
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
  __builtin_amdgcn_sched_barrier(0);
  copy(s0, wave);
  copy(s1, wave + kPWaves);
  if constexpr (NS > 2) copy(s2, wave + 2 * kPWaves);
  if constexpr (NS > 3) copy(s3, wave + 3 * kPWaves);
  for (int c = wave; c < steps; c += NS * kPWaves) {  // (steps past the end multiply zeros)
    step(s0, c);
    step(s1, c + kPWaves);
    if constexpr (NS > 2) step(s2, c + 2 * kPWaves);
    if constexpr (NS > 3) step(s3, c + 3 * kPWaves);
    folds(NS);
  }
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));  // copies past the end write zeros into the stages
  if constexpr (DT == kF32) {
    fold(total, acc);
    fold(acc, total);
  }
  __syncthreads();
  rows_finish<DT, NP, NJ, T::kSlots>(a, it, c0, wave, s0, s1, acc);
}

// The same with the operands through registers, for any alignment: a wave loads the step after the next while it
// writes the next one's slots into its own stage and multiplies it.
template <int DT, int NP, int NJ>
__global__ __launch_bounds__(kPThreads) void product_rows_staged_kernel(ProductArgs a) {
  using T = RowsTile<NP, NJ, 1>;
  using S = typename Elem<DT>::S;
  constexpr int kEps = 16 / sizeof(S), kDepth = kPStep / sizeof(S);
  const int b = static_cast<int>(blockIdx.x);
  if (b >= a.item_blocks) {
    fill_rows<DT>(a, b - a.item_blocks);
    return;
  }
  ProductItem it;
  const int width = a.gated ? T::kP / 2 : T::kP;
  const int col_tiles = (a.out_cols + width - 1) / width;
  if (!find_row_item(a, b, T::kQ, col_tiles, it)) return;
  __shared__ u32x4 s0[kPWaves * T::kSlots], s1[kPWaves * T::kSlots];
  const int lane = lane_id(), wave = wave_id(), r = lane & 15, g = lane >> 4;
  const int c0 = it.ct * width;
  const int last = a.out_cols - 1 - c0;
  const int slot = (lane & 7) ^ (lane >> 3);
  const S* at[T::kCopies];  // the lane's slot of the walk's first step
#pragma unroll
  for (int n = 0; n < T::kCopies; ++n) {
    const int y = n * 8 + (lane >> 3);
    if (n < T::kP / 8) {
      const int64_t row = a.gated ? min(y & (T::kP / 2 - 1), last) + (y >= T::kP / 2 ? static_cast<int64_t>(a.out_cols) : 0)
                                  : static_cast<int64_t>(min(y, last));
      at[n] = reinterpret_cast<const S*>(a.p) + it.w * a.p_group + (c0 + row) * a.p_ld + slot * kEps;
    } else {
      at[n] = reinterpret_cast<const S*>(a.q) + (static_cast<int64_t>(it.row) + min(y - T::kP, it.m - 1)) * a.q_ld +
              slot * kEps;
    }
  }
  const int steps = (it.depth + kDepth - 1) / kDepth;
  struct Step {
    u32x4 v[T::kCopies];
  };
  auto load = [&](Step& v, int c) {
    const int have = it.depth - c * kDepth - slot * kEps;
#pragma unroll
    for (int n = 0; n < T::kCopies; ++n) v.v[n] = load_slot<DT>(at[n] + static_cast<int64_t>(c) * kDepth, have);
  };
  f32x4 acc[NP][NJ] = {}, total[NP][NJ] = {};
  int chain = 0;  // steps since the last fold
  auto folds = [&](int n) {
    if (DT == kF32 && (chain += n) >= kFold) {
      fold(total, acc);
      chain = 0;
    }
  };
  auto step = [&](const Step& v, u32x4* st) {
    u32x4* mine = st + wave * T::kSlots;
#pragma unroll
    for (int n = 0; n < T::kCopies; ++n) mine[n * kWave + lane] = v.v[n];
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      u32x4 fp[NP], fq[NJ];
#pragma unroll
      for (int i = 0; i < NP; ++i) fp[i] = mine[(i * 16 + r) * 8 + ((4 * u + g) ^ (r & 7))];
#pragma unroll
      for (int j = 0; j < NJ; ++j) fq[j] = mine[(T::kP + j * 16 + r) * 8 + ((4 * u + g) ^ (r & 7))];
#pragma unroll
      for (int i = 0; i < NP; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[i][j] = Elem<DT>::mfma(fp[i], fq[j], acc[i][j]);
    }
    __builtin_amdgcn_wave_barrier();
  };
  Step v0, v1;
  load(v0, wave);
  load(v1, wave + kPWaves);
  for (int c = wave; c < steps; c += 2 * kPWaves) {
    step(v0, s0);
    load(v0, c + 2 * kPWaves);
    step(v1, s1);
    load(v1, c + 3 * kPWaves);
    folds(2);
  }
  if constexpr (DT == kF32) {
    fold(total, acc);
    fold(acc, total);
  }
  __syncthreads();
  rows_finish<DT, NP, NJ, T::kSlots>(a, it, c0, wave, s0, s1, acc);
}

template <int DT>
static hipError_t rows_launch(const TileShape& t, const ProductArgs& a, hipStream_t s) {
  constexpr int n = 16 / dtype_bytes(DT);
  if ((a.gated && t.bn < 32) || a.splits != 1) return hipErrorInvalidValue;
  const unsigned blocks = static_cast<unsigned>(a.item_blocks + a.fill_blocks);
  if (t.form == TileShape::kRowsStaged) {
    if (t.bm == 16 && t.bn == 32) product_rows_staged_kernel<DT, 2, 1><<<blocks, kPThreads, 0, s>>>(a);
    else if (t.bm == 32 && t.bn == 32) product_rows_staged_kernel<DT, 2, 2><<<blocks, kPThreads, 0, s>>>(a);
    else return hipErrorInvalidValue;
    return hipGetLastError();
  }
  if (a.p_ld % n != 0 || a.q_ld % n != 0 || a.p_group % n != 0 || a.depth % n != 0) return hipErrorInvalidValue;
  // Three stages where the contraction is long (16 KB: 32 steps per wave), two where the third one's copies are a good part
  // of a short walk. One row, swiglu weights, us with two and with three: 88 workgroups, bf16, 1024 columns 5.0 and 5.4, 2048
  // 6.9 and 7.1, 4096 10.5 and 10.5, 8192 17.9 and 16.7, fp32, 1024 columns 7.6 and 7.5, 4096 20.6 and 17.7, 8192 39.2 and
  // 35.1; 352 workgroups, bf16, 2048 columns 12.7 and 13.4, 4096 24.3 and 25.5, 8192 49.0 and 49.1, fp32, 2048 columns 25.2 and
  // 27.0, 8192 91.0 and 90.9; 512 workgroups, fp32, 4096 columns 62.8 and 60.4. (Against it: 20 rows, 2048 -> 4096 in fp32 13.2
  // and 12.4.)
  const bool long_walk = a.depth >= 16384 / dtype_bytes(DT);
  if (t.bm == 16 && t.bn == 16) product_rows_kernel<DT, 1, 1, 4><<<blocks, kPThreads, 0, s>>>(a);
  else if (t.bm == 16 && t.bn == 32 && long_walk) product_rows_kernel<DT, 2, 1, 3><<<blocks, kPThreads, 0, s>>>(a);
  else if (t.bm == 16 && t.bn == 32) product_rows_kernel<DT, 2, 1, 2><<<blocks, kPThreads, 0, s>>>(a);
  else if (t.bm == 32 && t.bn == 32) product_rows_kernel<DT, 2, 2, 2><<<blocks, kPThreads, 0, s>>>(a);
  else if (t.bm == 64 && t.bn == 64) product_rows_kernel<DT, 4, 4, 2><<<blocks, kPThreads, 0, s>>>(a);
  else return hipErrorInvalidValue;
  return hipGetLastError();
}

hipError_t launch_product_rows(int dtype, const TileShape& t, const ProductArgs& a, hipStream_t s) {
  switch (dtype) {
    case kF32: return rows_launch<kF32>(t, a, s);
    case kF16: return rows_launch<kF16>(t, a, s);
    case kBF16: return rows_launch<kBF16>(t, a, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace smx
