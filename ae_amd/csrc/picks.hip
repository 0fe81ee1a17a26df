// Routing for training and serving: each token's best experts with their weights, the picks' order by expert, and the
// gradient of the logits.
//
//   pick_kernel        L lanes a token with PL experts each: scores, groups, the k best, their weights; and where order
//                      is asked for, each pick's rank among the picks of its expert in the workgroup's tokens, with the
//                      workgroup's counts per expert. One workgroup does it all for few tokens.
//   pick_scan_kernel   many workgroups: counts per workgroup and expert -> the picks of an expert before a workgroup's
//   pick_place_kernel  place = the expert's first + those before the workgroup's + the rank
//   pick_grad_kernel   the gradient of a token's logits
//
// Everything is counted in integers and in the order of the picks, so the order is the stable one on every run.
//
// Bound by the instructions of the choice, not by the logits' bytes (8191 tokens over 256 experts in fp32: 8.4 MB, 2 us): 4
// tokens a wave, about 490 vector instructions a token with groups and a bias, 200 without. The gradient is bound by the
// comparison of each of a lane's experts with each pick (153 instructions a token over 256 experts with 8 picks, 272 in the
// dense form; issued at four cycles each they take 16 and 29 us of 65536 tokens). Measured, in bf16 unless said:
//   1 token, 64 experts, 6 picks                                         4.4 us, one launch
//   8191 tokens, 256 experts in 8 groups, bias, 8 picks, fp32            picks 15, places 7.0 us (at first 33, and 12 in two)
//   65536 tokens, the same                                               68 us with the order, 50 without
//   65536 tokens, 256 experts, 8 picks, no groups, no bias               41 and 24 us, gradient 19 (of all scores: 29)
//   16384 tokens, 64 experts, 6 picks                                    picks 8.0, places 5.4, gradient 5.4 us
#include <algorithm>

#include "blocks.h"

namespace smx {
namespace {

constexpr int kPickThreads = 512;     // most of a workgroup that picks
constexpr int kGradThreads = 256;
constexpr int kMaxK = 16;
constexpr int kMaxE = 1024;
constexpr int kMaxGroups = 64;
constexpr int kEntry = kMaxK + 2;     // slots of a token's picks: two more, whose distances are looked at
constexpr int kBlockPicks = 1024;     // picks whose ranks a workgroup holds
constexpr int kPlaceThreads = 512;
constexpr int kScanCols = 16;         // experts of a workgroup that scans

struct PickArgs {
  const char* logits;
  int64_t ld, T;
  int E, k, ng, tg, gs;
  bool sigmoid, renorm, grad_dense;
  float scale;
  const float* bias;
  float* weights;
  int32_t* ids;
  int32_t* places;     // null: no order
  int32_t* order;
  int64_t* offsets;
  int32_t* counts;     // [blocks][pitch] picks of the workgroup per expert (E: of nobody)
  int32_t* totals;     // [E + 1]
  int wave_tokens;     // consecutive tokens of a wave
  int blocks, pitch;
  bool scanned;        // counts hold the picks before the workgroup's by now
  int bits;            // of an expert's number, E among them
  const float* grad_w;
  char* grad;
};

__device__ __forceinline__ void wave_sync() {  // what this wave's lanes wrote to LDS is there for its other lanes
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// v, unknown to the compiler: what a rare branch derives from it stays in the branch, where a wave that does not take it
// spends nothing on it (a wave takes few tokens, so what is moved out of its loop costs as much as what is in it).
__device__ __forceinline__ int opaque(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

// Values in an order of unsigned numbers: -inf is 0 (nobody's pick), NaN the largest, -0 as +0.
__device__ __forceinline__ uint32_t key_of(float v) {
  if (v != v) return 0xffffffffu;
  if (v == -__builtin_inff()) return 0u;
  const uint32_t u = __float_as_uint(v + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) {
  if (k == 0u) return -__builtin_inff();
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);  // (the largest key is a NaN)
}
__device__ __forceinline__ uint64_t key_of(double v) {
  if (v != v) return ~uint64_t{0};
  if (v == -__builtin_inf()) return 0u;
  const uint64_t u = __builtin_bit_cast(uint64_t, v + 0.0);
  return (u >> 63) ? ~u : (u | (uint64_t{1} << 63));
}

// The sum of a group's two best choices (next 0: there is one). Sums behind the largest finite number are that: they lie as near
// as can be, and 64 bits tell them apart.
__device__ __forceinline__ uint32_t key_of_two(uint32_t best, uint32_t next) {
  if (best == 0u) return 0u;
  constexpr float kMost = 0x1.fffffep+127f;
  const float s = value_of(best) + (next != 0u ? value_of(next) : 0.0f);
  return s != s ? 0xffffffffu : key_of(fminf(fmaxf(s, -kMost), kMost));
}

template <int L> __device__ __forceinline__ float sum_over(float v) {
  return group_reduce<L>(v, [](float a, float b) { return a + b; });
}
template <int L> __device__ __forceinline__ float max_over(float v) {
  return group_reduce<L>(v, [](float a, float b) { return fmaxf(a, b); });
}
template <int L> __device__ __forceinline__ uint32_t max_over(uint32_t v) {
  auto step = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
  v = step(v, static_cast<uint32_t>(dpp<kDppXor1>(static_cast<int>(v))));
  v = step(v, static_cast<uint32_t>(dpp<kDppXor2>(static_cast<int>(v))));
  v = step(v, static_cast<uint32_t>(dpp<kDppHalfMirror>(static_cast<int>(v))));
  v = step(v, static_cast<uint32_t>(dpp<kDppMirror>(static_cast<int>(v))));
  if constexpr (L == kWave) {
    const int s = static_cast<int>(v);
    v = step(step(static_cast<uint32_t>(__builtin_amdgcn_readlane(s, 0)), static_cast<uint32_t>(__builtin_amdgcn_readlane(s, 16))),
             step(static_cast<uint32_t>(__builtin_amdgcn_readlane(s, 32)), static_cast<uint32_t>(__builtin_amdgcn_readlane(s, 48))));
  }
  return v;
}

// PL consecutive logits of a row from e on; -inf behind its end. `whole`: rows and base of aligned runs of PL.
template <int DT, int PL>
__device__ __forceinline__ void load_run(const char* base, int64_t at, int e, int E, bool whole, float (&v)[PL]) {
  using S = typename Elem<DT>::S;
  const S* p = reinterpret_cast<const S*>(base) + at + e;
  if (whole) {
    struct alignas(PL * sizeof(S) < 16 ? PL * sizeof(S) : 16) Run { S s[PL]; } r = {};
    const bool in = e < E;
    if (in) r = *reinterpret_cast<const Run*>(p);
#pragma unroll
    for (int i = 0; i < PL; ++i) v[i] = in ? Elem<DT>::to_f32(r.s[i]) : -__builtin_inff();
  } else {
    const int rest = opaque(E - e);
#pragma unroll
    for (int i = 0; i < PL; ++i) v[i] = i < rest ? Elem<DT>::to_f32(p[i]) : -__builtin_inff();
  }
}

__device__ __forceinline__ float sigmoid_of(float x) {
  const float e = expf(-fabsf(x));
  return (x < 0.0f ? e : 1.0f) / (1.0f + e);  // NaN stays NaN
}

// The same and exp for comparisons only: an instruction each, off by |x| 2^-23 and 2^-22 of themselves.
__device__ __forceinline__ float quick_exp(float x) { return __builtin_amdgcn_exp2f(x * 0x1.715476p+0f); }
__device__ __forceinline__ float quick_sigmoid(float x) {
  const float e = quick_exp(-fabsf(x));
  return (x < 0.0f ? e : 1.0f) * __builtin_amdgcn_rcpf(1.0f + e);
}

// LDS of a wave: the picks of its tokens; the choices of its tokens by key while groups are compared,
// or the listed ones in 64 bits, or those of one token.
template <int L, int PL> struct PickLds {
  static constexpr int kTokens = kWave / L;
  alignas(8) int entry[kTokens * kEntry];
  union {
    uint64_t fine[kTokens * kEntry];        // the listed choices in 64 bits
    uint32_t choice[kTokens][L * PL + 16];  // (tokens begin in other banks)
    uint64_t exact[L * PL];
  };
  uint32_t group[kTokens][kMaxGroups];
};

// The picks of one token by its choices in 64 bits (without a bias the logits themselves): the whole wave's work, for tokens
// whose choices the keys cannot tell apart.
template <int DT, bool kBiased>
__device__ __forceinline__ void pick_exactly(const PickArgs& a, int64_t t, uint64_t* key, int* entry) {
  using S = typename Elem<DT>::S;
  const int lane = opaque(lane_id());
  const S* row = reinterpret_cast<const S*>(a.logits) + t * a.ld;
  auto top_of = [](uint64_t v) {  // the wave's largest: the upper halves first
    const uint32_t high = static_cast<uint32_t>(v >> 32), top = max_over<kWave>(high);
    return static_cast<uint64_t>(top) << 32 | max_over<kWave>(high == top ? static_cast<uint32_t>(v) : 0u);
  };
  double m = 0.0, z = 1.0;
  if (kBiased && !a.sigmoid) {
    float top = -__builtin_inff();
    for (int e = lane; e < a.E; e += kWave) top = fmaxf(top, Elem<DT>::to_f32(row[e]));
    m = max_over<kWave>(top);
    z = 0.0;
    for (int e = lane; e < a.E; e += kWave) z += exp(static_cast<double>(Elem<DT>::to_f32(row[e])) - m);
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) z += __shfl_xor(z, off, kWave);
  }
  auto score = [&](int e) {
    const double x = Elem<DT>::to_f32(row[e]);
    return a.sigmoid ? 1.0 / (1.0 + exp(-x)) : exp(x - m) / z;
  };
  for (int e = lane; e < a.E; e += kWave) {
    const float x = Elem<DT>::to_f32(row[e]);
    if constexpr (kBiased) key[e] = x == -__builtin_inff() ? 0u : key_of(score(e) + static_cast<double>(a.bias[e]));
    else key[e] = key_of(static_cast<double>(x));
  }
  wave_sync();
  if (a.tg < a.ng) {
    uint64_t mine = 0u;
    if (lane < a.ng) {
      uint64_t best = 0u, next = 0u;
      int at = 0, after = 0;
      for (int j = 0, r = lane % a.gs; j < a.gs; ++j, r = r + 1 == a.gs ? 0 : r + 1) {  // (each lane from another bank on)
        const int i = lane * a.gs + r;
        const uint64_t c = key[i];
        if (c > best) {
          next = best;
          after = at;
          best = c;
          at = i;
        } else if (c > next) {
          next = c;
          after = i;
        }
      }
      // scores and biases each on their own: the sums of biases are exact, so groups that tie tie here
      mine = best;
      if (kBiased && next != 0u)
        mine = key_of((score(at) + score(after)) + (static_cast<double>(a.bias[at]) + static_cast<double>(a.bias[after])));
    }
    int before = 0;
    for (int g = 0; g < a.ng; ++g) {
      const uint64_t o = static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(mine >> 32), g))) << 32 |
                         static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(mine), g));
      before += o > mine || (o == mine && g < lane);
    }
    const uint64_t kept = ballot(lane < a.ng && before < a.tg);
    for (int e = lane; e < a.E; e += kWave)
      if (!((kept >> (e / a.gs)) & 1u)) key[e] = 0u;
    wave_sync();
  }
  for (int j = 0; j < a.k; ++j) {
    uint64_t best = 0u;
    int at = a.E;
    for (int e = lane; e < a.E; e += kWave)
      if (key[e] > best) {
        best = key[e];
        at = e;
      }
    const uint64_t top = top_of(best);
    // ties: the lowest expert
    const int low = static_cast<int>(~max_over<kWave>(top != 0u && best == top ? ~static_cast<uint32_t>(at) : ~static_cast<uint32_t>(a.E)));
    if (low < a.E && at == low && best == top) key[at] = 0u;
    if (lane == 0) entry[j] = low;
    wave_sync();
  }
}

// Exclusive prefix sums over n <= 1025 counts in LDS, by the whole workgroup (of at least one wave).
__device__ __forceinline__ void block_scan(int32_t* v, int n, int32_t* waves) {
  const int threads = static_cast<int>(blockDim.x), per = (n + threads - 1) / threads;
  const int first = static_cast<int>(threadIdx.x) * per;
  int sum = 0;
  for (int i = 0; i < per; ++i) sum += first + i < n ? v[first + i] : 0;
  const int incl = wave_incl_scan(sum);
  if (lane_id() == kWave - 1) waves[wave_id()] = incl;
  __syncthreads();
  int before = incl - sum;
  for (int w = 0; w < wave_id(); ++w) before += waves[w];
  for (int i = 0; i < per; ++i) {
    if (first + i >= n) break;
    const int c = v[first + i];
    v[first + i] = before;
    before += c;
  }
  __syncthreads();
}

// Waves of a SIMD at least. Four tokens a wave, 16 experts and their biases a lane take just over 128 registers, which leaves a CU
// one workgroup of 8 waves instead of two (65536 tokens over 256 experts in groups 90 us for 67, 8191 the same); the others
// take less, or nothing from it.
template <int L, int PL, bool kBiased> constexpr int pick_waves() { return L == 16 && PL == 16 && kBiased ? 4 : 1; }

// The keys that the rounds compare are the choices' with the expert's number in their low bits, so that one comparison finds
// an expert, takes it out and settles ties:
//   plain logits of 16 bits  all ten bits of it (1023 - e): their fp32 images have 13 low bits that say nothing. The keys of a
//                            token differ, and are exact.
//   otherwise                the number within the lane (PL - 1 - i, up to four bits). Lanes that tie in the rest of the key
//                            are settled by their order. What these bits and fp32 itself leave open is looked at afterwards.
template <int DT, int L, int PL, bool kBiased>
__global__ __launch_bounds__(kPickThreads, (pick_waves<L, PL, kBiased>())) void pick_kernel(PickArgs a, bool whole) {
  constexpr int kTokens = kWave / L;
  constexpr bool kExact = DT != kF32 && !kBiased;
  constexpr uint32_t kCode = kExact ? kMaxE - 1 : PL - 1;
  using Lds = PickLds<L, PL>;
  extern __shared__ __attribute__((aligned(16))) char shared[];
  const int waves = static_cast<int>(blockDim.x) / kWave, wave = wave_id(), lane = lane_id();
  Lds& lds = reinterpret_cast<Lds*>(shared)[wave];
  int32_t* counts = reinterpret_cast<int32_t*>(shared + waves * sizeof(Lds));  // [waves][E + 1], then the first of each expert
  int32_t* local = counts + (waves + 1) * (a.E + 1);                           // expert and rank of the workgroup's picks
  const int seg = lane / L, l = lane % L, E = a.E, k = a.k;
  const bool ordered = a.places != nullptr;
  int32_t* mine = counts + wave * (E + 1);
  const int64_t block_first = static_cast<int64_t>(blockIdx.x) * waves * a.wave_tokens;
  const int64_t first = block_first + static_cast<int64_t>(wave) * a.wave_tokens;
  const int64_t last = first + a.wave_tokens < a.T ? first + a.wave_tokens : a.T;
  int* entry = lds.entry + seg * kEntry;
  auto row_of = [&](int64_t t) { return (t < last ? t : last - 1) * a.ld; };
  float b[PL], far = 0.0f;  // biases, and the largest finite one
  if constexpr (kBiased) {
    load_run<kF32, PL>(reinterpret_cast<const char*>(a.bias), 0, l * PL, E, whole && (reinterpret_cast<uintptr_t>(a.bias) & 15) == 0, b);
#pragma unroll
    for (int i = 0; i < PL; ++i)
      if (fabsf(b[i]) < __builtin_inff()) far = fmaxf(far, fabsf(b[i]));
    far = max_over<L>(far);
  }
  if (ordered) {
    for (int e = lane; e <= E; e += kWave) mine[e] = 0;
    wave_sync();
  }
  for (int64_t t0 = first; t0 < last; t0 += kTokens) {
    const int64_t t = t0 + seg, at = row_of(t);
    const bool live = t < last;
    float v[PL];
    load_run<DT, PL>(a.logits, at, l * PL, E, whole, v);
    float m = 0.0f, z = 1.0f;
    if (!a.sigmoid && (kBiased || !a.renorm)) {
      m = v[0];
#pragma unroll
      for (int i = 1; i < PL; ++i) m = fmaxf(m, v[i]);
      m = max_over<L>(m);
      z = 0.0f;
#pragma unroll
      for (int i = 0; i < PL; ++i) z += l * PL + i < E ? expf(v[i] - m) : 0.0f;
      z = sum_over<L>(z);
    }
    const float rz = 1.0f / z;
    uint32_t key[PL];
#pragma unroll
    for (int i = 0; i < PL; ++i) {
      if constexpr (kBiased) {
        const float s = a.sigmoid ? quick_sigmoid(v[i]) : quick_exp(v[i] - m) * rz;
        key[i] = v[i] == -__builtin_inff() ? 0u : key_of(s + b[i]);
      } else {
        key[i] = key_of(v[i]);
      }
      if (kExact && key[i] != 0u) key[i] = (key[i] & ~kCode) | (kMaxE - 1 - (l * PL + i));
    }
    auto of_token = [&](bool flag) {  // the token's lanes that raise it
      const uint64_t v = ballot(flag);
      return L == kWave ? v : (v >> (seg * L)) & ((uint64_t{1} << (L % kWave)) - 1);
    };
    bool close = false;  // groups too near for 32 bits
    if (a.tg < a.ng) {
      uint64_t kept = 0u;
      float low = __builtin_inff(), high = -__builtin_inff();
      const int share = a.gs / PL;  // lanes of a group
      if (share * PL == a.gs && (share & (share - 1)) == 0 && share <= 16) {
        // whole lanes a group: the two best of each lane's, joined over the group's lanes, and ranked over the token's
        uint32_t best = key[0], next = 0u;
#pragma unroll
        for (int i = 1; i < PL; ++i) {
          const uint32_t less = best < key[i] ? best : key[i];
          next = next > less ? next : less;
          best = best > key[i] ? best : key[i];
        }
        auto join = [&](auto ctrl) {
          const uint32_t ob = static_cast<uint32_t>(dpp<decltype(ctrl)::value>(static_cast<int>(best)));
          const uint32_t on = static_cast<uint32_t>(dpp<decltype(ctrl)::value>(static_cast<int>(next)));
          const uint32_t less = best < ob ? best : ob;
          next = next > on ? next : on;
          next = next > less ? next : less;
          best = best > ob ? best : ob;
        };
        using std::integral_constant;
        if (share >= 2) join(integral_constant<int, kDppXor1>{});
        if (share >= 4) join(integral_constant<int, kDppXor2>{});
        if (share >= 8) join(integral_constant<int, kDppHalfMirror>{});
        if (share >= 16) join(integral_constant<int, kDppMirror>{});
        if constexpr (kBiased) best = key_of_two(best, next);
        const bool real = l * PL < E;
        bool keep;
        if constexpr (L == kWave) {
          int before = 0;
          for (int g = 0; g < a.ng; ++g) {
            const uint32_t other = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(best), g * share));
            before += other > best || (other == best && g * share < (l & -share));
          }
          keep = before < a.tg;
        } else {
          int before = 0;  // lanes whose group comes first (of groups that tie neither does)
          auto turn = [&](auto steps) {
            constexpr int kRor = 0x120 + decltype(steps)::value;  // row_ror: lane i has lane i - steps'
            before += static_cast<uint32_t>(dpp<kRor>(static_cast<int>(best))) > best;
          };
          turn(integral_constant<int, 1>{}); turn(integral_constant<int, 2>{}); turn(integral_constant<int, 3>{});
          turn(integral_constant<int, 4>{}); turn(integral_constant<int, 5>{}); turn(integral_constant<int, 6>{});
          turn(integral_constant<int, 7>{}); turn(integral_constant<int, 8>{}); turn(integral_constant<int, 9>{});
          turn(integral_constant<int, 10>{}); turn(integral_constant<int, 11>{}); turn(integral_constant<int, 12>{});
          turn(integral_constant<int, 13>{}); turn(integral_constant<int, 14>{}); turn(integral_constant<int, 15>{});
          keep = (before >> __builtin_ctz(share)) < a.tg;
          if (!kExact && share * a.tg < __builtin_popcountll(of_token(real && keep && best != 0u))) close = true;
        }
        if (real && keep) low = value_of(best);
        if (real && !keep) high = value_of(best);
        if (!keep) {
#pragma unroll
          for (int i = 0; i < PL; ++i) key[i] = 0u;
        }
      } else {
        const int lo = opaque(l);
#pragma unroll
        for (int i = 0; i < PL; ++i) lds.choice[seg][lo * PL + i] = key[i];
        wave_sync();
        for (int g = lo; g < a.ng; g += L) {
          uint32_t best = 0u, next = 0u;
          for (int i = 0, r = lo % a.gs; i < a.gs; ++i, r = r + 1 == a.gs ? 0 : r + 1) {  // (each lane from another bank on)
            const uint32_t c = lds.choice[seg][g * a.gs + r], less = best < c ? best : c;
            next = next > less ? next : less;
            best = best > c ? best : c;
          }
          if constexpr (kBiased) best = key_of_two(best, next);
          lds.group[seg][g] = best;
        }
        wave_sync();
        for (int g0 = 0; g0 < a.ng; g0 += L) {
          const int g = g0 + lo;
          bool keep = false;
          if (g < a.ng) {
            const uint32_t c = lds.group[seg][g];
            int before = 0;
            for (int o = 0; o < a.ng; ++o) {
              const uint32_t other = lds.group[seg][o];
              before += other > c || (other == c && o < g);
            }
            keep = before < a.tg;
            if (keep) low = fminf(low, value_of(c));
            else high = fmaxf(high, value_of(c));
          }
          kept |= of_token(keep) << g0;
        }
        int g = lo * PL / a.gs, rest = lo * PL - g * a.gs;
#pragma unroll
        for (int i = 0; i < PL; ++i) {
          if (!((kept >> (g & 63)) & 1u)) key[i] = 0u;
          if (++rest == a.gs) {
            rest = 0;
            ++g;
          }
        }
        wave_sync();
      }
      if constexpr (kBiased) {
        low = -max_over<L>(-low);
        high = max_over<L>(high);
        // a group's choice is the sum of two scores, each off by 2^-18 at most (a sigmoid by 2^-21), and of two biases; three
        // roundings
        if (low - high <= (a.sigmoid ? 0x1p-19f : 0x1p-16f) + 0x1p-21f * far) close = true;
      }
    }
    if constexpr (!kExact) {
#pragma unroll
      for (int i = 0; i < PL; ++i) key[i] = key[i] == 0u ? 0u : (key[i] & ~kCode) | static_cast<uint32_t>(PL - 1 - i);
    }
    uint32_t pick = 0u;  // lane j: the key of pick j
    const int listing = k < L ? k + 1 : L;  // entries that have a lane; one more is listed
    if constexpr (kExact) {
      for (int j = 0; j < k; ++j) {
        uint32_t top = key[0];
#pragma unroll
        for (int i = 1; i < PL; ++i) top = key[i] > top ? key[i] : top;
        const uint32_t all = max_over<L>(top);
        pick = l == j ? all : pick;
#pragma unroll
        for (int i = 0; i < PL; ++i) key[i] = key[i] == all ? 0u : key[i];
      }
      if (l < k) entry[l] = pick != 0u ? static_cast<int>(kMaxE - 1 - (pick & kCode)) : E;
    } else {
      for (int j = 0; j <= listing; ++j) {
        uint32_t top = key[0];
#pragma unroll
        for (int i = 1; i < PL; ++i) top = key[i] > top ? key[i] : top;
        const uint32_t all = max_over<L>(top);
        const uint64_t who = of_token((top ^ all) <= kCode && all != 0u);
        const bool winner = who != 0u && l == __builtin_ctzll(who);
        const uint32_t gone = winner ? top : 1u;  // (no key)
#pragma unroll
        for (int i = 0; i < PL; ++i) key[i] = key[i] == gone ? 0u : key[i];
        if (winner || (who == 0u && l == 0)) entry[j] = winner ? l * PL + static_cast<int>(PL - 1 - (top & kCode)) : E;
      }
    }
    wave_sync();
    using S = typename Elem<DT>::S;
    const S* row = reinterpret_cast<const S*>(a.logits) + at;
    if constexpr (!kExact) {
      auto choice_of = [&](float x, float p) {  // as the keys have it, before it was cut
        if constexpr (!kBiased) return x;
        else return (a.sigmoid ? quick_sigmoid(x) : quick_exp(x - m) * rz) + p;
      };
      // How far two choices are off together, or one of them and any that the list does not hold. A sigmoid: exp, two
      // roundings (2^-22 of it, and of small ones less than that). A softmax, of the largest: exp of an argument rounded
      // twice, two products, and the sum, 22 roundings and its terms' (2^-18). The key: a rounding, and the bits that it
      // lacks (2^-19).
      auto reach = [&](float c, float d) {
        if constexpr (!kBiased) return 0x1p-19f * (fabsf(c) + fabsf(d)) + 1e-37f;
        else return (a.sigmoid ? 0x1p-20f : 0x1p-17f * rz) + 0x1.2p-19f * (fabsf(c) + fabsf(d)) + 1e-37f;
      };
      // Which neighbours in the list the keys cannot tell apart: lane j looks at entries j and j + 1. They are linked, equal or
      // not: what lies behind a tie may still be larger than it.
      const int e = l < listing ? entry[l] : E, n = l < listing ? entry[l + 1] : E;
      bool linked = false, equal = false;
      float x = 0.0f, p = 0.0f, c = 0.0f;  // logit, bias and choice of entry j
      if (e < E && n < E) {
        x = Elem<DT>::to_f32(row[e]);
        const float y = Elem<DT>::to_f32(row[n]);
        float q = 0.0f;
        if constexpr (kBiased) {
          p = a.bias[e];
          q = a.bias[n];
        }
        c = choice_of(x, p);
        const float d = choice_of(y, q);
        linked = c - d <= reach(c, d);
        equal = x == y && p == q;
      }
      const uint64_t links = of_token(linked && live), apart = of_token(linked && !equal && live);
      const bool inside = apart & ((uint64_t{1} << k) - 1);  // among the picks and the one behind them
      bool open = ((links >> (k - 1)) & 1u) && (k == L || ((links >> k) & 1u));  // from the last pick past what the list closes
      if (ballot(open) != 0u) {
        // Where all that the last pick cannot be told from are its equals, the list holds the first of them, in their order, and
        // all that are larger: nothing is open. (A router of zeros is such a case, and 16-bit logits that tie.) What is not
        // listed is not larger; the tenth more is for roundings.
        const int at_last = seg * L + k - 1;
        const float xk = __shfl(x, at_last, kWave), pk = __shfl(p, at_last, kWave), ck = __shfl(c, at_last, kWave);
        const uint32_t below = key_of(ck - 1.1f * reach(ck, ck)) & ~kCode, least = below != 0u ? below : 1u;
        bool other = apart & ((uint64_t{2} << k) - 1);
        if constexpr (PL == 16) load_run<DT, PL>(a.logits, at, opaque(l * PL), E, whole, v);  // (kept, they take 16 registers of every token)
#pragma unroll
        for (int i = 0; i < PL; ++i) {
          bool same = v[i] == xk;
          if constexpr (kBiased) same = same && b[i] == pk;
          other |= key[i] >= least && !same;
        }
        open = open && of_token(other) != 0u;
      }
      // Whole tokens again in 64 bits: where groups are near, or the set of the picks is open past what the list holds.
      // (A softmax's sum takes the whole token anyway.)
      uint64_t again = ballot(live && (close || open || (kBiased && !a.sigmoid && inside)));
      if (ballot(inside) & ~again) {
        // otherwise the list itself in 64 bits, the one behind the last pick among it, and each to its rank
        const bool listed = e < E;
        uint64_t exact = 0u;
        if (listed) {
          const double w = Elem<DT>::to_f32(row[e]);
          exact = key_of(kBiased ? 1.0 / (1.0 + exp(-w)) + static_cast<double>(a.bias[e]) : w);
        }
        if (l < listing) lds.fine[seg * kEntry + l] = exact;
        wave_sync();
        int rank = 0;
        for (int j = 0; j < listing; ++j) {
          const uint64_t o = lds.fine[seg * kEntry + j];
          rank += o > exact || (o == exact && o != 0u && entry[j] < e);
        }
        wave_sync();
        if (listed && live && inside) entry[rank] = e;
        wave_sync();
      }
      while (again != 0u) {
        const int s = __builtin_ctzll(again) / L;
        again &= L == kWave ? 0u : ~(((uint64_t{1} << (L % kWave)) - 1) << (s * L));
        wave_sync();
        pick_exactly<DT, kBiased>(a, t0 + s, lds.exact, lds.entry + s * kEntry);
      }
    }
    // the weights: lane j has pick j
    const int e = l < k ? entry[l] : E;
    const bool some = e < E;
    float x = -__builtin_inff();
    if (some) x = kExact ? value_of((pick >> 31) != 0u ? pick & ~kCode : pick | kCode) : Elem<DT>::to_f32(row[e]);
    float s;
    if (a.renorm) {
      // ratios of scores, scaled by the largest so that they do not vanish together
      const float lead = a.sigmoid ? fminf(x, 0.0f) : x;
      const float most = max_over<L>(some ? lead : -__builtin_inff());
      s = some ? expf(lead - most) : 0.0f;
      if (a.sigmoid && some) s = (x != x ? x : s) / (1.0f + expf(-fabsf(x)));
      s = s / sum_over<L>(s);
      if (kBiased && !a.sigmoid && z != z) s = z;  // (of a NaN score nobody need be picked)
    } else {
      s = a.sigmoid ? sigmoid_of(x) : expf(x - m) / z;
    }
    if (live && l < k) {
      a.weights[t * k + l] = some ? a.scale * s : 0.0f;
      a.ids[t * k + l] = some ? e : -1;
    }
    if (ordered) {
      // lane p has pick p of the wave's tokens
      const int of = lane / k, j = lane - of * k;
      const bool valid = of < kTokens && t0 + of < last;
      const int who = valid ? lds.entry[of * kEntry + j] : 0;
      const uint64_t same = same_expert_lanes(who, valid, a.bits);
      if (valid) {
        const uint64_t lower = same & ((uint64_t{1} << lane) - 1);
        const int rank = mine[who] + __builtin_popcountll(lower);
        local[static_cast<int>(t0 + of - block_first) * k + j] = (rank << 16) | who;
        wave_sync();
        if ((same >> lane) == 1u) mine[who] = rank + 1;
      }
      wave_sync();
    }
    wave_sync();
  }
  if (!ordered) return;
  __syncthreads();
  const bool alone = gridDim.x == 1;
  int32_t* starts = counts + waves * (E + 1);
  for (int e = threadIdx.x; e <= E; e += static_cast<int>(blockDim.x)) {
    int sum = 0;
    for (int w = 0; w < waves; ++w) {
      const int c = counts[w * (E + 1) + e];
      counts[w * (E + 1) + e] = sum;
      sum += c;
    }
    starts[e] = alone ? sum : 0;
    if (!alone && e == E)
      for (int pad = E + 1; pad < a.pitch; ++pad) a.counts[static_cast<int64_t>(blockIdx.x) * a.pitch + pad] = 0;
    if (!alone) a.counts[static_cast<int64_t>(blockIdx.x) * a.pitch + e] = sum;
  }
  __syncthreads();
  if (alone) {
    block_scan(starts, E + 1, reinterpret_cast<int32_t*>(shared));
    for (int e = threadIdx.x; e <= E; e += static_cast<int>(blockDim.x)) a.offsets[e] = starts[e];
  }
  const int64_t rest = a.T - block_first;
  const int tokens = rest < static_cast<int64_t>(waves) * a.wave_tokens ? static_cast<int>(rest) : waves * a.wave_tokens;
  for (int i = threadIdx.x; i < tokens * k; i += static_cast<int>(blockDim.x)) {
    const int who = local[i] & 0xffff, w = i / (a.wave_tokens * k);
    const int place = starts[who] + counts[w * (E + 1) + who] + (local[i] >> 16);
    a.places[block_first * k + i] = alone && who == E ? ~place : place;
    if (alone) a.order[place] = who == E ? ~i : i;
  }
}

// counts [blocks][pitch] -> exclusive prefix sums over the workgroups, and the totals. A workgroup takes kScanCols experts;
// 64 threads an expert take a share of the workgroups each.
__global__ __launch_bounds__(kScanCols * kWave) void pick_scan_kernel(PickArgs a) {
  __shared__ int32_t sums[kWave][kScanCols + 1];
  const int col = static_cast<int>(threadIdx.x) % kScanCols, share = static_cast<int>(threadIdx.x) / kScanCols;
  const int n = a.E + 1, e = static_cast<int>(blockIdx.x) * kScanCols + col;
  const int per = (a.blocks + kWave - 1) / kWave, first = share * per;
  const int end = first + per < a.blocks ? first + per : a.blocks;
  int32_t* p = a.counts + e;
  int sum = 0;
  if (e < n) {
#pragma unroll 8
    for (int i = first; i < end; ++i) sum += p[static_cast<int64_t>(i) * a.pitch];
  }
  sums[share][col] = sum;
  __syncthreads();
  const int lane = lane_id(), wave = wave_id();  // a wave adds up the shares of an expert
  const int mine = sums[lane][wave], incl = wave_incl_scan(mine);
  sums[lane][wave] = incl - mine;
  if (lane == kWave - 1 && static_cast<int>(blockIdx.x) * kScanCols + wave < n) a.totals[blockIdx.x * kScanCols + wave] = incl;
  __syncthreads();
  if (e >= n) return;
  int before = sums[share][col];
#pragma unroll 8
  for (int i = first; i < end; ++i) {
    const int c = p[static_cast<int64_t>(i) * a.pitch];
    p[static_cast<int64_t>(i) * a.pitch] = before;
    before += c;
  }
}

// The workgroup takes the picks of one that picked, whose number is its own. Of few it adds up the counts before it, and all
// of them, by itself: four experts a thread, the threads of an expert a share of the workgroups each.
__global__ __launch_bounds__(kPlaceThreads) void pick_place_kernel(PickArgs a, int block_picks) {
  __shared__ int32_t starts[kMaxE + 4], base[kMaxE + 4];
  __shared__ int32_t waves[kPlaceThreads / kWave];
  const int n = a.E + 1, tid = static_cast<int>(threadIdx.x);
  const int64_t block = blockIdx.x, picks = a.T * a.k, pick = block * block_picks + tid;  // (block_picks <= kBlockPicks)
  constexpr int kEach = kBlockPicks / kPlaceThreads;
  int id[kEach], rank[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const bool some = tid + i * kPlaceThreads < block_picks && pick + i * kPlaceThreads < picks;
    id[i] = some ? a.ids[pick + i * kPlaceThreads] : 0;
    rank[i] = some ? a.places[pick + i * kPlaceThreads] : -1;
  }
  if (a.scanned) {
    for (int e = tid; e < n; e += kPlaceThreads) {
      starts[e] = a.totals[e];
      base[e] = a.counts[block * a.pitch + e];
    }
  } else {
    for (int e = tid; e < a.pitch; e += kPlaceThreads) starts[e] = base[e] = 0;
    __syncthreads();
    typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
    constexpr int kBatch = 20;  // loads on their way at once
    const int quads = a.pitch / 4, shares = kPlaceThreads / quads, share = tid / quads, quad = tid - share * quads;
    if (share < shares) {
      i32x4 all = {0, 0, 0, 0}, before = {0, 0, 0, 0};
      for (int i0 = share; i0 < a.blocks; i0 += kBatch * shares) {
        i32x4 c[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          const int i = i0 + j * shares;
          c[j] = i < a.blocks ? *reinterpret_cast<const i32x4*>(a.counts + static_cast<int64_t>(i) * a.pitch + 4 * quad) : i32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          all += c[j];
          if (i0 + j * shares < block) before += c[j];
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {  // (integers: any order gives the same)
        if (all[j] != 0) atomicAdd(&starts[4 * quad + j], all[j]);
        if (before[j] != 0) atomicAdd(&base[4 * quad + j], before[j]);
      }
    }
  }
  __syncthreads();
  block_scan(starts, n, waves);
  if (block == 0)
    for (int e = tid; e < n; e += kPlaceThreads) a.offsets[e] = starts[e];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    if (rank[i] < 0) continue;
    const int who = id[i] < 0 ? a.E : id[i], place = starts[who] + base[who] + rank[i];
    const int64_t mine = pick + i * kPlaceThreads;
    a.places[mine] = id[i] < 0 ? ~place : place;
    a.order[place] = static_cast<int32_t>(id[i] < 0 ? ~mine : mine);
  }
}

__global__ __launch_bounds__(kPickThreads) void no_picks_kernel(int64_t* offsets, int n) {
  const int e = static_cast<int>(blockIdx.x) * kPickThreads + static_cast<int>(threadIdx.x);
  if (e < n) offsets[e] = 0;
}

// With p the weights before the scale, g = scale * grad_w, D = sum over the picks of p g:
//   softmax              s_e ([e picked] g_e - D)   over all experts
//   softmax, renormed    p_j (g_j - D)              at the picks
//   sigmoid              s_j (1 - s_j) g_j          at the picks
//   sigmoid, renormed    p_j (1 - s_j) (g_j - D)    at the picks
template <int DT, int L, int PL>
__global__ __launch_bounds__(kGradThreads) void pick_grad_kernel(PickArgs a, bool whole) {
  constexpr int kTokens = kWave / L;
  using S = typename Elem<DT>::S;
  __shared__ float ds[kGradThreads / kWave][kTokens][kMaxK];
  __shared__ int es[kGradThreads / kWave][kTokens][kMaxK];
  const int wave = wave_id(), lane = lane_id(), seg = lane / L, l = lane % L, E = a.E, k = a.k;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (kGradThreads / kWave) * kTokens;
  for (int64_t t0 = (static_cast<int64_t>(blockIdx.x) * (kGradThreads / kWave) + wave) * kTokens; t0 < a.T; t0 += step) {
    const int64_t t = t0 + seg < a.T ? t0 + seg : a.T - 1;
    const bool live = t0 + seg < a.T;
    const S* row = reinterpret_cast<const S*>(a.logits) + t * a.ld;
    float v[PL], m = 0.0f, z = 1.0f;
    if (a.grad_dense) {
      load_run<DT, PL>(a.logits, t * a.ld, l * PL, E, whole, v);
      m = v[0];
#pragma unroll
      for (int i = 1; i < PL; ++i) m = fmaxf(m, v[i]);
      m = max_over<L>(m);
      z = 0.0f;
#pragma unroll
      for (int i = 0; i < PL; ++i) {
        v[i] = v[i] == -__builtin_inff() ? 0.0f : expf(v[i] - m);
        z += v[i];
      }
      z = sum_over<L>(z);
    }
    const int id = l < k ? a.ids[t * k + l] : -1;
    const bool some = id >= 0 && id < E;
    const float g = some ? a.scale * a.grad_w[t * k + l] : 0.0f;
    const float x = some ? Elem<DT>::to_f32(row[id]) : -__builtin_inff();
    float p, d, dot = 0.0f;
    if (a.renorm) {
      const float lead = a.sigmoid ? fminf(x, 0.0f) : x;
      const float most = max_over<L>(some ? lead : -__builtin_inff());
      p = some ? expf(lead - most) : 0.0f;
      if (a.sigmoid && some) p = (x != x ? x : p) / (1.0f + expf(-fabsf(x)));
      p = p / sum_over<L>(p);
      dot = sum_over<L>(some ? p * g : 0.0f);
      d = p * (g - dot);
      if (a.sigmoid) d *= sigmoid_of(-x);
    } else if (a.sigmoid) {
      d = sigmoid_of(x) * sigmoid_of(-x) * g;
    } else {
      p = some ? expf(x - m) / z : 0.0f;
      d = p * g;
      dot = sum_over<L>(some ? d : 0.0f);
    }
    if (l < k) {
      ds[wave][seg][l] = d;
      es[wave][seg][l] = some ? id : -1;
    }
    wave_sync();
    float o[PL];
#pragma unroll
    for (int i = 0; i < PL; ++i) o[i] = a.grad_dense ? (v[i] == 0.0f ? 0.0f : -(v[i] / z) * dot) : 0.0f;
    for (int j = 0; j < k; ++j) {
      const int at = es[wave][seg][j] - l * PL;
      const float dj = ds[wave][seg][j];
#pragma unroll
      for (int i = 0; i < PL; ++i) o[i] += at == i ? dj : 0.0f;
    }
    if (live) {
      S* out = reinterpret_cast<S*>(a.grad) + t * E + l * PL;
      if (whole) {
        struct alignas(PL * sizeof(S) < 16 ? PL * sizeof(S) : 16) Run { S s[PL]; } r;
#pragma unroll
        for (int i = 0; i < PL; ++i) r.s[i] = round_to<DT>(o[i]);
        if (l * PL < E) *reinterpret_cast<Run*>(out) = r;
      } else {
#pragma unroll
        for (int i = 0; i < PL; ++i)
          if (l * PL + i < E) out[i] = round_to<DT>(o[i]);
      }
    }
    wave_sync();
  }
}

// ---- host ----------------------------------------------------------------------------------------

struct PickShape { int lanes, each; };

// A wave a token where there are few and each takes long: its chain of instructions is shorter, though there are more in all
// (256 experts in 8 groups with a bias, fp32: 1 token 11.1 -> 9.3 us, 1024 17.4 -> 15.5, 2048 20.6 and 20.0, 4096 23.3 -> 26.9).
constexpr int64_t kFewTokens = 1024;

PickShape pick_shape(int64_t T, int64_t E) {
  if (T <= kFewTokens && E > 64 && E <= 128) return {64, 2};
  if (T <= kFewTokens && E > 128 && E <= 256) return {64, 4};
  if (E <= 16) return {16, 1};
  if (E <= 64) return {16, 4};
  if (E <= 128) return {16, 8};
  if (E <= 256) return {16, 16};
  if (E <= 512) return {64, 8};
  return {64, 16};
}

struct PickPlan {
  int waves, wave_tokens, pitch;
  bool scan;
  int64_t blocks, totals, total;  // workgroups; offset of the totals (behind the counts); bytes in all
};

// Workgroups that add up the counts by themselves: (workgroups) x (experts) up to this. With 256 x 260 the placing kernel takes
// 7.1 us that way, and 4.1 behind a scan of 4.8 and another launch; with 512 x 260 the scan is ahead.
constexpr int64_t kOwnCounts = 1 << 17;

PickPlan pick_plan(int64_t T, int64_t E, int64_t k) {
  const PickShape f = pick_shape(T, E);
  const int tokens = kWave / f.lanes;
  PickPlan p{};
  p.waves = E <= 256 ? kPickThreads / kWave : kPickThreads / kWave / 2;  // (64 KB of LDS)
  p.waves = static_cast<int>(std::min<int64_t>(p.waves, std::max<int64_t>(1, (T + tokens - 1) / tokens)));
  const int64_t step = p.waves * tokens;                                // tokens that a workgroup takes at once
  const int64_t most = std::max<int64_t>(1, kBlockPicks / (step * k));  // such steps whose ranks a workgroup can hold
  const int64_t spread = 256 * (E <= 256 ? 1 : 2);                      // workgroups for many tokens
  int64_t steps = std::max<int64_t>(1, (T + spread * step - 1) / (spread * step));
  // one workgroup, while its steps take less than another kernel: of 64 experts two (42 tokens 7.5 us for 8.8, 85 9.4 for 9.0), of
  // 16 four (128 tokens 7.5 for 8.0, 256 11.6 for 8.2), of more one (64 tokens over 256 experts in two 19.8 us for 16.0)
  const int64_t alone = E <= 16 ? 4 : E <= 64 ? 2 : 1;
  if (T <= alone * step) steps = (T + step - 1) / step;
  steps = std::max<int64_t>(1, std::min(steps, most));
  p.wave_tokens = static_cast<int>(steps * tokens);
  p.blocks = (T + steps * step - 1) / (steps * step);
  p.pitch = static_cast<int>((E + 4) / 4 * 4);
  p.scan = p.blocks * p.pitch > kOwnCounts;
  p.totals = (p.blocks * p.pitch * 4 + 255) / 256 * 256;
  p.total = p.blocks > 1 ? p.totals + (E + 1) * 4 : 0;
  return p;
}

bool whole_runs(const void* p, int64_t pitch, int64_t E, int64_t es, int each) {
  const int64_t run = std::min<int64_t>(16, each * es);
  return E % each == 0 && aligned_to(p, run) && pitch * es % run == 0;
}

template <int DT, int L, int PL>
hipError_t launch_pick(const PickArgs& a, const PickPlan& p, bool whole, hipStream_t s) {
  size_t lds = p.waves * sizeof(PickLds<L, PL>);
  if (a.places) lds += (static_cast<size_t>(p.waves) + 1) * (a.E + 1) * 4 + static_cast<size_t>(p.waves) * p.wave_tokens * a.k * 4;
  const unsigned blocks = static_cast<unsigned>(p.blocks);
  const int threads = p.waves * kWave;
  if (a.bias) pick_kernel<DT, L, PL, true><<<blocks, threads, lds, s>>>(a, whole);
  else pick_kernel<DT, L, PL, false><<<blocks, threads, lds, s>>>(a, whole);
  return hipGetLastError();
}

template <int DT, int L, int PL>
hipError_t launch_pick_grad(const PickArgs& a, bool whole, hipStream_t s) {
  const int64_t step = kGradThreads / L;
  const unsigned blocks = static_cast<unsigned>(std::min<int64_t>((a.T + step - 1) / step, 2048));
  pick_grad_kernel<DT, L, PL><<<blocks, kGradThreads, 0, s>>>(a, whole);
  return hipGetLastError();
}

template <bool kGrad, int DT>
hipError_t launch_typed(const PickArgs& a, const PickPlan& p, bool whole, hipStream_t s) {
  const PickShape f = pick_shape(kGrad ? kFewTokens + 1 : a.T, a.E);
  auto go = [&](auto lanes, auto each) {
    constexpr int L = decltype(lanes)::value, PL = decltype(each)::value;
    if constexpr (kGrad) return launch_pick_grad<DT, L, PL>(a, whole, s);
    else return launch_pick<DT, L, PL>(a, p, whole, s);
  };
  using std::integral_constant;
  if (f.lanes == 16) {
    switch (f.each) {
      case 1: return go(integral_constant<int, 16>{}, integral_constant<int, 1>{});
      case 4: return go(integral_constant<int, 16>{}, integral_constant<int, 4>{});
      case 8: return go(integral_constant<int, 16>{}, integral_constant<int, 8>{});
      default: return go(integral_constant<int, 16>{}, integral_constant<int, 16>{});
    }
  }
  if constexpr (!kGrad) {
    if (f.each == 2) return go(integral_constant<int, 64>{}, integral_constant<int, 2>{});
    if (f.each == 4) return go(integral_constant<int, 64>{}, integral_constant<int, 4>{});
  }
  return f.each == 8 ? go(integral_constant<int, 64>{}, integral_constant<int, 8>{}) : go(integral_constant<int, 64>{}, integral_constant<int, 16>{});
}

template <bool kGrad>
hipError_t launch_picks(int dtype, const PickArgs& a, const PickPlan& p, bool whole, hipStream_t s) {
  switch (dtype) {
    case kF32: return launch_typed<kGrad, kF32>(a, p, whole, s);
    case kF16: return launch_typed<kGrad, kF16>(a, p, whole, s);
    default: return launch_typed<kGrad, kBF16>(a, p, whole, s);
  }
}

int check_picks(int64_t T, int64_t E, int64_t k, int dtype, int scoring) {
  if (T < 0 || E <= 0 || k <= 0 || k > E || !known_dtype(dtype) || (scoring != SMX_SCORE_SOFTMAX && scoring != SMX_SCORE_SIGMOID))
    return SMX_ERR_INVALID_ARG;
  if (E > kMaxE || k > kMaxK || T > INT32_MAX / k) return SMX_ERR_UNSUPPORTED;
  return SMX_OK;
}

}  // namespace
}  // namespace smx

using namespace smx;

extern "C" {

size_t smx_route_workspace_size(int64_t T, int64_t E, int64_t k) {
  if (check_picks(T, E, k, kF32, SMX_SCORE_SOFTMAX) != SMX_OK) return 0;
  return static_cast<size_t>(pick_plan(T, E, k).total);
}

int smx_route(const void* logits, int64_t logits_stride, int dtype, int64_t T, int64_t E, int64_t k, int scoring,
              const float* bias, int64_t num_groups, int64_t top_groups, int renormalize, float scale, float* weights,
              int32_t* ids, int32_t* places, int32_t* order, int64_t* offsets, void* workspace, size_t workspace_bytes,
              void* stream) {
  const int rc = check_picks(T, E, k, dtype, scoring);
  if (rc != SMX_OK) return rc;
  if (logits_stride < E || num_groups <= 0 || E % num_groups != 0 || top_groups <= 0 || top_groups > num_groups ||
      k > E / num_groups * top_groups || !(scale - scale == 0.0f))
    return SMX_ERR_INVALID_ARG;
  if (num_groups > kMaxGroups) return SMX_ERR_UNSUPPORTED;
  const bool ordered = places != nullptr;
  if ((order != nullptr) != ordered && T > 0) return SMX_ERR_INVALID_ARG;
  if (ordered && !offsets) return SMX_ERR_INVALID_ARG;
  if (T > 0 && (!logits || !weights || !ids || (offsets && !ordered))) return SMX_ERR_INVALID_ARG;
  const int64_t es = dtype_bytes(dtype);
  if (!aligned_to(logits, es) || !aligned_to(bias, 4) || !aligned_to(weights, 4) || !aligned_to(ids, 4) || !aligned_to(places, 4) ||
      !aligned_to(order, 4) || !aligned_to(offsets, 8) || !aligned_to(workspace, 16))
    return SMX_ERR_MISALIGNED;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const PickPlan p = pick_plan(T, E, k);
  PickArgs a{};
  a.T = T;
  a.E = static_cast<int>(E);
  a.k = static_cast<int>(k);
  a.places = places;
  a.order = order;
  a.offsets = offsets;
  a.ids = ids;
  a.blocks = static_cast<int>(p.blocks);
  a.pitch = p.pitch;
  if (ordered && p.total > 0) {
    if (!workspace || workspace_bytes < static_cast<size_t>(p.total)) return SMX_ERR_WORKSPACE;
    a.counts = static_cast<int32_t*>(workspace);
    a.totals = reinterpret_cast<int32_t*>(static_cast<char*>(workspace) + p.totals);
  }
  if (T == 0) {
    if (!offsets) return SMX_OK;
    no_picks_kernel<<<static_cast<unsigned>((E + kPickThreads) / kPickThreads), kPickThreads, 0, s>>>(offsets, a.E + 1);
    return static_cast<int>(hipGetLastError());
  }
  a.logits = static_cast<const char*>(logits);
  a.ld = logits_stride;
  a.ng = static_cast<int>(num_groups);
  a.tg = static_cast<int>(top_groups);
  a.gs = static_cast<int>(E / num_groups);
  a.sigmoid = scoring == SMX_SCORE_SIGMOID;
  a.renorm = renormalize != 0;
  a.scale = scale;
  a.bias = bias;
  a.weights = weights;
  a.wave_tokens = p.wave_tokens;
  while ((E >> a.bits) != 0) ++a.bits;
  hipError_t err = launch_picks<false>(dtype, a, p, whole_runs(logits, logits_stride, E, es, pick_shape(T, E).each), s);
  if (err != hipSuccess || !ordered || p.blocks == 1) return static_cast<int>(err);
  if (p.scan) {
    pick_scan_kernel<<<static_cast<unsigned>((E + kScanCols) / kScanCols), kScanCols * kWave, 0, s>>>(a);
    err = hipGetLastError();
    if (err != hipSuccess) return static_cast<int>(err);
    a.scanned = true;
  }
  pick_place_kernel<<<static_cast<unsigned>(p.blocks), kPlaceThreads, 0, s>>>(a, static_cast<int>(p.waves * p.wave_tokens * k));
  return static_cast<int>(hipGetLastError());
}

int smx_route_grad(const float* grad_weights, const void* logits, int64_t logits_stride, int dtype, int64_t T, int64_t E,
                   int64_t k, int scoring, int renormalize, float scale, const int32_t* ids, void* grad_logits, void* stream) {
  const int rc = check_picks(T, E, k, dtype, scoring);
  if (rc != SMX_OK) return rc;
  if (logits_stride < E || !(scale - scale == 0.0f)) return SMX_ERR_INVALID_ARG;
  if (T == 0) return SMX_OK;
  if (!grad_weights || !logits || !ids || !grad_logits) return SMX_ERR_INVALID_ARG;
  const int64_t es = dtype_bytes(dtype);
  if (!aligned_to(logits, es) || !aligned_to(grad_logits, es) || !aligned_to(grad_weights, 4) || !aligned_to(ids, 4)) return SMX_ERR_MISALIGNED;
  PickArgs a{};
  a.T = T;
  a.E = static_cast<int>(E);
  a.k = static_cast<int>(k);
  a.logits = static_cast<const char*>(logits);
  a.ld = logits_stride;
  a.sigmoid = scoring == SMX_SCORE_SIGMOID;
  a.renorm = renormalize != 0;
  a.grad_dense = !a.sigmoid && !a.renorm;
  a.scale = scale;
  a.ids = const_cast<int32_t*>(ids);
  a.grad_w = grad_weights;
  a.grad = static_cast<char*>(grad_logits);
  const int each = pick_shape(kFewTokens + 1, E).each;
  const bool whole = whole_runs(logits, logits_stride, E, es, each) && whole_runs(grad_logits, E, E, es, each);
  return static_cast<int>(launch_picks<true>(dtype, a, PickPlan{}, whole, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
