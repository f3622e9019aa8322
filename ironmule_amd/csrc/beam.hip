// MI355X (gfx950) kernels of beam selection and their C ABI (include/ironmule_paged.h): the best
// continuations of each group of beams over the whole vocabulary.

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <string>

#include "../../include/ironmule_paged.h"
#include "common.h"
#include "runtime.h"

namespace {

using namespace imq_dev;

using imq_rt::aligned;
using imq_rt::current_device;
using imq_rt::fail;
using imq_rt::ok;

constexpr int kWaves = 4, kThreads = 64 * kWaves;  // of a slice's workgroup
constexpr int kMergeThreads = 1024;
constexpr int kMaxCount = IMQ_BEAM_MAX_COUNT, kMaxBeams = IMQ_BEAM_MAX_BEAMS;
constexpr int kSome = 512, kRankStep = 8;  // values that wave_best gathers, and compares with at a time
constexpr float kLog2e = 1.44269504088896340736f;

// A row's slice as select_slice_kernel leaves it: the largest value, the sum of exp(x - largest), and
// the ranks (rank_of) of the `count` best values in order; 0 where there are fewer.
struct Slices {
  double* sum;
  uint64_t* rank;
  float* most;
  int32_t slices;
};

// (value, token) as one number that orders values descending and equal ones by token: the value's
// bits made monotone above the token's complement.  Never 0.
__device__ __forceinline__ uint32_t monotone(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);  // (-0 as 0)
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t rank_of(float x, int token) { return ((uint64_t)monotone(x) << 32) | (uint32_t)~token; }
__device__ __forceinline__ float value_of(uint32_t u) { return __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u); }
__device__ __forceinline__ int token_of(uint64_t rank) { return (int)~(uint32_t)rank; }

__device__ __forceinline__ uint64_t wave_most(uint64_t v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    const uint64_t o = __shfl_xor(v, d);
    v = o > v ? o : v;
  }
  return v;
}

__device__ __forceinline__ double wave_total(double v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
  return v;
}

__device__ __forceinline__ int lanes_below(uint64_t mask) {  // set bits below this lane's
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// LDS that the lanes of one wavefront hand each other: its accesses complete in order, the compiler must
// not move them.
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// The `count` best of the wavefront's 64 E values (and of the `have` in best[]) in order into best[];
// returns how many there are (values of -inf and NaN are none).  most: the lane's largest value; token(e): of its
// e-th; `some`: kSome + kRankStep places of LDS.
//
// The last of best[], where it is full, or else the count-th largest of the lanes' own largest values bounds
// the count-th largest of all from below; of the latter the upper 16 bits come from 16 ballots.  Few values pass
// it: they are gathered in LDS, cut down to
// those that the exact bound passes if they are over 64, and for each the better ones are counted.  Where more
// than kSome pass (many equal values), the best is taken count times.
// (Taken count times always, workgroup by workgroup: 61 us where this takes 11, for eight of each of 32 rows of
// 262144 bf16 values.)
template <int E, typename TOKEN>
__device__ __forceinline__ int wave_best(const float (&x)[E], float most, TOKEN token, int count, int have, uint64_t* best,
                                         uint64_t* some) {
  const int lane = threadIdx.x & 63;
  const uint64_t old = lane < have ? best[lane] : 0ull;
  uint32_t top = most > -INFINITY ? monotone(most) : 0u;
  uint32_t bound = 0;
  if (have == count) {
    bound = __builtin_amdgcn_readlane((uint32_t)(old >> 32), count - 1);
    if (!__any(top >= bound)) return have;
  } else {
    top = max(top, (uint32_t)(old >> 32));
#pragma unroll 1
    for (uint32_t bit = 1u << 31; bit >= 1u << 16; bit >>= 1)
      if (__popcll(__ballot(top >= (bound | bit))) >= count) bound |= bit;
  }
  // as a value; 0: fewer lanes than count have any
  const float least = bound ? value_of(bound) : -INFINITY;
  int passed = 0;
  auto gather = [&](bool pass, uint64_t rank) {
    const uint64_t mask = __ballot(pass);
    if (mask == 0) return;
    const int at = passed + lanes_below(mask);
    if (pass && at < kSome) some[at] = rank;
    passed += __popcll(mask);
  };
  gather(old != 0 && (uint32_t)(old >> 32) >= bound, old);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const bool pass = x[e] > -INFINITY && x[e] >= least;
    if (__any(pass)) gather(pass, pass ? rank_of(x[e], token(e)) : 0ull);
  }
  if (passed <= kSome) {
    wave_fence();
    if (passed > 64) {  // the values' bound exactly, from the gathered ones, eight a lane; those below it fall out
      uint64_t mine[kSome / 64];
      bound = 0;
#pragma unroll
      for (int k = 0; k < kSome / 64; ++k) mine[k] = 64 * k + lane < passed ? some[64 * k + lane] : 0ull;
#pragma unroll 1
      for (uint32_t bit = 1u << 31; bit; bit >>= 1) {
        int n = 0;
#pragma unroll
        for (int k = 0; k < kSome / 64; ++k) n += __popcll(__ballot((uint32_t)(mine[k] >> 32) >= (bound | bit)));
        if (n >= count) bound |= bit;
      }
      wave_fence();
      passed = 0;
#pragma unroll
      for (int k = 0; k < kSome / 64; ++k) gather(mine[k] != 0 && (uint32_t)(mine[k] >> 32) >= bound, mine[k]);
    }
    if (lane < kRankStep) some[passed + lane] = 0ull;
    wave_fence();
    for (int i = lane; i < passed; i += 64) {
      const uint64_t mine = some[i];
      int better = 0;
      for (int j = 0; j < passed; j += kRankStep) {
        uint64_t other[kRankStep];
#pragma unroll
        for (int k = 0; k < kRankStep; ++k) other[k] = some[j + k];
#pragma unroll
        for (int k = 0; k < kRankStep; ++k) better += other[k] > mine;
      }
      if (better < count) best[better] = mine;
    }
    wave_fence();
    return min(passed, count);
  }
  uint64_t below = ~0ull;  // ranks from here on are taken
  int n = 0;
  for (; n < count; ++n) {
    uint64_t mine = old < below ? old : 0ull;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint64_t r = rank_of(x[e], token(e));
      if (x[e] > -INFINITY && r < below && r > mine) mine = r;
    }
    below = wave_most(mine);
    if (below == 0) break;
    if (lane == 0) best[n] = below;
  }
  wave_fence();
  return n;
}

// The row's values v0 .. v0 + N - 1, -inf past the row's end: one load where they are all inside, wherever the row
// starts (which values a lane has must not depend on that: rows of the same values have to have the same sums,
// to the last bit, for their ties to be ties).
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

template <bool BF16>
__device__ __forceinline__ void load_values(const void* at, int v0, int vocab, float* x) {
  constexpr int N = BF16 ? 8 : 4;
  if (v0 + N <= vocab) {
    const u32x4_any u = *static_cast<const u32x4_any*>(at);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (BF16)
        x[2 * e] = bf16_bits_to_f32(u[e] & 0xffffu), x[2 * e + 1] = bf16_bits_to_f32(u[e] >> 16);
      else
        x[e] = __uint_as_float(u[e]);
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < N; ++e) {
    x[e] = -INFINITY;
    if (v0 + e < vocab)
      x[e] = BF16 ? bf16_bits_to_f32(static_cast<const uint16_t*>(at)[e]) : static_cast<const float*>(at)[e];
  }
}

// A workgroup per slice of a row, a quarter of it a wavefront, `blocks` times 64 E values.  Bound by each wavefront's chain,
// with two wavefronts for each SIMD: its block's loads, then the sums, then the candidates, nothing of the next step
// under the one before (32 rows of 262144 bf16 values, 15 MB, in 12 us: 1.3 TB/s).
template <bool BF16, int E>
__global__ __launch_bounds__(kThreads) void select_slice_kernel(const void* __restrict__ logits, int64_t ld, int vocab,
                                                                int count, const int32_t* __restrict__ finished, int blocks,
                                                                Slices s) {
  constexpr int N = BF16 ? 8 : 4, SIZE = BF16 ? 2 : 4;
  __shared__ uint64_t best[kWaves][kMaxCount], some[kWaves][kSome + kRankStep];
  __shared__ float tops[kWaves];
  __shared__ double sums[kWaves];
  __shared__ int counts[kWaves];
  const int row = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (finished && finished[row]) return;
  const char* const values = static_cast<const char*>(logits) + row * ld * SIZE;
  const int first = ((int)blockIdx.x * kWaves + wave) * 64 * E * blocks + lane * N;
  float most = -INFINITY;
  double sum = 0.0;  // of exp(x - most), of the lane's values
  int have = 0;
  for (int block = 0; block < blocks; ++block) {
    const int v0 = first + 64 * E * block;
    float x[E];
#pragma unroll
    for (int i = 0; i < E / N; ++i)
      load_values<BF16>(values + ((int64_t)v0 + 64 * N * i) * SIZE, v0 + 64 * N * i, vocab, x + N * i);
    float mine = -INFINITY;
#pragma unroll
    for (int e = 0; e < E; ++e) mine = fmaxf(mine, x[e]);
    const float higher = fmaxf(most, wave_max(mine)), base = higher == -INFINITY ? 0.0f : higher;
    if (block) sum *= (double)__builtin_amdgcn_exp2f((most - base) * kLog2e);
    most = higher;
    // Eight at a time in fp32 (a NaN stays one).  The difference first: base * log2(e) as a number of its own is
    // rounded to its own size, which every term would carry, and is infinite for a base of the lowest finite
    // value; the difference is as good as its own size, and the largest value's term is 1.
#pragma unroll
    for (int e = 0; e < E; e += 8) {
      float part = 0.0f;
#pragma unroll
      for (int k = 0; k < 8; ++k) part += __builtin_amdgcn_exp2f((x[e + k] - base) * kLog2e);
      sum += (double)part;
    }
    have = wave_best<E>(x, mine, [&](int e) { return v0 + 64 * N * (e / N) + e % N; }, count, have, best[wave], some[wave]);
  }
  sum = wave_total(sum);
  if (lane == 0) tops[wave] = most, sums[wave] = sum, counts[wave] = have;
  __syncthreads();
  const int64_t at = (int64_t)row * s.slices + blockIdx.x;
  if (threadIdx.x == 0) {
    const float all = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    double total = 0.0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) total += tops[w] == all || sums[w] != sums[w] ? sums[w] : sums[w] * exp((double)tops[w] - all);
    s.most[at] = all;
    s.sum[at] = total;
  }
  // the wavefronts' lists as one: a thread per entry counts the better ones, by bisection of each list
  const int list = threadIdx.x / kMaxCount, entry = threadIdx.x % kMaxCount;
  int all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) all += counts[w];
  if (entry < counts[list]) {
    const uint64_t mine = best[list][entry];
    int better = entry;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      int lo = 0, hi = w == list ? 0 : counts[w];  // the first entry that is worse
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (best[w][mid] > mine) lo = mid + 1; else hi = mid;
      }
      better += lo;
    }
    if (better < count) s.rank[at * count + better] = mine;
  }
  for (int i = all + threadIdx.x; i < count; i += kThreads) s.rank[at * count + i] = 0ull;
}

struct SelectArgs {
  const float* scores;
  const int32_t* finished;
  int32_t eos, beams, count;
  float* out_scores;
  int32_t *out_parents, *out_tokens, *out_finished;
};

// A workgroup per group.  A wavefront per beam at a time: the beam's log sum, and the best of its slices'
// candidates in order; then a thread per (beam, entry) counts the better ones of the other beams.  A key is
// (value - largest) + (score - log sum of exp(value - largest)): the largest value alone may be of any size.
__global__ __launch_bounds__(kMergeThreads) void select_merge_kernel(Slices s, SelectArgs a) {
  constexpr int kE = 8;
  __shared__ double shift[kMaxBeams];  // score - log sum, of a finished beam the score
  __shared__ float tops[kMaxBeams];    // the largest value, of a finished beam 0
  __shared__ int counts[kMaxBeams];
  __shared__ uint64_t best[kMaxBeams][kMaxCount];
  __shared__ uint64_t some[kMergeThreads / 64][kSome + kRankStep];
  const int group = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int b = wave; b < a.beams; b += kMergeThreads / 64) {
    const int row = group * a.beams + b;
    const float score = a.scores[row];
    int have = 0;
    if (a.finished && a.finished[row]) {
      if (lane == 0) shift[b] = (double)score, tops[b] = 0.0f, best[b][0] = rank_of(0.0f, a.eos);
      have = isfinite(score) ? 1 : 0;
    } else {
      const int64_t at = (int64_t)row * s.slices;
      float most = -INFINITY;
      for (int i = lane; i < s.slices; i += 64) most = fmaxf(most, s.most[at + i]);
      most = wave_max(most);
      double sum = 0.0;
      for (int i = lane; i < s.slices; i += 64) {
        const float m = s.most[at + i];
        const double z = s.sum[at + i];
        sum += m == -INFINITY && z == 0.0 ? 0.0 : z * exp((double)m - (most == -INFINITY ? 0.0f : most));
      }
      sum = wave_total(sum);
      const double v = (double)score - log(sum);
      if (lane == 0) shift[b] = v, tops[b] = most;
      if (isfinite(v) && isfinite(most)) {  // (a score, a value or a sum that is not finite: nothing is offered)
        const int all = s.slices * a.count;
        for (int i0 = 0; i0 < all; i0 += 64 * kE) {
          float x[kE], mine = -INFINITY;
          int token[kE];
#pragma unroll
          for (int e = 0; e < kE; ++e) {
            const int i = i0 + 64 * e + lane;
            const uint64_t r = i < all ? s.rank[at * a.count + i] : 0ull;
            x[e] = r ? value_of((uint32_t)(r >> 32)) : -INFINITY;
            token[e] = token_of(r);
            mine = fmaxf(mine, x[e]);
          }
          have = wave_best<kE>(x, mine, [&](int e) { return token[e]; }, a.count, have, best[b], some[wave]);
        }
      }
    }
    if (lane == 0) counts[b] = have;
  }
  __syncthreads();
  int all = 0;
  for (int b = 0; b < a.beams; ++b) all += counts[b];
  auto key_of = [&](int b, int i) { return ((double)value_of((uint32_t)(best[b][i] >> 32)) - (double)tops[b]) + shift[b]; };
  for (int item = threadIdx.x; item < a.beams * a.count; item += kMergeThreads) {
    const int b = item / a.count, i = item % a.count;
    if (i >= counts[b]) continue;
    const double mine = key_of(b, i);
    int better = i;
    for (int o = 0; o < a.beams && better < a.count; ++o) {
      int lo = 0, hi = o == b ? 0 : counts[o];
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        const double theirs = key_of(o, mid);
        if (theirs > mine || (theirs == mine && o < b)) lo = mid + 1; else hi = mid;
      }
      better += lo;
    }
    if (better >= a.count) continue;
    const int at = group * a.count + better, row = group * a.beams + b, token = token_of(best[b][i]);
    a.out_scores[at] = (float)mine;
    a.out_parents[at] = row;
    a.out_tokens[at] = token;
    a.out_finished[at] = token == a.eos || (a.finished && a.finished[row]) ? 1 : 0;
  }
  for (int i = all + threadIdx.x; i < a.count; i += kMergeThreads) {
    const int at = group * a.count + i;
    a.out_scores[at] = -INFINITY;
    a.out_parents[at] = a.out_tokens[at] = -1;
    a.out_finished[at] = 0;
  }
}

int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

int32_t check_sizes(int32_t groups, int32_t beams, int32_t vocab, int32_t count) {
  if (groups < 1 || beams < 1 || vocab < 1 || count < 1) return fail(IMQ_EINVAL, "groups, beams, vocab and count must be >= 1");
  if (groups > IMQ_BEAM_MAX_GROUPS || beams > IMQ_BEAM_MAX_BEAMS || count > IMQ_BEAM_MAX_COUNT)
    return fail(IMQ_EUNSUPPORTED, "too many groups, beams or continuations");
  if (vocab > (1 << 24)) return fail(IMQ_EUNSUPPORTED, "the vocabulary is too large");
  return IMQ_OK;
}

// How the rows are cut: about 2048 wavefronts over all of them, two for each of the card's SIMDs, each of whole
// blocks of 64 values a lane, or of one of 32 or 8 where that is enough.
struct Cut {
  int each, blocks, slices;
};

Cut cut_rows(int64_t rows, int32_t vocab) {
  const int64_t values = ceil_div(vocab, std::max<int64_t>(1, 2048 / rows));  // of a wavefront
  Cut c;
  c.each = values > 64 * 32 ? 64 : values > 64 * 8 ? 32 : 8;
  c.blocks = std::max(1, ceil_div(values, 64 * c.each));
  c.slices = ceil_div(vocab, (int64_t)kThreads * c.each * c.blocks);
  return c;
}

// The parts of the workspace: sums, ranks and maxima of the rows' slices.
size_t lay_out(int64_t rows, int32_t vocab, int32_t count, char* base, Slices* s) {
  const int64_t slices = cut_rows(rows, vocab).slices;
  const size_t sums = rows * slices * 8, ranks = rows * slices * count * 8;
  if (s)
    *s = Slices{reinterpret_cast<double*>(base), reinterpret_cast<uint64_t*>(base + sums),
                reinterpret_cast<float*>(base + sums + ranks), (int32_t)slices};
  return sums + ranks + rows * slices * 4;
}

}  // namespace

extern "C" {

size_t imq_beam_select_workspace(int32_t groups, int32_t beams, int32_t vocab, int32_t count) {
  if (check_sizes(groups, beams, vocab, count) != IMQ_OK) return 0;
  return lay_out((int64_t)groups * beams, vocab, count, nullptr, nullptr);
}

int32_t imq_beam_select(const void* logits, int64_t ld, int32_t dtype, const float* scores, const int32_t* finished,
                        int32_t eos, int32_t groups, int32_t beams, int32_t vocab, int32_t count, float* out_scores,
                        int32_t* out_parents, int32_t* out_tokens, int32_t* out_finished, void* workspace,
                        size_t workspace_bytes, void* stream) {
  int32_t code = check_sizes(groups, beams, vocab, count);
  if (code != IMQ_OK) return code;
  if (dtype != IMQ_F32 && dtype != IMQ_BF16) return fail(IMQ_EINVAL, "the logits must be fp32 or bf16");
  if (ld < vocab) return fail(IMQ_EINVAL, "ld must be >= vocab");
  if (finished && (eos < 0 || eos >= vocab)) return fail(IMQ_EINVAL, "eos must be a token where beams may be finished");
  if (!logits || !scores || !out_scores || !out_parents || !out_tokens || !out_finished)
    return fail(IMQ_EINVAL, "null pointer");
  if (!aligned(logits, dtype == IMQ_F32 ? 4 : 2)) return fail(IMQ_EINVAL, "the logits are misaligned");
  const int64_t rows = (int64_t)groups * beams;
  if (rows > 65535) return fail(IMQ_EUNSUPPORTED, "too many beams in all");
  if (!workspace || !aligned(workspace, 16) || workspace_bytes < lay_out(rows, vocab, count, nullptr, nullptr))
    return fail(IMQ_EINVAL, "the workspace is too small or not 16-byte aligned");
  if (!current_device(&code)) return code;
  hipStream_t st = static_cast<hipStream_t>(stream);
  Slices s;
  lay_out(rows, vocab, count, static_cast<char*>(workspace), &s);
  const Cut cut = cut_rows(rows, vocab);
  const auto slice = dtype == IMQ_F32 ? (cut.each == 64   ? select_slice_kernel<false, 64>
                                         : cut.each == 32 ? select_slice_kernel<false, 32>
                                                          : select_slice_kernel<false, 8>)
                                      : (cut.each == 64   ? select_slice_kernel<true, 64>
                                         : cut.each == 32 ? select_slice_kernel<true, 32>
                                                          : select_slice_kernel<true, 8>);
  hipLaunchKernelGGL(slice, dim3(s.slices, (uint32_t)rows), dim3(kThreads), 0, st, logits, ld, vocab, count, finished,
                     cut.blocks, s);
  const SelectArgs a{scores, finished, eos, beams, count, out_scores, out_parents, out_tokens, out_finished};
  hipLaunchKernelGGL(select_merge_kernel, dim3(groups), dim3(kMergeThreads), 0, st, s, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(IMQ_ELAUNCH, std::string("beam selection launch failed: ") + hipGetErrorString(e));
  return ok();
}

}  // extern "C"
