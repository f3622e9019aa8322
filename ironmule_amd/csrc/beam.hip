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

constexpr int kThreads = 256;
constexpr int kEach = 16;                    // values of a thread
constexpr int kSlice = kThreads * kEach;     // values of a workgroup
constexpr float kLog2e = 1.44269504088896340736f;

// A row's slice as select_slice_kernel leaves it: the largest value, the sum of exp(x - largest), and
// the `count` best (value, token), the largest value first, equal ones by token; token -1 where there
// are fewer.
struct Slices {
  float* most;
  double* sum;
  float* value;
  int32_t* token;
  int32_t slices;
};

// (value, token) as one number that orders values descending and equal ones by token: the value's
// bits made monotone above the token's complement.  Never 0.
__device__ __forceinline__ uint64_t rank_of(float x, int token) {
  uint32_t u = __float_as_uint(x + 0.0f);  // (-0 as 0)
  u = (u & 0x80000000u) ? ~u : u | 0x80000000u;
  return ((uint64_t)u << 32) | (uint32_t)~token;
}
__device__ __forceinline__ float value_of(uint64_t rank) {
  const uint32_t u = (uint32_t)(rank >> 32);
  return __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u);
}

__device__ __forceinline__ uint64_t wave_most(uint64_t v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    const uint64_t o = __shfl_xor(v, d);
    v = o > v ? o : v;
  }
  return v;
}

template <bool BF16>
__global__ __launch_bounds__(kThreads) void select_slice_kernel(const void* __restrict__ logits, int64_t ld, int vocab,
                                                                int count, Slices s) {
  __shared__ uint64_t best[kThreads / 64];
  __shared__ float tops[kThreads / 64];
  __shared__ double sums[kThreads / 64];
  const int row = blockIdx.y, tid = threadIdx.x, wave = tid >> 6;
  float x[kEach];
  float most = -INFINITY;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int v = blockIdx.x * kSlice + i * kThreads + tid;
    x[i] = -INFINITY;
    if (v < vocab)
      x[i] = BF16 ? bf16_bits_to_f32(static_cast<const uint16_t*>(logits)[row * ld + v])
                  : static_cast<const float*>(logits)[row * ld + v];
    most = fmaxf(most, x[i]);
  }
  most = wave_max(most);
  if ((tid & 63) == 0) tops[wave] = most;
  __syncthreads();
  most = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  const float base = most == -INFINITY ? 0.0f : most;
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) sum += (double)exp2f((x[i] - base) * kLog2e);  // (a NaN stays one)
#pragma unroll
  for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
  if ((tid & 63) == 0) sums[wave] = sum;
  __syncthreads();
  const int64_t at = (int64_t)row * s.slices + blockIdx.x;
  if (tid == 0) {
    s.most[at] = most;
    s.sum[at] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
  }
  uint64_t below = ~0ull;  // ranks from here on are taken
  for (int c = 0; c < count; ++c) {
    uint64_t mine = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const uint64_t r = rank_of(x[i], blockIdx.x * kSlice + i * kThreads + tid);
      if (x[i] > -INFINITY && r < below && r > mine) mine = r;
    }
    mine = wave_most(mine);
    if ((tid & 63) == 0) best[wave] = mine;
    __syncthreads();
    uint64_t all = best[0];
#pragma unroll
    for (int w = 1; w < kThreads / 64; ++w) all = best[w] > all ? best[w] : all;
    if (tid == 0) {
      s.value[at * count + c] = all ? value_of(all) : -INFINITY;
      s.token[at * count + c] = all ? (int32_t)~(uint32_t)all : -1;
    }
    below = all;
    __syncthreads();
  }
}

struct SelectArgs {
  const float* scores;
  const int32_t* finished;
  int32_t eos, beams, count;
  float* out_scores;
  int32_t *out_parents, *out_tokens, *out_finished;
};

// A workgroup per group: the beams' log sums, then the best of the slices' candidates one after
// another.
__global__ __launch_bounds__(kThreads) void select_merge_kernel(Slices s, SelectArgs a) {
  __shared__ double shift[IMQ_BEAM_MAX_BEAMS];  // score - log sum, or -inf: the beam offers nothing
  __shared__ double keys[kThreads / 64];
  __shared__ int64_t places[kThreads / 64];
  const int group = blockIdx.x, tid = threadIdx.x;
  for (int b = tid >> 6; b < a.beams; b += kThreads / 64) {
    const int row = group * a.beams + b, lane = tid & 63;
    float most = -INFINITY;
    for (int i = lane; i < s.slices; i += 64) most = fmaxf(most, s.most[(int64_t)row * s.slices + i]);
    most = wave_max(most);
    const float base = most == -INFINITY ? 0.0f : most;
    double sum = 0.0;
    for (int i = lane; i < s.slices; i += 64) {
      const float m = s.most[(int64_t)row * s.slices + i];
      const double z = s.sum[(int64_t)row * s.slices + i];
      sum += m == -INFINITY && z == 0.0 ? 0.0 : z * exp((double)m - base);
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    if (lane == 0) {
      const double v = (double)a.scores[row] - ((double)base + log(sum));
      shift[b] = sum > 0.0 && isfinite(v) ? v : -INFINITY;
    }
  }
  __syncthreads();
  const int per_row = s.slices * a.count, all = a.beams * per_row;
  double below = INFINITY;
  int64_t past = -1;  // of equal keys, places up to here are taken
  for (int c = 0; c < a.count; ++c) {
    double key = -INFINITY;
    int64_t place = INT64_MAX;  // beam << 32 | token
    auto offer = [&](double k, int64_t p) {
      if (!(k < below || (k == below && p > past))) return;
      if (k > key || (k == key && p < place)) key = k, place = p;
    };
    for (int i = tid; i < all; i += kThreads) {
      const int b = i / per_row, row = group * a.beams + b;
      if (a.finished && a.finished[row]) continue;
      const int token = s.token[(int64_t)row * per_row + i % per_row];
      if (token < 0 || shift[b] == -INFINITY) continue;
      offer(shift[b] + (double)s.value[(int64_t)row * per_row + i % per_row], ((int64_t)b << 32) | token);
    }
    if (a.finished && tid < a.beams && a.finished[group * a.beams + tid]) {
      const float score = a.scores[group * a.beams + tid];
      if (isfinite(score)) offer((double)score, ((int64_t)tid << 32) | a.eos);
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) {
      const double k = __shfl_xor(key, d);
      const int64_t p = __shfl_xor(place, d);
      if (k > key || (k == key && p < place)) key = k, place = p;
    }
    if ((tid & 63) == 0) keys[tid >> 6] = key, places[tid >> 6] = place;
    __syncthreads();
    key = keys[0];
    place = places[0];
#pragma unroll
    for (int w = 1; w < kThreads / 64; ++w)
      if (keys[w] > key || (keys[w] == key && places[w] < place)) key = keys[w], place = places[w];
    below = key;
    past = place;
    if (tid == 0) {
      const int at = group * a.count + c;
      const bool some = key > -INFINITY;
      const int row = group * a.beams + (int)(place >> 32), token = (int)(uint32_t)place;
      a.out_scores[at] = some ? (float)key : -INFINITY;
      a.out_parents[at] = some ? row : -1;
      a.out_tokens[at] = some ? token : -1;
      a.out_finished[at] = some && (token == a.eos || (a.finished && a.finished[row])) ? 1 : 0;
    }
    __syncthreads();
  }
}

int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }
size_t round_up(size_t v, size_t a) { return (v + a - 1) / a * a; }

int32_t check_sizes(int32_t groups, int32_t beams, int32_t vocab, int32_t count) {
  if (groups < 1 || beams < 1 || vocab < 1 || count < 1) return fail(IMQ_EINVAL, "groups, beams, vocab and count must be >= 1");
  if (groups > IMQ_BEAM_MAX_GROUPS || beams > IMQ_BEAM_MAX_BEAMS || count > IMQ_BEAM_MAX_COUNT)
    return fail(IMQ_EUNSUPPORTED, "too many groups, beams or continuations");
  if (vocab > (1 << 24)) return fail(IMQ_EUNSUPPORTED, "the vocabulary is too large");
  return IMQ_OK;
}

// The parts of the workspace: sums, maxima, values, tokens of the rows' slices.
size_t lay_out(int64_t rows, int32_t vocab, int32_t count, char* base, Slices* s) {
  const int64_t slices = ceil_div(vocab, kSlice);
  const size_t sums = round_up(rows * slices * 8, 16), tops = round_up(rows * slices * 4, 16);
  const size_t list = round_up(rows * slices * count * 4, 16);
  if (s)
    *s = Slices{reinterpret_cast<float*>(base + sums), reinterpret_cast<double*>(base),
                reinterpret_cast<float*>(base + sums + tops), reinterpret_cast<int32_t*>(base + sums + tops + list),
                (int32_t)slices};
  return sums + tops + 2 * list;
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
  const auto slice = dtype == IMQ_F32 ? select_slice_kernel<false> : select_slice_kernel<true>;
  hipLaunchKernelGGL(slice, dim3(s.slices, (uint32_t)rows), dim3(kThreads), 0, st, logits, ld, vocab, count, s);
  const SelectArgs a{scores, finished, eos, beams, count, out_scores, out_parents, out_tokens, out_finished};
  hipLaunchKernelGGL(select_merge_kernel, dim3(groups), dim3(kThreads), 0, st, s, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(IMQ_ELAUNCH, std::string("beam selection launch failed: ") + hipGetErrorString(e));
  return ok();
}

}  // extern "C"
