// MI355X (gfx950) kernels of the paged KV cache and their C ABI (include/ironmule_paged.h): pages
// shared out to requests, their reordering, the norm and rotary embedding of new tokens into pages,
// and attention over pages.

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include <algorithm>
#include <string>

#include "../../include/ironmule_paged.h"
#include "common.h"
#include "runtime.h"

namespace {

using namespace imq_dev;

using imq_rt::aligned;
using imq_rt::current_device;
using imq_rt::DeviceInfo;
using imq_rt::fail;
using imq_rt::ok;

constexpr int kThreads = 256;

__device__ __forceinline__ int clamp_int(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }

// ------------------------------------------------------------ pages for new tokens
//
// One workgroup shares out the pages, so that a page's number depends only on the request's place:
// the k-th page asked for (requests in order, a request's columns in order) is the k-th lowest page
// with no references.
//   1. A thread per request: its columns to write, its first page if others hold it too.
//   2. A thread per column to write, 1024 at a time: whether it needs a page; a scan over the threads
//      gives its rank, left in the table as -2 - rank.
//   3. The free pages, kWindow at a time in LDS, by a scan over the references (which ends where enough
//      are found); then a thread per column again: rank -> page, or -1 again for a refused request.
// Requests are taken or refused between the two by the sums of what was asked for.
constexpr int kReserveThreads = 1024;
constexpr int kWindow = 8192;  // free pages listed at a time
constexpr int kMaxRequests = IMQ_PAGED_MAX_REQUESTS;

struct ReserveArgs {
  int32_t* tables;
  const int32_t* lengths;
  int32_t* refs;
  const int32_t* counts;
  int32_t *starts, *ends, *status, *copies;
  int32_t requests, columns, pages, shift, rows;
};

__device__ __forceinline__ int wave_scan(int v) {  // inclusive
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int u = __shfl_up(v, d);
    if ((int)(threadIdx.x & 63) >= d) v += u;
  }
  return v;
}

// Inclusive scan over the workgroup's WAVES wavefronts; *total gets the sum.  `part`: WAVES ints of
// LDS, free again when the call returns.
template <int WAVES>
__device__ __forceinline__ int group_scan(int v, int* part, int* total) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  v = wave_scan(v);
  if (lane == 63) part[wave] = v;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    const int p = part[w];
    before += w < wave ? p : 0;
    all += p;
  }
  __syncthreads();
  *total = all;
  return v + before;
}

__global__ __launch_bounds__(kReserveThreads) void reserve_kernel(ReserveArgs a) {
  __shared__ int part[kReserveThreads / 64];
  __shared__ int list[kWindow];
  __shared__ int last_item[kMaxRequests];   // columns to write, up to and with this request
  __shared__ int first_col[kMaxRequests];
  __shared__ int old_page[kMaxRequests];    // the shared page this request leaves, -1 none
  __shared__ int new_page[kMaxRequests];
  __shared__ int before_wants[kMaxRequests], after_wants[kMaxRequests];
  __shared__ int bad_table[kMaxRequests], refused[kMaxRequests];
  const int tid = threadIdx.x;
  const bool mine = tid < a.requests;
  const int waves = kReserveThreads / 64;

  // 1. a thread per request
  int len = 0, count = 0, items = 0, old = -1;
  bool malformed = false;
  if (mine) {
    len = a.lengths[tid];
    count = a.counts[tid];
    malformed = len < 0 || count < 0 || (int64_t)len + count > ((int64_t)a.columns << a.shift);
    if (malformed) count = 0;
    const int first = malformed ? 0 : len >> a.shift;
    if (count) {
      items = ((len + count - 1) >> a.shift) - first + 1;
      const int cur = a.tables[(int64_t)tid * a.columns + first];
      if (cur >= 0 && cur < a.pages && a.refs[cur] > 1) old = cur;
    }
    first_col[tid] = first;
    old_page[tid] = old;
    new_page[tid] = -1;
    before_wants[tid] = after_wants[tid] = 0;
    bad_table[tid] = 0;
  }
  int all_items, all_rows;
  const int upto = group_scan<waves>(items, part, &all_items);
  if (mine) last_item[tid] = upto;
  // rows asked for: more than there are count as one more, which keeps the sums in 32 bits
  const int rows_upto = group_scan<waves>(count < a.rows ? count : a.rows + (count > a.rows), part, &all_rows);
  __syncthreads();

  auto request_of = [&](int item) {  // the first request whose last column lies past `item`
    int lo = 0, hi = a.requests - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (last_item[mid] > item) hi = mid; else lo = mid + 1;
    }
    return lo;
  };

  // 2. a thread per column to write
  int wanted = 0;
  for (int base = 0; base < all_items; base += kReserveThreads) {
    const int item = base + tid;
    int r = 0, place = 0, need = 0;
    int32_t* entry = nullptr;
    if (item < all_items) {
      r = request_of(item);
      place = item - (r ? last_item[r - 1] : 0);
      entry = a.tables + (int64_t)r * a.columns + first_col[r] + place;
      const int cur = *entry;
      const bool held = cur >= 0 && cur < a.pages;
      need = !held || (place == 0 && old_page[r] >= 0);
      if (held && place && a.refs[cur] > 1) bad_table[r] = 1;
    }
    int sum;
    const int rank = wanted + group_scan<waves>(need, part, &sum);  // inclusive
    if (entry) {
      if (need) *entry = -2 - (rank - 1);
      if (place == 0) before_wants[r] = rank - need;
      if (item + 1 == last_item[r]) after_wants[r] = rank;
    }
    wanted += sum;
  }

  // 3. the free pages
  int cursor = 0;  // pages below it are listed already, or in use
  auto fill = [&](int most) {  // lists up to min(most, kWindow) free pages; returns how many
    int have = 0;
    const int want = most < kWindow ? most : kWindow;
    int at = cursor & ~3;
    while (at < a.pages && have < want) {
      const int p = at + 4 * tid;
      int free[4], sum;
      int4 v = make_int4(1, 1, 1, 1);
      if (p + 3 < a.pages) {
        v = *reinterpret_cast<const int4*>(a.refs + p);
      } else {
        if (p < a.pages) v.x = a.refs[p];
        if (p + 1 < a.pages) v.y = a.refs[p + 1];
        if (p + 2 < a.pages) v.z = a.refs[p + 2];
      }
      free[0] = v.x == 0 && p >= cursor;
      free[1] = v.y == 0 && p + 1 >= cursor;
      free[2] = v.z == 0 && p + 2 >= cursor;
      free[3] = v.w == 0 && p + 3 >= cursor;
      const int n = free[0] + free[1] + free[2] + free[3];
      int to = have + group_scan<waves>(n, part, &sum) - n;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (free[e]) {
          if (to < want) list[to] = p + e;
          ++to;
        }
      have += sum;
      at += 4 * kReserveThreads;
    }
    __syncthreads();
    if (have > want) have = want;
    if (have) cursor = list[have - 1] + 1;
    return have;
  };
  int found = 0;
  while (found < wanted) {
    const int n = fill(wanted - found);
    found += n;
    if (n == 0) break;
    if (found < wanted) __syncthreads();  // the list is filled again
  }
  const bool one_window = wanted <= kWindow;

  // taken or refused
  int state = 0;
  if (mine) {
    const bool short_of = after_wants[tid] > before_wants[tid] && after_wants[tid] > found;
    state = malformed || bad_table[tid] ? 2 : short_of ? 1 : count && rows_upto > a.rows ? 3 : 0;
    refused[tid] = state != 0;
    a.status[tid] = state;
    a.ends[tid] = state ? len : len + count;
  }
  int all_taken;
  const int taken = group_scan<waves>(state ? 0 : count, part, &all_taken);
  if (mine) a.starts[tid + 1] = taken;
  if (tid == 0) a.starts[0] = 0;
  __syncthreads();

  // rank -> page
  cursor = 0;
  int window = 0;
  do {
    const int n = one_window ? found : fill(wanted - window);
    for (int item = tid; item < all_items; item += kReserveThreads) {
      const int r = request_of(item), place = item - (r ? last_item[r - 1] : 0);
      int32_t* const entry = a.tables + (int64_t)r * a.columns + first_col[r] + place;
      const int rank = -2 - *entry;
      if (rank < 0) continue;
      if (refused[r]) {
        *entry = place == 0 ? old_page[r] : -1;
      } else if (rank >= window && rank < window + n) {
        const int page = list[rank - window];
        *entry = page;
        a.refs[page] = 1;
        if (place == 0) new_page[r] = page;
      }
    }
    window += n;
    if (n == 0) break;
    __syncthreads();
  } while (window < found);
  __syncthreads();
  if (mine) {
    int from = -1, to = -1;
    if (old >= 0 && state == 0) {
      atomicSub(a.refs + old, 1);
      if (len & ((1 << a.shift) - 1)) from = old, to = new_page[tid];
    }
    a.copies[2 * tid] = from;
    a.copies[2 * tid + 1] = to;
  }
}

// The rows' positions and slots, and the copies of shared pages: the first `row_groups` workgroups take
// 256 rows each, the others share the copies out in pieces of 4 KB.
constexpr int kPiece = 4096;
__global__ __launch_bounds__(kThreads) void rows_kernel(const int32_t* __restrict__ tables,
                                                        const int32_t* __restrict__ lengths,
                                                        const int32_t* __restrict__ starts,
                                                        const int32_t* __restrict__ copies, int32_t* __restrict__ positions,
                                                        int32_t* __restrict__ slots, char* __restrict__ pool, int requests,
                                                        int columns, int pages, int shift, int rows, int row_groups,
                                                        int planes, int64_t page_bytes) {
  __shared__ int table[2 * kMaxRequests + 1];
  __shared__ int part[kThreads / 64];
  const int tid = threadIdx.x;
  if ((int)blockIdx.x < row_groups) {
    for (int i = tid; i <= requests; i += kThreads) table[i] = starts[i];
    __syncthreads();
    const int row = blockIdx.x * kThreads + tid;
    if (row >= rows) return;
    int position = -1, slot = -1;
    if (row < table[requests]) {
      int lo = 0, hi = requests - 1;  // the last request that starts at or before the row
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (table[mid] <= row) lo = mid; else hi = mid - 1;
      }
      position = lengths[lo] + row - table[lo];
      slot = (tables[(int64_t)lo * columns + (position >> shift)] << shift) | (position & ((1 << shift) - 1));
    }
    positions[row] = position;
    slots[row] = slot;
    return;
  }
  // the requests that copy, in order
  int copied = 0;
  for (int base = 0; base < requests; base += kThreads) {
    const int r = base + tid;
    const int from = r < requests ? copies[2 * r] : -1, to = r < requests ? copies[2 * r + 1] : -1;
    const int some = from >= 0;
    int sum;
    const int at = copied + group_scan<kThreads / 64>(some, part, &sum) - 1;
    if (some) table[2 * at] = from, table[2 * at + 1] = to;
    copied += sum;
  }
  __syncthreads();
  const int pieces = (int)((page_bytes + kPiece - 1) / kPiece);
  const int64_t all = (int64_t)copied * planes * pieces;
  for (int64_t i = blockIdx.x - row_groups; i < all; i += gridDim.x - row_groups) {
    const int piece = (int)(i % pieces), which = (int)(i / pieces % copied);
    const int64_t plane = i / pieces / copied, offset = (int64_t)piece * kPiece + 16 * tid;
    if (offset >= page_bytes) continue;
    *reinterpret_cast<uint4*>(pool + (plane * pages + table[2 * which + 1]) * page_bytes + offset) =
        *reinterpret_cast<const uint4*>(pool + (plane * pages + table[2 * which]) * page_bytes + offset);
  }
}

// ------------------------------------------------------------ reordering of requests
//
// A workgroup takes some columns of every request: it reads them all into LDS, then writes each
// request's from its parent's and counts the pages that come and go.  The counts are integers, so
// the order of the additions does not matter.  The lengths follow in a launch of their own: every
// workgroup reads the parents' old ones.
constexpr int kReorderEntries = 8192;  // table entries of a workgroup, 32 KB of LDS

__global__ __launch_bounds__(kThreads) void reorder_kernel(int32_t* __restrict__ tables,
                                                           const int32_t* __restrict__ lengths,
                                                           int32_t* __restrict__ refs,
                                                           const int32_t* __restrict__ parents, int requests, int columns,
                                                           int pages, int shift, int width) {
  __shared__ int old[kReorderEntries];
  const int c0 = blockIdx.x * width, wide = min(width, columns - c0), entries = requests * wide;
  for (int e = threadIdx.x; e < entries; e += kThreads)
    old[e] = tables[(int64_t)(e / wide) * columns + c0 + e % wide];
  __syncthreads();
  for (int e = threadIdx.x; e < entries; e += kThreads) {
    const int r = e / wide, c = e % wide, p = parents[r];
    if (p == r || p < -1 || p >= requests) continue;
    const int before = old[e];
    int after = -1;
    if (p >= 0 && (int64_t)lengths[p] > ((int64_t)(c0 + c) << shift)) after = old[p * wide + c];
    if (after < 0 || after >= pages) after = -1;
    if (before == after) continue;
    if (before >= 0 && before < pages) atomicSub(refs + before, 1);
    if (after >= 0) atomicAdd(refs + after, 1);
    tables[(int64_t)r * columns + c0 + c] = after;
  }
}

__global__ __launch_bounds__(kMaxRequests) void reorder_lengths_kernel(int32_t* __restrict__ lengths,
                                                                       const int32_t* __restrict__ parents, int requests) {
  const int r = threadIdx.x;
  int length = 0;
  bool change = false;
  if (r < requests) {
    const int p = parents[r];
    change = p != r && p >= -1 && p < requests;
    if (change && p >= 0) length = lengths[p];
  }
  __syncthreads();
  if (change) lengths[r] = length;
}

// ------------------------------------------------------------ norm, rotary, rows into pages
//
// A workgroup per row, a wavefront per head at a time; lane l holds dimensions l, l + 64, .. of the
// head, so that the pairs (d, d + head_dim / 2) that turn together lie in one lane.
template <int D>
__global__ __launch_bounds__(kThreads) void write_kernel(const uint16_t* __restrict__ q, int64_t ldq,
                                                         const uint16_t* __restrict__ k, int64_t ldk,
                                                         const uint16_t* __restrict__ v, int64_t ldv,
                                                         const uint16_t* __restrict__ q_norm,
                                                         const uint16_t* __restrict__ k_norm,
                                                         const int32_t* __restrict__ positions,
                                                         const int32_t* __restrict__ slots, uint16_t* __restrict__ q_out,
                                                         int64_t ldo, uint16_t* __restrict__ k_pages,
                                                         uint16_t* __restrict__ v_pages, int Hq, int Hkv, int shift,
                                                         int64_t tokens, double log2_theta, float eps) {
  constexpr int H = D / 2, N = D / 64;
  __shared__ float turn[2][H];
  const int row = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int slot = slots[row];
  if (slot < 0 || slot >= tokens) return;
  if (threadIdx.x < H) {
    double sn, cs;
    sincos((double)positions[row] * exp2(-(double)threadIdx.x * (log2_theta / H)), &sn, &cs);
    turn[0][threadIdx.x] = (float)sn;
    turn[1][threadIdx.x] = (float)cs;
  }
  __syncthreads();
  const int page = slot >> shift, offset = slot & ((1 << shift) - 1);
  for (int hh = wave; hh < Hq + 2 * Hkv; hh += kThreads / 64) {
    const bool is_q = hh < Hq, is_v = hh >= Hq + Hkv;
    const int head = is_q ? hh : is_v ? hh - Hq - Hkv : hh - Hq;
    const uint16_t* const src = is_q ? q + row * ldq + head * D : is_v ? v + row * ldv + head * D : k + row * ldk + head * D;
    uint16_t* const dst = is_q ? q_out + row * ldo + head * D
                               : (is_v ? v_pages : k_pages) + ((((int64_t)page * Hkv + head) << shift) + offset) * D;
    if (is_v) {
#pragma unroll
      for (int i = 0; i < N; ++i) dst[lane + 64 * i] = src[lane + 64 * i];
      continue;
    }
    const uint16_t* const weight = is_q ? q_norm : k_norm;
    float x[N], ss = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      x[i] = bf16_bits_to_f32(src[lane + 64 * i]);
      ss = fmaf(x[i], x[i], ss);
    }
    const float inv = 1.0f / sqrtf(wave_sum(ss) / (float)D + eps);
#pragma unroll
    for (int i = 0; i < N; ++i)
      x[i] = bf16_bits_to_f32(f32_to_bf16_bits(x[i] * inv * bf16_bits_to_f32(weight[lane + 64 * i])));
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const float lo = x[i], hi = x[i + N / 2], s = turn[0][lane + 64 * i], c = turn[1][lane + 64 * i];
      dst[lane + 64 * i] = f32_to_bf16_bits(lo * c - hi * s);
      dst[lane + 64 * i + H] = f32_to_bf16_bits(lo * s + hi * c);
    }
  }
}

// ------------------------------------------------------------ attention over pages
//
// The rows of a request and the query heads of one KV head are taken together as G n queries (row i,
// head g of the group: query i G + g).  A wavefront takes a tile of 16 queries of one KV head and
// walks the keys 32 at a time.  Scores are K Q^T on v_mfma_f32_16x16x32_bf16, so that a lane holds
// keys of one query: P^T is then the B operand of V^T P^T without leaving its lane (keys 4 g .. of two
// 16-key tiles).  K goes from its page to the A operand directly; V goes through LDS by rows and is
// read transposed.
typedef __bf16 bf16x2v __attribute__((ext_vector_type(2)));

struct AttendArgs {
  const uint16_t *q, *k_pages, *v_pages;
  const int32_t *tables, *starts, *ends;
  uint16_t* out;
  int64_t ldq, ldo;
  int32_t rows, requests, columns, pages, shift, Hq, Hkv, group, window;
  float scale_log2;  // scale * log2(e)
};

// The request whose tile `tile` is (tiles of `width` queries, requests in order), the tile's place in
// it, its first row and its number of rows; false past the last tile.  The whole wavefront agrees.
__device__ __forceinline__ bool find_tile(const AttendArgs& a, int tile, int width, int* request, int* place, int* first,
                                          int* count) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int base = 0; base < a.requests; base += 64) {
    const int r = base + lane;
    int lo = 0, n = 0;
    if (r < a.requests) {
      lo = clamp_int(a.starts[r], 0, a.rows);
      n = clamp_int(a.starts[r + 1], lo, a.rows) - lo;
    }
    const int tiles = (n * a.group + width - 1) / width;
    const int upto = before + wave_scan(tiles);
    const uint64_t past = __ballot(upto > tile);
    if (past) {
      const int at = __ffsll((unsigned long long)past) - 1;
      *request = base + at;
      // (clamped: starts that do not ascend must not lead outside the request)
      *place = clamp_int(tile - __builtin_amdgcn_readlane(upto - tiles, at), 0, __builtin_amdgcn_readlane(tiles, at) - 1);
      *first = __builtin_amdgcn_readlane(lo, at);
      *count = __builtin_amdgcn_readlane(n, at);
      return true;
    }
    before = __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {  // v_cvt_pk_bf16_f32
  bf16x2v r;
  r.x = (__bf16)lo;
  r.y = (__bf16)hi;
  return __builtin_bit_cast(uint32_t, r);
}

typedef __attribute__((address_space(3))) s16x4_t* lds_s16x4;

// The bf16 pair `w` with infinities and NaNs as zeros; *odd gets a bit set if there were any.
__device__ __forceinline__ uint32_t finite_pair(uint32_t w, uint32_t* odd) {
  const bool lo = (w & 0x7f80u) == 0x7f80u, hi = (w & 0x7f800000u) == 0x7f800000u;
  *odd |= lo || hi;
  return (lo ? 0u : w & 0xffffu) | (hi ? 0u : w & 0xffff0000u);
}

template <int D>
__global__ __launch_bounds__(64) void attend_rows_kernel(AttendArgs a) {
  constexpr int T = D / 32, P = D / 8, C = D / 16;  // k-steps of a score, 16-byte pieces of a row, 16-dim tiles
  __shared__ __attribute__((aligned(16))) char vl[32 * 2 * D];
  const int head = blockIdx.x % a.Hkv, lane = threadIdx.x, n = lane & 15, g = lane >> 4;
  int request, place, first, count;
  if (!find_tile(a, blockIdx.x / a.Hkv, 16, &request, &place, &first, &count)) return;
  const int end = clamp_int(a.ends[request], 0, a.columns << a.shift);
  const int query = 16 * place + n, row = query / a.group;
  const bool live = row < count;
  const int position = end - count + row;
  const int tile_first = end - count + (16 * place) / a.group;
  const int tile_last = min(end - 1, end - count + (16 * place + 15) / a.group);
  const int low = a.window ? max(0, tile_first - a.window + 1) : 0;
  const int64_t q_head = (int64_t)head * a.group + query % a.group;

  bf16x8_t qf[T];
#pragma unroll
  for (int t = 0; t < T; ++t) {
    u32x4_t w = {0u, 0u, 0u, 0u};
    if (live) w = *reinterpret_cast<const u32x4_t*>(a.q + (first + row) * a.ldq + q_head * D + 32 * t + 8 * g);
    qf[t] = __builtin_bit_cast(bf16x8_t, w);
  }
  f32x4_t o[C];
#pragma unroll
  for (int c = 0; c < C; ++c) o[c] = f32x4_t{};
  float top = -INFINITY, sum = 0.0f;
  const int32_t* const table = a.tables + (int64_t)request * a.columns;
  const int mask = (1 << a.shift) - 1;

  for (int k0 = low & ~31; k0 <= tile_last; k0 += 32) {
    // the two 16-key groups' pages (a page holds a multiple of 16 tokens)
    int page[2];
    bool held[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int key = k0 + 16 * b;
      page[b] = key <= tile_last ? table[key >> a.shift] : -1;
      held[b] = page[b] >= 0 && page[b] < a.pages;
      page[b] = held[b] ? page[b] : 0;
    }
    f32x4_t s[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int64_t at = ((((int64_t)page[b] * a.Hkv + head) << a.shift) + ((k0 + 16 * b) & mask) + n) * D;
      s[b] = f32x4_t{};
#pragma unroll
      for (int t = 0; t < T; ++t) {
        const u32x4_t w = *reinterpret_cast<const u32x4_t*>(a.k_pages + at + 32 * t + 8 * g);
        s[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, w), qf[t], s[b], 0, 0, 0);
      }
    }
    // V to LDS: rows that no query sees are zeros, whatever their page holds.  Where some queries see a
    // key and others do not, a probability of zero must not meet an infinity or a NaN: such values
    // are zeros in LDS, and are added below for the queries that see them.
    const bool edge = k0 + 31 > tile_first || (a.window && k0 <= tile_last - a.window);
    uint32_t odd = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 32 * P / 64; ++i) {
      const int p = lane + 64 * i, r = p / P, b = r >> 4, key = k0 + r;
      u32x4_t w = {0u, 0u, 0u, 0u};
      if (held[b] && key >= low && key <= tile_last)
        w = *reinterpret_cast<const u32x4_t*>(a.v_pages + ((((int64_t)page[b] * a.Hkv + head) << a.shift) + (key & mask)) * D + 8 * (p % P));
      if (edge) {
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = finite_pair(w[e], &odd);
      }
      *reinterpret_cast<u32x4_t*>(vl + r * 2 * D + 16 * (p % P)) = w;
    }
    __syncthreads();
    float most = top;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = k0 + 16 * b + 4 * g + e;
        const bool seen = live && held[b] && key <= position && (!a.window || key > position - a.window);
        s[b][e] = seen ? s[b][e] * a.scale_log2 : -INFINITY;
        most = fmaxf(most, s[b][e]);  // (a NaN score comes back through its exponential)
      }
    most = max_xor32(max_xor16(most));
    const float base = most == -INFINITY ? 0.0f : most;
    const float keep = exp2f(top - base);
    top = most;
    sum *= keep;
    float p[2][4];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        p[b][e] = exp2f(s[b][e] - base);
        sum += p[b][e];
      }
    const u32x4_t pw = {pack_bf16(p[0][0], p[0][1]), pack_bf16(p[0][2], p[0][3]), pack_bf16(p[1][0], p[1][1]),
                        pack_bf16(p[1][2], p[1][3])};
    const bf16x8_t pf = __builtin_bit_cast(bf16x8_t, pw);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      o[c] *= keep;
      // lane i of each 16 reads 8 bytes of row i / 4; the transposed read gives it the four rows' value
      // of dimension i
      char* const from = vl + (4 * g + (n >> 2)) * 2 * D + 32 * c + 8 * (n & 3);
      const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)from);
      const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(from + 16 * 2 * D));
      const bf16x8_t vf = __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
      o[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf, o[c], 0, 0, 0);
    }
    if (__any(odd)) {
      for (int r = 0; r < 32; ++r) {
        const int b = r >> 4, key = k0 + r;
        if (!held[b] || key < low || key > tile_last) continue;
        const float mine = (r & 16) ? ((r & 2) ? ((r & 1) ? p[1][3] : p[1][2]) : ((r & 1) ? p[1][1] : p[1][0]))
                                    : ((r & 2) ? ((r & 1) ? p[0][3] : p[0][2]) : ((r & 1) ? p[0][1] : p[0][0]));
        const float pr = __shfl(mine, n + 16 * ((r >> 2) & 3));
        const bool seen = live && key <= position && (!a.window || key > position - a.window);
        const uint16_t* const from = a.v_pages + ((((int64_t)page[b] * a.Hkv + head) << a.shift) + (key & mask)) * D;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t v = from[16 * c + 4 * g + e];
            if (seen && (v & 0x7f80u) == 0x7f80u) o[c][e] += pr * bf16_bits_to_f32(v);
          }
      }
    }
  }
  sum = add_xor32(add_xor16(sum));
  if (!live) return;
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  uint16_t* const to = a.out + (first + row) * a.ldo + q_head * D;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const u32x2_t four = {pack_bf16(o[c][0] * inv, o[c][1] * inv), pack_bf16(o[c][2] * inv, o[c][3] * inv)};
    *reinterpret_cast<u32x2_t*>(to + 16 * c + 4 * g) = four;
  }
}

// ------------------------------------------------------------ host side

int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

int32_t launched(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(IMQ_ELAUNCH, std::string(what) + " launch failed: " + hipGetErrorString(e));
  return ok();
}

int32_t check_page_size(int32_t page_size) {
  if (page_size < IMQ_PAGED_MIN_PAGE || page_size > IMQ_PAGED_MAX_PAGE || (page_size & (page_size - 1)))
    return fail(IMQ_EUNSUPPORTED, "a page holds a power of two of 16 to 1024 tokens");
  return IMQ_OK;
}

int32_t check_tables(int32_t requests, int32_t columns, int32_t pages, int32_t page_size) {
  const int32_t code = check_page_size(page_size);
  if (code != IMQ_OK) return code;
  if (requests < 1 || columns < 1 || pages < 1) return fail(IMQ_EINVAL, "requests, columns and pages must be >= 1");
  if (requests > IMQ_PAGED_MAX_REQUESTS) return fail(IMQ_EUNSUPPORTED, "too many requests");
  if (columns > IMQ_PAGED_MAX_COLUMNS) return fail(IMQ_EUNSUPPORTED, "too many columns");
  // positions and slots are 32-bit
  if ((int64_t)columns * page_size > (1 << 30) || (int64_t)pages * page_size > INT32_MAX)
    return fail(IMQ_EUNSUPPORTED, "more tokens than positions and slots can number");
  return IMQ_OK;
}

int32_t check_cache(const imq_paged_cache* c) {
  if (!c) return fail(IMQ_EINVAL, "the cache is null");
  const int32_t code = check_tables(c->requests, c->columns, c->pages, c->page_size);
  if (code != IMQ_OK) return code;
  if (!c->tables || !c->lengths || !c->refs) return fail(IMQ_EINVAL, "null pointer");
  if (!aligned(c->tables, 4) || !aligned(c->lengths, 4) || !aligned(c->refs, 16))
    return fail(IMQ_EINVAL, "tables and lengths must be 4-byte aligned, refs 16-byte aligned");
  return IMQ_OK;
}

int32_t check_heads(int32_t rows, int32_t Hq, int32_t Hkv, int32_t head_dim) {
  if (rows < 0 || rows > IMQ_PAGED_MAX_ROWS) return fail(IMQ_EINVAL, "rows out of range");
  if (Hq < 1 || Hkv < 1 || Hq % Hkv) return fail(IMQ_EINVAL, "need Hkv >= 1 dividing Hq");
  if (Hq > IMQ_PAGED_MAX_HEADS) return fail(IMQ_EUNSUPPORTED, "too many heads");
  if (head_dim != 128 && head_dim != 256) return fail(IMQ_EUNSUPPORTED, "the head size must be 128 or 256");
  return IMQ_OK;
}

bool row_stride(int64_t ld, int64_t width) { return ld >= width && ld % 8 == 0; }

}  // namespace

extern "C" {

int32_t imq_paged_reserve(const imq_paged_cache* cache, const int32_t* counts, const imq_paged_chunk* chunk,
                          void* pool, int32_t planes, int64_t page_bytes, void* stream) {
  int32_t code = check_cache(cache);
  if (code != IMQ_OK) return code;
  if (!counts || !chunk) return fail(IMQ_EINVAL, "null pointer");
  if (chunk->rows < 0 || chunk->rows > IMQ_PAGED_MAX_ROWS) return fail(IMQ_EINVAL, "rows out of range");
  if (!chunk->starts || !chunk->ends || !chunk->status || !chunk->copies ||
      (chunk->rows && (!chunk->positions || !chunk->slots)))
    return fail(IMQ_EINVAL, "null pointer");
  if (pool) {
    if (planes < 1) return fail(IMQ_EINVAL, "planes must be >= 1");
    if (page_bytes < 16 || page_bytes % 16 || !aligned(pool, 16))
      return fail(IMQ_EINVAL, "the pool must be 16-byte aligned, its pages multiples of 16 bytes");
  }
  if (!current_device(&code)) return code;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int shift = __builtin_ctz(cache->page_size);
  ReserveArgs a{cache->tables, cache->lengths, cache->refs, counts, chunk->starts, chunk->ends, chunk->status,
                chunk->copies, cache->requests, cache->columns, cache->pages, shift, chunk->rows};
  hipLaunchKernelGGL(reserve_kernel, dim3(1), dim3(kReserveThreads), 0, st, a);
  code = launched("reserve");
  if (code != IMQ_OK) return code;
  const int row_groups = ceil_div(chunk->rows, kThreads);
  int copy_groups = 0;
  if (pool) copy_groups = (int)std::min<int64_t>(1024, cache->requests * (int64_t)planes * ((page_bytes + kPiece - 1) / kPiece));
  if (row_groups + copy_groups == 0) return ok();
  hipLaunchKernelGGL(rows_kernel, dim3(row_groups + copy_groups), dim3(kThreads), 0, st, cache->tables, cache->lengths,
                     chunk->starts, chunk->copies, chunk->positions, chunk->slots, static_cast<char*>(pool),
                     cache->requests, cache->columns, cache->pages, shift, chunk->rows, row_groups, planes, page_bytes);
  return launched("reserve rows");
}

int32_t imq_paged_reorder(const imq_paged_cache* cache, const int32_t* parents, void* stream) {
  int32_t code = check_cache(cache);
  if (code != IMQ_OK) return code;
  if (!parents) return fail(IMQ_EINVAL, "null pointer");
  if (!current_device(&code)) return code;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int width = std::min(cache->columns, std::min(256, kReorderEntries / cache->requests));
  hipLaunchKernelGGL(reorder_kernel, dim3(ceil_div(cache->columns, width)), dim3(kThreads), 0, st, cache->tables,
                     cache->lengths, cache->refs, parents, cache->requests, cache->columns, cache->pages,
                     __builtin_ctz(cache->page_size), width);
  hipLaunchKernelGGL(reorder_lengths_kernel, dim3(1), dim3(kMaxRequests), 0, st, cache->lengths, parents, cache->requests);
  return launched("reorder");
}

int32_t imq_paged_write(const uint16_t* q, int64_t ldq, const uint16_t* k, int64_t ldk, const uint16_t* v,
                        int64_t ldv, const uint16_t* q_norm, const uint16_t* k_norm, const int32_t* positions,
                        const int32_t* slots, uint16_t* q_out, int64_t ldo, uint16_t* k_pages, uint16_t* v_pages,
                        int32_t rows, int32_t Hq, int32_t Hkv, int32_t head_dim, int32_t pages, int32_t page_size,
                        double theta, float eps, void* stream) {
  int32_t code = check_heads(rows, Hq, Hkv, head_dim);
  if (code == IMQ_OK) code = check_page_size(page_size);
  if (code != IMQ_OK) return code;
  if (pages < 1 || (int64_t)pages * page_size > INT32_MAX) return fail(IMQ_EINVAL, "pages out of range");
  if (!(eps >= 0.0f) || !(theta > 1.0)) return fail(IMQ_EINVAL, "eps must be >= 0 and theta > 1");
  const int64_t qd = (int64_t)Hq * head_dim, kd = (int64_t)Hkv * head_dim;
  if (!row_stride(ldq, qd) || !row_stride(ldk, kd) || !row_stride(ldv, kd) || !row_stride(ldo, qd))
    return fail(IMQ_EINVAL, "a row stride must be a multiple of 8 and at least the row's values");
  if (rows == 0) return ok();
  if (!positions || !slots) return fail(IMQ_EINVAL, "null pointer");
  for (const void* p : {(const void*)q, (const void*)k, (const void*)v, (const void*)q_norm, (const void*)k_norm,
                        (const void*)q_out, (const void*)k_pages, (const void*)v_pages})
    if (!p || !aligned(p, 16)) return fail(IMQ_EINVAL, "rows, norm weights and pages must be non-null and 16-byte aligned");
  if (!current_device(&code)) return code;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int shift = __builtin_ctz(page_size);
  const auto kernel = head_dim == 128 ? write_kernel<128> : write_kernel<256>;
  hipLaunchKernelGGL(kernel, dim3(rows), dim3(kThreads), 0, st, q, ldq, k, ldk, v, ldv, q_norm, k_norm, positions, slots,
                     q_out, ldo, k_pages, v_pages, Hq, Hkv, shift, (int64_t)pages << shift, log2(theta), eps);
  return launched("paged write");
}

size_t imq_paged_attention_workspace(int32_t rows, int32_t requests, int32_t Hq, int32_t Hkv, int32_t head_dim,
                                     int32_t max_context, int32_t window) {
  return 0;
}

int32_t imq_paged_attention(const uint16_t* q, int64_t ldq, const uint16_t* k_pages, const uint16_t* v_pages,
                            const int32_t* tables, const int32_t* starts, const int32_t* ends, uint16_t* out,
                            int64_t ldo, int32_t rows, int32_t requests, int32_t columns, int32_t pages,
                            int32_t page_size, int32_t Hq, int32_t Hkv, int32_t head_dim, int32_t max_context,
                            int32_t window, float scale, void* workspace, size_t workspace_bytes, void* stream) {
  int32_t code = check_heads(rows, Hq, Hkv, head_dim);
  if (code == IMQ_OK) code = check_tables(requests, columns, pages, page_size);
  if (code != IMQ_OK) return code;
  if (window < 0) return fail(IMQ_EINVAL, "the window must be >= 0");
  if (max_context < 1) return fail(IMQ_EINVAL, "max_context must be >= 1");
  if (!(scale > 0.0f) || !(scale < INFINITY)) return fail(IMQ_EINVAL, "the scale must be positive and finite");
  const int64_t qd = (int64_t)Hq * head_dim;
  if (!row_stride(ldq, qd) || !row_stride(ldo, qd))
    return fail(IMQ_EINVAL, "a row stride must be a multiple of 8 and at least the row's values");
  if (rows == 0) return ok();
  if (!tables || !starts || !ends) return fail(IMQ_EINVAL, "null pointer");
  for (const void* p : {(const void*)q, (const void*)k_pages, (const void*)v_pages, (const void*)out})
    if (!p || !aligned(p, 16)) return fail(IMQ_EINVAL, "rows and pages must be non-null and 16-byte aligned");
  if (!current_device(&code)) return code;
  const int group = Hq / Hkv;
  AttendArgs a{q, k_pages, v_pages, tables, starts, ends, out, ldq, ldo, rows, requests, columns, pages,
               __builtin_ctz(page_size), Hq, Hkv, group, window, scale * 1.44269504088896340736f};
  // tiles of 16 queries: at most one part-full one for each request with rows
  const int64_t tiles = std::min<int64_t>(rows, requests) + (int64_t)rows * group / 16;
  const auto kernel = head_dim == 128 ? attend_rows_kernel<128> : attend_rows_kernel<256>;
  hipLaunchKernelGGL(kernel, dim3((uint32_t)(tiles * Hkv)), dim3(64), 0, static_cast<hipStream_t>(stream), a);
  return launched("paged attention");
}

}  // extern "C"
