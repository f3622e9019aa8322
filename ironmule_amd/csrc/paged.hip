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
//   2. A thread per COLUMNS columns to write: which need a page; a scan over the threads gives their
//      ranks, left in the table as -2 - rank.
//   3. The free pages, WINDOW at a time in LDS, by a scan over the references (which ends where enough
//      are found); then a thread per COLUMNS columns again: rank -> page, or -1 again for a refused request.
// Requests are taken or refused between the two by the sums of what was asked for.
//
// Bound by its chain of loads and barriers, and in a large cache by the references, which one CU reads
// at about 150 GB/s (512 KB for 131072 pages).  One column and four references a thread at a time are best
// for a step's few columns (eight beams 5.6 us, 9.6 with eight and 16), four and 16 for many prompts' (a
// round of 764 requests 46; 50 with eight and 16, 104 with one and four).  Columns in turn among a wavefront's
// lanes, for neighbouring accesses, took 150: a lane's next column is then many requests on.
constexpr int kReserveThreads = 1024, kReserveWaves = kReserveThreads / 64;
constexpr int kMaxRequests = IMQ_PAGED_MAX_REQUESTS;

struct ReserveArgs {
  int32_t* tables;
  const int32_t* lengths;
  int32_t* refs;
  const int32_t* counts;
  int32_t *starts, *ends, *status, *copies;
  int32_t requests, columns, pages, shift, rows;
};

// Inclusive sum over the wavefront's lanes up to each: within each 16 by shifts, then lane 15 of a row
// into the next one, then lane 31 into the upper half.
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr 1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast 15, into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row_bcast 31, into rows 2 and 3
  return v;
}

// Inclusive sums over a workgroup of WAVES wavefronts, one barrier each: the two halves of `part` take turns,
// and nobody writes one of them again before the barrier of the other.
template <int WAVES>
struct GroupScan {
  int (*part)[WAVES];
  int turn = 0;
  __device__ __forceinline__ int operator()(int v, int* total) {
    const int wave = threadIdx.x >> 6;
    int* const mine = part[turn];
    turn ^= 1;
    v = wave_scan(v);
    if ((threadIdx.x & 63) == 63) mine[wave] = v;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const int p = mine[w];
      before += w < wave ? p : 0;
      all += p;
    }
    *total = all;
    return v + before;
  }
};

template <int COLUMNS, int REFS, int WINDOW>
__global__ __launch_bounds__(kReserveThreads) void reserve_kernel(ReserveArgs a) {
  __shared__ int part[2][kReserveWaves];
  __shared__ int list[WINDOW];
  __shared__ int last_item[kMaxRequests];  // columns to write, up to and with this request
  __shared__ int first_col[kMaxRequests];
  __shared__ int old_page[kMaxRequests];   // the shared page this request leaves, -1 none
  __shared__ int new_page[kMaxRequests];
  __shared__ int before_wants[kMaxRequests], after_wants[kMaxRequests];
  __shared__ int flags[kMaxRequests];      // 1: a shared page past its tokens; 2: refused
  const int tid = threadIdx.x;
  const bool mine = tid < a.requests;
  GroupScan<kReserveWaves> scan{part};
  auto four_refs = [&](int p) {
    int4 v = make_int4(1, 1, 1, 1);
    if (p + 3 < a.pages) {
      v = *reinterpret_cast<const int4*>(a.refs + p);
    } else {
      if (p < a.pages) v.x = a.refs[p];
      if (p + 1 < a.pages) v.y = a.refs[p + 1];
      if (p + 2 < a.pages) v.z = a.refs[p + 2];
    }
    return v;
  };
  auto free_of = [&](int p) {  // which of the REFS pages from p on are free
    int4 v[REFS / 4];
#pragma unroll
    for (int i = 0; i < REFS / 4; ++i) v[i] = four_refs(p + 4 * i);
    uint32_t free = 0;
#pragma unroll
    for (int i = 0; i < REFS / 4; ++i)
      free |= (uint32_t)((v[i].x == 0) | (v[i].y == 0) << 1 | (v[i].z == 0) << 2 | (v[i].w == 0) << 3) << (4 * i);
    return free;
  };
  const uint32_t first_free = free_of(REFS * tid);  // (on its way over the first step's loads)

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
    flags[tid] = 0;
  }
  int all_items;
  const int upto = scan(items, &all_items);
  if (mine) last_item[tid] = upto;
  // rows asked for: more than there are count as one more, which keeps the sums in 32 bits
  int all_rows;
  const int rows_upto = scan(count < a.rows ? count : a.rows + (count > a.rows), &all_rows);

  auto request_of = [&](int item) {  // the first request whose last column lies past the item
    int lo = 0, hi = a.requests - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (last_item[mid] > item) hi = mid; else lo = mid + 1;
    }
    return lo;
  };
  // The columns to write `item` .. item + COLUMNS - 1, the first of request lo: work(j, request, number in it,
  // whether
  // its last, entry).
  auto for_items = [&](int item, int lo, auto work) {
#pragma unroll
    for (int j = 0; j < COLUMNS; ++j) {
      if (item + j >= all_items) break;
      while (last_item[lo] <= item + j) ++lo;
      const int place = item + j - (lo ? last_item[lo - 1] : 0);
      work(j, lo, place, item + j + 1 == last_item[lo], a.tables + (int64_t)lo * a.columns + first_col[lo] + place);
    }
  };

  // 2. the columns that need a page
  int wanted = 0;
  for (int base = 0; base < all_items; base += COLUMNS * kReserveThreads) {
    const int item = base + COLUMNS * tid;
    const int lo = request_of(item);
    int32_t current[COLUMNS], need[COLUMNS] = {}, sum;
    for_items(item, lo, [&](int j, int, int, bool, int32_t* entry) { current[j] = *entry; });
    int n = 0;
    for_items(item, lo, [&](int j, int r, int place, bool, int32_t*) {
      const bool held = current[j] >= 0 && current[j] < a.pages;
      need[j] = !held || (place == 0 && old_page[r] >= 0);
      n += need[j];
      if (held && place && a.refs[current[j]] > 1) flags[r] = 1;
    });
    int rank = wanted + scan(n, &sum) - n;
    for_items(item, lo, [&](int j, int r, int place, bool last, int32_t* entry) {
      if (need[j]) *entry = -2 - rank;
      if (place == 0) before_wants[r] = rank;
      rank += need[j];
      if (last) after_wants[r] = rank;
    });
    wanted += sum;
  }

  // 3. the free pages: lists up to min(most, WINDOW) from `cursor` on; returns how many
  int cursor = 0;
  auto fill = [&](int most) {
    int have = 0;
    const int want = most < WINDOW ? most : WINDOW;
    for (int at = cursor & ~3; at < a.pages && have < want; at += REFS * kReserveThreads) {
      const int p = at + REFS * tid;
      uint32_t free = at == 0 ? first_free : free_of(p);
      if (p < cursor) free &= cursor - p < 32 ? ~0u << (cursor - p) : 0u;
      const int n = __popc(free);
      int sum, to = have + scan(n, &sum) - n;
      for (; free; free &= free - 1, ++to)
        if (to < want) list[to] = p + __builtin_ctz(free);
      have += sum;
    }
    __syncthreads();
    if (have > want) have = want;
    if (have) cursor = list[have - 1] + 1;
    return have;
  };
  const bool one_window = wanted <= WINDOW;
  int found;
  if (one_window) {
    found = wanted ? fill(wanted) : 0;
  } else {
    int n = 0, all;
    for (int p = REFS * tid; p < a.pages; p += REFS * kReserveThreads) n += __popc(free_of(p));
    scan(n, &all);
    found = min(wanted, all);
  }
  __syncthreads();

  // taken or refused
  int state = 0;
  if (mine) {
    const bool short_of = after_wants[tid] > before_wants[tid] && after_wants[tid] > found;
    state = malformed || flags[tid] ? 2 : short_of ? 1 : count && rows_upto > a.rows ? 3 : 0;
    if (state) flags[tid] = 2;
    a.status[tid] = state;
    a.ends[tid] = state ? len : len + count;
  }
  int all_taken;
  const int taken = scan(state ? 0 : count, &all_taken);
  if (mine) a.starts[tid + 1] = taken;
  if (tid == 0) a.starts[0] = 0;

  // rank -> page
  int window = 0, listed = one_window ? found : 0;  // the list holds ranks window .. window + listed - 1
  for (int base = 0; base < all_items; base += COLUMNS * kReserveThreads) {
    const int item = base + COLUMNS * tid;
    const int lo = request_of(item);
    int32_t code[COLUMNS] = {};
    for_items(item, lo, [&](int j, int, int, bool, int32_t* entry) { code[j] = *entry; });
    for (;;) {
      bool later = false;
      for_items(item, lo, [&](int j, int r, int place, bool, int32_t* entry) {
        const int rank = -2 - code[j];
        if (rank < 0) return;
        if (flags[r]) {
          *entry = place == 0 ? old_page[r] : -1;
        } else if (rank >= window + listed) {
          later = true;
          return;
        } else {
          const int page = list[rank - window];
          *entry = page;
          a.refs[page] = 1;
          if (place == 0) new_page[r] = page;
        }
        code[j] = 0;
      });
      if (one_window || !__syncthreads_or(later)) break;
      window += listed;
      listed = fill(found - window);
      if (listed == 0) break;
    }
  }
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
  __shared__ int part[2][kThreads / 64];
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
  GroupScan<kThreads / 64> scan{part};
  int copied = 0;
  for (int base = 0; base < requests; base += kThreads) {
    const int r = base + tid;
    const int from = r < requests ? copies[2 * r] : -1, to = r < requests ? copies[2 * r + 1] : -1;
    const int some = from >= 0;
    int sum;
    const int at = copied + scan(some, &sum) - 1;
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
// A workgroup takes some columns of every request: it reads them all into LDS, with each request's
// parent and how many columns that one holds, then writes each request's from its parent's and counts the
// pages that come and go.  The counts are integers, so the order of the additions does not matter.  One
// workgroup does small tables and the lengths with them; for larger ones the lengths follow in a launch
// of their own, since every workgroup reads the parents' old ones.  (With up to 8192 entries and 256 threads a
// workgroup 73 requests of 258 columns took 14 us.)
constexpr int kReorderEntries = 8192;  // table entries of a workgroup, 32 KB of LDS
constexpr int kReorderThreads = 1024;

__device__ __forceinline__ bool changes(int r, int parent, int requests) {
  return parent != r && parent >= -1 && parent < requests;
}

__global__ __launch_bounds__(kReorderThreads) void reorder_kernel(int32_t* __restrict__ tables, int32_t* __restrict__ lengths,
                                                                  int32_t* __restrict__ refs,
                                                                  const int32_t* __restrict__ parents, int requests,
                                                                  int columns, int pages, int shift, int log2_width,
                                                                  int whole) {
  __shared__ int old[kReorderEntries];
  __shared__ int parent[kMaxRequests], held[kMaxRequests];  // the columns that the request will hold
  const int width = 1 << log2_width, c0 = blockIdx.x << log2_width, entries = requests << log2_width, tid = threadIdx.x;
  int length = 0;
  if (tid < requests) {
    const int p = parents[tid];
    if (p >= 0 && p < requests) length = lengths[p];
    parent[tid] = p;
    held[tid] = length > 0 ? (int)(((int64_t)length + (1 << shift) - 1) >> shift) : 0;
  }
#pragma unroll 4
  for (int e = tid; e < entries; e += kReorderThreads) {
    const int r = e >> log2_width, c = c0 + (e & (width - 1));
    old[e] = c < columns ? tables[(int64_t)r * columns + c] : -1;
  }
  __syncthreads();
#pragma unroll 4
  for (int e = tid; e < entries; e += kReorderThreads) {
    const int r = e >> log2_width, in = e & (width - 1), p = parent[r];
    if (c0 + in >= columns || !changes(r, p, requests)) continue;
    const int before = old[e];
    int after = p >= 0 && c0 + in < held[r] ? old[(p << log2_width) + in] : -1;
    if (after < 0 || after >= pages) after = -1;
    if (before == after) continue;
    if (before >= 0 && before < pages) atomicSub(refs + before, 1);
    if (after >= 0) atomicAdd(refs + after, 1);
    tables[(int64_t)r * columns + c0 + in] = after;
  }
  if (whole && tid < requests && changes(tid, parent[tid], requests)) lengths[tid] = length;
}

__global__ __launch_bounds__(kMaxRequests) void reorder_lengths_kernel(int32_t* __restrict__ lengths,
                                                                       const int32_t* __restrict__ parents, int requests) {
  const int r = threadIdx.x;
  int length = 0;
  bool change = false;
  if (r < requests) {
    const int p = parents[r];
    change = changes(r, p, requests);
    if (change && p >= 0) length = lengths[p];
  }
  __syncthreads();
  if (change) lengths[r] = length;
}

// ------------------------------------------------------------ norm, rotary, rows into pages
//
// A workgroup per row, D / 16 lanes per head; lane l holds dimensions 8 l .. 8 l + 7 of the head and those
// D / 2 further on, so that the pairs that turn together lie in one lane and every load and store is 16
// bytes.  The first heads' loads are in flight while the row's angles are computed (in double: positions
// are large, and the angle is the product).  Two roundings to bf16, as imq_qk_norm_rope: the norm's result
// (what the model's norm gives) and the turned value.
// Bound by memory: 4099 rows of 32 heads of 256 (134 MB read and written) in 22.5 us where they are in the
// last-level cache, in 28 with new ones; single
// 2-byte values a lane took 34.  The slot is looked at after the loads: before them, 32.  256 to 512
// threads are alike there, 320 and more best for a few rows (five rows 3.8 us, 4.2 with 256); a number of
// threads by the row's heads 26.
constexpr int kWriteThreads = 384;

typedef __bf16 bf16x2v __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {  // v_cvt_pk_bf16_f32
  bf16x2v r;
  r.x = (__bf16)lo;
  r.y = (__bf16)hi;
  return __builtin_bit_cast(uint32_t, r);
}

__device__ __forceinline__ float octets(const uint4 w, int i) {  // value i of eight bf16 values
  const uint32_t word = i < 2 ? w.x : i < 4 ? w.y : i < 6 ? w.z : w.w;
  return __uint_as_float(i & 1 ? word & 0xffff0000u : word << 16);
}

template <int D>
__global__ __launch_bounds__(kWriteThreads) void write_kernel(const uint16_t* q, int64_t ldq,
                                                              const uint16_t* __restrict__ k, int64_t ldk,
                                                              const uint16_t* __restrict__ v, int64_t ldv,
                                                              const uint16_t* __restrict__ q_norm,
                                                              const uint16_t* __restrict__ k_norm,
                                                              const int32_t* __restrict__ positions,
                                                              const int32_t* __restrict__ slots,
                                                              uint16_t* q_out, int64_t ldo,
                                                              uint16_t* __restrict__ k_pages,
                                                              uint16_t* __restrict__ v_pages, int Hq, int Hkv,
                                                              int shift, int64_t tokens, double log2_theta, float eps) {
  constexpr int H = D / 2, L = D / 16;  // L lanes a head
  __shared__ __align__(16) float turn[2][H];
  const int row = blockIdx.x, slot = slots[row], in = threadIdx.x % L;
  const int heads = Hq + 2 * Hkv, stride = kWriteThreads / L;
  int hh = threadIdx.x / L;
  uint4 lo, hi;
  const auto load = [&] {
    const uint16_t* const src = hh < Hq         ? q + row * ldq + hh * D
                                : hh < Hq + Hkv ? k + row * ldk + (hh - Hq) * D
                                                : v + row * ldv + (hh - Hq - Hkv) * D;
    lo = *reinterpret_cast<const uint4*>(src + 8 * in);
    hi = *reinterpret_cast<const uint4*>(src + H + 8 * in);
  };
  if (hh < heads) load();
  for (int d = threadIdx.x; d < H; d += kWriteThreads) {
    double sn, cs;
    sincos((double)positions[row] * exp2(-(double)d * (log2_theta / H)), &sn, &cs);
    turn[0][d] = (float)sn;
    turn[1][d] = (float)cs;
  }
  __syncthreads();
  if (slot < 0 || slot >= tokens) return;
  const int64_t page = slot >> shift, offset = slot & ((1 << shift) - 1);
  while (hh < heads) {
    const bool is_q = hh < Hq, is_v = hh >= Hq + Hkv;
    const int head = is_q ? hh : is_v ? hh - Hq - Hkv : hh - Hq;
    uint16_t* const dst = is_q ? q_out + row * ldo + head * D
                               : (is_v ? v_pages : k_pages) + (((page * Hkv + head) << shift) + offset) * D;
    uint4 lo_out = lo, hi_out = hi;
    if (!is_v) {
      float x[16], ss = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = octets(lo, i);
        x[8 + i] = octets(hi, i);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
      for (int step = 1; step < L; step *= 2) ss += __shfl_xor(ss, step);
      const float inv = 1.0f / sqrtf(ss / (float)D + eps);
      const uint16_t* const weight = is_q ? q_norm : k_norm;
      const uint4 w_lo = *reinterpret_cast<const uint4*>(weight + 8 * in);
      const uint4 w_hi = *reinterpret_cast<const uint4*>(weight + H + 8 * in);
      uint32_t made[2][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t a = pack_bf16(x[2 * i] * inv * octets(w_lo, 2 * i), x[2 * i + 1] * inv * octets(w_lo, 2 * i + 1));
        const uint32_t b = pack_bf16(x[8 + 2 * i] * inv * octets(w_hi, 2 * i), x[9 + 2 * i] * inv * octets(w_hi, 2 * i + 1));
        const float2 s = *reinterpret_cast<const float2*>(&turn[0][8 * in + 2 * i]);
        const float2 c = *reinterpret_cast<const float2*>(&turn[1][8 * in + 2 * i]);
        const float a0 = __uint_as_float(a << 16), a1 = __uint_as_float(a & 0xffff0000u);
        const float b0 = __uint_as_float(b << 16), b1 = __uint_as_float(b & 0xffff0000u);
        made[0][i] = pack_bf16(a0 * c.x - b0 * s.x, a1 * c.y - b1 * s.y);
        made[1][i] = pack_bf16(a0 * s.x + b0 * c.x, a1 * s.y + b1 * c.y);
      }
      lo_out = make_uint4(made[0][0], made[0][1], made[0][2], made[0][3]);
      hi_out = make_uint4(made[1][0], made[1][1], made[1][2], made[1][3]);
    }
    *reinterpret_cast<uint4*>(dst + 8 * in) = lo_out;
    *reinterpret_cast<uint4*>(dst + H + 8 * in) = hi_out;
    hh += stride;
    if (hh < heads) load();
  }
}

// ------------------------------------------------------------ attention over pages
//
// The rows of a request and the query heads of one KV head are taken together as G n queries (row i,
// head g of the group: query i G + g), in tiles.  The work is shared out on the device, where the
// lengths are: every workgroup adds up the key blocks of the requests' tiles and finds its own part.  Tiles
// that several workgroups share leave fp32 partial results, which a second launch, by the same sums,
// adds up in the order of their keys.
struct AttendArgs {
  const uint16_t *q, *k_pages, *v_pages;
  const int32_t *tables, *starts, *ends;
  uint16_t* out;
  int64_t ldq, ldo;
  float* partial;     // (slot, KV head, query of the tile, head_dim)
  float2* state;      // (slot, KV head, query of the tile): the maximum (of scale_log2 q.k) and the sum
  int32_t rows, requests, columns, pages, shift, Hq, Hkv, group, window;
  int32_t fewest, most;  // the queries n group of a request that this launch serves
  int32_t units;      // parts to share the work out in, per KV head
  int32_t slots;      // partial results there is room for, per KV head
  int32_t grain;      // log2 of the blocks that are counted as one (see attend_grain)
  float scale_log2;   // scale * log2(e)
};

// A request as the launch sees it: its first row and its rows, its tokens, its tiles of WIDTH queries,
// the first block of BLOCK keys that any of them sees, and the blocks, in grains, from there to its end.
struct Request {
  int first, count, end, tiles, block0, blocks;
};

template <int WIDTH, int BLOCK>
__device__ __forceinline__ Request read_request(const AttendArgs& a, int r) {
  Request q = {0, 0, 0, 0, 0, 0};
  if (r < a.requests) {
    q.first = clamp_int(a.starts[r], 0, a.rows);
    q.count = clamp_int(a.starts[r + 1], q.first, a.rows) - q.first;
    q.end = clamp_int(a.ends[r], 0, a.columns << a.shift);
    const int queries = q.count * a.group;
    q.tiles = queries < a.fewest || queries > a.most ? 0 : (queries + WIDTH - 1) / WIDTH;
    q.block0 = (a.window ? max(0, q.end - q.count - a.window + 1) : 0) / BLOCK;
    int blocks = (q.end + BLOCK - 1) / BLOCK - q.block0;
    // (a tile of many queries goes over its own rows' windows only)
    if (WIDTH > 16 && a.window) blocks = min(blocks, (a.window + (WIDTH - 2) / a.group) / BLOCK + 2);
    q.blocks = max(1, (blocks + (1 << a.grain) - 1) >> a.grain);
  }
  return q;
}

// The request of lane `at`, in every lane.
__device__ __forceinline__ Request from_lane(const Request& q, int at) {
  return Request{__builtin_amdgcn_readlane(q.first, at), __builtin_amdgcn_readlane(q.count, at),
                 __builtin_amdgcn_readlane(q.end, at),   __builtin_amdgcn_readlane(q.tiles, at),
                 __builtin_amdgcn_readlane(q.block0, at), __builtin_amdgcn_readlane(q.blocks, at)};
}

// The 64 requests that a wavefront looked at last, one a lane.
template <int WIDTH, int BLOCK>
struct Lanes {
  const AttendArgs& a;
  Request q;
  int base;
  __device__ __forceinline__ explicit Lanes(const AttendArgs& args) : a(args), base(-1) {}
  __device__ __forceinline__ void read(int from) {
    if (from == base) return;
    base = from;
    q = read_request<WIDTH, BLOCK>(a, from + (threadIdx.x & 63));
  }
};

// The requests' tiles one after another, each as long as `weight` says of its request: a line along which
// the work of a KV head is shared out.
template <typename LANES, typename WEIGHT>
struct Line {
  LANES& lanes;
  WEIGHT weight;
  int upto;  // the line up to and with the lane's request
  int before = 0, total = 0;

  __device__ __forceinline__ void read(int base) {
    lanes.read(base);
    upto = before + wave_scan(lanes.q.tiles * weight(lanes.q));
  }
  __device__ __forceinline__ Line(LANES& l, WEIGHT w) : lanes(l), weight(w) {
    for (int base = 0;; base += 64) {
      before = total;
      read(base);
      total = __builtin_amdgcn_readlane(upto, 63);
      if (base + 64 >= lanes.a.requests) break;
    }
  }
  // The request at point x of the line: its number and where it starts; false past the end.
  __device__ __forceinline__ bool find(int x, Request* q, int* number, int* start) {
    const int requests = lanes.a.requests;
    if (requests > 64) {  // (another line may have moved the lanes on)
      before = 0;
      read(0);
      for (int base = 64; x >= __builtin_amdgcn_readlane(upto, 63) && base < requests; base += 64) {
        before = __builtin_amdgcn_readlane(upto, 63);
        read(base);
      }
    }
    const uint64_t past = __ballot(upto > x);
    if (!past) return false;
    const int at = __ffsll((unsigned long long)past) - 1;
    *q = from_lane(lanes.q, at);
    *number = lanes.base + at;
    *start = __builtin_amdgcn_readlane(upto, at) - q->tiles * weight(*q);
    return true;
  }
};

__device__ __forceinline__ int wave_total(int v) { return __builtin_amdgcn_readlane(wave_scan(v), 63); }

__device__ __forceinline__ int wave_highest(int v) {  // (of values >= 0; as wave_scan)
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false));
  return __builtin_amdgcn_readlane(v, 63);
}

struct BlocksOf {
  __device__ __forceinline__ int operator()(const Request& q) const { return q.blocks; }
};

struct One {
  __device__ __forceinline__ int operator()(const Request&) const { return 1; }
};

__device__ __forceinline__ int ceil_of(int a, int b) { return (a + b - 1) / b; }

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) s16x4_t* lds_s16x4;
typedef __attribute__((address_space(3))) u32x4_t* lds_u32x4;
typedef __attribute__((address_space(3))) f32x4_t* lds_f32x4;
typedef __attribute__((address_space(3))) char* lds_char;
__device__ __forceinline__ uint32_t lds_at(char* p) { return (uint32_t)(uintptr_t)(lds_char)p; }
// (page numbers of a whole wavefront, which no kernel that reads them writes: loaded by the scalar unit)
typedef const __attribute__((address_space(4))) int32_t* scalar_ints;

// The bf16 pair `w` with infinities and NaNs as zeros; *odd gets a bit set if there were any.
__device__ __forceinline__ uint32_t finite_pair(uint32_t w, uint32_t* odd) {
  const bool lo = (w & 0x7f80u) == 0x7f80u, hi = (w & 0x7f800000u) == 0x7f800000u;
  *odd |= lo || hi;
  return (lo ? 0u : w & 0xffffu) | (hi ? 0u : w & 0xffff0000u);
}

typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t max_pair(uint32_t a, uint32_t b) {  // v_pk_max_u16
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, a), __builtin_bit_cast(u16x2_t, b)));
}

// Few queries per request (decode steps, short chunks): tiles of 16 queries of one KV head.  The line of
// blocks is cut into `units` equal parts whatever tiles they belong to, a workgroup takes one, tile
// after tile, and each of its four wavefronts a quarter of a tile's keys there, 32 at a time.
// Scores are K Q^T on v_mfma_f32_16x16x32_bf16, so that a lane holds keys of one query: P^T is then
// the B operand of V^T P^T without leaving its lane (keys 4 g .. of two 16-key tiles), as two terms of bf16
// (2^-15 of a probability are lost, about as in the slots' decode attention: where values of both signs all
// but cancel, one term's 2^-8 would be most of the result; the second product hides under the loads, 32
// requests of up to 8000 tokens 113.8 us and 114.2 with it, one of 777 11.5 and 11.6).  K goes from
// its page to the A operand directly; V goes through the wavefront's own LDS by rows, 32-byte pieces
// swizzled, and is read transposed.  The next block's K loads are issued as soon as this block's are
// used, its V loads when this block's have gone to LDS: 16 KB (head size 128) in flight per wavefront
// over the softmax and P V, and no barrier before the wavefronts' results are joined.
// Bound by memory: 32 requests of up to 8000 tokens, 32 heads on 8 of 128 (669 MB), in 110 us, 6.1 TB/s, and 5 us
// for the second launch; 16 heads on 8 of 256 (1.33 GB) in 211 us with it, 6.3 TB/s.  One of 777 tokens 7.8 and
// 5.0 us: the chain of starts, lengths, table and keys, each a load after the last.  Parts of four blocks: a request of 8000 tokens 17 us instead of 14.
constexpr int kRowsTile = 16, kRowsBlock = 32, kRowsLeast = 8;
constexpr int kRowsMost = 32;  // queries of a request that rows_workgroup is there for
template <int D>
constexpr int kWorkgroups = D == 128 ? 512 : 256;  // as many as are resident

// The length of a part of the line.
__device__ __forceinline__ int part_length(const AttendArgs& a, int total, int least) {
  return max(least, (total + a.units - 1) / a.units);
}

// The LDS of a workgroup of either kind: four arrays of 16 KB (of their own: a read of one does not wait for
// the loads into another), for attend_rows a block's values of each wavefront and then its result.
constexpr int kArray = 16384;

// Wavefront w's part of it.
template <int D>
__device__ __forceinline__ lds_char part_of(int w, uint32_t at0, uint32_t at1, uint32_t at2, uint32_t at3) {
  if (D == 128) return (lds_char)(uintptr_t)((w & 2 ? at1 : at0) + (w & 1) * (32 * 2 * D));
  return (lds_char)(uintptr_t)(w & 2 ? (w & 1 ? at3 : at2) : w & 1 ? at1 : at0);
}

template <bool ONCE>
__device__ __forceinline__ u32x4_t load_piece(const char* at) {
  const u32x4_t* const p = reinterpret_cast<const u32x4_t*>(at);
  return ONCE ? __builtin_nontemporal_load(p) : *p;
}

template <int D, bool ONCE>
__device__ __forceinline__ void attend_rows(const AttendArgs& a, int head, const Request& s, int request, int place, int from,
                                            int to, int slot, char* l0, char* l1, char* l2, char* l3, float (*tops)[16],
                                            float (*sums)[16]) {
  constexpr int T = D / 32, P = D / 8, C = D / 16;  // k-steps of a score, 16-byte pieces of a row, 16-dim tiles
  constexpr int V = 32 * P / 64;                    // 16-byte pieces of a block's values per lane
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int query = 16 * place + n, row = query / a.group;
  const bool live = row < s.count;
  const int begin = s.end - s.count;  // position of the request's first row
  const int position = begin + row;
  const int tile_first = begin + (16 * place) / a.group;
  const int tile_last = min(s.end - 1, begin + (16 * place + 15) / a.group);
  const int low = a.window ? max(0, tile_first - a.window + 1) : 0;
  const int64_t q_head = (int64_t)head * a.group + query % a.group;

  const uint32_t at0 = lds_at(l0), at1 = lds_at(l1), at2 = D == 128 ? 0u : lds_at(l2), at3 = D == 128 ? 0u : lds_at(l3);
  // the wavefront's blocks: its quarter of those between from and to that the tile sees
  from = max(from, low / kRowsBlock);
  to = tile_last < low ? from : min(to, tile_last / kRowsBlock + 1);
  const int per_wave = (to - from + 3) >> 2;
  int at = __builtin_amdgcn_readfirstlane(min(to, from + wave * per_wave));
  const int stop = __builtin_amdgcn_readfirstlane(min(to, from + (wave + 1) * per_wave));

  f32x4_t o[C];
#pragma unroll
  for (int c = 0; c < C; ++c) o[c] = f32x4_t{};
  float top = -INFINITY, sum = 0.0f;

  if (at < stop) {
    bf16x8_t qf[T];
#pragma unroll
    for (int t = 0; t < T; ++t) {
      u32x4_t w = {0u, 0u, 0u, 0u};
      if (live) w = *reinterpret_cast<const u32x4_t*>(a.q + (s.first + row) * a.ldq + q_head * D + 32 * t + 8 * g);
      qf[t] = __builtin_bit_cast(bf16x8_t, w);
    }
    const scalar_ints table = (scalar_ints)(a.tables + (int64_t)request * a.columns);
    const int mask = (1 << a.shift) - 1;
    const uint32_t k_lane = 2 * (n * D + 8 * g), v_lane = 2 * ((lane / P) * D + 8 * (lane % P));
    const lds_char vl = part_of<D>(wave, at0, at1, at2, at3);

    // the pages of a block's two 16-key groups (a page holds a multiple of 16 tokens).  (Plain numbers, no
    // array: as one they went to LDS, for whose layout the compiler has every workgroup read the launch's
    // packet in host memory, one after another: 15 us for 256 of them.)
    auto page_of = [&](int block, int b) { return table[min(block * 32 + 16 * b, tile_last) >> a.shift]; };
    auto held = [&](int page) { return (uint32_t)page < (uint32_t)a.pages; };
    auto group_offset = [&](int page, int block, int b) {  // bytes; a bad page reads as page 0
      page = held(page) ? page : 0;
      return 2 * ((((int64_t)page * a.Hkv + head) << a.shift) + ((block * 32 + 16 * b) & mask)) * D;
    };
    u32x4_t kr[2][T], vr[V];
    auto load_k = [&](int page0, int page1, int block) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const char* const base = reinterpret_cast<const char*>(a.k_pages) + group_offset(b ? page1 : page0, block, b);
#pragma unroll
        for (int t = 0; t < T; ++t) kr[b][t] = load_piece<ONCE>(base + k_lane + 64 * t);
      }
    };
    auto load_v = [&](int page0, int page1, int block) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const char* const base = reinterpret_cast<const char*>(a.v_pages) + group_offset(b ? page1 : page0, block, b);
#pragma unroll
        for (int i = 0; i < V / 2; ++i)
          vr[b * (V / 2) + i] = load_piece<ONCE>(base + v_lane + 1024 * i);
      }
    };
    int now0 = page_of(at, 0), now1 = page_of(at, 1);
    int next0 = page_of(min(at + 1, stop - 1), 0), next1 = page_of(min(at + 1, stop - 1), 1);
    load_k(now0, now1, at);
    load_v(now0, now1, at);
    for (; at < stop; ++at) {
      const int ahead = min(at + 1, stop - 1), k0 = 32 * at;
      f32x4_t sc[2];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        sc[b] = f32x4_t{};
#pragma unroll
        for (int t = 0; t < T; ++t)
          sc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, kr[b][t]), qf[t], sc[b], 0, 0, 0);
      }
      load_k(next0, next1, ahead);
      // Where some queries see a key of the block and others do not, or none does: keys masked, values that
      // nothing sees zeros whatever their page holds, and infinities and NaNs, which a probability of
      // zero must not meet, zeros too; those are added below for the queries that see them.
      const bool edge = k0 + 31 > tile_first || k0 < low || (a.window && k0 <= tile_last - a.window) ||
                        !held(now0) || !held(now1);
      uint32_t odd = 0;
      if (edge) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int key = k0 + (64 / P) * i + lane / P;
          const bool some = held(i / (V / 2) ? now1 : now0) && key >= low && key <= tile_last;
#pragma unroll
          for (int e = 0; e < 4; ++e) vr[i][e] = some ? finite_pair(vr[i][e], &odd) : 0u;
        }
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int r = (64 / P) * i + lane / P, piece = lane % P;
        *(lds_u32x4)(vl + r * 2 * D + 32 * ((piece >> 1) ^ (r & 7)) + 16 * (piece & 1)) = vr[i];
      }
      load_v(next0, next1, ahead);
      const int after0 = page_of(min(at + 2, stop - 1), 0), after1 = page_of(min(at + 2, stop - 1), 1);
      float most = top;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sc[b][e] *= a.scale_log2;
          if (edge) {
            const int key = k0 + 16 * b + 4 * g + e;
            if (!(held(b ? now1 : now0) && key <= position && (!a.window || key > position - a.window))) sc[b][e] = -INFINITY;
          }
          most = fmaxf(most, sc[b][e]);  // (a NaN score comes back through its exponential)
        }
      most = max_xor32(max_xor16(most));
      const float base = most == -INFINITY ? 0.0f : most;
      const float keep = __builtin_amdgcn_exp2f(top - base);
      top = most;
      sum *= keep;
      float p[2][4];
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          p[b][e] = __builtin_amdgcn_exp2f(sc[b][e] - base);
          sum += p[b][e];
        }
      // The probabilities as two terms of bf16 each: the first cut off, the second what is left and 2^-20 of it all
      // (which scales every output alike), so that it is above zero where the first one is: an infinite value times
      // a zero or a negative number would be a NaN, or one with the first product.
      u32x4_t pw, rest;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float even = p[i / 2][2 * (i % 2)], odd_one = p[i / 2][2 * (i % 2) + 1];
        const uint32_t e = __float_as_uint(even), o1 = __float_as_uint(odd_one);
        pw[i] = __builtin_amdgcn_perm(o1, e, 0x07060302);
        rest[i] = pack_bf16(fmaf(even, 1.0f + 0x1p-20f, -__uint_as_float(e & 0xffff0000u)),
                            fmaf(odd_one, 1.0f + 0x1p-20f, -__uint_as_float(o1 & 0xffff0000u)));
      }
      const bf16x8_t pf = __builtin_bit_cast(bf16x8_t, pw), pr = __builtin_bit_cast(bf16x8_t, rest);
      __builtin_amdgcn_wave_barrier();  // (a wavefront's LDS accesses complete in order)
#pragma unroll
      for (int c = 0; c < C; ++c) {
        o[c] *= keep;
        // lane i of each 16 reads 8 bytes of row i / 4; the transposed read gives it the four rows' value
        // of dimension i
        const int r = 4 * g + (n >> 2);
        const lds_char v0 = vl + r * 2 * D + 32 * (c ^ (r & 7)) + 8 * (n & 3);
        const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)v0);
        const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(v0 + 16 * 2 * D));
        const bf16x8_t vf = __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        o[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf, o[c], 0, 0, 0);
        o[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pr, o[c], 0, 0, 0);
      }
      __builtin_amdgcn_wave_barrier();
      if (__any(odd)) {
        for (int r = 0; r < 32; ++r) {
          const int b = r >> 4, key = k0 + r;
          if (!held(b ? now1 : now0) || key < low || key > tile_last) continue;
          const float mine = b ? ((r & 2) ? ((r & 1) ? p[1][3] : p[1][2]) : ((r & 1) ? p[1][1] : p[1][0]))
                               : ((r & 2) ? ((r & 1) ? p[0][3] : p[0][2]) : ((r & 1) ? p[0][1] : p[0][0]));
          const float chance = __shfl(mine, n + 16 * ((r >> 2) & 3));
          const bool seen = live && key <= position && (!a.window || key > position - a.window);
          const uint16_t* const v = a.v_pages + group_offset(b ? now1 : now0, at, b) / 2 + (r & 15) * D;
#pragma unroll
          for (int c = 0; c < C; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t bits = v[16 * c + 4 * g + e];
              if (seen && (bits & 0x7f80u) == 0x7f80u) o[c][e] += chance * bf16_bits_to_f32(bits);
            }
        }
      }
      now0 = next0, now1 = next1;
      next0 = after0, next1 = after1;
    }
    sum = add_xor32(add_xor16(sum));
  }

  // the four wavefronts' results joined: each by its distance from the common maximum
  if (lane < 16) {
    tops[wave][lane] = top;
    sums[wave][lane] = sum;
  }
  __syncthreads();  // (and every wavefront is through with its values in LDS)
  const float most = fmaxf(fmaxf(tops[0][n], tops[1][n]), fmaxf(tops[2][n], tops[3][n]));
  const float scale = exp2f(top - (most == -INFINITY ? 0.0f : most));
#pragma unroll
  for (int c = 0; c < C; ++c)
    ((lds_f32x4)part_of<D>(wave, at0, at1, at2, at3))[c * 64 + lane] = o[c] * scale;  // (tile of 16 dims, lane)
  __syncthreads();
  float total = 0.0f;
#pragma unroll
  for (int w = 0; w < 4; ++w) total += sums[w][n] * exp2f(tops[w][n] - (most == -INFINITY ? 0.0f : most));
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  const int64_t result = ((int64_t)slot * a.Hkv + head) * 16 + n;
#pragma unroll
  for (int i = 0; i < C / 4; ++i) {
    const int c = wave + 4 * i;
    f32x4_t v = ((lds_f32x4)part_of<D>(0, at0, at1, at2, at3))[c * 64 + lane];
#pragma unroll
    for (int w = 1; w < 4; ++w) v += ((lds_f32x4)part_of<D>(w, at0, at1, at2, at3))[c * 64 + lane];
    if (!live) continue;
    if (slot < 0) {
      const u32x2_t four = {pack_bf16(v.x * inv, v.y * inv), pack_bf16(v.z * inv, v.w * inv)};
      *reinterpret_cast<u32x2_t*>(a.out + (s.first + row) * a.ldo + q_head * D + 16 * c + 4 * g) = four;
    } else {
      *reinterpret_cast<f32x4_t*>(a.partial + result * D + 16 * c + 4 * g) = v;
    }
  }
  if (slot >= 0 && live && wave == 0 && g == 0) a.state[result] = make_float2(most, total);
}

// Workgroup `index` of a launch over tiles of few queries.
template <int D, bool ONCE>
__device__ __forceinline__ void rows_workgroup(const AttendArgs& a, int index, char* l0, char* l1, char* l2, char* l3,
                                               float (*tops)[16], float (*sums)[16]) {
  const int unit = index / a.Hkv, head = index % a.Hkv;
  Lanes<kRowsTile, kRowsBlock> lanes(a);
  if (a.units == 0) {  // whole tiles (rows_alone)
    Line<Lanes<kRowsTile, kRowsBlock>, One> tiles(lanes, One());
    Request q;
    int request, start;
    if (!tiles.find(unit, &q, &request, &start) || unit < start || unit - start >= q.tiles) return;
    attend_rows<D, ONCE>(a, head, q, request, unit - start, q.block0, q.block0 + (q.blocks << a.grain), -1, l0, l1, l2, l3, tops,
                         sums);
    return;
  }
  Line<Lanes<kRowsTile, kRowsBlock>, BlocksOf> line(lanes, BlocksOf());
  const int part = part_length(a, line.total, kRowsLeast);
  if ((int64_t)unit * part >= line.total) return;
  const int x0 = unit * part, x1 = min(line.total, x0 + part);
  for (int x = x0; x < x1;) {
    Request q;
    int request, start;
    if (!line.find(x, &q, &request, &start)) return;
    const int place = (x - start) / q.blocks, in = (x - start) % q.blocks;
    if (x < start || place >= q.tiles) return;  // (sums that starts which do not ascend have wrapped)
    const int length = min(q.blocks - in, x1 - x);
    // a tile not whole here: the workgroup's first partial result, or its last
    const int slot = length == q.blocks ? -1 : 2 * unit + (x != x0);
    if (x != x0) __syncthreads();
    attend_rows<D, ONCE>(a, head, q, request, place, q.block0 + (in << a.grain), q.block0 + ((in + length) << a.grain), slot,
                         l0, l1, l2, l3, tops, sums);
    x += length;
  }
}

// The partial results of a tile added up: a group of D / 4 lanes takes four queries, and of up to
// kMergeAlone partial results all, four at a time; of more, as many groups share the queries as there
// are groups, each every so manieth, and their sums are added in LDS.  The queries are those of the passes
// `pass`, `pass` + `step`, .. over the tile.  (A pass over maxima first, and LDS always, took 14 us where this
// takes 6.)
constexpr int kMergeAlone = 8;

template <int D>
struct MergeSpace {
  float4 sums[kThreads / (D / 4)][4][D / 4];
  float tops[kThreads / (D / 4)][4], totals[kThreads / (D / 4)][4];
};

template <int WIDTH, int D, typename SLOT>
__device__ __forceinline__ void merge_part(const AttendArgs& a, const Request& s, int place, int head, int pass, int step,
                                           int parts, SLOT slot_of, MergeSpace<D>& space) {
  constexpr int L = D / 4, NG = kThreads / L;
  const int lane = threadIdx.x % L, group = threadIdx.x / L;
  const int share = parts <= kMergeAlone ? 1 : NG, mine = group % share, many = 4 * (NG / share);
  const int64_t slot_step = (int64_t)a.Hkv * WIDTH;
  for (int qb = many * pass; qb < WIDTH; qb += many * step) {
    if ((WIDTH * place + qb) / a.group >= s.count) return;
    const int q = qb + 4 * (group / share);  // and the three behind it
    const bool some = q < WIDTH && (WIDTH * place + q) / a.group < s.count;
    const int64_t at = (int64_t)head * WIDTH + q;
    float most[4], total[4];
    float4 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      most[j] = -INFINITY;
      total[j] = 0.0f;
      v[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    // (rows behind the request's last one have places of their own that hold anything: not used)
    for (int i0 = some ? mine : parts; i0 < parts; i0 += 4 * share) {
      float2 st[4][4];
      float4 u[4][4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int64_t from = at + slot_of(min(i0 + k * share, parts - 1)) * slot_step;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          st[k][j] = a.state[from + j];
          u[k][j] = *reinterpret_cast<const float4*>(a.partial + (from + j) * D + 4 * lane);
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float higher = most[j];
#pragma unroll
        for (int k = 0; k < 4; ++k) higher = fmaxf(higher, i0 + k * share < parts ? st[k][j].x : -INFINITY);
        const float base = higher == -INFINITY ? 0.0f : higher, keep = exp2f(most[j] - base);
        most[j] = higher;
        total[j] *= keep;
        v[j].x *= keep, v[j].y *= keep, v[j].z *= keep, v[j].w *= keep;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (i0 + k * share < parts) {
            const float w = exp2f(st[k][j].x - base);
            total[j] = fmaf(st[k][j].y, w, total[j]);
            v[j].x = fmaf(u[k][j].x, w, v[j].x);
            v[j].y = fmaf(u[k][j].y, w, v[j].y);
            v[j].z = fmaf(u[k][j].z, w, v[j].z);
            v[j].w = fmaf(u[k][j].w, w, v[j].w);
          }
      }
    }
    auto write = [&](int j, const float4& r, float sum) {
      const int query = WIDTH * place + q + j, row = query / a.group;
      if (row >= s.count) return;
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      const u32x2_t four = {pack_bf16(r.x * inv, r.y * inv), pack_bf16(r.z * inv, r.w * inv)};
      *reinterpret_cast<u32x2_t*>(a.out + (s.first + row) * a.ldo + ((int64_t)head * a.group + query % a.group) * D + 4 * lane) = four;
    };
    if (share == 1) {
      if (some)
#pragma unroll
        for (int j = 0; j < 4; ++j) write(j, v[j], total[j]);
      continue;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      space.sums[group][j][lane] = v[j];
      if (lane == 0) space.tops[group][j] = most[j], space.totals[group][j] = total[j];
    }
    __syncthreads();
    if (some && group < 4) {  // one of the four queries each
      const int j = group;
      float higher = -INFINITY, sum = 0.0f;
      float4 r = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int k = 0; k < NG; ++k) higher = fmaxf(higher, space.tops[k][j]);
      const float base = higher == -INFINITY ? 0.0f : higher;
#pragma unroll
      for (int k = 0; k < NG; ++k) {
        const float w = exp2f(space.tops[k][j] - base);
        const float4 x = space.sums[k][j][lane];
        sum = fmaf(space.totals[k][j], w, sum);
        r.x = fmaf(x.x, w, r.x);
        r.y = fmaf(x.y, w, r.y);
        r.z = fmaf(x.z, w, r.z);
        r.w = fmaf(x.w, w, r.w);
      }
      write(j, r, sum);
    }
    __syncthreads();
  }
}

// After rows_workgroup: a workgroup per boundary between two parts of the line; those inside a tile
// share its queries.
template <int D>
__device__ __forceinline__ void merge_rows(const AttendArgs& a, int index, MergeSpace<D>& space) {
  const int head = index % a.Hkv, unit = index / a.Hkv + 1;
  Lanes<kRowsTile, kRowsBlock> lanes(a);
  Line<Lanes<kRowsTile, kRowsBlock>, BlocksOf> line(lanes, BlocksOf());
  const int part = part_length(a, line.total, kRowsLeast);
  if ((int64_t)unit * part >= line.total) return;
  Request q;
  int request, start;
  if (!line.find(unit * part, &q, &request, &start)) return;
  const int place = (unit * part - start) / q.blocks, tile = start + place * q.blocks;
  if (tile == unit * part) return;
  const int first = tile / part, last = (tile + q.blocks - 1) / part;  // the parts that hold some of it
  if (unit * part < start || place >= q.tiles || last >= a.units) return;  // (as in rows_workgroup)
  merge_part<kRowsTile, D>(a, q, place, head, unit - first - 1, last - first, last - first + 1,
                           [&](int i) { return (int64_t)(2 * (first + i) + (i == 0 && tile > first * part)); }, space);
}

// Many queries per request (chunks of prompts): tiles of 128 queries of one KV head, each of a workgroup's
// four wavefronts 32 of them; the key blocks go through LDS, shared by the four and twice there, the loads
// of the next one in flight over the current one's work and one barrier per block.  Scores are K Q^T on
// v_mfma_f32_32x32x16_bf16 and P^T the B operand of V^T P^T without leaving its lane, as above (keys 4 h ..
// and 8 + 4 h .. of 16), rounded to one term of bf16 (2^-8 of it at most): a second one is half as many
// matrix instructions again, which bound these tiles (1024 tokens of 16384: 272 us, and 375 with it; heads
// of 256 with windows 53 and 63).  The running maximum follows only when a score passes it
// by 2^8: until then the probabilities are up to 256, which costs no accuracy, and the sums need not be scaled
// again.  K lies in LDS by rows of 16-byte pieces, V by rows of 64-byte ones, both swizzled so that the rows
// that a read takes at a time lie in different banks (the 32-byte pieces of attend_rows and K's by row & 7 had
// every read conflict once: half of the LDS cycles).
//
// A tile is cut into splits of at most `chunk` blocks (tile_chunk).  Tiles of requests that have several
// splits come first, and a request's last tiles, the longest, before its first ones.
//
// Bound by the matrix cores' power and by what a wavefront can issue between their instructions: 8192 tokens
// of 32 heads of 128 in 515 to 530 us (1040 to 1070 TFLOP/s; a library product of 8192^3 reaches 1200), where the
// cores are busy 54 % of the time at 1.8 GHz.  A block takes 1.0 us (heads of 256) or 1.1 (128) alone on a CU and
// two workgroups there do one each in 2.1; an edge takes 0.5 us more; a workgroup's start and end take 5 us,
// the second launch 5 and its partial results' traffic.  So no tile is split where the longest context has
// kTileAlone keys, or twice that and there are tiles for a quarter of the CUs (512 queries of 32 heads over
// 1024 keys 24 us, 28 with a second launch).
constexpr int kTile = 128, kTileLeast = 256, kTileAlone = 1024;  // (keys)
constexpr float kSlack = 8.0f;
constexpr int kCUs = 256;
constexpr int kAhead = 4, kAheadV = 4;  // operands of K and of V^T that are in registers or on their way there

template <int D>
constexpr int tile_block() {
  return D == 128 ? 64 : 32;  // keys
}

struct TilePart {
  Request q;
  int request, place, split, splits, slot;  // splits: of the request's longest tile; slot: of the tile's first
};

struct SplitsOf {  // a request's splits of a tile: where there is one only, or more
  int chunk, several;
  __device__ __forceinline__ int operator()(const Request& q) const {
    const int splits = ceil_of(q.blocks, chunk);
    return (splits > 1) == several ? splits : 0;
  }
};

// The blocks of a split.  Three choices: whole tiles; as many splits of each as leave a CU to every one; and
// as many as are resident.  What each costs, in blocks (about 1 us): the longest split with its start and
// end (kStart), or what a CU has to do (with two workgroups on it they share it, and others wait for a
// quarter of the longest; with one, heads of 256, a last round may be short); and where tiles are split, the
// second launch and its partial results (kJoin).  512 queries of 32 heads on 8: whole over 1024 keys 27 us
// and split 32, over 4096 keys 75 and 55.
constexpr float kStart = 5.0f;
template <int D>
constexpr float kJoin = D == 128 ? 10.0f : 20.0f;
template <int D, typename LANES>
__device__ __forceinline__ int tile_chunk(LANES& lanes, int least) {
  const AttendArgs& a = lanes.a;
  if (a.units == 0) return 1 << 30;
  least = max(1, least >> a.grain);
  int work = 0, tiles = 0, longest = 0;
  for (int base = 0; base < a.requests; base += 64) {
    lanes.read(base);
    work += wave_total(lanes.q.tiles * lanes.q.blocks);
    tiles += wave_total(lanes.q.tiles);
    longest = max(longest, wave_highest(lanes.q.tiles ? lanes.q.blocks : 0));
  }
  const int cus = max(1, kCUs / a.Hkv);
  const auto cost = [&](int splits, int blocks) {
    const float mean = (float)work / (float)splits + kStart;
    const float shared = D == 128 ? mean * (float)splits / (float)cus + 0.25f * (float)blocks : mean * (float)ceil_of(splits, cus);
    return fmaxf((float)blocks + kStart, shared);
  };
  const int fine = max(least, ceil_of(work, a.units));
  if (fine >= longest) return 1 << 30;
  const int coarse = max(fine, ceil_of(longest, max(1, cus / tiles)));
  int splits_fine = 0, splits_coarse = 0;
  for (int base = 0; base < a.requests; base += 64) {
    lanes.read(base);
    splits_fine += wave_total(lanes.q.tiles * ceil_of(lanes.q.blocks, fine));
    splits_coarse += wave_total(lanes.q.tiles * ceil_of(lanes.q.blocks, coarse));
  }
  const float whole = cost(tiles, longest), with_coarse = cost(splits_coarse, min(coarse, longest)) + kJoin<D>;
  const float with_fine = cost(splits_fine, fine) + kJoin<D>;
  if (whole <= fminf(with_coarse, with_fine)) return 1 << 30;
  return with_coarse < with_fine ? coarse : fine;
}

// Split number `unit`; request -1 past the last one.
template <typename LANES>
__device__ __forceinline__ TilePart find_part(LANES& lanes, int unit, int chunk) {
  Line<LANES, SplitsOf> split(lanes, SplitsOf{chunk, 1});
  TilePart p;
  p.request = -1;
  const bool several = unit < split.total;
  int start = 0, number = -1, x = unit;
  bool found;
  if (several) {
    found = split.find(x, &p.q, &number, &start);
  } else {
    x -= split.total;
    Line<LANES, SplitsOf> whole(lanes, SplitsOf{chunk, 0});
    found = whole.find(x, &p.q, &number, &start);
  }
  if (!found) return p;
  p.splits = several ? ceil_of(p.q.blocks, chunk) : 1;
  const int in = (x - start) / p.splits;
  p.split = (x - start) - in * p.splits;
  p.slot = several ? unit - p.split : 0;
  p.place = p.q.tiles - 1 - in;
  // (sums that starts which do not ascend have wrapped must not lead outside the request or the workspace)
  if (p.place >= 0 && in >= 0 && (!several || (p.slot >= 0 && p.slot + p.splits <= lanes.a.slots))) p.request = number;
  return p;
}

// A tile's blocks: from *first on, as many as are returned, of KEYS keys.
template <int KEYS>
__device__ __forceinline__ int tile_blocks(const AttendArgs& a, const Request& q, int place, int* tile_first, int* tile_last,
                                           int* low, int* first) {
  const int begin = q.end - q.count;
  *tile_first = begin + (kTile * place) / a.group;
  *tile_last = min(q.end - 1, begin + (kTile * place + kTile - 1) / a.group);
  *low = a.window ? max(0, *tile_first - a.window + 1) : 0;
  *first = *low / KEYS;
  return *tile_last < *low ? 0 : *tile_last / KEYS + 1 - *first;
}

// Workgroup `index` of a launch over tiles of many queries.
template <int D>
__device__ __forceinline__ void tile_workgroup(const AttendArgs& a, int index, char* k0l, char* k1l, char* v0l, char* v1l) {
  constexpr int KEYS = tile_block<D>(), B = KEYS / 32, T = D / 16, C = D / 32, P = D / 8;
  constexpr int MINE = KEYS / 4, L = MINE * P / 64;  // keys of a block that a wavefront loads, 1 KB at a time
  constexpr int GROUPS = KEYS / 16;
  static_assert(KEYS * 2 * D == kArray, "a block's keys, or its values, fill an array");
  __shared__ __attribute__((aligned(16))) int odd_waves[4];
  const int head = index % a.Hkv, lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Lanes<kTile, KEYS> lanes(a);
  const int chunk = tile_chunk<D>(lanes, kTileLeast / KEYS);
  const TilePart s = find_part(lanes, index / a.Hkv, chunk);
  if (s.request < 0) return;
  int tile_first, tile_last, low, block0;
  const int all = tile_blocks<KEYS>(a, s.q, s.place, &tile_first, &tile_last, &low, &block0);
  const int splits = max(1, ceil_of(ceil_of(all, 1 << a.grain), chunk));  // of this tile
  if (s.split >= splits) return;
  const int query = kTile * s.place + 32 * wave + n, row = query / a.group;
  const bool live = row < s.q.count;
  const int position = s.q.end - s.q.count + row;
  const int64_t q_head = (int64_t)head * a.group + query % a.group;
  const int per_split = ceil_of(all, splits);
  const int from = __builtin_amdgcn_readfirstlane(block0 + min(all, s.split * per_split));
  const int stop = __builtin_amdgcn_readfirstlane(block0 + min(all, (s.split + 1) * per_split));

  f32x16_t o[C];
#pragma unroll
  for (int c = 0; c < C; ++c) o[c] = f32x16_t{};
  float top = -INFINITY, sum = 0.0f;  // (in units of raw scores times scale_log2)

  if (from < stop) {
    const int32_t* const table = a.tables + (int64_t)s.request * a.columns;
    const int mask = (1 << a.shift) - 1;
    // The pages of 64 groups of 16 keys, one a lane, and of the 64 after those: loaded long before they are
    // used.  (A scalar load for each block cost its whole latency: LDS reads wait for scalar loads too.)
    constexpr int AHEAD = 64 / GROUPS;  // blocks
    auto read_pages = [&](int block) __attribute__((always_inline)) {
      return table[min(block * KEYS + 16 * lane, tile_last) >> a.shift];
    };
    int seen = from, pages_now = read_pages(from), pages_next = read_pages(from + AHEAD);
    // Of a block: the page of this wavefront's keys (a bad one read as page 0), and which 16-key groups have a
    // bad page.
    auto move_pages = [&](int block) __attribute__((always_inline)) {
      if (min(block, stop - 1) - seen >= AHEAD) {
        seen += AHEAD;
        pages_now = pages_next;
        pages_next = read_pages(seen + AHEAD);
      }
    };
    auto look_up = [&](int block, int* page, uint32_t* bad) __attribute__((always_inline)) {  // (after move_pages)
      block = min(block, stop - 1);
      const int at = (block - seen) * GROUPS;
      const int p = __builtin_amdgcn_readlane(pages_now, at + wave * MINE / 16);
      *page = (uint32_t)p < (uint32_t)a.pages ? p : 0;
      *bad = (uint32_t)(__ballot((uint32_t)pages_now >= (uint32_t)a.pages) >> at) & ((1u << GROUPS) - 1);
    };
    // Memory -> LDS, 1 KB a load: lane l gets the 16 bytes at l.  The swizzle is in where the lane reads: of
    // row r it takes the piece that belongs in its place.  A wavefront's MINE keys lie in one page.
    uint32_t k_from[L], v_from[L];
#pragma unroll
    for (int i = 0; i < L; ++i) {
      const int in = (64 / P) * i + lane / P, r = wave * MINE + in, piece = lane % P;
      k_from[i] = in * 2 * D + 16 * (piece ^ (r & 15));
      v_from[i] = in * 2 * D + 64 * ((piece >> 2) ^ (r & 3)) + 16 * (piece & 3);
    }
    auto source = [&](const uint16_t* pages, int page, int block) __attribute__((always_inline)) {
      block = min(block, stop - 1);
      const int64_t at = ((((int64_t)page * a.Hkv + head) << a.shift) + ((block * KEYS + wave * MINE) & mask)) * D;
      return buffer_rsrc(pages + at, MINE * 2 * D);
    };
    auto load_kb = [&](__amdgpu_buffer_rsrc_t rsrc, int i, const uint32_t* lane_from, char* to) __attribute__((always_inline)) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rsrc, (__attribute__((address_space(3))) void*)(to + wave * MINE * 2 * D + 1024 * i), 16, lane_from[i], 0, 0, 0);
    };
    auto load = [&](const uint16_t* pages, int page, int block, const uint32_t* lane_from, char* to) __attribute__((always_inline)) {
      const __amdgpu_buffer_rsrc_t rsrc = source(pages, page, block);
#pragma unroll
      for (int i = 0; i < L; ++i) load_kb(rsrc, i, lane_from, to);
    };
    // Where some queries see a key of the block and others do not, or none does (see attend_rows)
    auto is_edge = [&](int block, uint32_t bad) __attribute__((always_inline)) {
      const int k0 = block * KEYS;
      return bad || k0 + KEYS - 1 > tile_first || k0 < low || (a.window && k0 <= tile_last - a.window);
    };
    bf16x8_t qf[T];
    const uint32_t k_lane = n * 2 * D + 16 * (h ^ (n & 15));
    auto scores = [&](const char* kb, uint32_t at, int t, f32x16_t* sc) __attribute__((always_inline)) {
#pragma unroll
      for (int b = 0; b < B; ++b) {
        const u32x4_t w = *reinterpret_cast<const u32x4_t*>(kb + 32 * b * 2 * D + (at ^ (32 * t)));
        sc[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, w), qf[t], t ? sc[b] : f32x16_t{}, 0, 0, 0);
      }
    };
    // K and V as the matrix instructions take them: of K the keys 32 b .. + 31 and dimensions 16 t .. + 15
    // (j = B t + b), of V^T the dimensions 32 c .. + 31 and keys 16 u .. + 15 (j = C u + c)
    auto key_operand = [&](const char* kb, uint32_t at, int j) __attribute__((always_inline)) {
      return __builtin_bit_cast(bf16x8_t, *reinterpret_cast<const u32x4_t*>(kb + 32 * (j % B) * 2 * D + (at ^ (32 * (j / B)))));
    };
    uint32_t v_lane[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 4 * h + ((lane & 15) >> 2);
      v_lane[i] = r * 2 * D + 64 * (i ^ (r & 3)) + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);
    }
    auto value_operand = [&](const char* vb, int j) __attribute__((always_inline)) {
      const char* const at = vb + v_lane[j % C % 4] + 64 * (j % C / 4 * 4) + 16 * (j / C) * 2 * D;
      const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)at);
      const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(at + 8 * 2 * D));
      return __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    auto highest = [&](const f32x16_t* sc) __attribute__((always_inline)) {  // (a NaN score comes back through its exponential)
      float most = -INFINITY;
#pragma unroll
      for (int b = 0; b < B; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) most = fmaxf(most, sc[b][i]);
      return most;
    };
    // One block: its scores in sc, its values in vb; the next one's keys are in kb, its scores become
    // `ahead`.  The keys after that go to k_free, the next values to v_free.
    f32x16_t scores0[B], scores1[B];
    float most;                      // of the block's scores
    int page1, page2;                // the next block's page, and the one's after that
    uint32_t bad0, bad1, bad2;       // this block's bad groups, and those of the two
    auto turn = [&](int block, f32x16_t* sc, f32x16_t* ahead, const char* kb, char* k_free, char* vb,
                    char* v_free) __attribute__((always_inline)) {
      // this wavefront's part of the next keys and of these values has landed; past the barrier every
      // wavefront's has, and nobody reads the free arrays
      wait_vmem();
      __builtin_amdgcn_s_barrier();
      __builtin_amdgcn_sched_barrier(0);
      move_pages(block + 3);
      const int k0 = KEYS * block;
      const bool edge = is_edge(block, bad0);
      int odd = 0;
      if (edge) {
        // (what only edges need is worked out here, not kept in registers over the loop)
        int l = lane, p = position;
        asm volatile("" : "+v"(l), "+v"(p));
        // An infinity or a NaN among the values?  (a probability of zero must not meet one)
        uint32_t exponents = 0;
#pragma unroll
        for (int i = 0; i < L; ++i) {
          const u32x4_t w = *reinterpret_cast<const u32x4_t*>(vb + wave * MINE * 2 * D + 1024 * i + 16 * l);
#pragma unroll
          for (int e = 0; e < 4; ++e) exponents = max_pair(exponents, w[e] & 0x7f807f80u);
        }
        // (not __syncthreads_or, which loads the size of the workgroup)
        const uint64_t any = __ballot((exponents & 0xffffu) == 0x7f80u || exponents >> 16 == 0x7f80u);
        if (lane == 0) odd_waves[wave] = any != 0;
        __syncthreads();
        const int4 odds = *reinterpret_cast<const int4*>(odd_waves);
        odd = odds.x | odds.y | odds.z | odds.w;
        if (odd) {
#pragma unroll
          for (int i = 0; i < L; ++i) {
            u32x4_t* const at = reinterpret_cast<u32x4_t*>(vb + wave * MINE * 2 * D + 1024 * i + 16 * l);
            u32x4_t w = *at;
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = finite_pair(w[e], &exponents);
            *at = w;
          }
          __syncthreads();
        }
        // the query sees the keys that are less than `span` before its own
        const int own = p - k0 - 4 * (l >> 5);
        const uint32_t span = a.window ? a.window : 0x7fffffff;
#pragma unroll
        for (int b = 0; b < B; ++b)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int key = 32 * b + 8 * (i >> 2) + (i & 3);
            sc[b][i] = (uint32_t)(own - key) < span ? sc[b][i] : -INFINITY;
          }
        if (bad0)
#pragma unroll
          for (int b = 0; b < B; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) sc[b][i] = (bad0 >> (2 * b + (i >> 3))) & 1 ? -INFINITY : sc[b][i];
        most = max_xor32(highest(sc));
      }
      most *= a.scale_log2;
      if (__any(most > top + kSlack)) {
        const float higher = fmaxf(most, top), base = higher == -INFINITY ? 0.0f : higher;
        const float keep = __builtin_amdgcn_exp2f(top - base);
        top = higher;
        sum *= keep;
#pragma unroll
        for (int c = 0; c < C; ++c) o[c] *= keep;
      }
      const float base = top == -INFINITY ? 0.0f : top;
      // The next block's scores, and this one's probabilities between them; then the values, and the next
      // block's maximum between them.  A wavefront issues in order: each matrix instruction here is followed
      // by the reads for one a few later and by as much arithmetic as fits under it.  Left to the
      // compiler, which read each operand just before its instruction: 8192 tokens 576 us, now 523.
      constexpr int N = T * B, M = C * KEYS / 16, PAIRS = 8 * B;  // matrix instructions of either kind
      uint32_t k_at = k_lane;
      asm volatile("" : "+v"(k_at));  // (one register, and an instruction for each read's address)
      u32x4_t pw[KEYS / 16];
      bf16x8_t kf[kAhead], vf[kAheadV];
      __amdgpu_buffer_rsrc_t k_source, v_source;
      static_assert(2 + 2 * L <= N, "the loads have their steps");
      auto probabilities = [&](int step) __attribute__((always_inline)) {
#pragma unroll
        for (int e = step * PAIRS / (N + M / 2); e < (step + 1) * PAIRS / (N + M / 2); ++e) {
          const int b = e / 8, i = 2 * (e % 8);
          const float lo = __builtin_amdgcn_exp2f(fmaf(sc[b][i], a.scale_log2, -base));
          const float hi = __builtin_amdgcn_exp2f(fmaf(sc[b][i + 1], a.scale_log2, -base));
          sum += lo;
          sum += hi;
          pw[2 * b + i / 8][i / 2 % 4] = pack_bf16(lo, hi);
        }
      };
#pragma unroll
      for (int j = 0; j < kAhead - 1; ++j) kf[j] = key_operand(kb, k_at, j);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if (j + kAhead - 1 < N) kf[(j + kAhead - 1) % kAhead] = key_operand(kb, k_at, j + kAhead - 1);
#pragma unroll
        for (int i = 0; i < kAheadV; ++i)
          if (j == N - kAheadV / 2 + i / 2) vf[i] = value_operand(vb, i);
        ahead[j % B] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[j % kAhead], qf[j / B], j < B ? f32x16_t{} : ahead[j % B], 0, 0, 0);
        probabilities(j);
        // (the next loads: their addresses, then 1 KB at a time)
        if (j == 0) k_source = source(a.k_pages, page2, block + 2);
        if (j == 1) v_source = source(a.v_pages, page1, block + 1);
        if (j >= 2 && j < 2 + L) load_kb(k_source, j - 2, k_from, k_free);
        if (j >= 2 + L && j < 2 + 2 * L) load_kb(v_source, j - 2 - L, v_from, v_free);
        __builtin_amdgcn_sched_barrier(0);
      }
      most = -INFINITY;  // (a NaN score comes back through its exponential)
#pragma unroll
      for (int j = 0; j < M; ++j) {
        o[j % C] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[j % kAheadV], __builtin_bit_cast(bf16x8_t, pw[j / C]), o[j % C], 0, 0, 0);
        if (j + kAheadV < M) vf[j % kAheadV] = value_operand(vb, j + kAheadV);
        if (j < M / 2) {
          probabilities(N + j);
        } else {
#pragma unroll
          for (int e = (2 * j - M) * 16 * B / M; e < (2 * j + 2 - M) * 16 * B / M; ++e) most = fmaxf(most, ahead[e / 16][e % 16]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      most = max_xor32(most);
      asm volatile("" : "+v"(most));  // (worked out here, not where it is used)
      const uint32_t bad = bad0;
      page1 = page2;
      bad0 = bad1;
      bad1 = bad2;
      look_up(block + 3, &page2, &bad2);
      if (odd) {
        int l = lane, p = live ? position : -1;
        asm volatile("" : "+v"(l), "+v"(p));
        for (int r = 0; r < KEYS; ++r) {
          const int key = k0 + r;
          if (((bad >> (r >> 4)) & 1) || key < low || key > tile_last) continue;
          const int which = 16 * (r >> 5) + 4 * ((r >> 3) & 3) + (r & 3);
          uint32_t word = 0;
#pragma unroll
          for (int e = 0; e < PAIRS; ++e) word = which >> 1 == e ? pw[e / 4][e % 4] : word;
          const float mine = __uint_as_float(which & 1 ? word & 0xffff0000u : word << 16);
          const float pr = __shfl(mine, (l & 31) + 32 * ((r >> 2) & 1));
          const bool seen = key <= p && (!a.window || key > p - a.window);
          const uint16_t* const v = a.v_pages + ((((int64_t)table[key >> a.shift] * a.Hkv + head) << a.shift) + (key & mask)) * D;
#pragma unroll
          for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const uint32_t bits = v[32 * c + 8 * (i >> 2) + 4 * (l >> 5) + (i & 3)];
              if (seen && (bits & 0x7f80u) == 0x7f80u) o[c][i] += pr * bf16_bits_to_f32(bits);
              if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // (few registers: the loop above needs them)
            }
        }
      }
    };

    int page0;
    look_up(from, &page0, &bad0);
    look_up(from + 1, &page1, &bad1);
    look_up(from + 2, &page2, &bad2);
    load(a.k_pages, page0, from, k_from, k0l);
    load(a.k_pages, page1, from + 1, k_from, k1l);
    load(a.v_pages, page0, from, v_from, v0l);
#pragma unroll
    for (int t = 0; t < T; ++t) {
      u32x4_t w = {0u, 0u, 0u, 0u};
      if (live) w = *reinterpret_cast<const u32x4_t*>(a.q + (s.q.first + row) * a.ldq + q_head * D + 16 * t + 8 * h);
      qf[t] = __builtin_bit_cast(bf16x8_t, w);
    }
    wait_vmem();
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int t = 0; t < T; ++t) scores(k0l, k_lane, t, scores0);
    most = max_xor32(highest(scores0));
    for (int block = from; block < stop; block += 2) {
      turn(block, scores0, scores1, k1l, k0l, v0l, v1l);
      if (block + 1 < stop) turn(block + 1, scores1, scores0, k0l, k1l, v1l, v0l);
    }
    wait_vmem();  // the loads past the last block, before the LDS is given up
    sum = add_xor32(sum);
  }
  if (!live) return;
  if (splits == 1) {
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    uint16_t* const to = a.out + (s.q.first + row) * a.ldo + q_head * D + 4 * h;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const u32x2_t four = {pack_bf16(o[c][i] * inv, o[c][i + 1] * inv), pack_bf16(o[c][i + 2] * inv, o[c][i + 3] * inv)};
        *reinterpret_cast<u32x2_t*>(to + 32 * c + 2 * i) = four;
      }
    return;
  }
  const int64_t result = ((int64_t)(s.slot + s.split) * a.Hkv + head) * kTile + 32 * wave + n;
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int i = 0; i < 16; i += 4)
      *reinterpret_cast<float4*>(a.partial + result * D + 32 * c + 2 * i + 4 * h) =
          make_float4(o[c][i], o[c][i + 1], o[c][i + 2], o[c][i + 3]);
  if (h == 0) a.state[result] = make_float2(top, sum);
}

// After tile_workgroup: a workgroup per split again, which takes its share of the tile's queries.
template <int D>
__device__ __forceinline__ void merge_tile(const AttendArgs& a, int index, MergeSpace<D>& space) {
  constexpr int KEYS = tile_block<D>();
  const int head = index % a.Hkv;
  Lanes<kTile, KEYS> lanes(a);
  const int chunk = tile_chunk<D>(lanes, kTileLeast / KEYS);
  const TilePart s = find_part(lanes, index / a.Hkv, chunk);
  if (s.request < 0 || s.splits == 1) return;
  int tile_first, tile_last, low, block0;
  const int all = tile_blocks<KEYS>(a, s.q, s.place, &tile_first, &tile_last, &low, &block0);
  const int splits = ceil_of(ceil_of(all, 1 << a.grain), chunk);
  if (splits <= 1 || s.split >= splits) return;
  const int64_t slot = s.slot;
  merge_part<kTile, D>(a, s.q, s.place, head, s.split, splits, splits, [&](int i) { return slot + i; }, space);
}

// A launch for requests of few queries, of many, or of both: `few_groups` and `many_groups` workgroups, those
// of many first: they are the longest, and the others, which wait for memory, share the CUs with the
// last of them.  A mixed batch of 24 requests in 87 us, 93 in turns of 32 and 102 the other way round.  (In turns
// of eight, one workgroup of each kind per XCD, half of an XCD's shader engines got all of the tiles: 144
// against 117 in turns of 32.)
enum { kFew = 1, kMany = 2, kFewOnce = 4 };  // (kFewOnce: kFew, whose keys and values one workgroup reads)

template <int D, int KINDS>
__global__ __launch_bounds__(kThreads, D == 128 ? 2 : 1) void attend_kernel(AttendArgs few, AttendArgs many, int many_groups) {
  __shared__ __attribute__((aligned(16))) char lds0[kArray], lds1[kArray];
  __shared__ float tops[4][16], sums[4][16];
  constexpr bool ONCE = KINDS == kFewOnce, FEW = KINDS == kFew || ONCE;
  if (FEW && D == 128) {
    rows_workgroup<D, ONCE>(few, blockIdx.x, lds0, lds1, nullptr, nullptr, tops, sums);
  } else {
    __shared__ __attribute__((aligned(16))) char lds2[kArray], lds3[kArray];
    const bool is_few = FEW || (KINDS == (kFew | kMany) && (int)blockIdx.x >= many_groups);
    const int index = KINDS == (kFew | kMany) && is_few ? blockIdx.x - many_groups : blockIdx.x;
    if (KINDS != kMany && is_few)
      rows_workgroup<D, ONCE>(few, index, lds0, lds1, lds2, lds3, tops, sums);
    else if (KINDS & kMany)
      tile_workgroup<D>(many, index, lds0, lds1, lds2, lds3);
  }
}

template <int D>
__global__ __launch_bounds__(kThreads) void merge_kernel(AttendArgs few, AttendArgs many, int few_groups) {
  __shared__ MergeSpace<D> space;
  if ((int)blockIdx.x < few_groups)
    merge_rows<D>(few, blockIdx.x, space);
  else
    merge_tile<D>(many, blockIdx.x - few_groups, space);
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

// A launch for the requests with `fewest` to `most` queries of a KV head, in tiles of `width` (0: none).  Per
// KV head: the tiles there may be, the parts their work is shared out in, the workgroups, and the partial
// results.
struct AttendLaunch {
  int64_t tiles, units, workgroups, slots;
  int32_t fewest, most, width;
};

struct AttendPlan {
  AttendLaunch few, many;
  bool once;  // one row for each request: its keys and values are read by one workgroup per KV head
};

// Of more keys and values than the last-level cache holds (256 MB), which are read once, nothing is kept in the
// caches: 32 steps over up to 8000 tokens (669 MB) in 115 us, 125 with plain loads.  Fewer stay there for
// the next call (32768 tokens, 134 MB: 31 us, and 33), and two tiles of a request share them (8 tokens each
// of four requests: 27 us, and 32).
constexpr int64_t kCached = 256ll << 20;

// The keys (of heads of 128) up to which tiles of few queries are left whole, one workgroup each and no second launch,
// rather than cut into equal parts of all their blocks.  One request: 512 keys 9.3 us and 11.3 cut, 777 equal, 1024
// 13.7 and 11.9; eight requests (64 workgroups): 512 keys 9.5 and 15.3, 1024 13.8 and 16.5, 2000 22.8
// and 22.1; 32 requests: 1024 17.8 and 23.8, 2000 29 and 33, 4000 68 and 62.  Longer requests of the launch fill the
// card with theirs: their queries count as well (a prompt of 1000 tokens in tables of 2048, 25 and 27).
int64_t rows_alone(int64_t workgroups) { return workgroups >= 128 ? 2048 : workgroups >= 32 ? 1024 : 768; }

// Requests of up to kRowsMost queries go to rows_workgroup, longer ones to tile_workgroup.  The
// host knows the sums only: where the average request stays within kRowsMost the first serves all, a chunk among
// many steps too (63 steps and a chunk of 449 tokens, all over 8000, 539 us; 323 and 96 in calls of their own).
// A workgroup with nothing to do costs its launch all the same (1000 of them 10 us): no more are launched than
// the longest context can give work to.  The device makes do with what there is, whatever the contexts.
AttendPlan plan_attend(int32_t rows, int32_t requests, int32_t Hq, int32_t Hkv, int32_t head_dim, int64_t max_context,
                       int32_t window) {
  const int64_t queries = (int64_t)rows * (Hq / Hkv), with = std::min(rows, requests);
  AttendPlan p;
  memset(&p, 0, sizeof(p));
  const bool all_few = queries <= kRowsMost * with, some_few = requests > 1;
  const int resident = head_dim == 128 ? kWorkgroups<128> : kWorkgroups<256>;
  // (a window's keys before the rows' own, and the parts of blocks at both ends)
  const int64_t keys = window ? std::min(max_context, (int64_t)window + rows) : max_context;
  p.once = all_few && rows <= requests && Hq / Hkv <= kRowsTile && with * keys * Hkv * head_dim * 4 > kCached;
  if (all_few || some_few) {
    AttendLaunch& l = p.few;
    l.width = kRowsTile;
    l.most = all_few ? INT32_MAX : kRowsMost;
    const int64_t all = with + queries / kRowsTile;  // of all rows: at most one part-full tile for each request
    // (beside longer requests only those of the others are here, which have at most kRowsMost queries)
    l.tiles = all_few ? all : std::min<int64_t>(all, (int64_t)with * (kRowsMost / kRowsTile));
    const int64_t line = l.tiles * (keys / kRowsBlock + 2);
    l.units = std::min<int64_t>(ceil_div(resident, Hkv),
                                ceil_div(line, kRowsLeast));
    if (keys * head_dim <= rows_alone(all * Hkv) * 128) l.units = 0;
    l.workgroups = l.units ? l.units : l.tiles;
    l.slots = l.units > 1 ? 2 * l.units : 0;  // a part's first tile and its last
  }
  if (!all_few) {
    AttendLaunch& l = p.many;
    l.width = kTile;
    l.fewest = some_few ? kRowsMost + 1 : 0;
    l.most = INT32_MAX;
    l.tiles = with + queries / kTile;
    const int keys_of = head_dim == 128 ? tile_block<128>() : tile_block<256>();
    // the chunk is the work over the units and a tile has its blocks over the chunk, rounded up, of splits: no more
    // than the units and the tiles together
    const int64_t sure = (queries - (some_few ? kRowsMost * with : 0)) / kTile;  // tiles that there are at least
    const bool whole = keys <= kTileAlone || (keys <= 2 * kTileAlone && 4 * sure * Hkv >= kCUs);
    const int64_t splits = whole ? 1 : ceil_div(keys / keys_of + 2, kTileLeast / keys_of);
    l.workgroups = std::min(ceil_div(resident, Hkv) + l.tiles, l.tiles * splits);
    l.units = l.workgroups - l.tiles;
    l.slots = std::min(l.workgroups, 2 * l.units);
  }
  return p;
}

// The partial results' part of a launch's workspace, then their maxima and sums.
size_t attend_space(const AttendLaunch& l, int32_t Hkv, int32_t head_dim) {
  return (size_t)l.slots * Hkv * l.width * (head_dim * 4 + 8);
}

// log2 of the blocks that the device counts as one: 0 unless the sums of the blocks of all tiles could pass 30 bits.
int attend_grain(const AttendLaunch& l, int64_t max_tokens) {
  const double most = (double)l.tiles * (double)(max_tokens / 32 + 1);
  int grain = 0;
  while (most / (double)(1ll << grain) >= (double)(1 << 30)) ++grain;
  return grain;
}

// A launch's fields of the arguments, its part of the workspace starting at `space`.
AttendArgs with_launch(AttendArgs a, const AttendLaunch& l, int head_dim, char* space) {
  a.fewest = l.fewest;
  a.most = l.most;
  a.units = (int32_t)l.units;
  a.slots = (int32_t)l.slots;
  a.grain = attend_grain(l, (int64_t)a.columns << a.shift);
  a.partial = reinterpret_cast<float*>(space);
  a.state = reinterpret_cast<float2*>(a.partial + (size_t)l.slots * a.Hkv * l.width * head_dim);
  return a;
}

template <int D>
void launch_attend(const AttendPlan& p, char* space, const AttendArgs& args, hipStream_t stream) {
  const AttendArgs few = with_launch(args, p.few, D, space);
  const AttendArgs many = with_launch(args, p.many, D, space + attend_space(p.few, args.Hkv, D));
  const int few_groups = (int)p.few.workgroups * args.Hkv, many_groups = (int)p.many.workgroups * args.Hkv;
  const auto kernel = !p.many.width  ? p.once ? attend_kernel<D, kFewOnce> : attend_kernel<D, kFew>
                      : !p.few.width ? attend_kernel<D, kMany>
                                     : attend_kernel<D, (kFew | kMany)>;
  hipLaunchKernelGGL(kernel, dim3(few_groups + many_groups), dim3(kThreads), 0, stream, few, many, many_groups);
  const int few_merges = p.few.slots ? (int)(p.few.units - 1) * args.Hkv : 0, many_merges = (int)p.many.slots * args.Hkv;
  if (few_merges + many_merges)
    hipLaunchKernelGGL(merge_kernel<D>, dim3(few_merges + many_merges), dim3(kThreads), 0, stream, few, many, few_merges);
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
  // at most this many columns: those that the rows fill, and two part-full ones for each request
  const int64_t most = chunk->rows / cache->page_size + 2 * (int64_t)cache->requests;
  const auto kernel = most <= 2 * kReserveThreads ? reserve_kernel<1, 4, 4096> : reserve_kernel<4, 16, 24576>;
  hipLaunchKernelGGL(kernel, dim3(1), dim3(kReserveThreads), 0, st, a);
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
  // columns of a workgroup: all where they fit, else 16 (or what fits), a 64-byte piece of a row
  int log2_width = 0;
  while ((1 << log2_width) < cache->columns) ++log2_width;
  const bool whole = ((int64_t)cache->requests << log2_width) <= kReorderEntries;
  if (!whole)
    for (log2_width = 4; (cache->requests << log2_width) > kReorderEntries;) --log2_width;
  hipLaunchKernelGGL(reorder_kernel, dim3(ceil_div(cache->columns, 1 << log2_width)), dim3(kReorderThreads), 0, st,
                     cache->tables, cache->lengths, cache->refs, parents, cache->requests, cache->columns, cache->pages,
                     __builtin_ctz(cache->page_size), log2_width, whole ? 1 : 0);
  if (!whole)
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
  hipLaunchKernelGGL(kernel, dim3(rows), dim3(kWriteThreads), 0, st, q, ldq, k, ldk, v, ldv, q_norm, k_norm, positions, slots,
                     q_out, ldo, k_pages, v_pages, Hq, Hkv, shift, (int64_t)pages << shift, log2(theta), eps);
  return launched("paged write");
}

size_t imq_paged_attention_workspace(int32_t rows, int32_t requests, int32_t Hq, int32_t Hkv, int32_t head_dim,
                                     int32_t max_context, int32_t window) {
  if (check_heads(rows, Hq, Hkv, head_dim) != IMQ_OK || rows == 0 || requests < 1 || max_context < 1) return 0;
  const AttendPlan plan = plan_attend(rows, requests, Hq, Hkv, head_dim, max_context, window);
  return attend_space(plan.few, Hkv, head_dim) + attend_space(plan.many, Hkv, head_dim);
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
  if (window >= (int64_t)columns * page_size) window = 0;  // (all that there can be: up to 2^30, so that sums of it stay in range)
  const AttendPlan plan = plan_attend(rows, requests, Hq, Hkv, head_dim,
                                      std::min<int64_t>(max_context, (int64_t)columns * page_size), window);
  const size_t nbytes = attend_space(plan.few, Hkv, head_dim) + attend_space(plan.many, Hkv, head_dim);
  if (nbytes && (!workspace || !aligned(workspace, 16) || workspace_bytes < nbytes))
    return fail(IMQ_EINVAL, "the workspace is too small or not 16-byte aligned");
  AttendArgs a{q, k_pages, v_pages, tables, starts, ends, out, ldq, ldo, nullptr, nullptr, rows, requests, columns, pages,
               __builtin_ctz(page_size), Hq, Hkv, Hq / Hkv, window, 0, 0, 0, 0, 0, scale * 1.44269504088896340736f};
  char* const space = static_cast<char*>(workspace);
  if (head_dim == 128)
    launch_attend<128>(plan, space, a, static_cast<hipStream_t>(stream));
  else
    launch_attend<256>(plan, space, a, static_cast<hipStream_t>(stream));
  return launched("paged attention");
}

}  // extern "C"
