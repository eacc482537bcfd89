// Block tables and slot maps from request lengths: one launch per step.
//
// Request b holds l0 = seq_lens[b] tokens in p0 = ceil(l0 / ps) pages and goes
// to l1 = max(l0 + new_lens[b], 0) tokens in p1 = ceil(l1 / ps) pages (at most
// the table's width P).  Pages given back (p1 .. p0 - 1 of a request that
// shrinks) are pushed on the stack of free pages, request by request; then the
// pages that growing requests need are popped from its top, request by request.
// So with the exclusive prefix sums RO (pages given back) and GO (pages needed)
// over the requests, the g-th page taken is stack entry A - 1 - g, A = free_count
// + all pages given back: an entry of free_pages, or, above free_count, a page
// given back by this very call, read from its owner's row of the table.
//
// Everything is a function of the inputs, and nothing that is written is read:
// rows are written at and above p0 only where a request grows, the stack at and
// above free_count, and seq_lens and free_count not at all.  So every workgroup
// forms the prefix sums by itself (B <= 4096 lengths: 32 KiB from L2) instead of
// waiting for one that does, any number of workgroups shares the tokens, and a
// call repeated on the same inputs writes the same values.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "common.h"

namespace fs {

constexpr int kPlanThreads = 512;
constexpr int kPlanMaxRequests = 4096;
constexpr int kPlanMaxGroups = 256;
constexpr uint32_t kMost = INT_MAX;                // sums stop here

__device__ __forceinline__ uint32_t sum(uint32_t x, uint32_t y) { return min(x + y, kMost); }

// A request's step; everything fits 32 bits (P * page_size < 2^31).
struct PlanReq {
  uint32_t l0, l1, n, p0, p1;
  __device__ __forceinline__ PlanReq(const fs_plan_args& a, int b) {
    const uint32_t ps = a.page_size, cap = (uint32_t)a.P * ps;
    const int d = a.new_lens[b];
    l0 = min((uint32_t)max(a.seq_lens[b], 0), cap);
    n = max(d, 0);
    l1 = d >= 0 ? l0 + n : l0 - min(l0, 0u - (uint32_t)d);
    p0 = pages(l0, ps);
    p1 = min(pages(l1, ps), (uint32_t)a.P);
  }
  static __device__ __forceinline__ uint32_t pages(uint32_t tokens, uint32_t ps) {
    const uint32_t q = tokens / ps;
    return q + (q * ps != tokens);
  }
  __device__ __forceinline__ uint32_t grow() const { return p1 > p0 ? p1 - p0 : 0; }
  __device__ __forceinline__ uint32_t give() const { return p0 > p1 ? p0 - p1 : 0; }
};

// Inclusive prefix sum over the wave, held at kMost.
__device__ __forceinline__ uint32_t wave_upto(uint32_t x) {
  auto from = [&](auto ctrl, auto rows) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
  };
#define FS_STEP(ctrl, rows) x = sum(x, from(std::integral_constant<int, ctrl>(), std::integral_constant<int, rows>()))
  FS_STEP(0x111, 0xf);                             // row_shr 1, 2, 4, 8: rows of 16 lanes
  FS_STEP(0x112, 0xf);
  FS_STEP(0x114, 0xf);
  FS_STEP(0x118, 0xf);
  FS_STEP(0x142, 0xa);                             // row_bcast 15, 31: the rows below
  FS_STEP(0x143, 0xc);
#undef FS_STEP
  return x;
}

// Largest b with cum[b] <= x, for an exclusive prefix cum[0..B] with cum[B] > x.
__device__ __forceinline__ int owner(const uint32_t* cum, int B, uint32_t x) {
  int lo = 0, hi = B;                              // cum[lo] <= x < cum[hi]
  while (hi - lo > 1) {
    const int m = (lo + hi) >> 1;
    if (cum[m] <= x) lo = m;
    else hi = m;
  }
  return lo;
}

__global__ __launch_bounds__(kPlanThreads) void plan_kernel(fs_plan_args a) {
  constexpr int NW = kPlanThreads / 64;
  // exclusive prefix sums of new tokens, pages needed and pages given back, and each request's tokens and pages before
  extern __shared__ uint32_t lds[];
  uint32_t *cu = lds, *go = cu + a.B + 1, *ro = go + a.B + 1, *l0 = ro + a.B + 1, *p0 = l0 + a.B;
  __shared__ uint32_t part[3][NW], lost_part[NW];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int per = (a.B + kPlanThreads - 1) / kPlanThreads;
  const int b0 = min(tid * per, a.B), b1 = min(b0 + per, a.B);
  const int fc = min(max(a.free_count[0], 0), a.F);
  uint32_t s[3] = {0, 0, 0};
  for (int b = b0; b < b1; ++b) {
    const PlanReq r(a, b);
    l0[b] = r.l0;
    p0[b] = r.p0;
    cu[b] = r.n;                                   // until the sums are known
    go[b] = r.l1;
    ro[b] = r.p1;
    s[0] = sum(s[0], r.n);
    s[1] = sum(s[1], r.grow());
    s[2] = sum(s[2], r.give());
  }
  uint32_t at[3], tot[3];
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    const uint32_t x = wave_upto(s[i]);
    if (lane == 63) part[i][wave] = x;
    at[i] = __builtin_amdgcn_update_dpp(0, (int)x, 0x138, 0xf, 0xf, false);   // wave_shr 1: the lanes below
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      before = w == wave ? all : before;
      all = sum(all, part[i][w]);
    }
    at[i] = sum(at[i], before);
    tot[i] = all;
  }
  const uint32_t avail = min(sum(fc, tot[2]), (uint32_t)a.F), ps = a.page_size;
  uint32_t lost = 0;
  for (int b = b0; b < b1; ++b) {
    const uint32_t n = cu[b], l1 = go[b], q0 = p0[b], q1 = ro[b], grow = q1 > q0 ? q1 - q0 : 0;
    const uint32_t got = min(avail > at[1] ? avail - at[1] : 0, grow), held = max(l0[b], (q0 + got) * ps);
    lost = sum(lost, l1 > held ? min(l1 - held, kMost) : 0);
    if (blockIdx.x == 0) {
      a.cu_lens[b] = at[0];
      a.seq_lens_out[b] = min(l1, kMost);
    }
    cu[b] = at[0];
    go[b] = at[1];
    ro[b] = at[2];
    at[0] = sum(at[0], n);
    at[1] = sum(at[1], grow);
    at[2] = sum(at[2], q0 > q1 ? q0 - q1 : 0);
  }
  if (tid == 0) {
    cu[a.B] = tot[0];
    go[a.B] = tot[1];
    ro[a.B] = tot[2];
  }
  lost = wave_upto(lost);
  if (lane == 63) lost_part[wave] = lost;
  __syncthreads();
  if (blockIdx.x == 0 && tid == 0) {
    uint32_t l = 0;
    for (int w = 0; w < NW; ++w) l = sum(l, lost_part[w]);
    a.cu_lens[a.B] = tot[0];
    a.lacking[0] = l;
    a.free_count_out[0] = avail > tot[1] ? avail - tot[1] : 0;
  }
  // pages that request b keeps or comes to (one of the two sums stands still)
  auto pages_after = [&](int b) { return p0[b] + (go[b + 1] - go[b]) - (ro[b + 1] - ro[b]); };
  // entry r of the pages given back: its owner's row of the table, above what the owner keeps
  auto given_page = [&](uint32_t r) {
    const int b = owner(ro, a.B, r);
    return a.block_table[(int64_t)b * a.t_sb + pages_after(b) + r - ro[b]];
  };
  // the g-th page taken, -1 past the stack's end
  auto taken_page = [&](uint32_t g) {
    if (g >= avail) return -1;
    const uint32_t k = avail - 1 - g;
    return k < (uint32_t)fc ? a.free_pages[k] : given_page(k - fc);
  };
  // The tokens, the pages taken and those given back are one list of items: few threads have more than one, so
  // their searches and loads wait side by side.
  const uint32_t T = a.T;
  const uint64_t items = (uint64_t)T + tot[1] + tot[2];
  for (uint64_t x = (uint64_t)blockIdx.x * kPlanThreads + tid; x < items; x += (uint64_t)gridDim.x * kPlanThreads) {
    if (x < T) {
      const uint32_t j = (uint32_t)x;
      int p = -1;
      int64_t slot = -1;
      if (j < tot[0]) {
        const int b = owner(cu, a.B, j);
        const uint32_t pos = l0[b] + (j - cu[b]), pg = pos / ps;   // below 2^32
        int page = -1;
        if (pg < p0[b]) page = a.block_table[(int64_t)b * a.t_sb + pg];
        else if (pg < pages_after(b)) page = taken_page(go[b] + pg - p0[b]);
        p = min(pos, kMost);
        if (page >= 0) slot = (int64_t)page * ps + (pos - pg * ps);
      }
      a.positions[j] = p;
      a.slots[j] = slot;
    } else if (x - T < tot[1]) {
      const uint32_t g = (uint32_t)(x - T);
      const int b = owner(go, a.B, g);
      a.block_table[(int64_t)b * a.t_sb + p0[b] + g - go[b]] = taken_page(g);
    } else {
      const uint32_t r = (uint32_t)(x - T - tot[1]);
      if (fc + r < (uint32_t)a.F) a.free_pages[fc + r] = given_page(r);
    }
  }
}

}  // namespace fs

using namespace fs;

extern "C" int fs_plan(const fs_plan_args* a, void* stream) {
  FS_CHECK_ARG(a != nullptr, "fs_plan: null args");
  FS_CHECK_ARG(a->block_table && a->seq_lens && a->new_lens && a->free_pages && a->free_count && a->cu_lens &&
                   a->seq_lens_out && a->positions && a->slots && a->free_count_out && a->lacking,
               "fs_plan: null tensor pointer");
  FS_CHECK_ARG(a->B >= 1 && a->P >= 1 && a->F >= 1 && a->T >= 0, "fs_plan: B=%d requests, P=%d pages per request, "
               "F=%d pages, T=%d tokens", a->B, a->P, a->F, a->T);
  FS_CHECK_ARG(a->page_size >= 1 && (int64_t)a->P * a->page_size <= INT_MAX && a->t_sb >= a->P,
               "fs_plan: page size %d, table of %d pages with row stride %lld", a->page_size, a->P, (long long)a->t_sb);
  FS_CHECK_SUPPORTED(a->B <= kPlanMaxRequests, "fs_plan: %d requests > %d", a->B, kPlanMaxRequests);
  // an item to a thread, with some for the pages that change hands
  const int64_t items = (int64_t)a->T + a->T / a->page_size + a->B;
  const int groups = (int)std::min<int64_t>((items + kPlanThreads - 1) / kPlanThreads, kPlanMaxGroups);
  const size_t bytes = (5 * (size_t)a->B + 3) * sizeof(uint32_t);
  if (int rc = fs_host::allow_dynamic_lds(plan_kernel, bytes, "fs_plan")) return rc;
  plan_kernel<<<groups, kPlanThreads, bytes, (hipStream_t)stream>>>(*a);
  return fs_host::launch_status("fs_plan");
}
