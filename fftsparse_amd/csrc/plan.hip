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
#include <climits>

#include "common.h"

namespace fs {

constexpr int kPlanThreads = 512;
constexpr int kPlanMaxRequests = 4096;
constexpr int kPlanTokensPerGroup = 1024;
constexpr int kPlanMaxGroups = 256;

struct PlanReq {
  int64_t l0, l1;
  int n, p0, p1;
};

__device__ __forceinline__ PlanReq plan_req(const fs_plan_args& a, int b) {
  PlanReq r;
  const int64_t cap = (int64_t)a.P * a.page_size;
  r.l0 = min(max((int64_t)a.seq_lens[b], (int64_t)0), cap);
  const int64_t d = a.new_lens[b];
  r.l1 = max(r.l0 + d, (int64_t)0);
  r.n = (int)max(d, (int64_t)0);
  r.p0 = (int)((r.l0 + a.page_size - 1) / a.page_size);
  r.p1 = (int)min((r.l1 + a.page_size - 1) / a.page_size, (int64_t)a.P);
  return r;
}

// Largest b with cum[b] <= x, for an exclusive prefix cum[0..B] with cum[B] > x.
__device__ __forceinline__ int owner(const int* cum, int B, int x) {
  int lo = 0, hi = B;                              // cum[lo] <= x < cum[hi]
  while (hi - lo > 1) {
    const int m = (lo + hi) >> 1;
    if (cum[m] <= x) lo = m;
    else hi = m;
  }
  return lo;
}

__global__ __launch_bounds__(kPlanThreads) void plan_kernel(fs_plan_args a) {
  // exclusive prefixes of new tokens, pages needed and pages given back; the
  // sums are formed in 64 bits and held at most at INT_MAX
  extern __shared__ int lds[];
  int* cu = lds;
  int* go = cu + a.B + 1;
  int* ro = go + a.B + 1;
  __shared__ int64_t part[3][kPlanThreads / 64];
  __shared__ int64_t lost_part[kPlanThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int per = (a.B + kPlanThreads - 1) / kPlanThreads;
  const int b0 = min(tid * per, a.B), b1 = min(b0 + per, a.B);
  int64_t s[3] = {0, 0, 0};
  for (int b = b0; b < b1; ++b) {
    const PlanReq r = plan_req(a, b);
    s[0] += r.n;
    s[1] += max(r.p1 - r.p0, 0);
    s[2] += max(r.p0 - r.p1, 0);
  }
  int64_t inc[3];
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    inc[i] = s[i];
    for (int o = 1; o < 64; o <<= 1) {
      const int64_t v = __shfl_up(inc[i], o, 64);
      if (lane >= o) inc[i] += v;
    }
    if (lane == 63) part[i][wave] = inc[i];
  }
  __syncthreads();
  int64_t pos[3], tot[3];
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    int64_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kPlanThreads / 64; ++w) {
      if (w < wave) before += part[i][w];
      all += part[i][w];
    }
    pos[i] = before + inc[i] - s[i];
    tot[i] = all;
  }
  auto cap = [](int64_t v) { return (int)min(v, (int64_t)INT_MAX); };
  const int fc = min(max(a.free_count[0], 0), a.F);
  const int avail = (int)min((int64_t)fc + tot[2], (int64_t)a.F);
  int64_t lost = 0;
  for (int b = b0; b < b1; ++b) {
    const PlanReq r = plan_req(a, b);
    cu[b] = cap(pos[0]);
    go[b] = cap(pos[1]);
    ro[b] = cap(pos[2]);
    const int64_t grow = max(r.p1 - r.p0, 0);
    const int64_t got = min(max((int64_t)avail - pos[1], (int64_t)0), grow);
    lost += max(r.l1 - max(r.l0, (r.p0 + got) * a.page_size), (int64_t)0);
    if (blockIdx.x == 0) {
      a.cu_lens[b] = cap(pos[0]);
      a.seq_lens_out[b] = cap(r.l1);
    }
    pos[0] += r.n;
    pos[1] += grow;
    pos[2] += max(r.p0 - r.p1, 0);
  }
  if (tid == 0) {
    cu[a.B] = cap(tot[0]);
    go[a.B] = cap(tot[1]);
    ro[a.B] = cap(tot[2]);
  }
  if (blockIdx.x == 0) {
    for (int o = 32; o > 0; o >>= 1) lost += __shfl_xor(lost, o, 64);
    if (lane == 0) lost_part[wave] = lost;
  }
  __syncthreads();
  if (blockIdx.x == 0 && tid == 0) {
    int64_t l = 0;
    for (int w = 0; w < kPlanThreads / 64; ++w) l += lost_part[w];
    a.cu_lens[a.B] = cap(tot[0]);
    a.lacking[0] = cap(l);
    a.free_count_out[0] = (int)max((int64_t)avail - tot[1], (int64_t)0);
  }
  const int total = cu[a.B], grown = go[a.B], given = ro[a.B];
  // entry r of the pages given back: its owner's row of the table, above what the owner keeps
  auto given_page = [&](int r) {
    const int b = owner(ro, a.B, r);
    return a.block_table[(int64_t)b * a.t_sb + plan_req(a, b).p1 + r - ro[b]];
  };
  // the g-th page taken, -1 past the stack's end
  auto taken_page = [&](int g) {
    const int at = avail - 1 - g;
    if (at < 0) return -1;
    return at < fc ? a.free_pages[at] : given_page(at - fc);
  };
  const int step = gridDim.x * kPlanThreads, first = blockIdx.x * kPlanThreads + tid;
  for (int j = first; j < a.T; j += step) {
    int p = -1;
    int64_t slot = -1;
    if (j < total) {
      const int b = owner(cu, a.B, j);
      const PlanReq r = plan_req(a, b);
      const int64_t at = r.l0 + (j - cu[b]);
      const int64_t pg = at / a.page_size;
      int page = -1;
      if (pg < r.p0) page = a.block_table[(int64_t)b * a.t_sb + pg];
      else if (pg < r.p1) page = taken_page(go[b] + (int)pg - r.p0);
      p = cap(at);
      if (page >= 0) slot = (int64_t)page * a.page_size + at % a.page_size;
    }
    a.positions[j] = p;
    a.slots[j] = slot;
  }
  for (int64_t g = first; g < grown; g += step) {
    const int b = owner(go, a.B, (int)g);
    a.block_table[(int64_t)b * a.t_sb + plan_req(a, b).p0 + (int)g - go[b]] = taken_page((int)g);
  }
  for (int64_t r = first; r < given && fc + r < a.F; r += step) a.free_pages[fc + r] = given_page((int)r);
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
  const int groups = min(max((a->T + kPlanTokensPerGroup - 1) / kPlanTokensPerGroup, 1), kPlanMaxGroups);
  const size_t bytes = 3 * (size_t)(a->B + 1) * sizeof(int);
  plan_kernel<<<groups, kPlanThreads, bytes, (hipStream_t)stream>>>(*a);
  return fs_host::launch_status("fs_plan");
}
