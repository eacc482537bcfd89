// Trees of drafted tokens: their positions and masks, the path that the model's choices keep, and
// the kept tokens' rows moved to their places in the cache.
//
// All three are bound by latency: a batch's tokens are some kilobytes, so what counts is the
// chain of loads that wait for each other.  One workgroup takes a request (its lengths, then its tokens,
// side by side).  Lines of parents and of children are followed in LDS, one by one at first, as far as trees go, and then by
// doubling: each round every token takes over what the token that it points to has, and that token's pointer, so a
// line of d takes log2 d rounds.  (One by one alone, a line of 1024 took 386 us for the masks and 55 for the path, 37
// and 12 so; by doubling alone trees of 16 took 4.2 and 4.5 us, 3.4 and 2.6 so.)
#include <algorithm>
#include <climits>
#include <new>
#include <utility>
#include <vector>

#include "common.h"

namespace fs {

constexpr int kTreeThreads = 256;
constexpr int kTreeMost = 1024;                    // tokens of a request that are looked at

// Request b's rows c0 .. c0 + n - 1, within 0 .. T; n <= 0: none.
struct TreeRows {
  int c0, n;
  __device__ __forceinline__ TreeRows(const int32_t* cu, int b, int T) {
    c0 = min(max(cu[b], 0), T);
    n = min(max(cu[b + 1], 0), T) - c0;
  }
};

// f of the rows behind the last request's, and before the first one's (a batch's later requests taken alone).
template <typename F>
__device__ __forceinline__ void rows_of_none(const int32_t* cu, int B, int T, F f) {
  const int c0 = min(max(cu[0], 0), T), c1 = min(max(cu[B], 0), T);
  for (int t = threadIdx.x; t < c0; t += kTreeThreads) f(t);
  for (int t = max(c0, c1) + (int)threadIdx.x; t < T; t += kTreeThreads) f(t);
}

constexpr int kSteps = 16;                         // one by one

// The k lowest of x's set bits (k below 1: none).
__device__ __forceinline__ uint64_t low_bits(uint64_t x, int k) {
  if (k >= (int)__popcll(x)) return x;
  int at = 0;                                      // the place of the bit after them
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) {
    const int c = (int)__popcll(x >> at & ((1ull << s) - 1));
    at += c <= k ? s : 0;
    k -= c <= k ? c : 0;
  }
  return x & ((1ull << at) - 1);
}

// rows[w][t]: word w of token t's mask.  After k rounds it holds t and its ancestors less than 16 2^k away, and up[t] is the one
// 16 2^k away.  Ancestors come in falling order, so the steps write each word once.  In a round a row may take over one that
// has grown in the same round already: what it gets beyond is ancestors as well.
// A parent's number is below its child's, so a row's bits stand in the order of the positions: a window leaves the row's highest
// bits, and the first tokens its lowest (256 trees of 4 to 250 tokens 6.2 us under a window and 4.9 without, a line of 1024 50 and 36).
__global__ __launch_bounds__(kTreeThreads) void tree_plan_kernel(fs_tree_plan_args a) {
  extern __shared__ uint64_t rows[];
  const int cap = 64 * a.words;                    // tokens of a tree
  int* par = reinterpret_cast<int*>(rows + (size_t)a.words * cap);
  const int tid = threadIdx.x, b = blockIdx.x;
  if (b == a.B) {                                  // rows that no request has
    rows_of_none(a.cu_lens, a.B, a.T, [&](int t) {
      a.positions[t] = -1;
      for (int w = 0; w < a.words; ++w) a.mask[(int64_t)t * a.words + w] = 0;
    });
    return;
  }
  const TreeRows r(a.cu_lens, b, a.T);
  const int64_t first = (int64_t)a.seq_lens[b] - r.n;
  const int most = min(r.n, cap);
  for (int t = tid; t < most; t += kTreeThreads) par[t] = a.parents[r.c0 + t];
  __syncthreads();
  constexpr int PER = kTreeMost / kTreeThreads;
  int up[PER];
  bool more = false;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int t = tid + i * kTreeThreads;
    up[i] = -1;
    if (t >= most) continue;
    int at = t, w = a.words;
    uint64_t word = 0;
    for (int s = 0; s < kSteps && at >= 0; ++s) {
      if (at >> 6 != w) {
        if (w < a.words) rows[w * cap + t] = word;
        while (--w > at >> 6) rows[w * cap + t] = 0;
        word = 0;
      }
      word |= 1ull << (at & 63);
      const int p = par[at];
      at = p < at ? p : -1;                        // a parent below 0, or not below the token: none
    }
    rows[w * cap + t] = word;
    while (--w >= 0) rows[w * cap + t] = 0;
    up[i] = max(at, -1);
    more |= at >= 0;
  }
  if (__syncthreads_or(more)) {
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (tid + i * kTreeThreads < most) par[tid + i * kTreeThreads] = up[i];   // now: the token that it is followed to
  }
  while (__syncthreads_or(more)) {
    int next[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int t = tid + i * kTreeThreads, p = t < most ? par[t] : -1;
      next[i] = -1;
      if (p < 0) continue;
      for (int w = 0; w <= p >> 6; ++w) rows[w * cap + t] |= rows[w * cap + p];
      next[i] = par[p];
    }
    __syncthreads();
    more = false;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int t = tid + i * kTreeThreads;
      if (t < most) par[t] = next[i];
      more |= next[i] >= 0;
    }
  }
  for (int t = tid; t < r.n; t += kTreeThreads) {
    int depth = -1;
    if (a.window == 0) {
      for (int w = 0; w < a.words; ++w) {
        const uint64_t x = t < most ? rows[w * cap + t] : 0;
        a.mask[(int64_t)(r.c0 + t) * a.words + w] = (int64_t)x;
        depth += __popcll(x);
      }
    } else {
      for (int w = 0; w < a.words; ++w) depth += t < most ? __popcll(rows[w * cap + t]) : 0;
      int from = (int)min(max(a.sinks - first, (int64_t)0), (int64_t)kTreeMost);   // bits of the first tokens,
      int to = max(depth + 1 - a.window, 0);       // and below the window
      for (int w = 0; w < a.words; ++w) {
        const uint64_t x = t < most ? rows[w * cap + t] : 0;
        a.mask[(int64_t)(r.c0 + t) * a.words + w] = (int64_t)(x & ~(low_bits(x, to) & ~low_bits(x, from)));
        from -= __popcll(x);
        to -= __popcll(x);
      }
    }
    a.positions[r.c0 + t] = t < most ? (int)(first + depth) : -1;
  }
}

// Every token that its parent's choice agrees with names itself to the parent, which keeps the lowest (`next`).  The tokens
// that the first one comes to, if it is a long path, are marked; on a path the numbers rise, so a token's place on it is
// the number of marks below.
template <typename I>
__global__ __launch_bounds__(kTreeThreads) void tree_accept_kernel(fs_tree_accept_args a) {
  constexpr int PER = kTreeMost / kTreeThreads, NW = kTreeThreads / 64;
  __shared__ int next[kTreeMost];
  __shared__ uint8_t marked[kTreeMost];
  __shared__ int marks[PER][NW], path[kSteps], steps, last;
  const int tid = threadIdx.x, b = blockIdx.x;
  if (b == a.B) {
    rows_of_none(a.cu_lens, a.B, a.T, [&](int t) { a.kept[t] = -1; });
    return;
  }
  const I *tokens = static_cast<const I*>(a.tokens), *chosen = static_cast<const I*>(a.chosen);
  const TreeRows r(a.cu_lens, b, a.T);
  const int most = min(r.n, a.most);
  if (tid == 0) last = 0;
  for (int t = tid; t < most; t += kTreeThreads) {
    next[t] = INT_MAX;
    marked[t] = t == 0;
  }
  __syncthreads();
  for (int t = tid; t < most; t += kTreeThreads) {
    const int p = a.parents[r.c0 + t];
    if (p < 0 || p >= t) continue;
    const I x = tokens[r.c0 + t];
    if (x < 0 || x == chosen[r.c0 + p]) atomicMin(&next[p], t);   // the least of them, in whatever order
  }
  __syncthreads();
  if (tid == 0) {
    int k = 0, t = 0;
    for (; t < most && k < kSteps; t = next[t]) path[k++] = t;
    steps = t < most ? -1 : k;                     // -1: it goes on
    if (t >= most) {
      a.kept_lens[b] = k;
      a.dropped[b] = k - max(r.n, 0);
      static_cast<I*>(a.next_tokens)[b] = k ? chosen[r.c0 + path[k - 1]] : (I)-1;
    }
  }
  __syncthreads();
  if (steps >= 0) {
    for (int t = tid; t < r.n; t += kTreeThreads) a.kept[r.c0 + t] = t < steps ? path[t] : -1;
    return;
  }
  // After k rounds the first 2^k tokens of the path are marked and next[t] is 2^k on.
  while (next[0] < most) {
    int on[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int t = tid + i * kTreeThreads, n = t < most ? next[t] : INT_MAX;
      on[i] = n < most ? next[n] : INT_MAX;
      if (n < most && marked[t]) marked[n] = 1;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (tid + i * kTreeThreads < most) next[tid + i * kTreeThreads] = on[i];
    __syncthreads();
  }
  uint64_t who[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int t = tid + i * kTreeThreads;
    who[i] = __ballot(t < most && marked[t]);
    if ((tid & 63) == 0) marks[i][tid >> 6] = (int)__popcll(who[i]);
  }
  __syncthreads();
  int count = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i)
    for (int w = 0; w < NW; ++w) {
      if (w == tid >> 6 && who[i] >> (tid & 63) & 1) a.kept[r.c0 + count + rank_below(who[i])] = tid + i * kTreeThreads;
      count += marks[i][w];
      if (w == tid >> 6 && marks[i][w] && (tid & 63) == 0) atomicMax(&last, i * kTreeThreads + w * 64 + 63 - (int)__builtin_clzll(who[i]));
    }
  for (int t = count + tid; t < r.n; t += kTreeThreads) a.kept[r.c0 + t] = -1;
  __syncthreads();
  if (tid == 0) {
    a.kept_lens[b] = count;
    a.dropped[b] = count - max(r.n, 0);
    static_cast<I*>(a.next_tokens)[b] = count ? chosen[r.c0 + last] : (I)-1;
  }
}

constexpr int kMoveLayers = 64;                    // of a launch
struct MoveKArgs {
  fs_cache_move_args a;
  int caches;                                      // that a workgroup takes
  char* cache[2 * kMoveLayers];                    // K and V of each layer
};

// A workgroup moves one request's rows in some of the caches, whose places it looks up once.  The pieces (cache, row, 16
// bytes) are taken in this order, 1024 at a time, and all of them are read before any is written: the place
// of row i may be that of a row j > i that another thread still has to read.  Pieces of later steps lie behind
// every place of their cache that is written by then: row j > i comes from behind j.
__global__ __launch_bounds__(kTreeThreads) void cache_move_kernel(MoveKArgs ka) {
  constexpr int HELD = 4;                          // pieces of a thread
  const fs_cache_move_args& a = ka.a;
  __shared__ int2 from[kTreeMost], to[kTreeMost];  // page and slot; page -1: stays
  __shared__ int lo, hi;
  const int tid = threadIdx.x, b = blockIdx.x;
  const TreeRows r(a.cu_lens, b, a.T);
  const int n = min(r.n, kTreeMost);
  const int64_t first = (int64_t)a.seq_lens[b] - r.n;
  if (tid == 0) {
    lo = INT_MAX;
    hi = -1;
  }
  __syncthreads();
  auto place = [&](int i) {
    const int64_t s = first + i;
    if (s < 0 || s >= (int64_t)a.P * a.page_size) return make_int2(-1, 0);
    const int pg = (int)s / a.page_size, e = a.block_table[b * a.t_sb + pg];
    return make_int2(e >= 0 && e < a.num_pages ? e : -1, (int)s - pg * a.page_size);
  };
  for (int i = tid; i < n; i += kTreeThreads) {
    const int j = a.kept[r.c0 + i];
    int2 f = make_int2(-1, 0), t = f;
    if (j > i && j < n) {
      f = place(j);
      t = place(i);
      if (f.x < 0 || t.x < 0) f.x = -1;
    }
    from[i] = f;
    to[i] = t;
    if (f.x >= 0) {
      atomicMin(&lo, i);
      atomicMax(&hi, i);
    }
  }
  __syncthreads();
  const int rows = hi + 1 - lo;
  if (rows <= 0) return;
  const uint32_t per_head = a.D * a.elem_bytes / 16, pieces = a.Hk * per_head, per_cache = rows * pieces;
  const int c0 = blockIdx.y * ka.caches, caches = min(ka.caches, 2 * a.layers - c0);
  // below 2^32: 8 caches of 1024 rows of 2^18 pieces
  for (uint32_t x0 = 0; x0 < caches * per_cache; x0 += HELD * kTreeThreads) {
    uint4 held[HELD];
    char* dst[HELD];
#pragma unroll
    for (int k = 0; k < HELD; ++k) {
      const uint32_t x = x0 + k * kTreeThreads + tid;
      dst[k] = nullptr;
      if (x < caches * per_cache) {
        const uint32_t c = x / per_cache, y = x - c * per_cache, i = y / pieces, z = y - i * pieces, h = z / per_head;
        const int2 f = from[lo + i], t = to[lo + i];
        if (f.x >= 0) {
          const bool v = (c0 + c) & 1;
          const int64_t sp = v ? a.v_sp : a.k_sp, ss = v ? a.v_ss : a.k_ss;
          char* at = ka.cache[c0 + c] + h * (v ? a.v_sh : a.k_sh) * a.elem_bytes + (z - h * per_head) * 16;
          held[k] = *reinterpret_cast<const uint4*>(at + (f.x * sp + f.y * ss) * a.elem_bytes);
          dst[k] = at + (t.x * sp + t.y * ss) * a.elem_bytes;
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < HELD; ++k)
      if (dst[k] != nullptr) *reinterpret_cast<uint4*>(dst[k]) = held[k];
  }
}

}  // namespace fs

using namespace fs;

// Part of an offset into the caches: lo to hi times `step` bytes.
struct Term {
  int64_t step, lo, hi;
};
// Whether some sum of the terms from t to `end`, the largest steps first, is less than `row` bytes from d: two caches d
// apart then have bytes in common, where the terms are what can lie between two of their rows.  Steps that hold all
// smaller ones (every layout that is a view of a dense tensor) leave one or two numbers to try for each; `tries`
// bounds the others (0: not known, taken as shared).
static bool shares(const Term* t, const Term* end, int64_t d, int64_t row, int& tries) {
  int64_t lo = 1 - row, hi = row - 1;              // what the terms after t reach
  if (t == end) return d >= lo && d <= hi;
  for (const Term* x = t + 1; x < end; ++x) {
    lo += x->step * x->lo;
    hi += x->step * x->hi;
  }
  auto down = [](int64_t a, int64_t b) { return a / b - (a % b < 0); };
  const int64_t from = std::max(t->lo, -down(hi - d, t->step)), to = std::min(t->hi, down(d - lo, t->step));
  for (int64_t c = from; c <= to; ++c)
    if (--tries < 0 || shares(t + 1, end, d - c * t->step, row, tries)) return true;
  return false;
}
// Whether the caches of a move have bytes in common.  Each is moved by workgroups of its own, so one that is named twice would be
// moved twice, in any order.
static bool caches_share(const fs_cache_move_args& a, const std::vector<std::pair<int64_t, bool>>& at) {
  const int64_t e = a.elem_bytes, row = a.D * e;
  const int64_t n[] = {a.layers, std::min<int64_t>(a.num_pages, INT_MAX), a.page_size, a.Hk};   // a table's numbers are below
  const int64_t st[2][4] = {{at.empty() ? a.k_sl * e : 0, a.k_sp * e, a.k_ss * e, a.k_sh * e},
                            {at.empty() ? a.v_sl * e : 0, a.v_sp * e, a.v_ss * e, a.v_sh * e}};
  // cache y of kind vy lies d bytes behind cache x of kind vx; layers: from another layer on (0: any)
  auto pair = [&](bool vx, bool vy, int64_t d, int layers) {
    Term t[8];
    int m = 0;
    auto add = [&](int64_t step, int64_t lo, int64_t hi) {
      if (step < 0) {
        step = -step;
        std::swap(lo, hi);
        lo = -lo;
        hi = -hi;
      }
      if (step == 0 || (lo == 0 && hi == 0)) return;
      for (int i = 0; i < m; ++i)
        if (t[i].step == step) {
          t[i].lo += lo;
          t[i].hi += hi;
          return;
        }
      t[m++] = {step, lo, hi};
    };
    for (int i = 0; i < 4; ++i) {
      if (i == 0 && layers) {
        add(st[vx][0], layers, n[0] - 1);
        continue;
      }
      add(st[vx][i], 0, n[i] - 1);
      add(st[vy][i], 1 - n[i], 0);
    }
    std::sort(t, t + m, [](const Term& x, const Term& y) { return x.step > y.step; });
    int tries = 1 << 16;
    return shares(t, t + m, d, row, tries);
  };
  if (at.empty())
    return (a.layers > 1 && (pair(false, false, 0, 1) || pair(true, true, 0, 1))) ||
           pair(false, true, (int64_t)((uintptr_t)a.v_cache - (uintptr_t)a.k_cache), 0);
  const size_t m = at.size();
  bool back = false;
  for (int v = 0; v < 2; ++v)
    for (int i = 1; i < 4; ++i) back |= st[v][i] < 0;
  if (back) {                                      // steps that run backwards: every two are looked at
    for (size_t x = 0; x < m; ++x)
      for (size_t y = x + 1; y < m; ++y)
        if (pair(at[x].second, at[y].second, at[y].first - at[x].first, 0)) return true;
    return false;
  }
  // f of every two caches that meet modulo s (0: as they lie): steps that s divides do not move them there, the others make
  // them as long as they are.  What does not meet is apart.
  auto meeting = [&](int64_t s, auto f) {
    int64_t len[2] = {row, row};
    for (int v = 0; v < 2; ++v)
      for (int i = 1; i < 4; ++i)
        if (s == 0 || st[v][i] % s) len[v] += st[v][i] * (n[i] - 1);
    std::vector<std::pair<int64_t, size_t>> by(m);
    for (size_t i = 0; i < m; ++i) by[i] = {s ? at[i].first % s : at[i].first, i};
    std::sort(by.begin(), by.end());
    for (size_t i = 0; i < m; ++i)
      for (size_t j = i + 1; j < (s ? i + m : m); ++j) {
        const auto &x = by[i], &y = by[j < m ? j : j - m];
        if (y.first + (j < m ? 0 : s) >= x.first + len[at[x.second].second]) break;
        if (f(x.second, y.second)) return true;
      }
    return false;
  };
  // Layers apart, of a page, or of a token: one of the steps separates nearly all (64 layers 3 to 20 us of host time; every two of the
  // 128 caches looked at 600).
  size_t least = 8 * m;
  int64_t best = 0;
  for (int i = 0; i < 4; ++i) {
    const int64_t s = i ? st[0][i] : 0;
    if (i && s == 0) continue;
    size_t count = 0;
    meeting(s, [&](size_t, size_t) { return ++count >= least; });
    if (count == 0) return false;
    if (count < least) {
      least = count;
      best = s;
    }
  }
  return meeting(best, [&](size_t x, size_t y) { return pair(at[x].second, at[y].second, at[y].first - at[x].first, 0); });
}

static int check_tree(const char* fn, int B, int T) {
  FS_CHECK_ARG(B >= 1 && T >= 0, "%s: B=%d requests, T=%d rows", fn, B, T);
  FS_CHECK_SUPPORTED(B <= 65535, "%s: %d requests > 65535", fn, B);
  return FS_OK;
}

extern "C" int fs_tree_plan(const fs_tree_plan_args* a, void* stream) {
  const char* fn = "fs_tree_plan";
  FS_CHECK_ARG(a != nullptr, "%s: null args", fn);
  if (int rc = check_tree(fn, a->B, a->T)) return rc;
  FS_CHECK_ARG(a->words >= 1, "%s: %d words", fn, a->words);
  FS_CHECK_ARG(a->window >= 0 && a->sinks >= 0, "%s: window %d and sinks %d must not be negative", fn, a->window, a->sinks);
  FS_CHECK_SUPPORTED(a->words <= kTreeMost / 64, "%s: trees of %d tokens > %d", fn, 64 * a->words, kTreeMost);
  if (a->T == 0) return FS_OK;
  FS_CHECK_ARG(a->parents && a->cu_lens && a->seq_lens && a->positions && a->mask, "%s: null tensor pointer", fn);
  const size_t bytes = (size_t)a->words * 64 * (a->words * sizeof(uint64_t) + sizeof(int));   // 132 KiB at most
  if (int rc = fs_host::allow_dynamic_lds(tree_plan_kernel, bytes, fn)) return rc;
  tree_plan_kernel<<<a->B + 1, kTreeThreads, bytes, (hipStream_t)stream>>>(*a);
  return fs_host::launch_status(fn);
}

extern "C" int fs_tree_accept(const fs_tree_accept_args* a, void* stream) {
  const char* fn = "fs_tree_accept";
  FS_CHECK_ARG(a != nullptr, "%s: null args", fn);
  if (int rc = check_tree(fn, a->B, a->T)) return rc;
  FS_CHECK_ARG(a->token_bytes == 4 || a->token_bytes == 8, "%s: tokens of %d bytes", fn, a->token_bytes);
  FS_CHECK_ARG(a->most >= 1, "%s: trees of %d tokens", fn, a->most);
  FS_CHECK_SUPPORTED(a->most <= kTreeMost, "%s: trees of %d tokens > %d", fn, a->most, kTreeMost);
  FS_CHECK_ARG(a->cu_lens && a->kept_lens && a->dropped && a->next_tokens &&
                   (a->T == 0 || (a->parents && a->tokens && a->chosen && a->kept)), "%s: null tensor pointer", fn);
  if (a->token_bytes == 8) tree_accept_kernel<int64_t><<<a->B + 1, kTreeThreads, 0, (hipStream_t)stream>>>(*a);
  else tree_accept_kernel<int32_t><<<a->B + 1, kTreeThreads, 0, (hipStream_t)stream>>>(*a);
  return fs_host::launch_status(fn);
}

extern "C" int fs_cache_move(const fs_cache_move_args* a, void* stream) {
  const char* fn = "fs_cache_move";
  FS_CHECK_ARG(a != nullptr, "%s: null args", fn);
  if (int rc = check_tree(fn, a->B, a->T)) return rc;
  FS_CHECK_ARG(a->layers >= 0 && a->Hk >= 1 && a->D >= 1 && a->P >= 1 && a->page_size >= 1 && a->num_pages >= 1,
               "%s: layers=%d Hk=%d D=%d P=%d page_size=%d num_pages=%lld", fn, a->layers, a->Hk, a->D, a->P, a->page_size,
               (long long)a->num_pages);
  FS_CHECK_ARG(a->elem_bytes == 1 || a->elem_bytes == 2 || a->elem_bytes == 4, "%s: elements of %d bytes", fn, a->elem_bytes);
  FS_CHECK_SUPPORTED((int64_t)a->Hk * a->D <= (1 << 20) && (int64_t)a->D * a->elem_bytes % 16 == 0,
                     "%s: rows of %d heads of %d unsupported (multiples of 16 bytes)", fn, a->Hk, a->D);
  FS_CHECK_SUPPORTED((int64_t)a->P * a->page_size <= INT_MAX, "%s: %d pages of %d tokens per request unsupported", fn,
                     a->P, a->page_size);
  if (a->T == 0 || a->layers == 0) return FS_OK;
  const bool arrays = a->k_caches != nullptr;
  const int64_t st[] = {a->k_sp, a->k_ss, a->k_sh, a->v_sp, a->v_ss, a->v_sh, arrays ? 0 : a->k_sl, arrays ? 0 : a->v_sl};
  for (int64_t x : st) FS_CHECK_ARG(x * a->elem_bytes % 16 == 0, "%s: strides must be multiples of 16 bytes", fn);
  FS_CHECK_ARG(arrays == (a->v_caches != nullptr) && a->block_table && a->cu_lens && a->seq_lens && a->kept && a->t_sb >= a->P,
               "%s: null tensor pointer, or row stride %lld of %d", fn, (long long)a->t_sb, a->P);
  auto cache = [&](bool v, int i) {
    return arrays ? static_cast<char*>((v ? a->v_caches : a->k_caches)[i])
                  : static_cast<char*>(v ? a->v_cache : a->k_cache) + i * (v ? a->v_sl : a->k_sl) * a->elem_bytes;
  };
  FS_CHECK_ARG(arrays || (a->k_cache && a->v_cache), "%s: caches must be given, 16-byte aligned", fn);
  for (int i = 0; i < a->layers; ++i)
    FS_CHECK_ARG(cache(false, i) && cache(true, i) && ((uintptr_t)cache(false, i) | (uintptr_t)cache(true, i)) % 16 == 0,
                 "%s: caches must be given, 16-byte aligned", fn);
  bool share = false;
  try {
    std::vector<std::pair<int64_t, bool>> at;      // address, whether of values
    for (int i = 0; arrays && i < a->layers; ++i)
      for (bool v : {false, true}) at.emplace_back((int64_t)(uintptr_t)cache(v, i), v);
    share = caches_share(*a, at);
  } catch (const std::bad_alloc&) {
    FS_CHECK_SUPPORTED(false, "%s: no host memory to look over %d layers", fn, a->layers);
  }
  FS_CHECK_ARG(!share, "%s: caches share storage; each is moved once: name it once", fn);
  for (int l0 = 0; l0 < a->layers; l0 += kMoveLayers) {
    MoveKArgs k{*a, 1, {}};
    const int n = std::min(a->layers - l0, kMoveLayers);
    for (int i = 0; i < 2 * n; ++i) k.cache[i] = cache(i & 1, l0 + i / 2);
    k.a.layers = n;
    // few requests: a cache each; else as many as leave two workgroups per CU (64 requests, 32 layers: 9.6 us either way)
    k.caches = (int)std::max<int64_t>(1, std::min<int64_t>(8, (int64_t)a->B * 2 * n / 512));
    cache_move_kernel<<<dim3(a->B, (2 * n + k.caches - 1) / k.caches), kTreeThreads, 0, (hipStream_t)stream>>>(k);
    if (int rc = fs_host::launch_status(fn)) return rc;
  }
  return FS_OK;
}
