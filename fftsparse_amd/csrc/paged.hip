// Attention of new tokens over a paged cache, and sliding-window attention with
// sinks on contiguous tensors, on bf16 / f16 MFMA (gfx950).
//
// Rows.  The query heads that read one KV head are put side by side: row r of
// (request, KV head) is new token r / G, query head hk G + r % G (G = Hq / Hk).
// So a single token fills a tile with the G heads that read the same keys, and a
// chunk's tile of 128 rows reads each key once for all of them.  A row tile sees
// the keys kbeg .. kend - 1 (the union of its rows' windows) and the first
// `sinks`; groups of 16 keys in between are not visited, and a key tile is four groups of the
// others in a row (the first tokens cost a group, not a tile).
//
// few_kernel (calls whose requests have at most 32 rows per KV head: single tokens) is bound by
// the cache being read.  256 workgroups (512 at head dim 64) take equal runs of all the call's key tiles
// (Ranges), so that they end together whatever the lengths are.  Each of a workgroup's 4
// waves streams keys of its own, 32 at a time, through a ring of two LDS tiles that
// only it uses: no barrier in the loop, and 24 to 32 KiB per wave are always on their way
// (96 KiB and more per CU).  S^T = K Q^T, P in registers, O^T += V^T P on
// v_mfma_f32_32x32x16, of which a single token uses G of 32 columns (about a tenth of the
// MFMA rate is taken); V is read transposed from LDS as it is stored.  Measured
// (bf16, D = 128, 32 / 8 heads): 32 requests of 16384 tokens 5.3 TB/s, 64 of 64 - 8192 4.4 TB/s,
// one of 131072 4.7 TB/s; a copy of 4 GiB takes 4.9 TB/s on the same card, but pool.hip's pass, which only reads as
// this one does, 6.7: what keeps the last quarter has not been found.  All 106 scalar registers are taken and 72 (D = 64,
// contiguous) to 102 (D = 128, paged) more are kept in lanes of vector registers; no
// vector register is spilled.
//
// many_kernel (tiles of 128 rows) is bound by MFMA: 4 waves of 32 rows share tiles of 64 keys,
// two tiles deep: S of the next tile and P V of the last one are interleaved with the
// exponentials of the current one.  A row tile's keys are taken in several pieces
// where that fills the GPU better (plan_pieces_kernel, from the lengths on the device).  Measured: 2048 new
// tokens over 32768 1.09 PFLOP/s; an 8192^3 GEMM takes 1.18 on the same card.
//
// Both leave the unnormalised sums of a row tile that was cut in the workspace, in
// 32 bits, with each row's maximum and sum; combine_kernel joins them, in an order that
// depends on the lengths only.
//
// Rounding: scores, maxima, sums and O are in 32 bits; P is rounded to the input type for the
// second product (its relative error, at most half a step of the type, averages out over the keys as the
// values' own does), and the row sum adds the rounded P, so that weights add up to one.  Against 64 bits (2-norm)
// bf16 is off by 1.8e-3 to 2.0e-3 (1.6e-3 to 1.7e-3 with P in 32 bits: the result's own rounding), f16 by 2.2e-4 to 2.8e-4
// (2.1e-4).  Sums stay below 2^34 of the largest |v| (P up to 2^8, 2^26 keys), so |v| up to 2^93 is safe.
//
// Groups of 16 keys are never split by a page (its size is a multiple of 16): a
// copy of one is addressed by one entry of the table.  A group that not all rows
// of the tile may read as a whole (the end of the request, the window's edge, a
// page that is none) is copied row by row, zeros in place of the rows that no row
// of the tile sees: nothing stands there that could spoil a sum.
#include <algorithm>
#include <cmath>
#include <climits>
#include <type_traits>

#include "attn_tile.h"

namespace fs {

constexpr int kFewWaves = 4;                        // of a workgroup of few_kernel (1 or 2, as many in all: 10% slower)
constexpr int kSlotsMany = 512;                     // workgroups that 256 CUs hold
constexpr int few_slots(int D) { return 256 * 4 / kFewWaves * (128 / D); }
constexpr int kPartsMany = 1024;                    // split pieces that the workspace holds
constexpr int kMaxRequests = 4096;
constexpr int kPlanThreads = 1024;

struct PagedKArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* out;
  int64_t q_sb, q_st, q_sh, o_sb, o_st, o_sh;   // request (contiguous tensors), token, head
  int64_t k_sp, k_sh, v_sp, v_sh;               // page (contiguous: batch), head
  int k_ss, v_ss;                               // slot
  const int32_t* table;                         // null: contiguous, the page of request b is b
  const int32_t* cu;
  const int32_t* lens;
  int64_t t_sb;
  int num_pages, B, T, Hq, Hk, G, Lq, Lk, P, page_size, window, sinks;
  uint32_t page_magic;                          // x / (page_size / 16) = mulhi(x, magic); 0: x
  float scale;
  // pieces, the last row tiles of a request first
  const int4* pieces;                           // [N] request, row tile, first key tile, slot (-1: the only piece)
  int4* splits;                                 // [Q] request, row tile, pieces, first slot
  int32_t* head;                                // N, Q, chunk, split pieces (of one KV head); null: nothing is split
  int max_splits;
  int slots;                                    // workgroups of few_kernel
  int row_tiles;                                // of a request (no list)
  float* part_o;                                // [slot][rows / 32][D / 32][4][64 lanes] 4 floats
  float* part_ml;                               // [slot][rows / 32][2][32]
};

// A wave-uniform load through the scalar unit: what no kernel of the launch writes.
template <typename E>
__device__ __forceinline__ E scalar_load(const E* p, int64_t i) {
  return ((const __attribute__((address_space(4))) E*)(uintptr_t)p)[i];
}

// A row tile's place and the keys it sees; everything wave-uniform.
struct RowTile {
  int row0, n, L;            // first row of q, new tokens, tokens
  int r0, nrows;             // rows r0 .. r0 + nrows - 1 of the request
  int p_lo, p_hi;            // positions of its first and last row
  int kbeg, kend;            // keys kbeg .. kend - 1 (and the first `sinks`) are seen by some row
  int ns, t0, nt;            // groups of 16 keys: 0 .. ns - 1, then t0 ..; nt tiles in all
  // first key of the i-th group that is visited
  __device__ __forceinline__ int key_of(int i) const { return (i < ns ? i : t0 + i - ns) * 16; }
};
struct Lengths {
  int row0, n, L;
};
__device__ __forceinline__ Lengths lengths_of(const PagedKArgs& a, int b) {
  if (a.table == nullptr) return {0, a.Lq, a.Lk};
  const int c0 = min(max(a.cu[b], 0), a.T), c1 = min(max(a.cu[b + 1], 0), a.T);
  return {c0, c1 - c0, min(max(a.lens[b], 0), a.P * a.page_size)};   // c1 < c0: no row (row numbers that fall)
}
template <int M, int TK>
__device__ __forceinline__ RowTile row_tile(const PagedKArgs& a, const Lengths& x, int rt) {
  RowTile u;
  u.row0 = x.row0;
  u.n = x.n;
  u.L = x.L;
  u.r0 = rt * M;
  u.nrows = min(M, u.n * a.G - u.r0);
  u.p_lo = u.L - u.n + u.r0 / a.G;
  u.p_hi = u.L - u.n + (u.r0 + max(u.nrows, 1) - 1) / a.G;
  u.kend = u.nrows > 0 ? max(u.p_hi + 1, 0) : 0;
  u.kbeg = a.window ? max(u.p_lo - a.window + 1, 0) : 0;
  u.ns = (min(a.sinks, u.kbeg) + 15) / 16;
  u.t0 = u.kbeg / 16;
  if (a.table != nullptr) u.t0 -= (u.t0 - u.ns) & 3;   // runs of 64 keys that pages of so many do not cut
  if (u.ns >= u.t0) u.ns = u.t0 = 0;
  u.nt = u.kend > 0 ? (u.ns + (u.kend + 15) / 16 - u.t0 + TK / 16 - 1) / (TK / 16) : 0;
  return u;
}

// Copies of 16-key groups into an LDS tile of rows of D elements: group g of it at byte
// 16 g * 2 D, swizzled as the operand reads expect.
template <int D, bool PAGED>
struct GroupCopy {
  static constexpr int ROWB = D * 2, CPR = D / 8, SWM = CPR - 1, LCPR = D == 128 ? 4 : 3;
  static constexpr int RPR = 1024 / ROWB;          // rows of a 1 KiB copy
  static constexpr int NI = 16 / RPR;              // copies of a group
  uint32_t koff[NI], voff[NI];
  const uint16_t *kp, *vp;
  const int32_t* row;                              // of the table
  int page;                                        // contiguous: the request
  __device__ __forceinline__ void place(const PagedKArgs& a, int b, int hk) {
    row = PAGED ? a.table + b * a.t_sb : nullptr;
    page = b;
    kp = a.k + hk * a.k_sh;
    vp = a.v + hk * a.v_sh;
  }
  __device__ __forceinline__ GroupCopy(const PagedKArgs& a, int lane) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int r = RPR * i + (lane >> LCPR);
      koff[i] = (uint32_t)(r * a.k_ss + kchunk(r, lane) * 8) * 2u;
      voff[i] = (uint32_t)(r * a.v_ss + vchunk(r, lane) * 8) * 2u;
    }
  }
  static __device__ __forceinline__ int kchunk(int r, int lane) { return (lane & SWM) ^ ((D == 128 ? r : r >> 1) & SWM); }
  static __device__ __forceinline__ int vchunk(int r, int lane) { return (lane & SWM) ^ v_swz<D>(r); }
  // the page of the table's row that holds key k0 (a multiple of 16), and the key's slot there
  static __device__ __forceinline__ int page_of(const PagedKArgs& a, int k0, int& slot) {
    if constexpr (!PAGED) {
      slot = k0;
      return 0;
    }
    const uint32_t x = (uint32_t)k0 >> 4;
    const uint32_t pg = a.page_magic ? __umulhi(x, a.page_magic) : x;
    slot = k0 - (int)pg * a.page_size;
    return (int)pg;
  }
  // the entry of page pg: the page's number in the cache, -1 for none
  __device__ __forceinline__ int entry(int pg) const { return PAGED ? scalar_load(row, pg) : page; }
  static __device__ __forceinline__ bool is_page(const PagedKArgs& a, int e) { return !PAGED || (uint32_t)e < (uint32_t)a.num_pages; }
  // some row of the tile sees some key of the group of key k0
  static __device__ __forceinline__ bool seen(const PagedKArgs& a, const RowTile& u, int k0) {
    return k0 < u.kend && (k0 + 15 >= u.kbeg || k0 < a.sinks);
  }
  // every key of n from k0 on is seen by some row
  static __device__ __forceinline__ bool whole(const PagedKArgs& a, const RowTile& u, int k0, int n) {
    return k0 + n <= u.kend && (k0 >= u.kbeg || k0 + n <= a.sinks);
  }
  // copies the group of key k0, at `slot` of page e (no page: e < 0); all: every key of it is seen
  template <bool V>
  __device__ __forceinline__ void issue(const PagedKArgs& a, const RowTile& u, uint32_t lds, int e, int slot, int k0,
                                        bool all) const {
    const int st = V ? a.v_ss : a.k_ss;
    const uint16_t* base = (V ? vp : kp) + max(e, 0) * (V ? a.v_sp : a.k_sp) + (int64_t)slot * st;
    if (all) {
#pragma unroll
      for (int i = 0; i < NI; ++i) dma16s(lds + i * 1024, base, V ? voff[i] : koff[i]);
    } else {
      int ln = (int)__lane_id();
      asm volatile("" : "+v"(ln));                 // keep this rare path's addresses out of the loop's preheader
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int r = RPR * i + (ln >> LCPR), key = k0 + r;
        const bool ok = e >= 0 && key < u.kend && (key >= u.kbeg || key < a.sinks);
        const uint16_t* row = ok ? base + (int64_t)r * st : reinterpret_cast<const uint16_t*>(kZeroRow);
        dma16(lds + i * 1024, row + (V ? vchunk(r, ln) : kchunk(r, ln)) * 8);
      }
    }
  }
};

// v and the value of the lane 32 apart (the same row's other keys)
__device__ __forceinline__ void lane_halves(float v, float& lo, float& hi) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  lo = __uint_as_float(r[0]);
  hi = __uint_as_float(r[1]);
}

// This lane's row of a 32-row part of a row tile.
struct LaneRow {
  int tok, g, p;             // token of the request, head of the group, position
  bool on;
};
template <typename A>
__device__ __forceinline__ LaneRow lane_row(const A& a, const RowTile& u, int r) {
  LaneRow w;
  const int rr = u.r0 + min(r, max(u.nrows, 1) - 1);  // rows past the tile's follow its last one
  w.tok = rr / a.G;
  w.g = rr - w.tok * a.G;
  w.p = u.L - u.n + w.tok;
  const int t = u.row0 + w.tok;
  w.on = r < u.nrows && t >= 0 && t < a.T;
  return w;
}

// Q^T fragments of a row (B operand of S^T = K Q^T): dims st*16 + hi*8 .. +7; zeros without a row
template <typename V8, int D>
__device__ __forceinline__ void load_q(const PagedKArgs& a, const RowTile& u, const LaneRow& w, int b, int hk, int hi,
                                       V8* qf) {
  const uint16_t* qp = a.q + b * a.q_sb + (int64_t)(u.row0 + w.tok) * a.q_st + (int64_t)(hk * a.G + w.g) * a.q_sh;
#pragma unroll
  for (int st = 0; st < D / 16; ++st) {
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (w.on) raw = *reinterpret_cast<const uint4*>(qp + st * 16 + hi * 8);
    qf[st] = __builtin_bit_cast(V8, raw);
  }
}

// whether some row of positions p_lo .. p_hi does not see some key of key0 .. key0 + n - 1
__device__ __forceinline__ bool needs_mask(const PagedKArgs& a, int p_lo, int p_hi, int key0, int n) {
  return key0 + n - 1 > p_lo || (a.window && key0 <= p_hi - a.window && key0 + n > a.sinks);
}
// -inf for the scores of the groups of 16 keys k0 and k1 (registers 0 - 7 and 8 - 15; register r: key ((r >> 2) & 1) * 8 +
// (r & 3) + hi * 4) that the row at p does not see; v0, v1: whether the groups are there.  A key of a group is hidden past
// `last`, and for n keys from `from` on (between the first tokens and the window).  Written without branches: with one for
// each edge the loop of many_kernel spilled 51 vector registers.
__device__ __forceinline__ void mask_keys(const PagedKArgs& a, f32x16_t& s, int p, int k0, int k1, int hi, bool v0, bool v1) {
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    __builtin_amdgcn_sched_barrier(0);             // the compares of one group at a time: they take scalar registers
    const int k = (g ? k1 : k0) + hi * 4, last = (g ? v1 : v0) ? p - k : -1;
    const int from = a.window ? max(a.sinks - k, 0) : 16;
    const uint32_t n = a.window ? (uint32_t)max(p - a.window - k + 1 - from, 0) : 0u;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const int c = (r >> 2) * 8 + (r & 3);
      s[8 * g + r] = c > last ? -INFINITY : s[8 * g + r];
      s[8 * g + r] = (uint32_t)(c - from) < n ? -INFINITY : s[8 * g + r];
    }
  }
}

// O^T of one row (this lane's dims dt * 32 + g4 * 8 + hi * 4 .. + 3) to the output
template <typename T>
__device__ __forceinline__ uint2 out_bits(float x0, float x1, float x2, float x3) {
  using Ops = MfmaOps<T>;
  return make_uint2((uint32_t)Ops::bits(x0) | ((uint32_t)Ops::bits(x1) << 16),
                    (uint32_t)Ops::bits(x2) | ((uint32_t)Ops::bits(x3) << 16));
}
template <typename T>
__device__ __forceinline__ void store_out(uint16_t* op, int d0, float x0, float x1, float x2, float x3) {
  *reinterpret_cast<uint2*>(op + d0) = out_bits<T>(x0, x1, x2, x3);
}
template <typename A>
__device__ __forceinline__ uint16_t* out_row(const A& a, const RowTile& u, const LaneRow& w, int b, int hk) {
  return a.out + b * a.o_sb + (int64_t)(u.row0 + w.tok) * a.o_st + (int64_t)(hk * a.G + w.g) * a.o_sh;
}

// What a kernel's end needs of its arguments, read from them only then.
struct LateArgs {
  uint16_t* out;
  int64_t o_sb, o_st, o_sh;
  float *part_o, *part_ml;
  int T, G;
  __device__ __forceinline__ LateArgs() {
    typedef const __attribute__((address_space(4))) PagedKArgs* kptr;
    kptr a = (kptr)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(a));
    out = a->out;
    o_sb = a->o_sb;
    o_st = a->o_st;
    o_sh = a->o_sh;
    part_o = a->part_o;
    part_ml = a->part_ml;
    T = a->T;
    G = a->G;
  }
};

// The piece of workgroup p: KV head, request, row tile, first key tile, key tiles, slot (-1: no other piece).
struct Piece {
  int hk, b, rt, begin, count, slot;
};

// How long a call takes, in key tiles' time: N pieces of at most c tiles of the W in all, `slots` at a time; a start
// per round of pieces and, where sums are joined, a launch, their writing and reading, and a turn for each of the most
// pieces of a row tile (without that, 16 tokens over 2048 were cut into single tiles: 33 us against 22; a
// launch at 1.5 cut a prompt of 700: 35 us against 29, at 9 left a batch of windows whole: 42 against 39).  One set
// serves both head dims, though a tile takes about half as long at 64: with all four twice as large there 64 tokens over
// 8192 took 34.7 us against 37.4, but 16 requests with chunks 71 against 61, windows of them 42.5 against 39.8, 64 tokens over
// 2048 23.5 against 22.8, and prompts of 300 to 2000 the same within 1%.
__device__ __forceinline__ float call_time(float N, float c, float W, float slots, float joined, float most) {
  constexpr float kStart = 1.5f, kJoin = 5.0f, kPiece = 0.014f, kTurn = 0.3f;
  const float rounds = ceilf(N / slots);
  return fminf(rounds * c, W / slots + c) + rounds * kStart + (joined > 0.f ? kJoin + joined * kPiece + most * kTurn : 0.f);
}
// The 16 numbers of key tiles per piece that are tried: an i-th part of the longest row tile's, and what gives about i
// rounds of pieces (U row tiles, of which each may leave a shorter piece).
__device__ __forceinline__ int chunk_choice(int i, int longest, float W, float U, float slots) {
  if (i < 8) return (longest + i) / (i + 1);
  const float s = slots * (float)(i - 7);
  return max(1, min(longest, (int)ceilf(W / (s - 0.5f * fminf(U, s)))));
}
// ceil(nt / c), at least 1; the division is exact below 2^22
__device__ __forceinline__ int parts_of(int nt, int c) { return max((int)((float)(nt + c - 1) / (float)c), 1); }

// The piece of this workgroup among n: XCD x, that is workgroups x, x + 8, .., takes a run of consecutive ones,
// row tiles of one head, whose keys its L2 then serves.  Past the last one: n.
__device__ __forceinline__ int piece_of(int n) {
  const int per = (n + 7) / 8, x = blockIdx.x & 7, i = blockIdx.x >> 3;
  return i < per ? x * per + i : n;
}

// Inclusive prefix sum over the wave (DPP: no LDS round trips).
__device__ __forceinline__ int wave_prefix(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);   // row_shr 1, 2, 4, 8: rows of 16 lanes
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);   // row_bcast 15, 31: the rows below
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
  return x;
}
// n / d for n < 2^30 with a quotient below 2^22 (one rounding of the reciprocal and one of the product: off by one at most)
__device__ __forceinline__ int small_quotient(int n, int d) {
  int q = (int)((float)n * __builtin_amdgcn_rcpf((float)d));
  const int r = n - q * d;
  return r < 0 ? q - 1 : r >= d ? q + 1 : q;
}

// few_kernel's work: the key tiles of all (KV head, request, row tile), one after another, are W (below 2^30, checked on the
// host); workgroup w takes the `per` tiles from w per on, so all end together whatever the lengths are, and a row
// tile's keys are cut where a range ends.  Every wave finds its place by itself, from the lengths: in a first step
// lane l adds the tiles of a group of requests, in a second one the lanes take one request each of the group that is
// looked for (one request per lane up to 64: the second step is the first).  It is kept short: a wave takes 4 cycles per
// instruction and its first copies wait for it.
template <int M, int TK>
struct Ranges {
  struct Request {
    Lengths x;
    int rts, nt;                                   // row tiles, and the key tiles that each is given (the most that any has)
  };
  const PagedKArgs& a;
  int lane, group;                                 // requests of a lane
  Request own;                                     // the lane's (last) one
  int before;                                      // tiles of the lanes below, for one KV head
  int W1, W, per;                                  // tiles of a KV head, of all, of a workgroup
  __device__ __forceinline__ Request request(int b) const {
    Request r{{0, 0, 0}, 0, 0};
    if (b >= a.B) return r;
    r.x = lengths_of(a, b);
    r.rts = r.x.n > 0 ? (r.x.n * a.G + M - 1) / M : r.x.n;
    const int all = (max(r.x.L, 1) + TK - 1) / TK;
    r.nt = all;                                    // its last row's keys; a row tile that sees none is written too
    if (a.window) {
      if (r.rts <= 1) r.nt = max(row_tile<M, TK>(a, r.x, 0).nt, 1);
      else r.nt = min(all, ((a.sinks + 15) / 16 + (a.window + (M + a.G - 2) / a.G + 14) / 16 + TK / 16) / (TK / 16) + 1);
    }
    return r;
  }
  // groups: a power of two
  __device__ __forceinline__ Ranges(const PagedKArgs& args, int groups) : a(args) {
    lane = lane_id();
    group = (a.B + 63) >> 6;
    int tiles = 0;
    bool falls = false;
    for (int k = 0; k < group; ++k) {
      own = request(lane * group + k);
      falls |= own.rts < 0;
      tiles += own.rts * own.nt;
    }
    if (__ballot(falls) != 0) tiles = 0;           // row numbers that fall: no row is written
    const int upto = wave_prefix(tiles);
    before = upto - tiles;
    W1 = __builtin_amdgcn_readlane(upto, 63);
    W = W1 * a.Hk;
    const int sh = 31 - __builtin_clz(groups);
    per = max((W + groups - 1) >> sh, 1);          // at least 2 or 4: one request of 1000 tokens 13.8, 17.2 us, not 12.2
  }
  // The row tile that tile `pos` (< W) of all belongs to: its first tile's place `start`, its key tiles nt.
  struct Place {
    Lengths x;
    int hk, b, rt, nt, start;
  };
  __device__ __forceinline__ Place find(int pos) const {
    Place w;
    w.hk = __builtin_amdgcn_readfirstlane(small_quotient(pos, W1));
    const int i = pos - w.hk * W1;
    Request r = own;
    int l = __popcll(__ballot(before <= i)) - 1, at = before;   // the last lane of those at the same place: it holds tiles
    w.b = l * group;
    if (group > 1) {                               // group <= 64
      const int base = __builtin_amdgcn_readlane(before, l);
      r = request(lane < group ? w.b + lane : a.B);
      const int tiles = r.rts * r.nt;
      at = base + wave_prefix(tiles) - tiles;
      l = (int)__builtin_ctzll(__ballot(at <= i && at + tiles > i));
      w.b += l;
    }
    w.nt = __builtin_amdgcn_readlane(r.nt, l);
    w.x.row0 = __builtin_amdgcn_readlane(r.x.row0, l);
    w.x.n = __builtin_amdgcn_readlane(r.x.n, l);
    w.x.L = __builtin_amdgcn_readlane(r.x.L, l);
    const int rts = __builtin_amdgcn_readlane(r.rts, l), from = w.hk * W1 + __builtin_amdgcn_readlane(at, l);
    const int x = rts > 1 ? (pos - from) / w.nt : 0;
    w.rt = rts - 1 - x;
    w.start = from + x * w.nt;
    return w;
  }
};

__device__ __forceinline__ bool find_piece(const PagedKArgs& a, Piece& w) {
  if (a.pieces != nullptr) {                       // plan_pieces_kernel's list
    const int N = scalar_load(a.head, 0), p = piece_of(N * a.Hk);
    if (p >= N * a.Hk) return false;
    w.hk = p / N;
    const int32_t* e = reinterpret_cast<const int32_t*>(a.pieces + (p - w.hk * N));
    w.b = scalar_load(e, 0);
    w.rt = scalar_load(e, 1);
    w.begin = scalar_load(e, 2);
    w.slot = scalar_load(e, 3);
    w.count = scalar_load(a.head, 2);
    if (w.slot >= 0) w.slot += w.hk * scalar_load(a.head, 3);
    return true;
  }
  const int R = a.B * a.row_tiles, p = piece_of(R * a.Hk);   // one piece per row tile
  if (p >= R * a.Hk) return false;
  w.hk = p / R;
  const int i = p - w.hk * R;
  w.b = i / a.row_tiles;
  w.rt = a.row_tiles - 1 - (i - w.b * a.row_tiles);
  w.begin = 0;
  w.slot = -1;
  w.count = INT_MAX;
  return true;
}

constexpr float kLog2e = 1.44269504088896340736f;
// f16 holds weights down to 2^-24; taken 2^7 times as large they reach from 2^15 (past the slack) to 2^-31 of the
// running maximum's weight
template <typename T> constexpr float kBias = std::is_same<T, f16_t>::value ? 7.0f : 0.0f;
// log2 e times the scale, above 0: a hidden key's -inf stays one.  (Scales below 0, whose sign would have to go into Q, made
// single tokens 4% slower and are refused.)
__device__ __forceinline__ float score_scale(const PagedKArgs& a) { return fmaxf(a.scale * kLog2e, 1e-30f); }
constexpr float kSlack = 8.0f;                     // a row's running max is raised past 2^8 only: few rescales of O

template <typename T, int D, bool PAGED, int NW>
__global__ __launch_bounds__(64 * NW) void few_kernel(PagedKArgs a) {
  using Ops = MfmaOps<T>;
  using V8 = typename Ops::V8;
  using Copy = GroupCopy<D, PAGED>;
  constexpr int TILE = 32 * D * 2;                 // bytes of 32 keys
  constexpr int RING = 4 * TILE;                   // of a wave: two K tiles, two V tiles
  constexpr int NI = 2 * Copy::NI;                 // copies of 32 keys
  __shared__ __attribute__((aligned(1024))) char lds[NW * RING];
  __shared__ float2 ml[NW][64];
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  char* ring = lds + wave * RING;
  const uint32_t ring0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)ring);
  const Ranges<32, 32 * NW> ranges(a, gridDim.x);
  const int first = blockIdx.x * ranges.per, end = min(first + ranges.per, ranges.W);
  if (first >= end) return;

  // A piece: a row tile, or the part of its keys that lies in the range.
  struct Seg {
    int hk, b, begin, cnt, slot;                   // slot: where a part's sums go (-1: the whole row tile)
    RowTile u;
    LaneRow me;
  } sg;
  V8 qf[D / 16];
  Copy cp(a, lane);
  // pages of the two groups of a step's keys (-1: none) and the keys' slots there
  struct Ent {
    int e[2], slot[2];
  } x0, x1, x2;
  // this wave's two groups of keys of each of the piece's tiles: the first one's place among those visited
  auto group_of = [&](int i) { return (sg.begin + i) * (2 * NW) + 2 * wave; };
  auto load_ent = [&](int i) {
    Ent x{{-1, -1}, {0, 0}};
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int k = sg.u.key_of(group_of(i) + g);
      if (i < sg.cnt && Copy::seen(a, sg.u, k)) x.e[g] = cp.entry(Copy::page_of(a, k, x.slot[g]));
    }
    return x;
  };
  auto there = [&](Ent& x) {                     // looked at a step after it is loaded
#pragma unroll
    for (int g = 0; g < 2; ++g)
      if (!Copy::is_page(a, x.e[g])) x.e[g] = -1;
  };
  auto issue = [&](auto v, int i, const Ent& x) {
    constexpr bool V = decltype(v)::value;
    const uint32_t at = ring0 + ((V ? 2 : 0) + (i & 1)) * TILE;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int k = sg.u.key_of(group_of(i) + g);
      cp.template issue<V>(a, sg.u, at + g * TILE / 2, x.e[g], x.slot[g], k, x.e[g] >= 0 && Copy::whole(a, sg.u, k, 16));
    }
  };
  auto issue_k = [&](int i, const Ent& x) { issue(std::integral_constant<bool, false>(), i, x); };
  auto issue_v = [&](int i, const Ent& x) { issue(std::integral_constant<bool, true>(), i, x); };
  // Begins the piece at tile pos: its rows of Q and its first two K tiles are requested.  Returns its tiles.
  auto open = [&](int pos) {
    const auto at = ranges.find(pos);
    const int count = min(at.start + at.nt, end) - pos;
    sg.hk = at.hk;
    sg.b = at.b;
    sg.begin = pos - at.start;
    sg.slot = count == at.nt ? -1 : 2 * blockIdx.x + (pos != first);   // a range's first piece or, not starting with it, its last
    sg.u = row_tile<32, 32 * NW>(a, at.x, at.rt);
    sg.me = lane_row(a, sg.u, l32);
    sg.cnt = min(count, sg.u.nt - sg.begin);
    if (sg.cnt > 0 && sg.u.key_of(group_of(sg.cnt - 1)) >= sg.u.kend) --sg.cnt;   // the last tile ends before this wave's keys
    cp.place(a, sg.b, sg.hk);
    load_q<V8, D>(a, sg.u, sg.me, sg.b, sg.hk, hi, qf);
    x0 = load_ent(0);
    x1 = load_ent(1);
    x2 = load_ent(2);
    there(x0);
    there(x1);
    if (sg.cnt > 0) issue_k(0, x0);
    if (sg.cnt > 1) issue_k(1, x1);
    return count;
  };
  constexpr int ROWB = Copy::ROWB, SWM = Copy::SWM;
  const uint32_t k_lane = (uint32_t)(l32 * ROWB + ((hi ^ ((D == 128 ? l32 : l32 >> 1) & SWM)) << 4));
  const int vrow = hi * 4 + ((lane & 15) >> 2);
  const uint32_t v_lane = (uint32_t)(vrow * ROWB + (lane & 1) * 8 +
                                     (((((lane >> 4) & 1) * 2 + ((lane & 3) >> 1)) ^ v_swz<D>(vrow)) << 4));
  const float sc = score_scale(a);
  int pos = first;
  pos += open(pos);
  while (true) {
    float m_run = -INFINITY, l_run = 0.f;
    f32x16_t o[D / 32];
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[dt][r] = 0.f;

    // Copies on their way at the top of step i: K(i), V(i), K(i+1), V(i+1), in this order (step 0: K(0), K(1), V(0), V(1));
    // K(i+2) and V(i+2) are requested as soon as their place is read.
#pragma unroll
    for (int st = 0; st < D / 16; ++st) asm volatile("" : "+v"(qf[st]));   // Q is here: the loop's waits count copies only
    if (sg.cnt > 0) issue_v(0, x0);
    if (sg.cnt > 1) issue_v(1, x1);
    for (int i = 0; i < sg.cnt; ++i) {
      if (i + 1 >= sg.cnt) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NI) : "memory");
      else if (i == 0) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * NI) : "memory");
      else asm volatile("s_waitcnt vmcnt(%0)" ::"n"(3 * NI) : "memory");
      const char* kt = ring + (i & 1) * TILE;
      f32x16_t s;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
      for (int st = 0; st < D / 16; ++st) s = Ops::mma(__builtin_bit_cast(V8, lds16(kt, k_lane ^ (uint32_t)(st << 5))), qf[st], s);
      there(x2);
      const Ent x3 = load_ent(i + 3);
      if (i + 2 < sg.cnt) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        issue_k(i + 2, x2);
      }
      {
        const int k0 = sg.u.key_of(group_of(i)), k1 = sg.u.key_of(group_of(i) + 1);
        if (x0.e[0] < 0 || x0.e[1] < 0 || k1 != k0 + 16 || needs_mask(a, sg.u.p_lo, sg.u.p_hi, k0, 32))
          mask_keys(a, s, sg.me.p, k0, k1, hi, x0.e[0] >= 0, x0.e[1] >= 0);
      }
      float mx = s[0], h0, h1;
#pragma unroll
      for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
      lane_halves(mx, h0, h1);
      mx = fmaxf(h0, h1) * sc;
      const bool up = mx > m_run + kSlack;
      const float al = up ? __builtin_amdgcn_exp2f(m_run - mx) : 1.0f;
      m_run = up ? mx : m_run;
      const float mu = (m_run == -INFINITY ? 0.f : m_run) - kBias<T>;
      V8 pb[2];
      float rs = 0.f;
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        float pv[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) pv[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * kk + j], sc, -mu));
        pb[kk] = Ops::pack(pv);
        rs = Ops::sum8(pb[kk], rs);
      }
      lane_halves(rs, h0, h1);
      l_run = l_run * al + (h0 + h1);
      if (__builtin_amdgcn_ballot_w64(al != 1.0f) != 0) {
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[dt][r] *= al;
      }
      if (i + 1 >= sg.cnt) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      else if (i == 0 && i + 2 >= sg.cnt) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NI) : "memory");
      else if (i == 0 || i + 2 >= sg.cnt) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * NI) : "memory");
      else asm volatile("s_waitcnt vmcnt(%0)" ::"n"(3 * NI) : "memory");
      const char* vt = ring + (2 + (i & 1)) * TILE;
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt) {
          const uint32_t lo = (v_lane ^ (uint32_t)(dt << 6)) + kk * 16 * ROWB;
          o[dt] = Ops::mma(__builtin_bit_cast(V8, join8(lds_tr8(vt, lo), lds_tr8(vt, lo + 8 * ROWB))), pb[kk], o[dt]);
        }
      if (i + 2 < sg.cnt) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        issue_v(i + 2, x2);
      }
      x0 = x1;
      x1 = x2;
      x2 = x3;
    }
    // ---- the waves' sums joined through LDS (the V tiles' place), wave w taking dims 32 w, 32 (w + NW) ..; the next piece's
    // first copies go out before
    constexpr int NV = D / 32;
    constexpr int SUMS = 2 * TILE;                 // of a wave's ring: [D / 32][4][64 lanes] 4 floats
    static_assert(NV * 4 * 64 * 16 == 2 * TILE, "the sums take the place of two V tiles");
#pragma unroll
    for (int dt = 0; dt < NV; ++dt)
#pragma unroll
      for (int g4 = 0; g4 < 4; ++g4)
        reinterpret_cast<float4*>(ring + SUMS)[(dt * 4 + g4) * 64 + lane] =
            make_float4(o[dt][4 * g4], o[dt][4 * g4 + 1], o[dt][4 * g4 + 2], o[dt][4 * g4 + 3]);
    ml[wave][lane] = make_float2(m_run, l_run);
    const LaneRow me = sg.me;
    const int slot = sg.slot;
    uint16_t* op = out_row(a, sg.u, me, sg.b, sg.hk);
    const bool more = pos < end;
    if (more) pos += open(pos);
    __syncthreads();
    if (me.on) {
      float m = -INFINITY, l = 0.f, f[NW];
#pragma unroll
      for (int w = 0; w < NW; ++w) m = fmaxf(m, ml[w][lane].x);
      const float mu = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        f[w] = __builtin_amdgcn_exp2f(ml[w][lane].x - mu);
        l += ml[w][lane].y * f[w];
      }
      const float inv = l != 0.f ? 1.0f / l : 0.f;
#pragma unroll
      for (int dt = wave; dt < NV; dt += NW)
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4) {
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int w = 0; w < NW; ++w) {
            const float4 x = reinterpret_cast<const float4*>(lds + w * RING + SUMS)[(dt * 4 + g4) * 64 + lane];
            acc.x += x.x * f[w];
            acc.y += x.y * f[w];
            acc.z += x.z * f[w];
            acc.w += x.w * f[w];
          }
          if (slot < 0) store_out<T>(op, dt * 32 + g4 * 8 + hi * 4, acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
          else reinterpret_cast<float4*>(a.part_o)[(((int64_t)slot * NV + dt) * 4 + g4) * 64 + lane] = acc;
        }
      if (slot >= 0 && wave == 0 && hi == 0) {
        a.part_ml[(int64_t)slot * 64 + l32] = m;
        a.part_ml[(int64_t)slot * 64 + 32 + l32] = l;
      }
    }
    if (!more) return;
    __syncthreads();                               // the sums are read: V tiles may come
  }
}

// The pieces' sums joined: 32 rows and 32 dims of a split row tile per workgroup.  A thread adds 4 dims of one row over every J-th
// piece (J as many threads as there are for an item), then the J sums are added in LDS; always in the same
// order.  Wave 0 looks up what the workgroup joins (mostly nothing).
constexpr int kJoinThreads = 256;
template <typename T, int D, int M>
__global__ __launch_bounds__(kJoinThreads) void combine_kernel(PagedKArgs a) {
  constexpr int QW = M / 32, NV = D / 32, NT = kJoinThreads, AHEAD = M == 32 ? 8 : 16;
  constexpr bool FEW = M == 32;
  __shared__ float4 part[NT];
  __shared__ float2 ml[NT];
  __shared__ int job[10];                          // pieces, first slot, second slot, KV head, request, row tile, lengths
  const int tid = threadIdx.x, dt = blockIdx.x % NV, qq = blockIdx.x / NV % QW, w = blockIdx.x / (NV * QW);
  if (tid < 64) {
    int np = 0;
    if constexpr (FEW) {
      // the row tile that the end of range w cuts, if it is the first that does
      const Ranges<M, 32 * kFewWaves> ranges(a, a.slots);
      const int cut = (w + 1) * ranges.per;
      if (cut < ranges.W) {
        const auto at = ranges.find(cut);
        if (at.start < cut && at.start >= w * ranges.per) {
          np = small_quotient(at.start + at.nt - 1, ranges.per) - w + 1;
          if (tid == 0) {
            job[1] = 2 * w + (at.start != w * ranges.per);
            job[2] = 2 * (w + 1);                  // the others are their ranges' first pieces
            job[3] = at.hk;
            job[4] = at.b;
            job[5] = at.rt;
            job[6] = at.x.row0;
            job[7] = at.x.n;
            job[8] = at.x.L;
          }
        }
      }
    } else {
      const int Q = scalar_load(a.head, 1), hk = w / a.max_splits, i = w - hk * a.max_splits;
      if (i < Q) {
        const int32_t* e = reinterpret_cast<const int32_t*>(a.splits + i);
        const int b = scalar_load(e, 0);
        const Lengths x = lengths_of(a, b);
        np = scalar_load(e, 2);
        if (tid == 0) {
          job[1] = (scalar_load(e, 3) + hk * scalar_load(a.head, 3)) * QW + qq;
          job[2] = job[1] + QW;
          job[3] = hk;
          job[4] = b;
          job[5] = scalar_load(e, 1);
          job[6] = x.row0;
          job[7] = x.n;
          job[8] = x.L;
        }
      }
    }
    if (tid == 0) job[0] = np;
  }
  __syncthreads();
  const int np = __builtin_amdgcn_readfirstlane(job[0]);
  if (np == 0) return;
  const int s0 = __builtin_amdgcn_readfirstlane(job[1]), s1 = __builtin_amdgcn_readfirstlane(job[2]);
  const int hk = __builtin_amdgcn_readfirstlane(job[3]), b = __builtin_amdgcn_readfirstlane(job[4]);
  const Lengths x = {__builtin_amdgcn_readfirstlane(job[6]), __builtin_amdgcn_readfirstlane(job[7]),
                     __builtin_amdgcn_readfirstlane(job[8])};
  const RowTile u = row_tile<M, 64>(a, x, __builtin_amdgcn_readfirstlane(job[5]));
  const int rows = min(u.nrows - qq * 32, 32);
  if (rows <= 0) return;
  const int items = rows * 8, J = NT / items;      // an item: row, and 4 dims: 32 dt + 4 c ..
  auto slot_of = [&](int j) { return (int64_t)(j == 0 ? s0 : s1 + (j - 1) * (FEW ? 2 : QW)); };
  const int jg = tid / items, it = tid - jg * items;
  const int c = it / rows, r = it - c * rows;
  float m = -INFINITY, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (jg < J)
    for (int j0 = jg; j0 < np; j0 += AHEAD * J) {
      float mj[AHEAD], lj[AHEAD];
      float4 xj[AHEAD];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        const int64_t s = slot_of(min(j0 + k * J, np - 1));
        mj[k] = a.part_ml[s * 64 + r];
        lj[k] = a.part_ml[s * 64 + 32 + r];
        xj[k] = reinterpret_cast<const float4*>(a.part_o)[((s * NV + dt) * 4 + (c >> 1)) * 64 + (c & 1) * 32 + r];
      }
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        if (j0 + k * J >= np) break;
        const float mn = fmaxf(m, mj[k]), mu = mn == -INFINITY ? 0.f : mn;
        const float f0 = __builtin_amdgcn_exp2f(m - mu), f1 = __builtin_amdgcn_exp2f(mj[k] - mu);
        m = mn;
        l = l * f0 + lj[k] * f1;
        acc.x = acc.x * f0 + xj[k].x * f1;
        acc.y = acc.y * f0 + xj[k].y * f1;
        acc.z = acc.z * f0 + xj[k].z * f1;
        acc.w = acc.w * f0 + xj[k].w * f1;
      }
    }
  if (J > 1) {
    part[tid] = acc;
    ml[tid] = make_float2(m, l);
    __syncthreads();
    for (int k = 1; jg == 0 && k < J; ++k) {
      const float2 o = ml[k * items + it];
      const float4 y = part[k * items + it];
      const float mn = fmaxf(m, o.x), mu = mn == -INFINITY ? 0.f : mn;
      const float f0 = __builtin_amdgcn_exp2f(m - mu), f1 = __builtin_amdgcn_exp2f(o.x - mu);
      m = mn;
      l = l * f0 + o.y * f1;
      acc.x = acc.x * f0 + y.x * f1;
      acc.y = acc.y * f0 + y.y * f1;
      acc.z = acc.z * f0 + y.z * f1;
      acc.w = acc.w * f0 + y.w * f1;
    }
  }
  const LaneRow me = lane_row(a, u, qq * 32 + r);
  if (jg > 0 || !me.on) return;
  const float inv = l != 0.f ? 1.0f / l : 0.f;
  store_out<T>(out_row(a, u, me, b, hk), dt * 32 + c * 4, acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
}

template <typename T, int D, bool PAGED>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void many_kernel(PagedKArgs a) {
  using Ops = MfmaOps<T>;
  using V8 = typename Ops::V8;
  using Copy = GroupCopy<D, PAGED>;
  constexpr int TK = 64, TILE = TK * D * 2;        // bytes of a K or V tile
  constexpr int ROWB = Copy::ROWB, SWM = Copy::SWM, GB = 16 * ROWB;
  // 64 KiB, so two workgroups share a CU (four tiles deep at head dim 64, in as much: 47.8 us against 44.8 for a batch of
  // windows)
  __shared__ __attribute__((aligned(1024))) char lds[2][2][TILE];   // [K, V][buffer]
  Piece pc;
  if (!find_piece(a, pc)) return;
  const RowTile u = row_tile<128, TK>(a, lengths_of(a, pc.b), pc.rt);
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const LaneRow me = lane_row(a, u, wave * 32 + l32);
  // positions of this wave's first and last row
  const int w_lo = u.L - u.n + (u.r0 + min(wave * 32, max(u.nrows, 1) - 1)) / a.G;
  const int w_hi = u.L - u.n + (u.r0 + min(wave * 32 + 31, max(u.nrows, 1) - 1)) / a.G;
  Copy cp(a, lane);
  cp.place(a, pc.b, pc.hk);
  const int cnt = min(pc.count, u.nt - pc.begin);
  // A tile's place: its first key (the first of this wave's group, where the tile's keys are not one run), and, kept as one
  // number, the page of the group that this wave copies (group w of each tile), whether the tile is one run of keys that
  // are all seen by some row (bit 4) and which groups are there (bits 0 - 3).  The table's
  // entries are loaded a step before they are looked at.  The loop's scalar instructions cost as vector ones do, so a
  // tile that is seen as a whole and lies in one page takes the short way (3-4% of a chunk's time).
  struct Raw {
    int key0, slot, e[4], all, one;                // one: all in one page
  };
  struct Tile {
    int key0, slot, page;
  };
  auto load_raw = [&](int i) {
    Raw x;
    const int g0 = (pc.begin + i) * 4;
    x.key0 = u.key_of(g0);
    x.all = i < cnt && (g0 >= u.ns || g0 + 4 <= u.ns) && Copy::whole(a, u, x.key0, TK);
    const int page = Copy::page_of(a, x.key0, x.slot);
    x.one = x.all && (!PAGED || x.slot + TK <= a.page_size);
    if (x.one) {
      x.e[0] = x.e[1] = x.e[2] = x.e[3] = cp.entry(page);
      x.slot += 16 * wave;
      return x;
    }
    if (PAGED && x.all && x.slot == 0 && a.page_size <= 32) {
      // four pages of 16 or two of 32, all below the request's last one
      const int two = a.page_size >> 5;
#pragma unroll
      for (int g = 0; g < 4; ++g) x.e[g] = cp.entry(page + (g >> two));
      x.slot = (16 * wave) & (a.page_size - 1);
      return x;
    }
    x.slot = 0;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int k = u.key_of(g0 + g);
      int slot = 0;
      x.e[g] = -1;
      if (i < cnt && Copy::seen(a, u, k)) x.e[g] = cp.entry(Copy::page_of(a, k, slot));
      if (g == wave) {
        x.slot = slot;
        if (!x.all) x.key0 = k;
      }
    }
    return x;
  };
  auto pack = [&](const Raw& x) {
    int own = x.e[0], there = (x.e[0] >= 0 && Copy::is_page(a, x.e[0])) ? 1 : 0;
    if (x.one) {
      there *= 15;
    } else {
#pragma unroll
      for (int g = 1; g < 4; ++g) {
        there |= (x.e[g] >= 0 && Copy::is_page(a, x.e[g])) ? 1 << g : 0;
        own = wave == g ? x.e[g] : own;
      }
    }
    return Tile{x.key0, x.slot, ((there >> wave & 1) ? own << 5 : -32) | (x.all ? 16 : 0) | there};
  };
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)&lds[0][0][0]) + wave * GB;
  auto issue = [&](auto v, int i, const Tile& x) {
    constexpr bool V = decltype(v)::value;
    cp.template issue<V>(a, u, lds0 + ((V ? 2 : 0) + (i & 1)) * TILE, x.page >> 5, x.slot, x.key0,
                         (x.page & 31) == 31);
  };
  auto issue_k = [&](int i, const Tile& x) { issue(std::integral_constant<bool, false>(), i, x); };
  auto issue_v = [&](int i, const Tile& x) { issue(std::integral_constant<bool, true>(), i, x); };

  V8 qf[D / 16];
  load_q<V8, D>(a, u, me, pc.b, pc.hk, hi, qf);
  const uint32_t k_lane = (uint32_t)(l32 * ROWB + ((hi ^ ((D == 128 ? l32 : l32 >> 1) & SWM)) << 4));
  const int vrow = hi * 4 + ((lane & 15) >> 2);
  const uint32_t v_lane = (uint32_t)(vrow * ROWB + (lane & 1) * 8 +
                                     (((((lane >> 4) & 1) * 2 + ((lane & 3) >> 1)) ^ v_swz<D>(vrow)) << 4));
  const float sc = score_scale(a);
  float m_run = -INFINITY, l_run = 0.f;
  f32x16_t o[D / 32];
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[dt][r] = 0.f;

  auto compute_s = [&](int buf, f32x16_t* s) {
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[kt][r] = 0.f;
#pragma unroll
    for (int st = 0; st < D / 16; ++st) {
      const uint32_t lo = k_lane ^ (uint32_t)(st << 5);
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
        s[kt] = Ops::mma(__builtin_bit_cast(V8, lds16(lds[0][buf] + kt * 32 * ROWB, lo)), qf[st], s[kt]);
    }
  };
  auto mask = [&](int i, f32x16_t* s, const Tile& t) {
    const int x = t.page, g0 = (pc.begin + i) * 4;
    if ((x & 31) == 31 && !needs_mask(a, w_lo, w_hi, t.key0, TK)) return;   // one test in most steps
    mask_keys(a, s[0], me.p, u.key_of(g0), u.key_of(g0 + 1), hi, x & 1, x & 2);
    mask_keys(a, s[1], me.p, u.key_of(g0 + 2), u.key_of(g0 + 3), hi, x & 4, x & 8);
  };
  auto exps = [&](const f32x16_t* s, V8* pb, float m_use) {
    float rs = 0.f;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      float pv[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) pv[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kk >> 1][8 * (kk & 1) + j], sc, -m_use));
      pb[kk] = Ops::pack(pv);
      rs = Ops::sum8(pb[kk], rs);
    }
    return rs;
  };
  auto pv_mma = [&](int buf, const V8* pb) {
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt) {
        const uint32_t lo = (v_lane ^ (uint32_t)(dt << 6)) + kk * 16 * ROWB;
        o[dt] = Ops::mma(__builtin_bit_cast(V8, join8(lds_tr8(lds[1][buf], lo), lds_tr8(lds[1][buf], lo + 8 * ROWB))),
                         pb[kk], o[dt]);
      }
  };
  // Step t: wait for K(t+1) and V(t-1), one barrier, copy K(t+2) over K(t) and V(t) over V(t-2); then S(t+1) and
  // P V(t-1) on MFMA between the exponentials of tile t; then O's rescale (rare) and the masks of tile t+1.
  f32x16_t sa[2], sb[2];
  V8 pa[4], pb[4];
  Tile x[3];                                       // of tiles t .. t+2, the last one packed from
  Raw raw;                                         // its entries
  typedef std::integral_constant<bool, true> yes;
  typedef std::integral_constant<bool, false> no;
  auto iter = [&](int t, f32x16_t* s_next, f32x16_t* s_cur, V8* p_prev, V8* p_cur, auto hasS, auto hasPV, auto hasE) {
    __builtin_amdgcn_s_setprio(0);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    x[2] = pack(raw);
    if (t + 2 < cnt) issue_k(t + 2, x[2]);
    if (t < cnt) issue_v(t, x[0]);
    raw = load_raw(t + 3);
    __builtin_amdgcn_s_setprio(2);
    float rs = 0.f, al = 1.0f;
    if constexpr (decltype(hasS)::value) compute_s((t + 1) & 1, s_next);
    if constexpr (decltype(hasPV)::value) pv_mma((t - 1) & 1, p_prev);
    if constexpr (decltype(hasE)::value) {
      float mx = s_cur[0][0], m0, m1;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s_cur[kt][r]);
      lane_halves(mx, m0, m1);
      mx = fmaxf(m0, m1) * sc;
      const bool up = mx > m_run + kSlack;
      al = up ? __builtin_amdgcn_exp2f(m_run - mx) : 1.0f;
      m_run = up ? mx : m_run;
      rs = exps(s_cur, p_cur, (m_run == -INFINITY ? 0.f : m_run) - kBias<T>);
    }
    if constexpr (decltype(hasS)::value && decltype(hasPV)::value && decltype(hasE)::value) {
      // one MFMA, then three VALU instructions, operand reads eight MFMAs ahead (6: 1.9% slower, 10: 65%; VPM 4: 0.5%)
      constexpr int NS = 2 * (D / 16), NM = NS + 4 * (D / 32), LA = 8, VPM = 3;
      __builtin_amdgcn_sched_group_barrier(0x100, LA, 0);
#pragma unroll
      for (int i = 0; i < NM; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        if (i + LA < NS) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        else if (i + LA < NM) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, VPM, 0);
      }
    }
    if constexpr (decltype(hasE)::value) {
      float r0, r1;
      lane_halves(rs, r0, r1);
      l_run = l_run * al + (r0 + r1);
      if (__builtin_amdgcn_ballot_w64(al != 1.0f) != 0) {
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[dt][r] *= al;   // O holds P V up to t-1 now
      }
    }
    if constexpr (decltype(hasS)::value) mask(t + 1, s_next, x[1]);
    x[0] = x[1];
    x[1] = x[2];
  };
  x[0] = pack(load_raw(0));
  x[1] = pack(load_raw(1));
  raw = load_raw(2);
  if (cnt > 0) issue_k(0, x[0]);
  if (cnt > 1) issue_k(1, x[1]);
  __builtin_amdgcn_s_waitcnt(0);
  if (wave * 32 >= u.nrows) {
    // A wave without rows (beside a single token, a request's last rows) only copies, in step with the others.  (The same for the
    // steps in which a wave's rows see nothing, at a window's edges, spilled registers in the loop: 5-25% slower.)
    auto copy = [&](auto v, int i) {
      constexpr bool V = decltype(v)::value;
      const int k = u.key_of((pc.begin + i) * 4 + wave);
      int slot = 0, e = Copy::seen(a, u, k) ? cp.entry(Copy::page_of(a, k, slot)) : -1;
      if (!Copy::is_page(a, e)) e = -1;
      cp.template issue<V>(a, u, lds0 + ((V ? 2 : 0) + (i & 1)) * TILE, e, slot, k, e >= 0 && Copy::whole(a, u, k, 16));
    };
    if (cnt > 0) __builtin_amdgcn_s_barrier();
    for (int t = 0; cnt > 0 && t <= cnt; ++t) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      if (t + 2 < cnt) copy(std::integral_constant<bool, false>(), t + 2);
      if (t < cnt) copy(std::integral_constant<bool, true>(), t);
    }
    return;
  }
  if (cnt > 0) {
    __builtin_amdgcn_s_barrier();
    compute_s(0, sa);
    mask(0, sa, x[0]);
    if (cnt > 1) iter(0, sb, sa, pb, pa, yes(), no(), yes());
    else iter(0, sb, sa, pb, pa, no(), no(), yes());
    int t = 1;
    for (; t + 2 < cnt; t += 2) {
      iter(t, sa, sb, pa, pb, yes(), yes(), yes());
      iter(t + 1, sb, sa, pb, pa, yes(), yes(), yes());
    }
    if (t + 1 < cnt) {                             // t odd, t + 1 = cnt - 1
      iter(t, sa, sb, pa, pb, yes(), yes(), yes());
      iter(t + 1, sb, sa, pb, pa, no(), yes(), yes());
      iter(t + 2, sa, sb, pa, pb, no(), yes(), no());
    } else if (t < cnt) {                          // t = cnt - 1, odd
      iter(t, sa, sb, pa, pb, no(), yes(), yes());
      iter(t + 1, sb, sa, pb, pa, no(), yes(), no());
    } else {                                       // cnt == 1: the final P V
      iter(t, sa, sb, pa, pb, no(), yes(), no());
    }
  }
  // this lane's row again, and the output's arguments: neither held a register in the loop
  int ln = lane;
  asm volatile("" : "+v"(ln));
  const LateArgs late;
  const LaneRow mine = lane_row(late, u, wave * 32 + (ln & 31));
  if (pc.slot >= 0) {
    if (!mine.on) return;
    const int64_t s = (int64_t)pc.slot * 4 + wave;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int g4 = 0; g4 < 4; ++g4)
        reinterpret_cast<float4*>(late.part_o)[((s * (D / 32) + dt) * 4 + g4) * 64 + ln] =
            make_float4(o[dt][4 * g4], o[dt][4 * g4 + 1], o[dt][4 * g4 + 2], o[dt][4 * g4 + 3]);
    if (ln < 32) {
      late.part_ml[s * 64 + ln] = m_run;
      late.part_ml[s * 64 + 32 + ln] = l_run;
    }
    return;
  }
  // The wave's rows through LDS (its part of the K tiles, which no wave reads past the last step's barrier), so that rows are
  // written whole (stored as they stand, 16 bytes of 32 rows at once: window of 256 over 2 x 1000 23.7 us against 22.7).
  const float inv = l_run != 0.f ? 1.0f / l_run : 0.f;
  const uint64_t op = mine.on ? (uint64_t)(uintptr_t)out_row(late, u, mine, pc.b, pc.hk) : 0;
  constexpr int CPR = D / 8, RPS = 64 / CPR;       // 16-byte chunks of a row, rows of a store
  static_assert(4 * 32 * ROWB == 2 * TILE, "the four waves' rows take the place of the K tiles");
  char* rows = &lds[0][0][0] + wave * 32 * ROWB;
  auto at = [](int r, int c) { return r * ROWB + ((c ^ ((D == 128 ? r : r >> 1) & SWM)) << 4); };
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int g4 = 0; g4 < 4; ++g4)
      *reinterpret_cast<uint2*>(rows + at(ln & 31, dt * 4 + g4) + (ln >> 5) * 8) =
          out_bits<T>(o[dt][4 * g4] * inv, o[dt][4 * g4 + 1] * inv, o[dt][4 * g4 + 2] * inv, o[dt][4 * g4 + 3] * inv);
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int i = 0; i < 32 / RPS; ++i) {
    const int r = i * RPS + ln / CPR, c = ln % CPR;
    const uint32_t lo = __shfl((uint32_t)op, r, 64), up = __shfl((uint32_t)(op >> 32), r, 64);
    const uint4 w = *reinterpret_cast<const uint4*>(rows + at(r, c));
    if (lo | up) reinterpret_cast<uint4*>((uintptr_t)((uint64_t)up << 32 | lo))[c] = w;
  }
}

// many_kernel's pieces of one KV head (all have the same), as a list.  The 16 choices of key tiles per piece are tried by a wave
// each.  One workgroup; its lists are read by the attention and the joining kernel.
template <int M, int TK>
__global__ __launch_bounds__(kPlanThreads) void plan_pieces_kernel(PagedKArgs a, int4* pieces, int4* pairs, int4* splits,
                                                                   int32_t* head, int max_pieces, int max_parts,
                                                                   int slots) {
  constexpr int NW = kPlanThreads / 64;
  constexpr int kHeld = 8192;                      // row tiles whose key tiles are kept in LDS
  __shared__ int base[kMaxRequests + 1], tiles[kHeld];
  __shared__ int wsum[3][NW], wmax[NW], falls;
  __shared__ float wtot[NW], cost[NW];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // inclusive prefix sum over the workgroup; the sum of all in `all`.  Barriers by the caller: one before and one after wsum[k]
  // is written
  auto upto = [&](int k, int x, int& all) {
    int before = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      before = w == wave ? all : before;
      all += wsum[k][w];
    }
    return x + before;
  };
  if (tid == 0) falls = 0;
  __syncthreads();
  int R = 0;
  for (int b0 = 0; b0 < a.B; b0 += kPlanThreads) {
    const int b = b0 + tid;
    int n = b < a.B ? lengths_of(a, b).n : 0;
    if (n < 0) falls = 1;                          // row numbers that fall: no row is written
    n = n > 0 ? (n * a.G + M - 1) / M : 0;
    const int x = wave_prefix(n);
    if (b0) __syncthreads();
    if (lane == 63) wsum[0][wave] = x;
    __syncthreads();
    int all;
    const int at = R + upto(0, x, all) - n;
    if (b < a.B) base[b] = at;
    R += all;
  }
  if (tid == 0) base[a.B] = R;
  __syncthreads();
  if (falls) R = 0;
  float total = 0.f;                               // an estimate: its rounding does not matter
  int longest = 1;
  for (int i = tid; i < R; i += kPlanThreads) {
    int lo = 0, hi = a.B;                          // the last request with base <= i
    while (hi - lo > 1) {
      const int m = (lo + hi) >> 1;
      if (base[m] <= i) lo = m;
      else hi = m;
    }
    const int rt = base[lo + 1] - 1 - i;           // the last row tiles, whose keys are the most, first
    const int nt = row_tile<M, TK>(a, lengths_of(a, lo), rt).nt;
    pairs[i] = make_int4(lo, rt, nt, 0);
    if (i < kHeld) tiles[i] = nt;
    total += (float)nt;
    longest = max(longest, nt);
  }
  total = wave_sum(total);
  for (int o = 32; o > 0; o >>= 1) longest = max(longest, __shfl_xor(longest, o, 64));
  if (lane == 0) {
    wtot[wave] = total;
    wmax[wave] = longest;
  }
  __syncthreads();
  total = 0.f;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    total += wtot[w];
    longest = max(longest, wmax[w]);
  }
  const float W = total * (float)a.Hk;
  auto chunk_of = [&](int i) { return chunk_choice(i, longest, W, (float)R * (float)a.Hk, (float)slots); };
  {
    const int c = chunk_of(wave);
    int n = 0, sp = 0;
    for (int i = lane; i < R; i += 64) {
      const int np = parts_of(i < kHeld ? tiles[i] : pairs[i].z, c);
      n += np;
      sp += np > 1 ? np : 0;
    }
    n = wave_prefix(n);
    sp = wave_prefix(sp);
    float t = call_time((float)n * (float)a.Hk, (float)c, W, (float)slots, (float)sp * (float)a.Hk,
                        (float)parts_of(longest, c));
    if (wave > 0 && (n > max_pieces || (int64_t)sp * a.Hk > max_parts)) t = INFINITY;
    if (lane == 63) cost[wave] = t;
  }
  __syncthreads();
  int best = 0;
  float least = cost[0];
#pragma unroll
  for (int w = 1; w < NW; ++w) {
    const float t = cost[w];
    best = t < least ? w : best;
    least = fminf(t, least);
  }
  const int c = chunk_of(best);
  int N = 0, S = 0, Q = 0;
  for (int i0 = 0; i0 < R; i0 += kPlanThreads) {
    const int i = i0 + tid;
    const int4 pr = i < R ? pairs[i] : make_int4(0, 0, 0, 0);
    const int np = i < R ? parts_of(pr.z, c) : 0, sp = np > 1 ? np : 0;
    const int x0 = wave_prefix(np), x1 = wave_prefix(sp), x2 = wave_prefix(sp > 0);
    if (i0) __syncthreads();
    if (lane == 63) {
      wsum[0][wave] = x0;
      wsum[1][wave] = x1;
      wsum[2][wave] = x2;
    }
    __syncthreads();
    int all0, all1, all2;
    const int n0 = N + upto(0, x0, all0) - np, s0 = S + upto(1, x1, all1) - sp, q = Q + upto(2, x2, all2) - 1;
    if (i < R) {
      if (sp) splits[q] = make_int4(pr.x, pr.y, np, s0);
      for (int j = 0; j < np; ++j) pieces[n0 + j] = make_int4(pr.x, pr.y, j * c, sp ? s0 + j : -1);
    }
    N += all0;
    S += all1;
    Q += all2;
  }
  if (tid == 0) {
    head[0] = N;
    head[1] = Q;
    head[2] = c;
    head[3] = S;
  }
}

// ---- host ---------------------------------------------------------------------

// Workspace of a call: the split pieces' sums, and before them, in calls of many_kernel, head, pairs, pieces and splits.
struct Work {
  int64_t max_pairs, max_pieces, max_splits;
  int max_parts, rows;
  size_t pairs, pieces, splits, ml, o, bytes;
};
static size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }
// row tiles of at most `rows` rows of B requests with T tokens in all; few: row tiles of 32, no lists
static Work work_of(bool few, int64_t T, int B, int Hk, int G, int D) {
  Work w{};
  w.rows = few ? 32 : 128;
  w.max_parts = few ? 2 * few_slots(D) : kPartsMany;
  if (!few) {
    w.max_pairs = T * G / w.rows + B;
    w.max_pieces = w.max_pairs + (w.max_parts + Hk - 1) / Hk;
    w.max_splits = std::min<int64_t>(w.max_pairs, std::max(w.max_parts / (2 * Hk), 1));
    w.pairs = 256;
    w.pieces = w.pairs + align256((size_t)w.max_pairs * 16);
    w.splits = w.pieces + align256((size_t)w.max_pieces * 16);
    w.ml = w.splits + align256((size_t)w.max_splits * 16);
  }
  w.o = w.ml + align256((size_t)w.max_parts * w.rows * 8);
  w.bytes = w.o + (size_t)w.max_parts * w.rows * D * 4;
  return w;
}
// Which kernel: single tokens and few rows of a KV head are bound by the keys' bytes.  At 64 rows few_kernel reads the keys
// twice: 16 tokens of one request of 2048 20 us against 22, but of 32 requests of 4096 201 against 117.  It counts key
// tiles of row tiles (of all KV heads) in 32 bits.
static bool few_rows(int64_t max_new, int G, int64_t row_tiles, int64_t keys) {
  return max_new * G <= 32 && row_tiles < (1ll << 30) / (keys / 32 + 2);
}
// What a caller is asked for.  It never falls as an argument grows, so a workspace of the largest call serves every other
// one: the lists are sized as for one KV head, which has the most row tiles and pieces; few_kernel's size is asked for
// where that is taken with one KV head too (few_rows then holds for any number: at most 32 rows of all heads, and
// row tiles counted from above), and it is the same for both head dims.  Either kernel's fits into many_kernel's.
static size_t work_bytes(int64_t max_new, int64_t T, int B, int Hq, int Hk, int D, int64_t keys) {
  if (few_rows(max_new, Hq, T * Hq / 32 + (int64_t)B * Hk, keys))
    return std::max(work_of(true, T, B, 1, Hq, 64).bytes, work_of(true, T, B, 1, Hq, 128).bytes);
  return work_of(false, T, B, 1, Hq, D).bytes;
}

template <typename T, int D, bool PAGED>
static int launch(PagedKArgs k, bool few, bool plan, const Work& w, char* work, int B, int Lq, hipStream_t s, const char* fn) {
  const int64_t rows = (int64_t)Lq * k.G;
  k.row_tiles = (int)((rows + w.rows - 1) / w.rows);
  int64_t grid = (int64_t)B * k.row_tiles * k.Hk;
  if (few || plan) {
    k.part_ml = reinterpret_cast<float*>(work + w.ml);
    k.part_o = reinterpret_cast<float*>(work + w.o);
  }
  if (few) {
    k.slots = few_slots(D);
    few_kernel<T, D, PAGED, kFewWaves><<<k.slots, 64 * kFewWaves, 0, s>>>(k);
    if (int rc = fs_host::launch_status(fn)) return rc;
    combine_kernel<T, D, 32><<<(k.slots - 1) * (D / 32), kJoinThreads, 0, s>>>(k);
    return fs_host::launch_status(fn);
  }
  if (plan) {
    int4* pieces = reinterpret_cast<int4*>(work + w.pieces);
    k.splits = reinterpret_cast<int4*>(work + w.splits);
    k.head = reinterpret_cast<int32_t*>(work);
    k.max_splits = (int)w.max_splits;
    grid = w.max_pieces * k.Hk;
    plan_pieces_kernel<128, 64><<<1, kPlanThreads, 0, s>>>(k, pieces, reinterpret_cast<int4*>(work + w.pairs), k.splits,
                                                           k.head, (int)w.max_pieces, w.max_parts, kSlotsMany);
    if (int rc = fs_host::launch_status(fn)) return rc;
    k.pieces = pieces;
  }
  many_kernel<T, D, PAGED><<<(unsigned)((grid + 7) / 8 * 8), 256, 0, s>>>(k);
  if (int rc = fs_host::launch_status(fn)) return rc;
  if (plan) {
    combine_kernel<T, D, 128><<<(unsigned)(w.max_splits * k.Hk * 4 * (D / 32)), kJoinThreads, 0, s>>>(k);
    return fs_host::launch_status(fn);
  }
  return FS_OK;
}
template <bool PAGED>
static int run(PagedKArgs k, int dtype, int D, bool few, bool plan, const Work& w, char* work, int B, int Lq, hipStream_t s,
               const char* fn) {
  k.G = k.Hq / k.Hk;
  k.window = k.window > (1 << 27) ? 1 << 27 : k.window;   // past the longest sequence: the same rule
  k.sinks = k.sinks > (1 << 27) ? 1 << 27 : k.sinks;
  if (dtype == FS_DTYPE_BF16)
    return D == 128 ? launch<bf16_t, 128, PAGED>(k, few, plan, w, work, B, Lq, s, fn)
                    : launch<bf16_t, 64, PAGED>(k, few, plan, w, work, B, Lq, s, fn);
  return D == 128 ? launch<f16_t, 128, PAGED>(k, few, plan, w, work, B, Lq, s, fn)
                  : launch<f16_t, 64, PAGED>(k, few, plan, w, work, B, Lq, s, fn);
}

}  // namespace fs

using namespace fs;

// checks that both entry points share
static int check_common(const char* fn, int dtype, int D, int Hq, int Hk, int B, int window, int sinks, float scale,
                        int64_t rows, const int64_t* strides, int ns, const void* const* ptrs, int np) {
  FS_CHECK_ARG(Hq >= 1 && Hk >= 1 && Hq % Hk == 0, "%s: Hq=%d must be a multiple of Hk=%d", fn, Hq, Hk);
  FS_CHECK_SUPPORTED(D == 128 || D == 64, "%s: head_dim %d unsupported (64 or 128)", fn, D);
  FS_CHECK_SUPPORTED(dtype == FS_DTYPE_BF16 || dtype == FS_DTYPE_F16, "%s: dtype %d unsupported (bf16/f16)", fn, dtype);
  FS_CHECK_ARG(window >= 0 && sinks >= 0, "%s: window %d and sinks %d must not be negative", fn, window, sinks);
  FS_CHECK_ARG(std::isfinite(scale) && scale >= 0.f, "%s: softmax_scale %g must be finite and not negative", fn, scale);
  FS_CHECK_SUPPORTED(rows * Hq < (1ll << 30) && Hk <= 4096, "%s: %lld rows of %d heads unsupported", fn,
                     (long long)rows, Hq);
  FS_CHECK_SUPPORTED(B <= kMaxRequests, "%s: %d requests > %d", fn, B, kMaxRequests);
  for (int i = 0; i < ns; ++i) FS_CHECK_ARG(strides[i] % 8 == 0, "%s: strides must be multiples of 8 elements", fn);
  for (int i = 0; i < np; ++i) {
    FS_CHECK_ARG(ptrs[i] != nullptr, "%s: null tensor pointer", fn);
    FS_CHECK_ARG((uintptr_t)ptrs[i] % 16 == 0, "%s: tensors must be 16-byte aligned", fn);
  }
  return FS_OK;
}

// the most new tokens of one request
static int64_t most_new(const fs_paged_attn_args& a) { return a.max_new > 0 && a.max_new < a.T ? a.max_new : a.T; }
static bool few_rows(const fs_paged_attn_args& a) {
  const int G = a.Hq / a.Hk;
  return few_rows(most_new(a), G, ((int64_t)a.T * G / 32 + a.B) * a.Hk, (int64_t)a.P * a.page_size);
}
static bool few_rows(const fs_window_attn_args& a) {
  const int G = a.Hq / a.Hk;
  return few_rows(a.Lq, G, ((int64_t)a.B * a.Lq * G / 32 + a.B) * a.Hk, a.Lk);
}
static Work work_of(const fs_paged_attn_args& a) { return work_of(few_rows(a), a.T, a.B, a.Hk, a.Hq / a.Hk, a.D); }
static Work work_of(const fs_window_attn_args& a) {
  return work_of(few_rows(a), (int64_t)a.B * a.Lq, a.B, a.Hk, a.Hq / a.Hk, a.D);
}

extern "C" size_t fs_paged_attn_work_bytes(const fs_paged_attn_args* a) {
  if (!a || a->B <= 0 || a->T <= 0 || a->Hk <= 0 || a->Hq < a->Hk || a->D <= 0) return 0;
  return work_bytes(most_new(*a), a->T, a->B, a->Hq, a->Hk, a->D, (int64_t)a->P * a->page_size);
}
extern "C" size_t fs_window_attn_work_bytes(const fs_window_attn_args* a) {
  if (!a || a->B <= 0 || a->Lq <= 0 || a->Hk <= 0 || a->Hq < a->Hk || a->D <= 0) return 0;
  return work_bytes(a->Lq, (int64_t)a->B * a->Lq, a->B, a->Hq, a->Hk, a->D, a->Lk);
}

extern "C" int fs_paged_attn(const fs_paged_attn_args* a, void* stream) {
  const char* fn = "fs_paged_attn";
  FS_CHECK_ARG(a != nullptr, "%s: null args", fn);
  FS_CHECK_ARG(a->B >= 1 && a->T >= 0 && a->P >= 1 && a->num_pages >= 1 && a->max_new >= 0,
               "%s: B=%d T=%d P=%d num_pages=%lld max_new=%d", fn, a->B, a->T, a->P, (long long)a->num_pages, a->max_new);
  FS_CHECK_SUPPORTED(a->page_size >= 16 && a->page_size <= 4096 && a->page_size % 16 == 0,
                     "%s: page size %d unsupported (multiples of 16 up to 4096)", fn, a->page_size);
  FS_CHECK_SUPPORTED(a->num_pages < (1 << 26), "%s: %lld pages unsupported", fn, (long long)a->num_pages);
  FS_CHECK_SUPPORTED((int64_t)a->P * a->page_size <= (1 << 26), "%s: %d pages of %d tokens per request unsupported",
                     fn, a->P, a->page_size);
  if (a->T == 0) return FS_OK;
  const int64_t st[] = {a->q_st, a->q_sh, a->o_st, a->o_sh, a->k_sp, a->k_ss, a->k_sh, a->v_sp, a->v_ss, a->v_sh};
  const void* const ptrs[] = {a->q, a->out, a->k_cache, a->v_cache, a->work};
  if (int rc = check_common(fn, a->dtype, a->D, a->Hq, a->Hk, a->B, a->window, a->sinks, a->softmax_scale, a->T, st, 10,
                            ptrs, 5))
    return rc;
  FS_CHECK_ARG(a->block_table && a->cu_lens && a->seq_lens && a->t_sb >= a->P &&
                   ((uintptr_t)a->block_table | (uintptr_t)a->cu_lens | (uintptr_t)a->seq_lens) % 4 == 0,
               "%s: block_table (row stride %lld of %d), cu_lens and seq_lens must be given, 4-byte aligned", fn,
               (long long)a->t_sb, a->P);
  // a copy's lane offsets are 32-bit byte offsets over 16 slots
  FS_CHECK_SUPPORTED(a->k_ss >= 0 && a->k_ss < (1 << 23) && a->v_ss >= 0 && a->v_ss < (1 << 23),
                     "%s: slot stride unsupported", fn);
  PagedKArgs k{};
  k.q = static_cast<const uint16_t*>(a->q);
  k.k = static_cast<const uint16_t*>(a->k_cache);
  k.v = static_cast<const uint16_t*>(a->v_cache);
  k.out = static_cast<uint16_t*>(a->out);
  k.q_st = a->q_st; k.q_sh = a->q_sh; k.o_st = a->o_st; k.o_sh = a->o_sh;
  k.k_sp = a->k_sp; k.k_ss = (int)a->k_ss; k.k_sh = a->k_sh; k.v_sp = a->v_sp; k.v_ss = (int)a->v_ss; k.v_sh = a->v_sh;
  k.table = a->block_table; k.cu = a->cu_lens; k.lens = a->seq_lens; k.t_sb = a->t_sb; k.num_pages = (int)a->num_pages;
  k.B = a->B; k.T = a->T; k.Hq = a->Hq; k.Hk = a->Hk; k.P = a->P; k.page_size = a->page_size;
  k.window = a->window; k.sinks = a->sinks; k.scale = a->softmax_scale;
  const uint32_t groups = a->page_size / 16;       // x / groups for x < 2^22, groups <= 256: mulhi is exact
  k.page_magic = groups > 1 ? (uint32_t)((1ull << 32) / groups + 1) : 0;
  const bool few = few_rows(*a);
  return run<true>(k, a->dtype, a->D, few, true, work_of(*a), static_cast<char*>(a->work), a->B, a->T, (hipStream_t)stream, fn);
}

extern "C" int fs_window_attn(const fs_window_attn_args* a, void* stream) {
  const char* fn = "fs_window_attn";
  FS_CHECK_ARG(a != nullptr, "%s: null args", fn);
  FS_CHECK_ARG(a->B >= 1 && a->Lq >= 1 && a->Lk >= 1, "%s: empty sequence", fn);
  FS_CHECK_SUPPORTED(a->Lk <= (1 << 26), "%s: %d keys unsupported", fn, a->Lk);
  const int64_t st[] = {a->q_sb, a->q_sh, a->q_sl, a->k_sb, a->k_sh, a->k_sl,
                        a->v_sb, a->v_sh, a->v_sl, a->o_sb, a->o_sh, a->o_sl};
  const void* const ptrs[] = {a->q, a->out, a->k, a->v, a->work};
  if (int rc = check_common(fn, a->dtype, a->D, a->Hq, a->Hk, a->B, a->window, a->sinks, a->softmax_scale,
                            (int64_t)a->B * a->Lq, st, 12, ptrs, 5))
    return rc;
  FS_CHECK_SUPPORTED(a->k_sl >= 0 && a->k_sl < (1 << 23) && a->v_sl >= 0 && a->v_sl < (1 << 23),
                     "%s: row stride unsupported", fn);
  PagedKArgs k{};
  k.q = static_cast<const uint16_t*>(a->q);
  k.k = static_cast<const uint16_t*>(a->k);
  k.v = static_cast<const uint16_t*>(a->v);
  k.out = static_cast<uint16_t*>(a->out);
  k.q_sb = a->q_sb; k.q_st = a->q_sl; k.q_sh = a->q_sh; k.o_sb = a->o_sb; k.o_st = a->o_sl; k.o_sh = a->o_sh;
  k.k_sp = a->k_sb; k.k_ss = (int)a->k_sl; k.k_sh = a->k_sh; k.v_sp = a->v_sb; k.v_ss = (int)a->v_sl; k.v_sh = a->v_sh;
  k.num_pages = a->B; k.B = a->B; k.Hq = a->Hq; k.Hk = a->Hk; k.Lq = a->Lq; k.Lk = a->Lk; k.page_size = a->Lk;
  k.window = a->window; k.sinks = a->sinks; k.scale = a->softmax_scale;
  k.T = a->Lq;
  const bool few = few_rows(*a);
  const Work w = work_of(*a);
  // Every sequence is as long here, so whether splitting keys pays is known.  In key tiles' time at D = 128: a call without a
  // plan lasts its longest row tile (slower where two share a CU), one with it its work evenly spread and 21 for the plan,
  // more pieces' starts and the joining.  Causal, 32 / 8 heads, 1100, 2000: 29.6, 52 us without, 38.9, 61 with; 8 / 2
  // heads, 900, 1500, 4000: 22.4, 33.7, 78 without, 24.4, 31.9, 58.7 with.  At D = 64 the sides meet at the same lengths: 32 / 8
  // heads, 1100, 2000: 21.3, 37.4 without, 28.5, 45.1 with; 8 / 2 heads, 900, 1500, 4000: 17.3, 25.8, 59.6 without, 19.3, 24.2,
  // 44.2 with; window of 1500, 1500, 2000, 4000: 25.8, 27.0, 28.2 without, 24.1, 27.2, 36.6 with.
  const int64_t tiles = ((int64_t)a->Lq * (a->Hq / a->Hk) + w.rows - 1) / w.rows * a->B * a->Hk;
  const int64_t most = a->window && a->window < a->Lk ? (int64_t)a->window + std::min(a->sinks, a->Lk) + w.rows : a->Lk;
  const int64_t mean = std::min(most, std::max<int64_t>(a->Lk - a->Lq / 2, most / 2));
  const bool plan = !few && tiles < kSlotsMany &&
                    most / 64.0 * (tiles <= kSlotsMany / 2 ? 1.1 : 1.35) > 21.0 + mean / 64.0 * tiles / (kSlotsMany / 2);
  return run<false>(k, a->dtype, a->D, few, plan, w, static_cast<char*>(a->work), a->B, a->Lq, (hipStream_t)stream, fn);
}
