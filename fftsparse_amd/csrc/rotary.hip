// Rotary positions, and the rotated keys and the values into a paged cache.
//
// The first R = 2 half dims of each query and key head are rotated in pairs
// (x1, x2) -> f (x1 c - x2 s, x2 c + x1 s) with c, s = cos, sin of pos *
// inv_freq[i]; pair i is dims (i, i + half), or (2 i, 2 i + 1) interleaved.
// The other dims are copied.  Angles are formed in 64 bits: in 32 the product
// alone is off by 2^-25 of the angle, 0.03 at position 10^6.  Their whole turns
// are taken off in 64 bits and the sine and cosine of the rest in 32 (its
// rounding is 2^-25 of a turn).  The rotation is in 32 bits, rounded once.
//
// One pass over q, k and v.  A workgroup takes a few tokens: their angles, one
// per (token, pair), go to LDS once and serve every head; then each thread moves
// 16-byte pieces (both of a pair's pieces where they are apart).  A thread keeps its
// place in the head and goes from head to head, so that no piece costs a
// division (found by one, the pieces' places cost more than their bytes in the
// interleaved layout, where a piece is 16 bytes and not two times 16).  Few tokens are bound by latency: 48 of them take
// 5.5 us, the launch and two round trips one after the other, positions and frequencies before the barrier, q, k and
// v behind it.
#include <algorithm>
#include <climits>

#include "common.h"

namespace fs {

constexpr int kRopeThreads = 256;
constexpr int kRopeMaxHalf = 128;
constexpr int kRopeMaxTokens = 4;                // of a workgroup

struct RopeKArgs {
  fs_rope_args a;
  int tokens;                                      // of a workgroup
};

template <typename T, int V>
__device__ __forceinline__ void load_piece(const T* p, float* x) {
  T e[V];
  if constexpr (V > 1) {
    const uint4 raw = *reinterpret_cast<const uint4*>(p);
    __builtin_memcpy(e, &raw, 16);
  } else {
    e[0] = *p;
  }
#pragma unroll
  for (int i = 0; i < V; ++i) x[i] = to_f32(e[i]);
}
template <typename T, int V>
__device__ __forceinline__ void store_piece(T* p, const float* x) {
  T e[V];
#pragma unroll
  for (int i = 0; i < V; ++i) e[i] = Conv<T>::store(x[i]);
  if constexpr (V > 1) {
    uint4 raw;
    __builtin_memcpy(&raw, e, 16);
    *reinterpret_cast<uint4*>(p) = raw;
  } else {
    *p = e[0];
  }
}

// V: elements of a piece, 16 bytes where every run of dims allows it, else 1.  32768 tokens, 32 / 8 heads of 128: bf16
// 126 us and f32 249 us (5.3 and 5.4 TB/s); 34 of the dims rotated, by single elements, bf16 421 us (426 interleaved): 1.6 TB/s.
template <typename T, int V, bool INTER>
__global__ __launch_bounds__(kRopeThreads) void rope_kernel(RopeKArgs ka) {
  constexpr bool TWO = !INTER || V == 1;           // a pair's elements are apart: two loads, two stores
  const fs_rope_args& a = ka.a;
  __shared__ float2 cs[kRopeMaxTokens * kRopeMaxHalf];
  __shared__ int64_t place[kRopeMaxTokens][2];     // a token's rows in the caches; -1: it has none
  __shared__ int taken[kRopeMaxTokens];            // 0: a row behind the last request
  const int tid = threadIdx.x;
  const int64_t t0 = (int64_t)blockIdx.x * ka.tokens;
  const int nt = (int)min((int64_t)ka.tokens, a.T - t0);
  auto pos_of = [&](int t) -> int64_t {
    return a.pos_bytes == 8 ? static_cast<const int64_t*>(a.positions)[t0 + t]
                            : (int64_t)static_cast<const int32_t*>(a.positions)[t0 + t];
  };
  if (tid < nt) {
    taken[tid] = pos_of(tid) >= 0;
    if (a.slots != nullptr) {
      const int64_t slot = a.slots[t0 + tid];
      const bool ok = slot >= 0 && slot < a.num_pages * a.page_size;
      const int64_t page = !ok ? 0 : slot <= INT_MAX ? (uint32_t)slot / (uint32_t)a.page_size : slot / a.page_size;
      const int64_t off = slot - page * a.page_size;
      place[tid][0] = ok ? page * a.kc_sp + off * a.kc_ss : -1;
      place[tid][1] = ok ? page * a.vc_sp + off * a.vc_ss : -1;
    }
  }
  for (int i = tid; i < nt * a.half; i += kRopeThreads) {
    const int t = i / a.half;
    double turns = (double)pos_of(t) * a.inv_freq[i - t * a.half] * 0.15915494309189533577;   // 1 / (2 pi)
    turns -= rint(turns);
    float s, c;
    sincospif(2.0f * (float)turns, &s, &c);
    cs[i] = make_float2(c * a.attention_factor, s * a.attention_factor);
  }
  __syncthreads();
  // pieces of a rotated head: one per pair of pieces (half layout) or per piece
  // (interleaved; single elements: per pair), then the dims that are copied
  const int rot = INTER ? (V > 1 ? 2 * a.half / V : a.half) : a.half / V;
  const int head = rot + (a.D - 2 * a.half) / V;
  const int apart = INTER ? 1 : a.half;            // elements between a pair's two loads
  // The rows of nt tokens of `rows` heads, `pieces` threads to a row: run(token, head, piece).  The workgroups of one
  // token (gridDim.y) share its rows, v's from the last one on.
  const int parts = gridDim.y, part = blockIdx.y;
  auto each = [&](int rows, int pieces, int part, auto&& run) {
    const int side = pieces < kRopeThreads ? kRopeThreads / pieces : 1;   // rows side by side
    const int mine = pieces < kRopeThreads ? tid / pieces : 0;
    if (mine >= side) return;
    for (int c = tid - mine * pieces; c < pieces; c += kRopeThreads) {
      int t = 0, h = mine + part * side;
      while (true) {
        while (h >= rows) {
          h -= rows;
          ++t;
        }
        if (t >= nt) break;
        if (taken[t]) run(t, h, c);
        h += parts * side;
      }
    }
  };
  each(a.Hq + a.Hk, head, part, [&](int t, int h, int c) {
    const bool turn = c < rot;
    const int d = turn ? (INTER ? c * (V > 1 ? V : 2) : c * V) : 2 * a.half + (c - rot) * V;
    const T* src;
    T* dst;
    if (h < a.Hq) {
      src = static_cast<const T*>(a.q) + (t0 + t) * a.q_st + h * a.q_sh + d;
      dst = static_cast<T*>(a.q_out) + (t0 + t) * a.qo_st + h * a.qo_sh + d;
    } else {
      h -= a.Hq;
      src = static_cast<const T*>(a.k) + (t0 + t) * a.k_st + h * a.k_sh + d;
      if (a.slots != nullptr) {
        const int64_t at = place[t][0];
        if (at < 0) return;                        // no place in the cache
        dst = static_cast<T*>(a.k_cache) + at + h * a.kc_sh + d;
      } else {
        dst = static_cast<T*>(a.k_out) + (t0 + t) * a.ko_st + h * a.ko_sh + d;
      }
    }
    float x1[V], y1[V];
    load_piece<T, V>(src, x1);
    if (!turn) {
      store_piece<T, V>(dst, x1);
      return;
    }
    if constexpr (TWO) {
      const float2* w = cs + t * a.half + c * V;
      float x2[V], y2[V];
      load_piece<T, V>(src + apart, x2);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float2 f = w[e];
        y1[e] = x1[e] * f.x - x2[e] * f.y;
        y2[e] = x2[e] * f.x + x1[e] * f.y;
      }
      store_piece<T, V>(dst, y1);
      store_piece<T, V>(dst + apart, y2);
    } else {
      const float2* w = cs + t * a.half + c * (V / 2);
#pragma unroll
      for (int e = 0; e < V / 2; ++e) {
        const float2 f = w[e];
        y1[2 * e] = x1[2 * e] * f.x - x1[2 * e + 1] * f.y;
        y1[2 * e + 1] = x1[2 * e + 1] * f.x + x1[2 * e] * f.y;
      }
      store_piece<T, V>(dst, y1);
    }
  });
  if (a.v == nullptr) return;
  each(a.Hk, a.D / V, parts - 1 - part, [&](int t, int h, int c) {
    const int64_t at = place[t][1];
    if (at < 0) return;
    float x[V];
    load_piece<T, V>(static_cast<const T*>(a.v) + (t0 + t) * a.v_st + h * a.v_sh + c * V, x);
    store_piece<T, V>(static_cast<T*>(a.v_cache) + at + h * a.vc_sh + c * V, x);
  });
}

template <typename T>
static int launch_rope(const fs_rope_args& a, hipStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const bool wide = a.D % V == 0 && (a.interleaved ? 2 * a.half : a.half) % V == 0;
  auto f = a.interleaved ? (wide ? rope_kernel<T, V, true> : rope_kernel<T, 1, true>)
                         : (wide ? rope_kernel<T, V, false> : rope_kernel<T, 1, false>);
  // Long calls: 2 tokens to a workgroup, 4 where a piece is 16 bytes (32768 tokens, half: 126 us against 131 with 4; 8191
  // interleaved, half of the head: 29.7 against 32.0 with 2).  Few tokens: their heads over several workgroups, so that a
  // thread has one piece to wait for.
  RopeKArgs k{a, a.T < 2048 ? 1 : a.interleaved ? 4 : 2};
  const int pieces = (wide && a.interleaved ? 2 * a.half / V : wide ? a.half / V : a.half) + (a.D - 2 * a.half) / (wide ? V : 1);
  const int side = std::max(kRopeThreads / pieces, 1);
  const int parts = a.T >= 1024 ? 1 : std::min((a.Hq + a.Hk + side - 1) / side, 16);
  f<<<dim3((a.T + k.tokens - 1) / k.tokens, parts), kRopeThreads, 0, s>>>(k);
  return fs_host::launch_status("fs_rope");
}

}  // namespace fs

using namespace fs;

extern "C" int fs_rope(const fs_rope_args* a, void* stream) {
  FS_CHECK_ARG(a != nullptr, "fs_rope: null args");
  FS_CHECK_ARG(a->T >= 0 && a->Hq >= 1 && a->Hk >= 1 && a->D >= 1 && a->half >= 1 && 2 * a->half <= a->D,
               "fs_rope: T=%d Hq=%d Hk=%d D=%d rotary dim %d", a->T, a->Hq, a->Hk, a->D, 2 * a->half);
  FS_CHECK_ARG(a->pos_bytes == 4 || a->pos_bytes == 8, "fs_rope: positions of %d bytes", a->pos_bytes);
  FS_CHECK_SUPPORTED(a->dtype == FS_DTYPE_F32 || a->dtype == FS_DTYPE_BF16 || a->dtype == FS_DTYPE_F16,
                     "fs_rope: dtype %d unsupported", a->dtype);
  FS_CHECK_SUPPORTED(a->half <= kRopeMaxHalf && a->D <= 512 && a->D % 8 == 0,
                     "fs_rope: head_dim %d, rotary dim %d unsupported (multiples of 8 up to 512, up to %d)", a->D,
                     2 * a->half, 2 * kRopeMaxHalf);
  FS_CHECK_SUPPORTED((a->Hq + 2 * (int64_t)a->Hk) * a->D <= (1 << 20), "fs_rope: %d + %d heads unsupported",
                     a->Hq, a->Hk);
  if (a->T == 0) return FS_OK;
  FS_CHECK_ARG(a->q && a->k && a->q_out && a->positions && a->inv_freq, "fs_rope: null tensor pointer");
  const bool cached = a->slots != nullptr;
  FS_CHECK_ARG(cached ? a->v && a->k_cache && a->v_cache && a->page_size >= 1 && a->num_pages >= 1
                      : a->k_out != nullptr && a->v == nullptr,
               "fs_rope: give slots with v and the caches, or k_out");
  const int64_t st[] = {a->q_st, a->q_sh, a->k_st, a->k_sh, a->v_st, a->v_sh, a->qo_st, a->qo_sh, a->ko_st, a->ko_sh,
                        a->kc_sp, a->kc_ss, a->kc_sh, a->vc_sp, a->vc_ss, a->vc_sh};
  for (int64_t x : st) FS_CHECK_ARG(x % 8 == 0, "fs_rope: strides must be multiples of 8 elements");
  const void* ptrs[] = {a->q, a->k, a->v, a->q_out, a->k_out, a->k_cache, a->v_cache};
  for (const void* p : ptrs) FS_CHECK_ARG((uintptr_t)p % 16 == 0, "fs_rope: tensors must be 16-byte aligned");
  FS_CHECK_ARG((uintptr_t)a->positions % a->pos_bytes == 0 && (uintptr_t)a->inv_freq % 8 == 0 &&
                   (uintptr_t)a->slots % 8 == 0, "fs_rope: positions, inv_freq and slots must be aligned to their size");
  const hipStream_t s = (hipStream_t)stream;
  switch (a->dtype) {
    case FS_DTYPE_BF16: return launch_rope<bf16_t>(*a, s);
    case FS_DTYPE_F16: return launch_rope<f16_t>(*a, s);
    default: return launch_rope<float>(*a, s);
  }
}
