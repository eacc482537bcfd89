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
// 16-byte pieces (both of a pair's pieces where they are apart).
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

// V: elements of a piece, 16 bytes where every run of dims allows it, else 1.
template <typename T, int V, bool INTER>
__global__ __launch_bounds__(kRopeThreads) void rope_kernel(RopeKArgs ka) {
  const fs_rope_args& a = ka.a;
  __shared__ float2 cs[kRopeMaxTokens * kRopeMaxHalf];
  const int tid = threadIdx.x;
  const int t0 = blockIdx.x * ka.tokens, nt = min(ka.tokens, a.T - t0);
  auto pos_of = [&](int t) -> int64_t {
    return a.pos_bytes == 8 ? static_cast<const int64_t*>(a.positions)[t0 + t]
                            : (int64_t)static_cast<const int32_t*>(a.positions)[t0 + t];
  };
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
  const int head = rot + (a.D - 2 * a.half) / V, vhead = a.D / V;
  const int rotated = (a.Hq + a.Hk) * head, token = rotated + (a.v != nullptr ? a.Hk * vhead : 0);
  for (int i = tid; i < nt * token; i += kRopeThreads) {
    const int tl = i / token, it = i - tl * token;
    const int64_t t = t0 + tl;
    if (pos_of(tl) < 0) continue;                  // a row behind the last request
    int64_t page = 0, off = 0;
    if (a.slots != nullptr && it >= a.Hq * head) {
      const int64_t slot = a.slots[t];
      page = slot / a.page_size;
      off = slot - page * a.page_size;
      if (slot < 0 || page >= a.num_pages) continue;   // no place in the cache
    }
    const T* src;
    T* dst;
    int c;
    bool turn = true;
    if (it < rotated) {
      const int h = it / head;
      c = it - h * head;
      turn = c < rot;
      if (h < a.Hq) {
        src = static_cast<const T*>(a.q) + t * a.q_st + h * a.q_sh;
        dst = static_cast<T*>(a.q_out) + t * a.qo_st + h * a.qo_sh;
      } else {
        const int hk = h - a.Hq;
        src = static_cast<const T*>(a.k) + t * a.k_st + hk * a.k_sh;
        dst = a.slots != nullptr ? static_cast<T*>(a.k_cache) + page * a.kc_sp + off * a.kc_ss + hk * a.kc_sh
                                 : static_cast<T*>(a.k_out) + t * a.ko_st + hk * a.ko_sh;
      }
    } else {
      const int hk = (it - rotated) / vhead;
      c = it - rotated - hk * vhead;
      turn = false;
      src = static_cast<const T*>(a.v) + t * a.v_st + hk * a.v_sh;
      dst = static_cast<T*>(a.v_cache) + page * a.vc_sp + off * a.vc_ss + hk * a.vc_sh;
    }
    const float2* w = cs + tl * a.half;
    if (!turn) {
      const int d = it < rotated ? 2 * a.half + (c - rot) * V : c * V;
      float x[V];
      load_piece<T, V>(src + d, x);
      store_piece<T, V>(dst + d, x);
    } else if constexpr (INTER) {
      constexpr int P = V > 1 ? V : 2;
      float x[P], y[P];
      if constexpr (V > 1) load_piece<T, V>(src + c * V, x);
      else {
        x[0] = to_f32(src[2 * c]);
        x[1] = to_f32(src[2 * c + 1]);
      }
#pragma unroll
      for (int e = 0; e < P / 2; ++e) {
        const float2 f = w[c * (P / 2) + e];
        y[2 * e] = x[2 * e] * f.x - x[2 * e + 1] * f.y;
        y[2 * e + 1] = x[2 * e + 1] * f.x + x[2 * e] * f.y;
      }
      if constexpr (V > 1) store_piece<T, V>(dst + c * V, y);
      else {
        dst[2 * c] = Conv<T>::store(y[0]);
        dst[2 * c + 1] = Conv<T>::store(y[1]);
      }
    } else {
      float x1[V], x2[V], y1[V], y2[V];
      load_piece<T, V>(src + c * V, x1);
      load_piece<T, V>(src + a.half + c * V, x2);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float2 f = w[c * V + e];
        y1[e] = x1[e] * f.x - x2[e] * f.y;
        y2[e] = x2[e] * f.x + x1[e] * f.y;
      }
      store_piece<T, V>(dst + c * V, y1);
      store_piece<T, V>(dst + a.half + c * V, y2);
    }
  }
}

template <typename T>
static int launch_rope(const fs_rope_args& a, hipStream_t s) {
  constexpr int V = 16 / sizeof(T);
  RopeKArgs k{a, a.T >= 2048 ? kRopeMaxTokens : 1};
  const unsigned grid = (unsigned)((a.T + k.tokens - 1) / k.tokens);
  const bool wide = a.D % V == 0 && (a.interleaved ? 2 * a.half : a.half) % V == 0;
  auto f = a.interleaved ? (wide ? rope_kernel<T, V, true> : rope_kernel<T, 1, true>)
                         : (wide ? rope_kernel<T, V, false> : rope_kernel<T, 1, false>);
  f<<<grid, kRopeThreads, 0, s>>>(k);
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
  FS_CHECK_SUPPORTED((int64_t)(a->Hq + 2 * (int64_t)a->Hk) * a->D <= (1 << 22), "fs_rope: %d + %d heads unsupported",
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
