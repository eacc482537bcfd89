// Attention of new tokens over a paged cache, and sliding-window attention with
// sinks on contiguous tensors: one wave per (token, query head), keys 64 at a
// time with a running maximum and sum.
#include <climits>

#include "common.h"

namespace fs {

struct PagedKArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* out;
  int64_t q_sb, q_st, q_sh, o_sb, o_st, o_sh;   // request (contiguous tensors), token, head
  int64_t k_sp, k_ss, k_sh, v_sp, v_ss, v_sh;   // page (contiguous: batch), slot, head
  const int32_t* table;                         // null: contiguous, the page of request b is b
  const int32_t* cu;
  const int32_t* lens;
  int64_t t_sb, num_pages;
  int B, T, Hq, Hk, Lq, Lk, P, page_size, window, sinks;
  float scale;
};

template <typename T, int D>
__global__ __launch_bounds__(64) void row_attn_kernel(PagedKArgs a) {
  __shared__ float qs[D];
  const int lane = threadIdx.x;
  const int h = blockIdx.x % a.Hq, t = blockIdx.x / a.Hq;
  const int hk = h / (a.Hq / a.Hk);
  int b, i, n, L;
  if (a.table != nullptr) {
    if (t >= a.cu[a.B]) return;
    int lo = 0, hi = a.B;
    while (hi - lo > 1) {
      const int m = (lo + hi) >> 1;
      if (a.cu[m] <= t) lo = m;
      else hi = m;
    }
    b = lo;
    i = t - a.cu[b];
    n = a.cu[b + 1] - a.cu[b];
    L = (int)min((int64_t)max(a.lens[b], 0), (int64_t)a.P * a.page_size);
  } else {
    b = t / a.Lq;
    i = t - b * a.Lq;
    n = a.Lq;
    L = a.Lk;
  }
  const int64_t row = a.table != nullptr ? t : i;
  const T* q = reinterpret_cast<const T*>(a.q) + b * a.q_sb + row * a.q_st + h * a.q_sh;
  for (int d = lane; d < D; d += 64) qs[d] = to_f32(q[d]);
  __syncthreads();
  const int p = L - n + i;
  float m = -INFINITY, l = 0.f, o[D / 64] = {};
  for (int k0 = 0; k0 <= p; k0 += 64) {
    const int s = k0 + lane;
    bool seen = s <= p && s < L && (a.window == 0 || s > p - a.window || s < a.sinks);
    const int pg = s / a.page_size;
    int64_t page = b;
    if (a.table != nullptr) {
      page = seen ? a.table[b * a.t_sb + pg] : 0;
      if (page < 0 || page >= a.num_pages) seen = false;
    }
    if (__ballot(seen) == 0) continue;
    const int slot = a.table != nullptr ? s - pg * a.page_size : s;
    float x = -INFINITY;
    if (seen) {
      const T* kr = reinterpret_cast<const T*>(a.k) + page * a.k_sp + slot * a.k_ss + hk * a.k_sh;
      float acc = 0.f;
      for (int c = 0; c < D; c += 8) {
        const uint4 raw = *reinterpret_cast<const uint4*>(kr + c);
        T e[8];
        __builtin_memcpy(e, &raw, 16);
#pragma unroll
        for (int j = 0; j < 8; ++j) acc += qs[c + j] * to_f32(e[j]);
      }
      x = acc * a.scale;
    }
    const float mn = fmaxf(m, wave_max(x));
    const float mu = mn == -INFINITY ? 0.f : mn;
    const float w = seen ? expf(x - mu) : 0.f;
    const float al = expf(m - mu);
    m = mn;
    l = l * al + wave_sum(w);
#pragma unroll
    for (int e = 0; e < D / 64; ++e) o[e] *= al;
    const int64_t vo = page * a.v_sp + slot * a.v_ss + hk * a.v_sh;
    const uint64_t any = __ballot(seen);
    for (int j = 0; j < 64; ++j) {
      if (!((any >> j) & 1)) continue;
      const float wj = __shfl(w, j, 64);
      const T* vr = reinterpret_cast<const T*>(a.v) + __shfl(vo, j, 64);
#pragma unroll
      for (int e = 0; e < D / 64; ++e) o[e] += wj * to_f32(vr[lane + 64 * e]);
    }
  }
  T* out = reinterpret_cast<T*>(a.out) + b * a.o_sb + row * a.o_st + h * a.o_sh;
  const float inv = l != 0.f ? 1.0f / l : 0.f;
#pragma unroll
  for (int e = 0; e < D / 64; ++e) out[lane + 64 * e] = Conv<T>::store(o[e] * inv);
}

static int run(const PagedKArgs& k, int dtype, int D, int64_t rows, hipStream_t s, const char* fn) {
  auto f = D == 64 ? (dtype == FS_DTYPE_BF16 ? row_attn_kernel<bf16_t, 64> : row_attn_kernel<f16_t, 64>)
                   : (dtype == FS_DTYPE_BF16 ? row_attn_kernel<bf16_t, 128> : row_attn_kernel<f16_t, 128>);
  f<<<(unsigned)(rows * k.Hq), 64, 0, s>>>(k);
  return fs_host::launch_status(fn);
}

}  // namespace fs

using namespace fs;

// checks that both entry points share
static int check_common(const char* fn, int dtype, int D, int Hq, int Hk, int window, int sinks, int64_t rows,
                        const int64_t* strides, int ns, const void* const* ptrs, int np) {
  FS_CHECK_ARG(Hq >= 1 && Hk >= 1 && Hq % Hk == 0, "%s: Hq=%d must be a multiple of Hk=%d", fn, Hq, Hk);
  FS_CHECK_SUPPORTED(D == 128 || D == 64, "%s: head_dim %d unsupported (64 or 128)", fn, D);
  FS_CHECK_SUPPORTED(dtype == FS_DTYPE_BF16 || dtype == FS_DTYPE_F16, "%s: dtype %d unsupported (bf16/f16)", fn, dtype);
  FS_CHECK_ARG(window >= 0 && sinks >= 0, "%s: window %d and sinks %d must not be negative", fn, window, sinks);
  FS_CHECK_SUPPORTED(rows * Hq < (1ll << 30) && Hk <= 4096, "%s: %lld rows of %d heads unsupported", fn,
                     (long long)rows, Hq);
  for (int i = 0; i < ns; ++i) FS_CHECK_ARG(strides[i] % 8 == 0, "%s: strides must be multiples of 8 elements", fn);
  for (int i = 0; i < np; ++i) {
    FS_CHECK_ARG(ptrs[i] != nullptr, "%s: null tensor pointer", fn);
    FS_CHECK_ARG((uintptr_t)ptrs[i] % 16 == 0, "%s: tensors must be 16-byte aligned", fn);
  }
  return FS_OK;
}

extern "C" size_t fs_paged_attn_work_bytes(const fs_paged_attn_args* a) { return a ? 16 : 0; }
extern "C" size_t fs_window_attn_work_bytes(const fs_window_attn_args* a) { return a ? 16 : 0; }

extern "C" int fs_paged_attn(const fs_paged_attn_args* a, void* stream) {
  const char* fn = "fs_paged_attn";
  FS_CHECK_ARG(a != nullptr, "%s: null args", fn);
  FS_CHECK_ARG(a->B >= 1 && a->T >= 0 && a->P >= 1 && a->num_pages >= 1 && a->max_new >= 0,
               "%s: B=%d T=%d P=%d num_pages=%lld max_new=%d", fn, a->B, a->T, a->P, (long long)a->num_pages, a->max_new);
  FS_CHECK_SUPPORTED(a->page_size >= 16 && a->page_size <= 4096 && a->page_size % 16 == 0,
                     "%s: page size %d unsupported (multiples of 16 up to 4096)", fn, a->page_size);
  FS_CHECK_SUPPORTED((int64_t)a->P * a->page_size <= (1 << 26), "%s: %d pages of %d tokens per request unsupported",
                     fn, a->P, a->page_size);
  if (a->T == 0) return FS_OK;
  const int64_t st[] = {a->q_st, a->q_sh, a->o_st, a->o_sh, a->k_sp, a->k_ss, a->k_sh, a->v_sp, a->v_ss, a->v_sh};
  const void* const ptrs[] = {a->q, a->out, a->k_cache, a->v_cache, a->work};
  if (int rc = check_common(fn, a->dtype, a->D, a->Hq, a->Hk, a->window, a->sinks, a->T, st, 10, ptrs, 5)) return rc;
  FS_CHECK_ARG(a->block_table && a->cu_lens && a->seq_lens && a->t_sb >= a->P &&
                   ((uintptr_t)a->block_table | (uintptr_t)a->cu_lens | (uintptr_t)a->seq_lens) % 4 == 0,
               "%s: block_table (row stride %lld of %d), cu_lens and seq_lens must be given, 4-byte aligned", fn,
               (long long)a->t_sb, a->P);
  PagedKArgs k{};
  k.q = static_cast<const uint16_t*>(a->q);
  k.k = static_cast<const uint16_t*>(a->k_cache);
  k.v = static_cast<const uint16_t*>(a->v_cache);
  k.out = static_cast<uint16_t*>(a->out);
  k.q_st = a->q_st; k.q_sh = a->q_sh; k.o_st = a->o_st; k.o_sh = a->o_sh;
  k.k_sp = a->k_sp; k.k_ss = a->k_ss; k.k_sh = a->k_sh; k.v_sp = a->v_sp; k.v_ss = a->v_ss; k.v_sh = a->v_sh;
  k.table = a->block_table; k.cu = a->cu_lens; k.lens = a->seq_lens; k.t_sb = a->t_sb; k.num_pages = a->num_pages;
  k.B = a->B; k.T = a->T; k.Hq = a->Hq; k.Hk = a->Hk; k.P = a->P; k.page_size = a->page_size;
  k.window = a->window; k.sinks = a->sinks; k.scale = a->softmax_scale;
  return run(k, a->dtype, a->D, a->T, (hipStream_t)stream, fn);
}

extern "C" int fs_window_attn(const fs_window_attn_args* a, void* stream) {
  const char* fn = "fs_window_attn";
  FS_CHECK_ARG(a != nullptr, "%s: null args", fn);
  FS_CHECK_ARG(a->B >= 1 && a->Lq >= 1 && a->Lk >= 1, "%s: empty sequence", fn);
  FS_CHECK_SUPPORTED(a->Lk <= (1 << 26), "%s: %d keys unsupported", fn, a->Lk);
  const int64_t st[] = {a->q_sb, a->q_sh, a->q_sl, a->k_sb, a->k_sh, a->k_sl,
                        a->v_sb, a->v_sh, a->v_sl, a->o_sb, a->o_sh, a->o_sl};
  const void* const ptrs[] = {a->q, a->out, a->k, a->v, a->work};
  if (int rc = check_common(fn, a->dtype, a->D, a->Hq, a->Hk, a->window, a->sinks, (int64_t)a->B * a->Lq, st, 12,
                            ptrs, 5))
    return rc;
  PagedKArgs k{};
  k.q = static_cast<const uint16_t*>(a->q);
  k.k = static_cast<const uint16_t*>(a->k);
  k.v = static_cast<const uint16_t*>(a->v);
  k.out = static_cast<uint16_t*>(a->out);
  k.q_sb = a->q_sb; k.q_st = a->q_sl; k.q_sh = a->q_sh; k.o_sb = a->o_sb; k.o_st = a->o_sl; k.o_sh = a->o_sh;
  k.k_sp = a->k_sb; k.k_ss = a->k_sl; k.k_sh = a->k_sh; k.v_sp = a->v_sb; k.v_ss = a->v_sl; k.v_sh = a->v_sh;
  k.num_pages = a->B; k.B = a->B; k.Hq = a->Hq; k.Hk = a->Hk; k.Lq = a->Lq; k.Lk = a->Lk; k.page_size = a->Lk;
  k.window = a->window; k.sinks = a->sinks; k.scale = a->softmax_scale;
  return run(k, a->dtype, a->D, (int64_t)a->B * a->Lq, (hipStream_t)stream, fn);
}
