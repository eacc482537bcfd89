// Entry points of paged and window attention, and the kernels' form over 16-bit keys and values without trees.
#include "paged_kernel.h"

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
static int form_of(const fs_paged_attn_args& a) { return (a.k_scale ? k8 : 0) | (a.mask ? kTree : 0); }
static Work work_of(const fs_paged_attn_args& a) {
  return work_of(few_rows(a), a.T, a.B, a.Hk, a.Hq / a.Hk, a.D, form_of(a));
}
static Work work_of(const fs_window_attn_args& a) {
  return work_of(few_rows(a), (int64_t)a.B * a.Lq, a.B, a.Hk, a.Hq / a.Hk, a.D, 0);
}

extern "C" size_t fs_paged_attn_work_bytes(const fs_paged_attn_args* a) {
  if (!a || a->B <= 0 || a->T <= 0 || a->Hk <= 0 || a->Hq < a->Hk || a->D <= 0) return 0;
  return work_bytes(most_new(*a), a->T, a->B, a->Hq, a->Hk, a->D, (int64_t)a->P * a->page_size, form_of(*a));
}
extern "C" size_t fs_window_attn_work_bytes(const fs_window_attn_args* a) {
  if (!a || a->B <= 0 || a->Lq <= 0 || a->Hk <= 0 || a->Hq < a->Hk || a->D <= 0) return 0;
  return work_bytes(a->Lq, (int64_t)a->B * a->Lq, a->B, a->Hq, a->Hk, a->D, a->Lk, 0);
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
  const bool e8 = a->k_scale != nullptr;
  FS_CHECK_ARG(e8 == (a->v_scale != nullptr) && ((uintptr_t)a->k_scale | (uintptr_t)a->v_scale) % 4 == 0,
               "%s: k_scale and v_scale come together, 4-byte aligned", fn);
  if (e8)
    for (int i = 4; i < 10; ++i) FS_CHECK_ARG(st[i] % 16 == 0, "%s: strides of an 8-bit cache must be multiples of 16 elements", fn);
  if (a->mask) {
    FS_CHECK_ARG((uintptr_t)a->mask % 8 == 0 && a->mask_words >= 1 && a->mask_words <= (1 << 20) && (uintptr_t)a->positions % 4 == 0,
                 "%s: mask of %d words per row, positions must be aligned to their size", fn, a->mask_words);
    FS_CHECK_ARG(!a->window || a->positions, "%s: a window over a tree needs the rows' positions", fn);
  }
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
  k.ks = a->k_scale; k.vs = a->v_scale;
  k.mask = reinterpret_cast<const uint32_t*>(a->mask); k.mask_words = 2 * a->mask_words; k.pos = a->positions;
  const uint32_t groups = a->page_size / 16;       // x / groups for x < 2^22, groups <= 256: mulhi is exact
  k.page_magic = groups > 1 ? (uint32_t)((1ull << 32) / groups + 1) : 0;
  const bool few = few_rows(*a);
  const Work w = work_of(*a);
  char* const work = static_cast<char*>(a->work);
  const hipStream_t s = (hipStream_t)stream;
  if (e8) return (a->mask ? run_tree8 : run_paged8)(k, a->dtype, a->D, few, w, work, a->B, a->T, s, fn);
  if (a->mask) return run_tree(k, a->dtype, a->D, few, w, work, a->B, a->T, s, fn);
  return run<true, 0>(k, a->dtype, a->D, few, true, w, work, a->B, a->T, s, fn);
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
  return run<false, 0>(k, a->dtype, a->D, few, plan, w, static_cast<char*>(a->work), a->B, a->Lq, (hipStream_t)stream, fn);
}
