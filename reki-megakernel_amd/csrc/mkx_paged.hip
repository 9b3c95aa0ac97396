// C ABI of the paged context cache (include/mkx.h): page map and rotary.
#include "mkx_paged.h"

#include "mkx_error.h"
#include "mkx_overlap.h"

using namespace mkx;

namespace {

#define HIPRC(where, x)                                                     \
  do {                                                                      \
    const hipError_t e_ = (x);                                              \
    if (e_ != hipSuccess) return set_error(MKX_EHIP, where, hipGetErrorString(e_)); \
  } while (0)

bool off16(const void* p) { return ((uintptr_t)p & 15u) != 0; }

int page_shift(int rows) {  // -1: not a page size
  for (int s = 4; s <= 8; ++s)
    if (rows == 1 << s) return s;
  return -1;
}

int type_of(const mkx_rope_args& a) { return a.dtype & ~(MKX_ROPE_POS64 | MKX_ROPE_NORM32); }

// The n tokens (or as many as there are) from t0 on
mkx_rope_args rope_from(mkx_rope_args a, int64_t t0, int64_t n) {
  auto skip = [&](const void* p, int64_t stride) { return (void*)((uintptr_t)p + 2 * (uintptr_t)(t0 * stride)); };
  a.T = (int)(a.T - t0 < n ? a.T - t0 : n);
  a.q = skip(a.q, a.q_stride_t), a.k = skip(a.k, a.k_stride_t), a.v = skip(a.v, a.v_stride_t);
  a.q_out = skip(a.q_out, a.qo_stride_t), a.k_out = skip(a.k_out, a.ko_stride_t);
  a.pos += a.dtype & MKX_ROPE_POS64 ? 2 * t0 : t0;
  if (a.slots != nullptr) a.slots += t0;
  return a;
}

hipError_t launch_rope(const mkx_rope_args& a, int shift, int tok, hipStream_t st) {
  const dim3 grid((unsigned)((a.T + tok - 1) / tok)), block(ROPE_BLOCK);
  if (type_of(a) == MKX_BF16) {
    if (a.HD == 128) hipLaunchKernelGGL((rope_kernel<BF16, 128>), grid, block, 0, st, a, shift, tok);
    else hipLaunchKernelGGL((rope_kernel<BF16, 64>), grid, block, 0, st, a, shift, tok);
  } else {
    if (a.HD == 128) hipLaunchKernelGGL((rope_kernel<FP16, 128>), grid, block, 0, st, a, shift, tok);
    else hipLaunchKernelGGL((rope_kernel<FP16, 64>), grid, block, 0, st, a, shift, tok);
  }
  return hipGetLastError();
}

}  // namespace

extern "C" {

int mkx_page_map(const mkx_page_map_args* a, void* stream) {
  const char* me = "mkx_page_map";
  if (!a) return set_error(MKX_EINVAL, me, "args is NULL");
  const int shift = page_shift(a->page_rows);
  if (shift < 0) return set_error(MKX_EINVAL, me, "page_rows must be 16, 32, 64, 128 or 256");
  if (a->B < 1 || a->B > MKX_MAX_SLOTS || a->cols < 1 || a->n_pages < 1 || a->max_tokens < 1)
    return set_error(MKX_EINVAL, me, "need 1 <= B <= MKX_MAX_SLOTS, cols >= 1, n_pages >= 1, max_tokens >= 1");
  if (((int64_t)a->cols << shift) > INT32_MAX || a->max_tokens > INT32_MAX - (1 << 24))
    return set_error(MKX_EINVAL, me, "cols * page_rows or max_tokens too large");
  if (a->table_stride < a->cols) return set_error(MKX_EINVAL, me, "table_stride smaller than cols");
  if (!a->add || !a->len_in || !a->ends_in || !a->table || !a->queue || !a->len_out || !a->ends_out || !a->cu ||
      !a->granted || !a->slot || !a->pos)
    return set_error(MKX_EINVAL, me, "a required pointer is NULL");
  if (((uintptr_t)a->slot & 7u) != 0) return set_error(MKX_EINVAL, me, "slot must be 8-byte aligned");
  if (a->len_out == a->len_in || a->ends_out == a->ends_in)
    return set_error(MKX_EINVAL, me, "len_out and ends_out must not be the inputs");
  // two tokens a thread: a workgroup's scan of the lengths is paid once for 512 tokens
  const int grid = (int)(((int64_t)a->max_tokens + 2 * MAP_BLOCK - 1) / (2 * MAP_BLOCK));
  hipLaunchKernelGGL(page_map_kernel, dim3(grid < 2048 ? grid : 2048), dim3(MAP_BLOCK), 0, (hipStream_t)stream, *a, shift);
  HIPRC(me, hipGetLastError());
  return MKX_OK;
}

int mkx_rope_axes(const mkx_rope_args* a, void* stream) {
  const char* me = "mkx_rope_axes";
  if (!a) return set_error(MKX_EINVAL, me, "args is NULL");
  if (a->HD != 64 && a->HD != 128) return set_error(MKX_EUNSUPPORTED, me, "HD must be 64 or 128");
  if (type_of(*a) != MKX_BF16 && type_of(*a) != MKX_FP16) return set_error(MKX_EUNSUPPORTED, me, "dtype must be MKX_BF16 or MKX_FP16");
  if (a->T < 0 || a->NQ < 0 || a->NK < 0 || a->NQ > 1024 || a->NK > 1024 || a->NQ + a->NK == 0 || a->axes < 1 || a->axes > 16)
    return set_error(MKX_EINVAL, me, "need T >= 0, heads of 0 .. 1024 (not both 0), axes of 1 .. 16");
  if (a->T > INT32_MAX - 64) return set_error(MKX_EINVAL, me, "T too large");
  if (!a->pos || !a->axis || !a->turns) return set_error(MKX_EINVAL, me, "pos, axis and turns are required");
  if (((uintptr_t)a->pos & (a->dtype & MKX_ROPE_POS64 ? 7u : 3u)) != 0) return set_error(MKX_EINVAL, me, "pos is not aligned to its numbers");
  if (a->pos_stride < a->T && a->axes > 1) return set_error(MKX_EINVAL, me, "pos_stride smaller than T");
  if (!(a->eps >= 0.f)) return set_error(MKX_EINVAL, me, "eps must not be negative");
  const bool store = a->slots != nullptr;
  int shift = 4;
  if (a->NQ > 0) {
    if (!a->q || !a->q_out || off16(a->q) || off16(a->q_out) || off16(a->q_norm) ||
        ((a->q_stride_t | a->q_stride_h | a->qo_stride_t | a->qo_stride_h) & 7))
      return set_error(MKX_EINVAL, me, "q, q_out: NULL, not 16-byte aligned, or a stride that is no multiple of 8");
    if (a->q_out == a->q && (a->qo_stride_t != a->q_stride_t || a->qo_stride_h != a->q_stride_h))
      return set_error(MKX_EINVAL, me, "q_out is q with other strides");
    if (a->qo_stride_h < a->HD || a->qo_stride_t < a->HD)
      return set_error(MKX_EINVAL, me, "q_out: a stride smaller than a head");
  }
  if (a->NK > 0) {
    if (!a->k || off16(a->k) || off16(a->k_norm) || ((a->k_stride_t | a->k_stride_h) & 7))
      return set_error(MKX_EINVAL, me, "k: NULL, not 16-byte aligned, or a stride that is no multiple of 8");
    if (a->NQ > 0 && a->q_out == a->k) return set_error(MKX_EINVAL, me, "q_out is k");
    if (store) {
      shift = page_shift(a->page_rows);
      if (shift < 0 || a->n_pages < 1) return set_error(MKX_EINVAL, me, "page_rows must be 16, 32, 64, 128 or 256, n_pages >= 1");
      if (!a->v || off16(a->v) || ((a->v_stride_t | a->v_stride_h) & 7) || !a->k_pages || !a->v_pages || off16(a->k_pages) ||
          off16(a->v_pages) || ((a->page_stride | a->row_stride | a->head_stride) & 7))
        return set_error(MKX_EINVAL, me, "v, pages: NULL, not 16-byte aligned, or a stride that is no multiple of 8");
      if (a->page_stride < a->HD || a->row_stride < a->HD || a->head_stride < a->HD)
        return set_error(MKX_EINVAL, me, "pages: a stride smaller than a head");
      if (a->k_pages == a->v_pages) return set_error(MKX_EINVAL, me, "k_pages and v_pages are the same");
    } else {
      if (!a->k_out || off16(a->k_out) || ((a->ko_stride_t | a->ko_stride_h) & 7))
        return set_error(MKX_EINVAL, me, "k_out: NULL, not 16-byte aligned, or a stride that is no multiple of 8");
      if (a->k_out == a->k && (a->ko_stride_t != a->k_stride_t || a->ko_stride_h != a->k_stride_h))
        return set_error(MKX_EINVAL, me, "k_out is k with other strides");
      if (a->NQ > 0 && (a->k_out == a->q_out || a->k_out == a->q))
        return set_error(MKX_EINVAL, me, "k_out is q's input or output");
      if (a->ko_stride_h < a->HD || a->ko_stride_t < a->HD)
        return set_error(MKX_EINVAL, me, "k_out: a stride smaller than a head");
    }
  }
  if (a->T == 0) return MKX_OK;
  const View q = {a->q, a->NQ, a->q_stride_t, a->q_stride_h}, k = {a->k, a->NK, a->k_stride_t, a->k_stride_h},
             v = {a->v, a->NK, a->v_stride_t, a->v_stride_h}, qo = {a->q_out, a->NQ, a->qo_stride_t, a->qo_stride_h},
             ko = {a->k_out, a->NK, a->ko_stride_t, a->ko_stride_h};
  auto shared = [&](const View& x, const View& y) { return share_elements(x, y, a->T, a->HD); };
  if (a->NQ > 0 && ((q.p != qo.p && shared(q, qo)) || (a->NK > 0 && (shared(k, qo) || (store && shared(v, qo))))))
    return set_error(MKX_EINVAL, me, "q_out shares elements with k or v, or with q without being q");
  if (a->NK > 0 && !store && ((k.p != ko.p && shared(k, ko)) || (a->NQ > 0 && (shared(q, ko) || shared(qo, ko)))))
    return set_error(MKX_EINVAL, me, "k_out shares elements with q or q_out, or with k without being k");
  // as many tokens a workgroup as leave its threads a unit each (30000 tokens of 4 + 1 heads of 128: 17.9 us, with one token
  // each 27.6, with half as many 21.6; 1100 tokens of 16 + 2 heads: one token each 4.5 us, four 5.4)
  const int units = (a->NQ + (store ? 2 : 1) * a->NK) * (a->HD / 16), fit = ROPE_BLOCK / units;
  const int tok = fit < 1 ? 1 : fit < ROPE_TOK ? fit : ROPE_TOK;
  // A launch has fewer than 2^32 threads (a larger grid wraps around without an error): 2^23 workgroups at a time
  const int64_t most = (int64_t)tok << 23;
  for (int64_t t0 = 0; t0 < a->T; t0 += most) HIPRC(me, launch_rope(rope_from(*a, t0, most), shift, tok, (hipStream_t)stream));
  return MKX_OK;
}

}  // extern "C"
