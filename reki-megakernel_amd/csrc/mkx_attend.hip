// C ABI of the paged attention (include/mkx.h).
#include <atomic>
#include <random>

#include "mkx_attend.h"

#include "mkx_error.h"
#include "mkx_overlap.h"

using namespace mkx;

namespace {

bool off16(const void* p) { return ((uintptr_t)p & 15u) != 0; }

// MKX_OK, or the failure of the sizes
int check_sizes(const mkx_attend_args* a, const char* me, int* shift) {
  if (!a) return set_error(MKX_EINVAL, me, "args is NULL");
  if (a->HD != 64 && a->HD != 128) return set_error(MKX_EUNSUPPORTED, me, "HD must be 64 or 128");
  if (a->dtype != MKX_BF16 && a->dtype != MKX_FP16) return set_error(MKX_EUNSUPPORTED, me, "dtype must be MKX_BF16 or MKX_FP16");
  *shift = -1;
  for (int s = 4; s <= 8; ++s)
    if (a->page_rows == 1 << s) *shift = s;
  if (*shift < 0) return set_error(MKX_EINVAL, me, "page_rows must be 16, 32, 64, 128 or 256");
  if (a->T < 0 || a->B < 1 || a->B > MKX_MAX_SLOTS || a->NK < 1 || a->NQ < a->NK || a->NQ > 1024 || a->NQ % a->NK)
    return set_error(MKX_EINVAL, me, "need T >= 0, 1 <= B <= MKX_MAX_SLOTS, NQ a multiple of NK, NQ <= 1024");
  if (a->row_stride < 0 || a->row_stride > (1 << 27)) return set_error(MKX_EINVAL, me, "row_stride must be 0 .. 2^27");
  if (a->cols < 1 || a->n_pages < 1 || ((int64_t)a->cols << *shift) > INT32_MAX - 1024 || (int64_t)a->T * a->NQ > INT32_MAX / 2)
    return set_error(MKX_EINVAL, me, "cols, n_pages or T * NQ out of range");
  if (a->window < 0 || a->sinks < 0 || (a->window > 0 && !a->causal) || (a->sinks > 0 && a->window == 0) || a->max_q < 0)
    return set_error(MKX_EINVAL, me, "window needs causal, sinks need a window, max_q must not be negative");
  return MKX_OK;
}

int cus_here(const char* me, int* cus) {
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e == hipSuccess) e = hipDeviceGetAttribute(cus, hipDeviceAttributeMultiprocessorCount, dev);
  if (e != hipSuccess) return set_error(MKX_EHIP, me, hipGetErrorString(e));
  if (*cus < 8) return set_error(MKX_EUNSUPPORTED, me, "fewer than 8 CUs");
  return MKX_OK;
}

// A tile has as many rows as the longest announced chunk needs, up to 256; a workgroup to a CU.
AttendLaunch launch_of(const mkx_attend_args* a, int shift, int cus) {
  AttendLaunch L = {};
  L.shift = shift;
  L.G = a->NQ / a->NK;
  const int64_t rows = (int64_t)(a->max_q < a->T ? a->max_q : a->T) * L.G;
  L.bm = rows <= 64 ? 64 : rows <= 128 ? 128 : 256;
  // A launch has fewer than 2^32 threads (a larger grid wraps around without an error): larger tiles for that many rows. With 256
  // rows there are at most 2^30 / 256 + MKX_MAX_SLOTS * 1024 of them, below 2^23.
  while (L.bm < 256 && ((int64_t)a->T * L.G / L.bm + a->B) * a->NK >= 1 << 23) L.bm *= 2;
  // Two tiles of 256 rows a CU and more go to workgroups of their own as CUs become free (8192-token prompt of 16 + 2 heads:
  // 285 us against 307 shared out), and so do more tiles than a workgroup can look through.
  const int64_t tiles = (int64_t)a->T * L.G / L.bm + a->B;
  L.tiles = (int)(tiles < ATT_TILES ? tiles : ATT_TILES);
  const int64_t units = (((int64_t)a->cols << shift) / 128 + 2) * 4 + ATT_BEGIN;  // of a tile, at most: the line's are 32-bit
  if (tiles <= ATT_TILES && tiles * a->NK * units < 1 << 30 && (L.bm < 256 || tiles * a->NK < 2 * cus)) L.parts = cus & ~7;
  return L;
}
int64_t ws_of(const mkx_attend_args* a, const AttendLaunch& L) {
  return L.parts == 0 ? 256 : a->HD == 128 ? Parts<128>::bytes(L.parts, L.bm) : Parts<64>::bytes(L.parts, L.bm);
}

template <class E, int HD>
hipError_t go(const mkx_attend_args& a, const AttendLaunch& L, hipStream_t st) {
  constexpr unsigned LDS = AttendLds<HD>::BYTES;
  if (L.parts > 0) {
    hipLaunchKernelGGL((attend_kernel<E, HD>), dim3(L.parts), dim3(ATT_BLOCK), LDS, st, a, L);
  } else {
    const int64_t tiles = (int64_t)a.T * L.G / L.bm + a.B;
    hipLaunchKernelGGL((attend_tiles_kernel<E, HD>), dim3((unsigned)(tiles * a.NK)), dim3(ATT_BLOCK), LDS, st, a, L);
  }
  return hipGetLastError();
}

// Stamps of launches: no two calls of a process share one, and what a workspace held before is none of them.
std::atomic<unsigned long long> g_stamp{0};
unsigned long long next_stamp() {
  static const unsigned long long seed = ((unsigned long long)std::random_device{}() << 32 | std::random_device{}()) | 1;
  return (seed + 2 * g_stamp.fetch_add(1, std::memory_order_relaxed)) * 0x9E3779B97F4A7C15ull;  // odd times odd: never 0
}

int attend(const char* me, const mkx_attend_args* a, const int32_t* granted, void* stream) {
  int shift;
  const int rc = check_sizes(a, me, &shift);
  if (rc != MKX_OK) return rc;
  if (!(a->scale > 0.f) || !(a->scale * 1.5f < __builtin_inff())) return set_error(MKX_EINVAL, me, "scale must be positive and finite");
  if (!a->q || !a->out || !a->k_pages || !a->v_pages || !a->table || !a->cu || !a->kv_len || !a->ws)
    return set_error(MKX_EINVAL, me, "a required pointer is NULL");
  if (off16(a->q) || off16(a->out) || off16(a->k_pages) || off16(a->v_pages) ||
      ((a->q_stride_t | a->q_stride_h | a->o_stride_t | a->o_stride_h | a->page_stride | a->row_stride | a->head_stride) & 7))
    return set_error(MKX_EINVAL, me, "q, out, pages: not 16-byte aligned, or a stride that is no multiple of 8");
  if (a->o_stride_t < a->HD || a->o_stride_h < a->HD || a->table_stride < a->cols)
    return set_error(MKX_EINVAL, me, "a stride of out or table is too small");
  if (a->out == a->q || a->out == a->k_pages || a->out == a->v_pages) return set_error(MKX_EINVAL, me, "out is an input");
  if (((uintptr_t)a->ws & 255u) != 0 || a->ws_bytes < 256)
    return set_error(MKX_EINVAL, me, "ws must be 256-byte aligned and hold mkx_page_attend_workspace() bytes");
  if (a->T == 0) return MKX_OK;
  if (share_elements({a->q, a->NQ, a->q_stride_t, a->q_stride_h}, {a->out, a->NQ, a->o_stride_t, a->o_stride_h}, a->T, a->HD))
    return set_error(MKX_EINVAL, me, "out shares elements with q");
  int cus;
  const int no_cus = cus_here(me, &cus);
  if (no_cus != MKX_OK) return no_cus;
  AttendLaunch L = launch_of(a, shift, cus);
  L.granted = granted;
  if (a->ws_bytes < ws_of(a, L)) return set_error(MKX_EINVAL, me, "ws_bytes smaller than mkx_page_attend_workspace()");
  try {
    L.stamp = next_stamp();
  } catch (...) {
    return set_error(MKX_EHIP, me, "no random numbers for the launch's stamp");
  }
  hipStream_t st = (hipStream_t)stream;
  const hipError_t e = a->dtype == MKX_BF16 ? (a->HD == 128 ? go<BF16, 128>(*a, L, st) : go<BF16, 64>(*a, L, st))
                                            : (a->HD == 128 ? go<FP16, 128>(*a, L, st) : go<FP16, 64>(*a, L, st));
  if (e != hipSuccess) return set_error(MKX_EHIP, me, hipGetErrorString(e));
  return MKX_OK;
}

}  // namespace

extern "C" {

int64_t mkx_page_attend_workspace(const mkx_attend_args* a) {
  const char* me = "mkx_page_attend_workspace";
  int shift, cus;
  if (check_sizes(a, me, &shift) != MKX_OK || cus_here(me, &cus) != MKX_OK) return -1;
  return ws_of(a, launch_of(a, shift, cus));
}

int mkx_page_attend(const mkx_attend_args* a, void* stream) { return attend("mkx_page_attend", a, nullptr, stream); }

int mkx_page_attend_granted(const mkx_attend_args* a, const int32_t* granted, void* stream) {
  return attend("mkx_page_attend_granted", a, granted, stream);
}

}  // extern "C"
