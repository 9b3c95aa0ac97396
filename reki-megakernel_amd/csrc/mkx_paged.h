// The paged context cache's bookkeeping and rotary: block tables and slots from request lengths, multi-axis RoPE with
// per-head norms and the store into pages.
#pragma once
#include <hip/hip_runtime.h>

#include "mkx.h"
#include "mkx_device.h"
#include "mkx_elem.h"
#include "mkx_scan.h"

namespace mkx {

// ---- block tables and slots -------------------------------------------------------------------------------------------
// Every workgroup sums all B lengths for itself (B <= 2048 numbers, from L2 after the first) and then fills its own part of
// the slots, so that one launch without any exchange between workgroups does: the work is latency, not bytes (12 bytes a
// token). Nothing that a workgroup reads is written by another one: new table entries lie behind the old ones, queue entries
// are read from the head and written behind the last free one. 16 requests of one token: 3.5 us of kernel, 64 requests of
// 14 K tokens with ended ones 5.2, 500 requests of 238 K tokens 6.8 (3 MB); with 64-bit sums through shuffles, a token at a
// time and the returned pages after them 4.4, 6.5 and 8.5.
constexpr int MAP_BLOCK = 256;
constexpr int MAP_PER = MKX_MAX_SLOTS / MAP_BLOCK;  // requests per thread at most

__device__ __forceinline__ int sat32(uint32_t v) { return (int)min(v, (uint32_t)INT32_MAX); }

__global__ __launch_bounds__(MAP_BLOCK) void page_map_kernel(mkx_page_map_args a, int shift) {
  constexpr int WAVES = MAP_BLOCK / 64;
  __shared__ int32_t s_cu[MKX_MAX_SLOTS];       // first token
  __shared__ int32_t s_pop[MKX_MAX_SLOTS];      // pages popped before it, -1: not granted
  __shared__ int32_t s_back[MKX_MAX_SLOTS];     // pages returned before it
  __shared__ int32_t s_len[MKX_MAX_SLOTS];      // old length
  __shared__ uint32_t s_sums[3 * WAVES], s_took[WAVES];
  const int tid = threadIdx.x, B = a.B, P = a.page_rows;
  const uint32_t N = (uint32_t)a.n_pages;
  const int per = (B + MAP_BLOCK - 1) / MAP_BLOCK, b0 = tid * per;
  const int len_max = a.cols << shift;
  const uint32_t head = (uint32_t)a.ends_in[0] % N, free_in = (uint32_t)min(max(a.ends_in[1], 0), a.n_pages);
  auto wrap = [&](uint32_t x) { return x >= N ? x - N : x; };  // of less than 2 N
  int len[MAP_PER], add[MAP_PER];
  bool done[MAP_PER];
  uint32_t sums[2] = {0, 0}, totals[2];  // tokens, returned pages
#pragma unroll
  for (int i = 0; i < MAP_PER; ++i) {
    len[i] = add[i] = 0;
    done[i] = false;
    if (i < per && b0 + i < B) {
      len[i] = min(max(a.len_in[b0 + i], 0), len_max);
      done[i] = a.done != nullptr && a.done[b0 + i] != 0;
      add[i] = done[i] ? 0 : max(a.add[b0 + i], 0);
      sums[0] = add_sat(sums[0], (uint32_t)add[i]);
      if (done[i]) sums[1] = add_sat(sums[1], (uint32_t)((len[i] + P - 1) >> shift));
    }
  }
  block_sums_sat<MAP_BLOCK>(sums, totals, s_sums);
  const int cu_end = sat32(totals[0]);
  // a request's need counts only where its table row and the token arrays hold it
  uint32_t at = sums[0], put = sums[1], pop[1] = {0}, needed[1];
  int cu[MAP_PER], need[MAP_PER];
  bool fits[MAP_PER];
#pragma unroll
  for (int i = 0; i < MAP_PER; ++i) {
    cu[i] = sat32(at);
    at = add_sat(at, (uint32_t)add[i]);
    const long long end = (long long)len[i] + add[i];
    fits[i] = !done[i] && end <= len_max && at <= (uint32_t)a.max_tokens;
    need[i] = fits[i] ? (int)((end + P - 1) >> shift) - ((len[i] + P - 1) >> shift) : 0;
    pop[0] = add_sat(pop[0], (uint32_t)need[i]);
  }
  block_sums_sat<MAP_BLOCK>(pop, needed, s_sums + 2 * WAVES);
  uint32_t took = 0;  // the end of the thread's last request that gets pages
#pragma unroll
  for (int i = 0; i < MAP_PER; ++i)
    if (i < per && b0 + i < B) {
      const int b = b0 + i;
      const uint32_t after = add_sat(pop[0], (uint32_t)need[i]);
      const bool ok = fits[i] && (need[i] == 0 || after <= free_in);
      s_cu[b] = cu[i];
      s_pop[b] = ok ? sat32(pop[0]) : -1;
      s_back[b] = sat32(put);
      s_len[b] = len[i];
      if (ok && need[i] > 0) took = after;
      pop[0] = after;
      put = add_sat(put, done[i] ? (uint32_t)((len[i] + P - 1) >> shift) : 0u);
      if (blockIdx.x == 0) {
        a.cu[b] = cu[i];
        a.granted[b] = ok;
        a.len_out[b] = done[i] ? 0 : len[i] + (ok ? add[i] : 0);
      }
    }
  // a request that is not granted takes all that need pages after it along: the last granted one's end is what is taken
  const unsigned long long takes = __ballot(took > 0);
  const uint32_t wave_took = takes ? (uint32_t)__builtin_amdgcn_readlane((int)took, 63 - __builtin_clzll(takes)) : 0;
  if ((tid & 63) == 0) s_took[tid >> 6] = wave_took;
  __syncthreads();
  if (blockIdx.x == 0 && tid == 0) {
    uint32_t taken = 0;
    for (int w = 0; w < WAVES; ++w) taken = max(taken, s_took[w]);
    a.cu[B] = cu_end;
    a.ends_out[0] = (int)wrap(head + taken);
    a.ends_out[1] = (int)min(N, add_sat(free_in - taken, totals[1]));
  }
  // returned pages go behind the free ones: the first that this thread moves is on its way while it does its tokens
  const int stride = gridDim.x * MAP_BLOCK, first = blockIdx.x * MAP_BLOCK + tid;
  const int n_back = (int)min(totals[1], N);
  auto returned = [&](int i) {
    const int b = last_at_or_below(s_back, B, i);
    return a.table[b * a.table_stride + (i - s_back[b])];
  };
  const int back = first < n_back ? returned(first) : 0;
  // Tokens, two of a thread at a time (their searches and loads side by side): the thread of a new page's first token writes its
  // table entry
  int top = 1;
  while (top < B) top <<= 1;
  for (int t0 = first; t0 < a.max_tokens; t0 += 2 * stride) {
    int t[2] = {t0, t0 + stride}, b[2] = {0, 0}, pos[2], page[2];
    for (int d = top >> 1; d > 0; d >>= 1)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int m = min(b[k] + d, B - 1);
        if (s_cu[m] <= t[k]) b[k] = m;
      }
    const int32_t* from[2];
    int32_t* entry[2];
    bool owned[2], first_of[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const bool in = t[k] < min(cu_end, a.max_tokens);
      const int len_b = s_len[b[k]], pop_b = s_pop[b[k]];
      pos[k] = in ? len_b + (t[k] - s_cu[b[k]]) : 0;
      owned[k] = in && pop_b >= 0;
      const int j = pos[k] >> shift, fresh = j - ((len_b + P - 1) >> shift);
      entry[k] = a.table + b[k] * a.table_stride + j;
      first_of[k] = owned[k] && fresh >= 0 && (pos[k] & (P - 1)) == 0;
      from[k] = !owned[k] ? a.queue : fresh >= 0 ? a.queue + wrap(head + (uint32_t)(pop_b + fresh)) : entry[k];
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) page[k] = *from[k];
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (t[k] < a.max_tokens) {
        if (first_of[k]) *entry[k] = page[k];
        a.slot[t[k]] = owned[k] && (uint32_t)page[k] < N ? ((long long)page[k] << shift) + (pos[k] & (P - 1)) : -1;
        a.pos[t[k]] = pos[k];
      }
  }
  const uint32_t tail = wrap(head + free_in);
  for (int i = first; i < n_back; i += stride) a.queue[wrap(tail + (uint32_t)i)] = i == first ? back : returned(i);
}

// ---- rotary ---------------------------------------------------------------------------------------------------------
// Bound by memory: a token's heads are read once and written once. A workgroup takes `tok` tokens; their angles are made
// once (a thread a pair: the turns in 64 bits, their fraction through sincospi in 32) and shared by all heads through
// LDS, and a thread moves 8 pairs of a head at a time (16 bytes of either half), so that a head is HD / 16 neighbouring
// lanes and its norm a sum over them. 30011 tokens of 32 + 8 heads of 128, stored: 133 us, 5.5 TB/s (a 2 GiB copy on this
// card 4.9); 16 tokens of 16 + 2 heads 3.3 us in a graph.
constexpr int ROPE_BLOCK = 256, ROPE_TOK = 16;  // threads; tokens of a workgroup at most

template <class E, int HD>
__global__ __launch_bounds__(ROPE_BLOCK) void rope_kernel(mkx_rope_args a, int shift, int tok) {
  constexpr int HALF = HD / 2, UH = HD / 16;  // units of a head
  __shared__ __align__(16) float s_cos[ROPE_TOK][HALF], s_sin[ROPE_TOK][HALF];
  const int t0 = blockIdx.x * tok, nt = min(tok, a.T - t0);
  const int heads = a.NQ + a.NK + (a.slots != nullptr ? a.NK : 0);
  for (int i = threadIdx.x; i < nt * HALF; i += ROPE_BLOCK) {
    const int t = i / HALF, p = i % HALF;
    int ax = a.axis[p];
    if (ax < 0 || ax >= a.axes) ax = 0;
    const int64_t at = ax * a.pos_stride + t0 + t;
    const double x = a.dtype & MKX_ROPE_POS64 ? (double)((const int64_t*)a.pos)[at] : (double)a.pos[at], w = a.turns[p];
    const double part = fma(x, w, -rint(x * w));  // the product unrounded: a far position keeps its fraction
    sincospif(2.0f * (float)(part - rint(part)), &s_sin[t][p], &s_cos[t][p]);
  }
  __syncthreads();
  const int per = heads * UH;
  for (int u = threadIdx.x; u < nt * per; u += ROPE_BLOCK) {
    const int tl = u / per, r = u % per, h = r / UH, c = (r % UH) * 8;
    const long long t = t0 + tl;
    const bool is_q = h < a.NQ, is_v = h >= a.NQ + a.NK;
    const uint16_t* src;
    uint16_t* dst = nullptr;
    const void* w = nullptr;
    if (is_q) {
      src = (const uint16_t*)a.q + t * a.q_stride_t + h * a.q_stride_h;
      dst = (uint16_t*)a.q_out + t * a.qo_stride_t + h * a.qo_stride_h;
      w = a.q_norm;
    } else {
      const int hk = h - a.NQ - (is_v ? a.NK : 0);
      src = is_v ? (const uint16_t*)a.v + t * a.v_stride_t + hk * a.v_stride_h
                 : (const uint16_t*)a.k + t * a.k_stride_t + hk * a.k_stride_h;
      if (a.slots != nullptr) {
        const long long s = a.slots[t];
        if (s >= 0 && (s >> shift) < a.n_pages)
          dst = (uint16_t*)(is_v ? a.v_pages : a.k_pages) + (s >> shift) * a.page_stride +
                (s & (a.page_rows - 1)) * a.row_stride + hk * a.head_stride;
      } else {
        dst = (uint16_t*)a.k_out + t * a.ko_stride_t + hk * a.ko_stride_h;
      }
      w = is_v ? nullptr : a.k_norm;
    }
    u32x4 vlo = ld16(src + c), vhi = ld16(src + HALF + c);
    if (!is_v) {
      float lo[8], hi[8];
      unpack8e<E>(vlo, lo);
      unpack8e<E>(vhi, hi);
      if (w != nullptr) {  // the same for every lane of a head
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(hi[i], hi[i], fmaf(lo[i], lo[i], ss));
        ss = quad_sum(ss);
        if (UH == 8) ss += dpp<0x141>(ss);  // row_half_mirror: the other quad of the half-row
        const float inv = rsqrtf(ss * (1.0f / HD) + a.eps);
        float wl[8], wh[8];
        if (a.dtype & MKX_ROPE_NORM32) {
          const float* wf = (const float*)w + c;
#pragma unroll
          for (int i = 0; i < 8; ++i) wl[i] = wf[i], wh[i] = wf[HALF + i];
        } else {
          unpack8e<E>(ld16((const uint16_t*)w + c), wl);
          unpack8e<E>(ld16((const uint16_t*)w + HALF + c), wh);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          lo[i] = lo[i] * inv * (1.0f + wl[i]);
          hi[i] = hi[i] * inv * (1.0f + wh[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float cs = s_cos[tl][c + i], sn = s_sin[tl][c + i], x = lo[i], y = hi[i];
        lo[i] = x * cs - y * sn;
        hi[i] = y * cs + x * sn;
      }
      vlo = pack8e<E>(lo);
      vhi = pack8e<E>(hi);
    }
    if (dst != nullptr) {
      *reinterpret_cast<u32x4*>(dst + c) = vlo;
      *reinterpret_cast<u32x4*>(dst + HALF + c) = vhi;
    }
  }
}

}  // namespace mkx
