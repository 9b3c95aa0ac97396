// Attention of a chunk of new tokens over the paged cache: o = softmax(scale q k^T over the visible keys) v, in one pass
// over the keys with the running maximum and sum of the softmax.
//
// Rows. The NQ / NK query heads that share a key head are rows of one matrix: row r of (request, key head) is token r / G,
// head r % G of the group, so that a key tile in LDS serves all of them and a single token fills G rows.
//
// Products. S^T = K Q^T and O^T = V^T P^T with v_mfma_f32_32x32x16: a lane then holds one row's scores (keys in its 16
// registers and in lane ^ 32), so maximum, sum and the rescaling of O are its own numbers and one exchange with lane ^ 32.
// The k index of the second product may be any order of the keys that both operands share; taken as the order in which
// the first product leaves them in the registers (register 8 s + j of lane half h holds key 16 s + 8 (j / 4) + 4 h + j % 4),
// P goes from the one product into the other without leaving its lane. V's operand in that order is two transposing LDS
// reads (ds_read_b64_tr_b16: 4 keys x 16 columns per 16 lanes).
//
// Bounds. Long histories of a few rows stream K and V at 6.7 TB/s (32 single tokens over 2000 to 32000 keys, 32 + 8 heads of
// 128: 330 us; a 2 GiB copy on this card 4.9 TB/s). Prompts run at 1.0 PFLOP/s (8192 tokens, 16 + 2 heads of 128, causal:
// 263 to 272 us; an 8192^3 bf16 product of the library 1.18) with the matrix cores busy for 52 % of the cycles, and the clock
// falls to 2.0 GHz: a loop whose exponentials were woven by hand between the products, and the DMAs one by one between
// those, waited less and took the same time (with no LDS reads, DMAs and maxima at all it would be 208 us). In between, a
// call is 2 us of plan, 2 of the first addresses, 2 to 3 for each piece's first keys, and 5 to 10 of joining cut tiles (16
// single tokens over 64 to 4096 keys: 21.5 us, 7.0 of them the keys' bytes).
//
// LDS. Tiles come by LDS DMA (16 bytes a lane, a wave's 64 lanes consecutive in LDS), so the bank swizzle is made by which
// 16 bytes of its row a lane fetches: K is read 16 rows x 16 bytes at a time, V 4 rows x 64 bytes (256 bytes a cycle, no
// bank twice: the conflict counter stays at 0 for both).
#pragma once
#include <hip/hip_runtime.h>

#include "mkx.h"
#include "mkx_device.h"
#include "mkx_elem.h"
#include "mkx_scan.h"

namespace mkx {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8v __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef const __attribute__((address_space(4))) int32_t* const_i32;  // uniform addresses: scalar loads

template <class E>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c);
template <>
__device__ __forceinline__ f32x16 mfma32<BF16>(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8v, a), __builtin_bit_cast(bf16x8v, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x16 mfma32<FP16>(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ u32x4 tr_pair(const char* __restrict__ p0, const char* __restrict__ p1) {  // __restrict__: not what a DMA in flight writes
  const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p0), b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p1);
  return __builtin_bit_cast(u32x4, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

constexpr int ATT_WAVES = 8, ATT_BLOCK = 64 * ATT_WAVES;
// Keys of a step: 64 KB of K and V. (Steps of half as many at 64 columns are bound by the latency of a step's chain of LDS
// reads, products and exponentials: 64 single tokens of 8 heads 55 us against 51.)
template <int HD>
constexpr int att_bn() { return HD == 128 ? 128 : 256; }
constexpr int ATT_TILES = 2048;   // row tiles that a launch shares out
constexpr float NEG_INF = -__builtin_inff();

template <int HD>
struct Swz {  // 16-byte chunk of a row -> its place in the row
  static __device__ __forceinline__ int k(int row) { return HD == 128 ? (row & 15) : ((row >> 1) & 7); }
  static __device__ __forceinline__ int v(int row) { return HD == 128 ? 4 * (row & 3) : 4 * ((row >> 1) & 1); }
};

// What the kernels know of a launch beside its arguments.
struct AttendLaunch {
  int shift, G, bm;          // log2 page_rows, heads of a group, rows of a tile (64, 128 or 256)
  int parts;                 // workgroups that share the work, a multiple of 8
  int tiles;                 // row tiles of a key head, at most
  unsigned long long stamp;  // of this launch: marks the partial results that are there
  const int32_t* granted;    // [B] 0: the request's rows see nothing; or NULL
};

// The arguments of the launch, read again from where they lie: kept in registers over a whole workgroup's work they spill.
typedef const __attribute__((address_space(4))) mkx_attend_args* args_ptr;
__device__ __forceinline__ args_ptr fresh(args_ptr p) {
  asm volatile("" : "+s"(p));
  return p;
}

typedef const __attribute__((address_space(4))) AttendLaunch* launch_ptr;
__device__ __forceinline__ launch_ptr launch_at(args_ptr p) {
  return (launch_ptr)((const __attribute__((address_space(4))) char*)p + sizeof(mkx_attend_args));
}
__device__ __forceinline__ AttendLaunch launch_args(args_ptr p) {
  const launch_ptr l = launch_at(p);
  return AttendLaunch{l->shift, l->G, l->bm, l->parts, l->tiles, l->stamp, nullptr};  // granted: read where the requests are, and no longer
}
static_assert(sizeof(mkx_attend_args) % 8 == 0, "AttendLaunch follows at its own alignment");

struct Request {
  int q0, nq, n;  // first token, tokens, cached keys
};
__device__ __forceinline__ Request request(args_ptr pa, int shift, int b) {
  const auto& a = *pa;
  const const_i32 cu = (const_i32)(uintptr_t)a.cu, kv = (const_i32)(uintptr_t)a.kv_len, granted = (const_i32)(uintptr_t)launch_at(fresh(pa))->granted;
  Request r;
  r.q0 = min(max(cu[b], 0), a.T);
  r.nq = max(min(cu[b + 1], a.T) - r.q0, 0);
  r.n = (int)min((int64_t)max(kv[b], 0), (int64_t)a.cols << shift);
  if (granted != nullptr && granted[b] == 0) r.n = 0;  // its tokens are not in the cache
  return r;
}

// One row tile of a (request, key head), and the keys that some row of it sees, [0, sinks) and [lo, hi).
struct Item {
  int h, pos0, nrows, q0, row0;  // key head; position of the request's first query, its rows, its first token; first row
  int hi, lo, sinks;
  int all_hi, all_lo;  // every row sees [all_lo, all_hi)
  const int32_t* table;
};
template <class A>
__device__ __forceinline__ Item make_item(A& a, const AttendLaunch& L, const Request& r, int b, int h, int row0) {
  Item it;
  it.h = h;
  it.pos0 = r.n - r.nq;
  it.nrows = r.nq * L.G;
  it.q0 = r.q0;
  it.row0 = row0;
  it.table = a.table + b * a.table_stride;
  it.hi = it.all_hi = r.n;
  it.lo = it.all_lo = it.sinks = 0;
  if (a.causal) {
    const int p0 = it.pos0 + row0 / L.G, p1 = it.pos0 + (min(row0 + L.bm, it.nrows) - 1) / L.G;
    it.hi = min(r.n, max(p1 + 1, 0));
    it.all_hi = min(it.hi, p0 + 1);
    if (a.window > 0) {
      // (rows ahead of the request's first key see nothing; from 0 on no difference leaves 32 bits)
      it.lo = min(max(max(p0, 0) - a.window + 1, 0), it.hi);
      it.all_lo = max(max(p1, 0) - a.window + 1, 0);
      it.sinks = min(a.sinks, it.lo);
    }
  }
  return it;
}

// The keys of an item in steps: first those that hold sinks, then those from lo on.
template <int BN>
struct Steps {
  int ns, t_lo, n;
  __device__ __forceinline__ Steps(const Item& it) {
    ns = (it.sinks + BN - 1) / BN;
    t_lo = max(it.lo / BN, ns);
    n = ns + max((it.hi + BN - 1) / BN - t_lo, 0);
  }
  __device__ __forceinline__ int key(int s) const { return (s < ns ? s : t_lo + (s - ns)) * BN; }
};

// What the steps of a piece need of the arguments, in scalar registers for as long: left to itself the compiler reads the
// arguments again in every step and waits for them.
template <class T>
__device__ __forceinline__ void pin(T& x) { asm volatile("" : "+s"(x)); }
struct Pages {
  const char *k, *v;  // of the item's head
  int64_t page_bytes;
  int32_t row_bytes, n_pages, cols, shift, sinks;
  template <class A>
  __device__ __forceinline__ Pages(A& a, const Item& it, int sh) {
    const int64_t head = 2 * it.h * a.head_stride;
    k = (const char*)a.k_pages + head;
    v = (const char*)a.v_pages + head;
    page_bytes = 2 * a.page_stride;
    row_bytes = 2 * (int32_t)a.row_stride;
    n_pages = a.n_pages;
    cols = a.cols;
    shift = sh;
    sinks = a.sinks;
    pin(k), pin(v), pin(page_bytes), pin(row_bytes), pin(n_pages), pin(cols), pin(shift), pin(sinks);
  }
  // where key j of page p is
  __device__ __forceinline__ int64_t at(int p, int j) const { return p * page_bytes + (int64_t)(j & ((1 << shift) - 1)) * row_bytes; }
};

// K and V rows of a step into LDS by DMA: lane l of a wave's 1 KB segment fetches the chunk that the swizzle puts at 16 l. A
// segment lies within 16 rows, so its page is a scalar; a lane's place in it is the same for all segments of a wave. The
// pages are read a step ahead, by a vector load that the wait for the step's DMAs covers: scalar loads would make every wait
// for LDS one for them too. Lanes whose key no row of the item sees lie outside their buffer and get zeros (0 x anything that a
// page may hold is 0 then). Buffer loads, since the compiler takes a DMA from a flat address for an LDS read too and lets every
// wait wait for everything (with both: 8192-token prompt 275 -> 265 us, mixed batch 79 -> 75).
template <int HD>
struct Loader {
  static constexpr int BN = att_bn<HD>(), RPS = 512 / HD, CH = HD / 8, N = BN / RPS / ATT_WAVES;  // rows, chunks of a row, segments of a wave
  static constexpr uint32_t OUT = 0x80000000u;  // behind a buffer's end
  uint32_t koff, voff;
  int wave, pages;  // lane i % N: page of segment i
  __device__ __forceinline__ void init(const Pages& g) {
    const int lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = wave * RPS + lane / CH, ch = lane % CH;
    static_assert(ATT_WAVES * RPS % 16 == 0, "the swizzle of a lane's row is the same in every segment");
    const uint32_t r = (uint32_t)(lane / CH) * (uint32_t)g.row_bytes;
    koff = r + 16 * (ch ^ Swz<HD>::k(row));
    voff = r + 16 * (ch ^ Swz<HD>::v(row));
  }
  __device__ __forceinline__ void fetch(const Pages& g, const Item& it, int key0) {
    const int seg = wave + (threadIdx.x & 63) % N * ATT_WAVES;
    pages = it.table[min((key0 + seg * RPS) >> g.shift, g.cols - 1)];
  }
  __device__ __forceinline__ void load(const Pages& g, const Item& it, char* kbuf, char* vbuf, int key0) {
    bool good = key0 + BN <= it.hi && (key0 >= it.lo || key0 + BN <= it.sinks);
    int page[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      page[i] = __builtin_amdgcn_readlane(pages, i);
      good = good && (unsigned)page[i] < (unsigned)g.n_pages;
    }
    auto dma = [&](const char* pages, int64_t off, uint32_t lane_off, char* to) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc(pages + off), (lds_void*)to, 16, lane_off, 0, 0, 0);
    };
    if (good) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int seg = wave + i * ATT_WAVES;
        const int64_t off = g.at(page[i], key0 + seg * RPS);
        dma(g.k, off, koff, kbuf + seg * 1024);
        dma(g.v, off, voff, vbuf + seg * 1024);
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int seg = wave + i * ATT_WAVES, first = key0 + seg * RPS, j = first + (threadIdx.x & 63) / CH;
        const bool in = (unsigned)page[i] < (unsigned)g.n_pages, ok = in && j < it.hi && (j >= it.lo || j < it.sinks);
        const int64_t off = in ? g.at(page[i], first) : 0;
        dma(g.k, off, ok ? koff : OUT, kbuf + seg * 1024);
        dma(g.v, off, ok ? voff : OUT, vbuf + seg * 1024);
      }
    }
  }
};

// A key that one row sees and another does not: were one of its values infinite or NaN, its product with the other row's weight
// of 0 would spoil that row. So in a step with such keys every wave looks at the values that it fetched itself; if any are
// not finite, they are 0 in the products (true is returned), and the rows that see their keys get them added as they are.
template <class E, int HD>
__device__ __forceinline__ bool tame_values(char* vbuf, int* flags) {
  constexpr int N = att_bn<HD>() * HD * 2 / 1024 / ATT_WAVES;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  uint32_t bad = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const u32x4 v = *reinterpret_cast<const u32x4*>(vbuf + (wave + i * ATT_WAVES) * 1024 + lane * 16);
#pragma unroll
    for (int k = 0; k < 4; ++k) bad |= E::not_finite(v[k]);
  }
  const bool mine = __any(bad != 0);
  if (mine)
    for (int i = 0; i < N; ++i) {
      u32x4* p = reinterpret_cast<u32x4*>(vbuf + (wave + i * ATT_WAVES) * 1024 + lane * 16);
      u32x4 v = *p;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t b = E::not_finite(v[k]);
        v[k] &= ~((b - (b >> 15)) | b);  // a sign bit spread over its half
      }
      *p = v;
    }
  if (lane == 0) flags[wave] = mine;
  wait_lds();
  exec_barrier();
  int any = 0;
#pragma unroll
  for (int w = 0; w < ATT_WAVES; ++w) any |= flags[w];
  return __builtin_amdgcn_readfirstlane(any) != 0;
}

// Where row `row` of an item goes, from column c on.
template <class A>
__device__ __forceinline__ uint16_t* out_row(A& a, const Item& it, int G, int row, int c) {
  const int tok = row / G;
  return (uint16_t*)a.out + (int64_t)(it.q0 + tok) * a.o_stride_t + (int64_t)(it.h * G + row % G) * a.o_stride_h + c;
}

// bits 0 .. n - 1 of 32 (none for n <= 0, all for n >= 32)
__device__ __forceinline__ uint32_t below(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }

// A wave's 32 rows against keys: running maximum m and sum l of the softmax in base 2 (l of this lane's keys alone), and O^T.
template <class E, int HD>
struct Rows {
  static constexpr int ND = HD / 32;
  u32x4 q[HD / 16];  // B operand of the first product: column lane % 32, elements 16 c + 8 (lane / 32) ..
  f32x16 o[ND];      // O^T: column lane % 32, element 32 d + 8 (i / 4) + 4 (lane / 32) + i % 4
  float m, l;
  int j_max, j_min;        // the row sees the keys j <= j_max that lie above j_min or are sinks
  int w_hi, w_full, w_lo, w_low;  // no row of the wave sees a key from w_hi on or, sinks aside, below w_low; every row sees
                                  // those below w_full and from w_lo on

  template <class A>
  __device__ __forceinline__ void init(A& a, const Item& it, int G, int row) {
    const int lane = threadIdx.x & 63;
    const int r = min(row + (lane & 31), it.nrows - 1), tok = r / G;
    j_max = a.causal ? min(it.pos0 + tok, it.hi - 1) : it.hi - 1;
    j_min = a.window > 0 ? max(it.pos0 + tok, 0) - a.window : -1;
    w_full = __builtin_amdgcn_readlane(j_max, 0) + 1;
    w_hi = row < it.nrows ? __builtin_amdgcn_readlane(j_max, 31) + 1 : 0;
    w_lo = __builtin_amdgcn_readlane(j_min, 31) + 1;
    w_low = __builtin_amdgcn_readlane(j_min, 0) + 1;
    const uint16_t* src = (const uint16_t*)a.q + (int64_t)(it.q0 + tok) * a.q_stride_t + (int64_t)(it.h * G + r % G) * a.q_stride_h + 8 * (lane >> 5);
#pragma unroll
    for (int c = 0; c < HD / 16; ++c) q[c] = ld16(src + 16 * c);
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
    m = NEG_INF;
    l = 0.f;
  }

  // Key j's values (v: its row of a page) that are infinite or NaN, added to the rows that see it
  __device__ __forceinline__ void add_not_finite(const uint16_t* v, int j, int sinks) {
    const bool see = (j <= j_max) & ((j > j_min) | (j < sinks));
    const int half = (threadIdx.x >> 5) & 1;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const u32x2 w = *reinterpret_cast<const u32x2*>(v + 32 * d + 2 * i + 4 * half);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t bad = E::not_finite(w[k]);
          float x, y;
          E::unpack2(w[k], x, y);
          o[d][i + 2 * k] += see && (bad & 0x8000u) ? x : 0.f;
          o[d][i + 2 * k + 1] += see && (bad >> 16) ? y : 0.f;
        }
      }
  }

  // KB blocks of 32 keys from key0 on, whose rows of K and V start at kbuf and vbuf
  template <int KB>
  __device__ __forceinline__ void step(const Item& it, int sinks, const char* kbuf, const char* vbuf, int key0, float c2) {
    if (key0 >= w_hi || (key0 + 32 * KB <= w_low && key0 >= sinks)) return;
    const int lane = threadIdx.x & 63, half = lane >> 5, l32 = lane & 31;
    f32x16 s[KB];
#pragma unroll
    for (int b = 0; b < KB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[b][i] = 0.f;
    const char* krow = kbuf + l32 * (HD * 2);
    const int ksw = (half ^ Swz<HD>::k(l32)) << 4;
#pragma unroll
    for (int c = 0; c < HD / 16; ++c)
#pragma unroll
      for (int b = 0; b < KB; ++b) {
        const u32x4 kf = *reinterpret_cast<const u32x4*>(krow + b * (32 * HD * 2) + (ksw ^ (c << 5)));
        s[b] = mfma32<E>(kf, q[c], s[b]);
      }
    // a quarter of the fragments is read ahead of the first product, then one for each product: left to itself the compiler
    // reads two, waits for them and multiplies (8192-token prompt 307 us against 293, in the form of four waves; a half or an
    // eighth ahead is 0 to 4 % slower)
    constexpr int KF = KB * (HD / 16), KPRE = KF / 4;
    __builtin_amdgcn_sched_group_barrier(0x100, KPRE, 0);
#pragma unroll
    for (int i = 0; i < KF - KPRE; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, KPRE, 0);
    // keys that the row does not see: -inf, whatever their product is. A lane's 32 keys of a block are bits of one number, and
    // a bit spread over a register selects (compares would take a pair of scalar registers each)
    if (key0 + 32 * KB > w_full || (key0 < w_lo && key0 + 32 * KB > it.sinks)) {
#pragma unroll
      for (int b = 0; b < KB; ++b) {
        const int k0 = key0 + 32 * b;
        const uint32_t bits = (below(j_max + 1 - k0) & (~below(j_min + 1 - k0) | below(sinks - k0))) >> (4 * half);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const uint32_t see = (uint32_t)((int32_t)(bits << (31 - (8 * (i / 4) + i % 4))) >> 31);
          s[b][i] = __uint_as_float((__float_as_uint(s[b][i]) & see) | (__float_as_uint(NEG_INF) & ~see));
        }
      }
    }
    float mx = NEG_INF;
#pragma unroll
    for (int b = 0; b < KB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[b][i]);
    mx = xor32_max(mx) * c2;  // c2 > 0
    // the maximum that the exponents refer to moves only when a score exceeds it by more than 8 (or there was none): the
    // probabilities stay below 2^8, their rounding is relative, and most steps leave O as it is
    if (__any(mx > m + 8.0f || m == NEG_INF)) {
      const float mn = fmaxf(m, mx);
      const float f = mn == NEG_INF ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= f;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] *= f;
    }
    const float ms = m == NEG_INF ? 0.f : -m;
    // The probabilities are rounded to the type of v, which the matrix cores take; their sum is of the unrounded ones. Each is off by
    // half a step of its own value at most, which leaves an error of 0.0015 (bf16) or 0.0002 (fp16) of the result's norm, as large
    // as the rounding of the result. A second product with what the rounding takes off would remove it, for half of the matrix
    // work again.
    u32x4 pf[2 * KB];
#pragma unroll
    for (int b = 0; b < KB; ++b)
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const float x = __builtin_amdgcn_exp2f(fmaf(s[b][i], c2, ms)), y = __builtin_amdgcn_exp2f(fmaf(s[b][i + 1], c2, ms));
        l += x + y;
        pf[2 * b + i / 8][(i % 8) / 2] = E::pack(x, y);
      }
    // transposing reads: lane i of a 16-lane group g names key 4 (g / 2) + i / 4, columns 16 (g % 2) + 4 (i % 4) ..
    const int vr = 4 * half + ((lane & 15) >> 2), vc = ((lane >> 4) & 1) * 32 + (lane & 3) * 8;  // row, byte of it
#pragma unroll
    for (int ks = 0; ks < 2 * KB; ++ks)
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        const int r0 = 16 * ks + vr, r1 = r0 + 8, byte = d * 64 + vc;
        const char* p0 = vbuf + r0 * (HD * 2) + (byte ^ (Swz<HD>::v(r0) << 4));
        const char* p1 = vbuf + r1 * (HD * 2) + (byte ^ (Swz<HD>::v(r1) << 4));
        o[d] = mfma32<E>(tr_pair(p0, p1), pf[ks], o[d]);
      }
    constexpr int VF = 2 * KB * ND, VPRE = VF < 4 ? VF : 4;
    __builtin_amdgcn_sched_group_barrier(0x100, 2 * VPRE, 1);
#pragma unroll
    for (int i = 0; i < VF - VPRE; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 1);
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 1);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, VPRE, 1);
  }
};

// ---- work ---------------------------------------------------------------------------------------------------------------
// A step's keys lie in LDS once for the workgroup's eight waves. Tiles of more than 128 rows give each wave 32 rows and all
// keys; smaller ones share their rows between waves that take different keys of the step (two waves up to 128 rows, four up
// to 64), joined through LDS at the end: with 256-row tiles alone, 16 single tokens (8 rows) took 41.6 us against 22.5, and 16
// chunks of 96 rows 42.6 against 37.5; a fourth form for up to 32 rows, with O's columns split too, was no faster.
// RW waves side by side in rows, KW in keys.
template <int HD, int RW>
struct Form {
  static constexpr int KW = 8 / RW, KB = att_bn<HD>() / 32 / KW;
};
__device__ __forceinline__ int form_of(int rows) { return rows <= 64 ? 2 : rows <= 128 ? 4 : 8; }
// What a step costs in units of about 1.3 us: tiles of 256 rows are bound by the products, small ones by the bytes of the keys.
__device__ __forceinline__ int cost_of(int rw) { return rw == 8 ? 4 : rw == 4 ? 3 : 2; }
// Units of a tile's beginning and end: the first keys' and the queries' way from memory, the result's. (0, 3, 6, 10 and 16 of
// them: mixed batch 89, 84.5, 79.6, 79.7, 81.8 us; 8192-token prompt 413, 358, 315, 306, 310.)
constexpr int ATT_BEGIN = 8;

// The work is shared out on the device, where the lengths are: `parts` workgroups, one a CU. With few tiles (up to a quarter
// of the parts) each tile gets parts of its own, as many as its keys deserve, and a workgroup has one piece of one tile. With more,
// the steps of all tiles, key head by key head, each with its cost, are one line that the parts share in equal lengths,
// however ragged the batch is. A tile with several pieces is joined through the workspace: a piece's O (not divided by the
// sum), maximum and sum go there, in 32 bits: to place 0 of the part if the tile began in an earlier one, otherwise to place
// 1. The workgroup whose piece is the last to be there joins them all, in the order of the keys. Nobody waits for anybody:
// data and stamps are written through to the coherence point and acknowledged before the stamps of the others are read, so
// at least one workgroup sees all of them.
template <int HD>
struct Parts {
  static __host__ __device__ constexpr int64_t stamps(int parts) { return ((int64_t)parts * 2 * 8 + 255) / 256 * 256; }
  static __host__ __device__ constexpr int64_t piece(int bm) { return (int64_t)bm * (HD + 2) * 4; }
  static __host__ __device__ constexpr int64_t bytes(int parts, int bm) { return stamps(parts) + 2 * parts * piece(bm); }
  static __device__ __forceinline__ unsigned long long* stamp(void* ws, int g, int place) { return (unsigned long long*)ws + 2 * g + place; }
  // O, [bm] maximum, [bm] sum. O is [bm][HD], or for tiles of 256 rows' form as their waves hold it: [wave][HD / 8][64 lanes][4]
  static __device__ __forceinline__ float* data(void* ws, int parts, int bm, int g, int place) {
    return (float*)((char*)ws + stamps(parts) + (2 * (int64_t)g + place) * piece(bm));
  }
};

__device__ __forceinline__ int udiv(int a, int b) { return (int)((uint32_t)a / (uint32_t)b); }

// Which steps of a tile lie in part g.
struct Cut {
  int start, share;  // the line's unit at which the tile's first step starts, and the units of a part; or, share == 0:
  int n, cost;       // steps, units of a step                             `cost` parts of its own, from part `start` on
  int each, more;    // of those parts: `each` steps, one more in the first `more`
  __device__ __forceinline__ int before(int x) const { return udiv(min(max(x - start, 0), n * cost) + cost - 1, cost); }  // steps that begin below unit x
  __device__ __forceinline__ int own(int p) const { return p * each + min(p, more); }
  __device__ __forceinline__ int lo(int g) const { return share ? before(g * share) : own(g - start); }
  __device__ __forceinline__ int hi(int g) const { return share ? before((g + 1) * share) : own(g + 1 - start); }
  __device__ __forceinline__ int first() const { return share ? udiv(start, share) : start; }
  __device__ __forceinline__ int last() const { return share ? udiv(start + n * cost - 1, share) : start + cost - 1; }
};

template <int HD>
struct AttendLds {
  // two stages of K and V
  static constexpr int TILE = att_bn<HD>() * HD * 2, NST = 2, STAGES = NST * 2 * TILE;
  static constexpr int RS = HD + 4;                                // floats between joined rows: banks
  static constexpr int JOIN = (8 * 32 * RS + 8 * 64) * 4;          // eight waves' 32 rows, maxima and sums
  static constexpr int REQS = STAGES > JOIN ? STAGES : JOIN;       // first token and keys of each request, ..
  static constexpr int FIRST = REQS + 4 * (2 * MKX_MAX_SLOTS + 4);  // .. tiles ahead of it (uint16), then a flag
  static constexpr int FLAGS = FIRST + 2 * MKX_MAX_SLOTS + 16;     // a number of each wave
  static constexpr int BYTES = FLAGS + 4 * ATT_WAVES;
  static_assert(BYTES <= 160 * 1024, "LDS of a CU");
};

// Rows r < nr of `waves` waves' results, po[wave][32][RS] and pm[wave][2][32], joined: to `out`, or to a piece.
template <class E, int HD, class Put>
__device__ __forceinline__ void join_rows(const float* po, const float* pm, int waves, int stride, int nr, Put put) {
  constexpr int TPR = HD / 4, RS = AttendLds<HD>::RS;
  for (int r = threadIdx.x / TPR; r < nr; r += ATT_BLOCK / TPR) {
    const int c = (threadIdx.x % TPR) * 4;
    float mm = NEG_INF, ll = 0.f;
    for (int w = 0; w < waves; ++w) mm = fmaxf(mm, pm[(w * stride + r / 32) * 64 + r % 32]);
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int w = 0; w < waves; ++w) {
      const int at = w * stride + r / 32;
      const float f = mm == NEG_INF ? 0.f : __builtin_amdgcn_exp2f(pm[at * 64 + r % 32] - mm);
      ll = fmaf(f, pm[at * 64 + 32 + r % 32], ll);
      const f32x4 x = *reinterpret_cast<const f32x4*>(po + (at * 32 + r % 32) * RS + c);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] = fmaf(f, x[i], acc[i]);
    }
    put(r, c, acc, mm, ll);
  }
}
template <class E>
__device__ __forceinline__ void put_out(uint16_t* dst, f32x4 o, float sum) {
  const float inv = sum > 0.f ? 1.0f / sum : 0.f;
  *reinterpret_cast<u32x2*>(dst) = u32x2{E::pack(o[0] * inv, o[1] * inv), E::pack(o[2] * inv, o[3] * inv)};
}

// Steps s0 .. s1 - 1 of one tile; part == NULL: they are all of it.
template <class E, int HD, int RW>
__device__ __forceinline__ void run_piece(args_ptr pa, const AttendLaunch& L, const Item& it, char* lds, int s0, int s1, float* part) {
  using F = Form<HD, RW>;
  constexpr int TILE = AttendLds<HD>::TILE, RS = AttendLds<HD>::RS;
  const auto& a = *fresh(pa);
  const Steps<att_bn<HD>()> st(it);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, half = lane >> 5, l32 = lane & 31;
  const int rw = wave % RW, kw = wave / RW;
  const float c2 = a.scale * 1.44269504088896340736f;
  constexpr int NST = AttendLds<HD>::NST, DMAS = 2 * Loader<HD>::N;  // of a wave and stage
  auto buf = [&](int s) { return lds + ((s - s0) & (NST - 1)) * (2 * TILE); };
  Loader<HD> ld;
  Rows<E, HD> rows;
  constexpr int ND = HD / 32;
  const Pages pg(a, it, L.shift);
  ld.init(pg);
  ld.fetch(pg, it, st.key(s0));
  rows.init(a, it, L.G, it.row0 + 32 * rw);  // ahead of the DMAs: they are waited for in order
#pragma unroll
  for (int i = 0; i < NST - 1; ++i)
    if (s0 + i < s1) {
      ld.load(pg, it, buf(s0 + i), buf(s0 + i) + TILE, st.key(s0 + i));
      ld.fetch(pg, it, st.key(s0 + i + 1));
    }
  for (int s = s0; s < s1; ++s) {
    if (s + NST - 2 < s1) wait_vm_le<(NST - 2) * DMAS>(); else wait_vm_le<0>();
    exec_barrier();  // the step's stage is there for all waves, and all are done with the one before it
    if (s + NST - 1 < s1) ld.load(pg, it, buf(s + NST - 1), buf(s + NST - 1) + TILE, st.key(s + NST - 1));
    ld.fetch(pg, it, st.key(s + NST));
    const int k0 = st.key(s);
    const bool tamed = ((k0 < it.hi && k0 + att_bn<HD>() > it.all_hi) || (k0 < it.all_lo && k0 + att_bn<HD>() > it.lo)) &&
                       tame_values<E, HD>(buf(s) + TILE, (int*)(lds + AttendLds<HD>::FLAGS));
    const char *kb = buf(s) + kw * F::KB * 32 * HD * 2, *vb = kb + TILE;
    const int key0 = k0 + kw * F::KB * 32;
    constexpr int KB = F::KB < 2 ? F::KB : 2;
#pragma unroll
    for (int k = 0; k < F::KB; k += KB) rows.template step<KB>(it, pg.sinks, kb + k * 32 * HD * 2, vb + k * 32 * HD * 2, key0 + 32 * k, c2);
    if (tamed)
      for (int j = key0; j < min(key0 + F::KB * 32, it.hi); ++j) {
        const int page = it.table[min(j >> pg.shift, pg.cols - 1)];
        if ((unsigned)page >= (unsigned)pg.n_pages || (j < it.lo && j >= it.sinks)) continue;
        const uint16_t* v = (const uint16_t*)(pg.v + pg.at(page, j));
        const u32x2 w = *reinterpret_cast<const u32x2*>(v + (lane % (HD / 4)) * 4);
        if (__any((E::not_finite(w[0]) | E::not_finite(w[1])) != 0)) rows.add_not_finite(v, j, pg.sinks);
      }
  }
  const float sum = xor32_sum(rows.l);
  const int nr = min(it.nrows - it.row0, 32 * RW);
  __syncthreads();  // the stages are free
  if constexpr (RW == 8) {
    const int r = 32 * rw + l32;
    if (part == nullptr && r < nr) {
      uint16_t* dst = out_row(a, it, L.G, it.row0 + r, 4 * half);
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 4) put_out<E>(dst + 32 * d + 2 * i, f32x4{rows.o[d][i], rows.o[d][i + 1], rows.o[d][i + 2], rows.o[d][i + 3]}, sum);
    }
    if (part != nullptr) {  // a wave's 1 KB at a time
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          st_sc1(part, (((wave * ND + d) * 4 + i / 4) * 64 + lane) * 16, __builtin_bit_cast(u32x4, f32x4{rows.o[d][i], rows.o[d][i + 1], rows.o[d][i + 2], rows.o[d][i + 3]}));
      if (half == 0) {
        st_sc1_b32(part, (L.bm * HD + r) * 4, __float_as_uint(rows.m));
        st_sc1_b32(part, (L.bm * HD + L.bm + r) * 4, __float_as_uint(sum));
      }
    }
  } else {
    float* po = (float*)lds;       // [KW][RW][32][RS]
    float* pm = po + 8 * 32 * RS;  // [KW][RW][2][32]
    const int at = kw * RW + rw;
    if (32 * rw + l32 < nr) {
      if (half == 0) {
        pm[at * 64 + l32] = rows.m;
        pm[at * 64 + 32 + l32] = sum;
      }
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          *reinterpret_cast<f32x4*>(po + (at * 32 + l32) * RS + 32 * d + 2 * i + 4 * half) = f32x4{rows.o[d][i], rows.o[d][i + 1], rows.o[d][i + 2], rows.o[d][i + 3]};
    }
    __syncthreads();
    join_rows<E, HD>(po, pm, F::KW, RW, nr, [&](int r, int c, f32x4 o, float mm, float ll) {
      if (part == nullptr) {
        put_out<E>(out_row(a, it, L.G, it.row0 + r, c), o, ll);
      } else {
        st_sc1(part, (r * HD + c) * 4, __builtin_bit_cast(u32x4, o));
        if (c == 0) {
          st_sc1_b32(part, (L.bm * HD + r) * 4, __float_as_uint(mm));
          st_sc1_b32(part, (L.bm * HD + L.bm + r) * 4, __float_as_uint(ll));
        }
      }
    });
    __syncthreads();
  }
}

// The pieces of a tile, all of them in the workspace, joined: by the rows (a wave takes rows of its own through all pieces), or,
// a long history of a few rows, by the pieces: wave w takes the pieces 4 w .. 4 w + 3 of every 32, and the waves' results are
// joined through LDS; whichever takes fewer rounds of loads. Four groups of rows of four pieces are on their way at once;
// HD / 4 lanes hold a row, the rows of a group lie side by side.
template <int HD>
struct Joined {
  static constexpr int TPR = HD / 4, RPG = 64 / TPR, NG = 4, ROWS = NG * RPG, U = 4;
  f32x4 o[NG];
  float m[NG], l[NG];
  __device__ __forceinline__ void init() {
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
      m[i] = NEG_INF;
      l[i] = 0.f;
    }
  }
  // rows r0 .. r0 + ROWS - 1 (those that exist) of the pieces of parts g .. g + n - 1, n <= U
  template <class Piece>
  __device__ __forceinline__ void add(int bm, int r0, int g, int n, Piece piece) {
    const int lane = threadIdx.x & 63, c = (lane % TPR) * 4;
    u32x4 x[U][NG];
    float pm[U][NG], pl[U][NG];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const float* p = k < n ? piece(g + k) : nullptr;
      if (p != nullptr) {
        const auto rs = rsrc(p);
#pragma unroll
        for (int i = 0; i < NG; ++i) {
          const int r = min(r0 + i * RPG + lane / TPR, bm - 1);
          pm[k][i] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, (bm * HD + r) * 4, 0, CPOL_SC1));
          pl[k][i] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, (bm * HD + bm + r) * 4, 0, CPOL_SC1));
          x[k][i] = __builtin_amdgcn_raw_buffer_load_b128(rs, (r * HD + c) * 4, 0, CPOL_SC1);
        }
      } else {
#pragma unroll
        for (int i = 0; i < NG; ++i) {
          pm[k][i] = NEG_INF;
          pl[k][i] = 0.f;
          x[k][i] = u32x4{0u, 0u, 0u, 0u};
        }
      }
    }
#pragma unroll
    for (int k = 0; k < U; ++k)
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        const float mn = fmaxf(m[i], pm[k][i]);
        const float f = mn == NEG_INF ? 0.f : __builtin_amdgcn_exp2f(m[i] - mn), h = mn == NEG_INF ? 0.f : __builtin_amdgcn_exp2f(pm[k][i] - mn);
        const f32x4 v = __builtin_bit_cast(f32x4, x[k][i]);
        m[i] = mn;
        l[i] = l[i] * f + pl[k][i] * h;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][j] = o[i][j] * f + v[j] * h;
      }
  }
};
template <class E, int HD>
__device__ __forceinline__ void join_pieces(args_ptr pa, const AttendLaunch& L, const Item& it, const Cut& cut, char* lds) {
  using J = Joined<HD>;
  constexpr int RS = AttendLds<HD>::RS;
  const auto& a = *fresh(pa);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, c = (lane % J::TPR) * 4;
  const int all = min(it.nrows - it.row0, L.bm), g0 = cut.first(), g1 = cut.last();
  auto piece = [&](int g) -> const float* {
    const int lo = cut.lo(g);
    return lo < cut.hi(g) ? Parts<HD>::data(a.ws, L.parts, L.bm, g, lo > 0 ? 0 : 1) : nullptr;
  };
  const int pieces = g1 - g0 + 1, chunks = (all + J::ROWS - 1) / J::ROWS;
  const int by_rows = (chunks + ATT_WAVES - 1) / ATT_WAVES * ((pieces + J::U - 1) / J::U);
  const int by_pieces = chunks * ((pieces + J::U * ATT_WAVES - 1) / (J::U * ATT_WAVES));
  if (by_rows <= by_pieces) {
    for (int r0 = wave * J::ROWS; r0 < all; r0 += ATT_WAVES * J::ROWS) {
      J j;
      j.init();
      for (int g = g0; g <= g1; g += J::U) j.add(L.bm, r0, g, min(g1 - g + 1, J::U), piece);
#pragma unroll
      for (int i = 0; i < J::NG; ++i) {
        const int r = r0 + i * J::RPG + lane / J::TPR;
        if (r < all) put_out<E>(out_row(a, it, L.G, it.row0 + r, c), j.o[i], j.l[i]);
      }
    }
    return;
  }
  float* po = (float*)lds;
  float* pm = po + 8 * 32 * RS;
  for (int r0 = 0; r0 < all; r0 += J::ROWS) {
    J j;
    j.init();
    for (int g = g0 + J::U * wave; g <= g1; g += J::U * ATT_WAVES) j.add(L.bm, r0, g, min(g1 - g + 1, J::U), piece);
#pragma unroll
    for (int i = 0; i < J::NG; ++i) {
      const int r = i * J::RPG + lane / J::TPR;
      *reinterpret_cast<f32x4*>(po + (wave * 32 + r) * RS + c) = j.o[i];
      if (c == 0) {
        pm[wave * 64 + r] = j.m[i];
        pm[wave * 64 + 32 + r] = j.l[i];
      }
    }
    __syncthreads();
    join_rows<E, HD>(po, pm, ATT_WAVES, 1, min(all - r0, J::ROWS),
                     [&](int r, int cc, f32x4 o, float, float ll) { put_out<E>(out_row(a, it, L.G, it.row0 + r0 + r, cc), o, ll); });
    __syncthreads();
  }
}

// The same for tiles of more than 128 rows: a wave joins the 32 rows that it holds in each piece, as it holds them.
template <class E, int HD>
__device__ __forceinline__ void join_large(args_ptr pa, const AttendLaunch& L, const Item& it, const Cut& cut) {
  constexpr int N = HD / 8;
  const auto& a = *fresh(pa);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, half = lane >> 5;
  const int r = 32 * wave + (lane & 31);
  f32x4 o[N];
  float m = NEG_INF, l = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int g = cut.first(); g <= cut.last(); ++g) {
    if (cut.lo(g) == cut.hi(g)) continue;
    const auto rs = rsrc(Parts<HD>::data(a.ws, L.parts, L.bm, g, cut.lo(g) > 0 ? 0 : 1));
    const float pm = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, (L.bm * HD + r) * 4, 0, CPOL_SC1));
    const float pl = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, (L.bm * HD + L.bm + r) * 4, 0, CPOL_SC1));
    u32x4 x[N];
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = __builtin_amdgcn_raw_buffer_load_b128(rs, ((wave * N + i) * 64 + lane) * 16, 0, CPOL_SC1);
    const float mn = fmaxf(m, pm);
    const float f = mn == NEG_INF ? 0.f : __builtin_amdgcn_exp2f(m - mn), h = mn == NEG_INF ? 0.f : __builtin_amdgcn_exp2f(pm - mn);
    m = mn;
    l = l * f + pl * h;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const f32x4 v = __builtin_bit_cast(f32x4, x[i]);
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j] = o[i][j] * f + v[j] * h;
    }
  }
  if (it.row0 + r < it.nrows) {
    uint16_t* dst = out_row(a, it, L.G, it.row0 + r, 4 * half);
#pragma unroll
    for (int i = 0; i < N; ++i) put_out<E>(dst + 8 * i, o[i], l);
  }
}

template <class E, int HD>
__device__ __forceinline__ void run_tile(args_ptr pa, const AttendLaunch& L, const Item& it, char* lds, int s0, int s1, float* part) {
  switch (form_of(min(it.nrows - it.row0, L.bm))) {
    case 2: run_piece<E, HD, 2>(pa, L, it, lds, s0, s1, part); break;
    case 4: run_piece<E, HD, 4>(pa, L, it, lds, s0, s1, part); break;
    default: run_piece<E, HD, 8>(pa, L, it, lds, s0, s1, part);
  }
}

// Many row tiles: one workgroup a (row tile, key head), heads fastest, the last tiles first. Request b's tiles start at slot cu[b] G / bm + b, which leaves room for every request's last, partial tile: a workgroup finds its request by a
// search of cu.
template <class E, int HD>
__global__ __launch_bounds__(ATT_BLOCK, 2) void attend_tiles_kernel(mkx_attend_args, AttendLaunch) {
  const args_ptr pa = (args_ptr)__builtin_amdgcn_kernarg_segment_ptr();
  const AttendLaunch L = launch_args(pa);
  const auto& a = *pa;
  extern __shared__ __align__(1024) char lds[];
  const const_i32 cu = (const_i32)(uintptr_t)a.cu;
  const int tile = (gridDim.x - 1 - blockIdx.x) / a.NK, h = (gridDim.x - 1 - blockIdx.x) % a.NK;
  auto slot = [&](int b) { return (int)((int64_t)min(max(cu[b], 0), a.T) * L.G / L.bm) + b; };
  int b = 0, e = a.B;
  while (e - b > 1) {
    const int m = (b + e) >> 1;
    if (slot(m) <= tile) b = m; else e = m;
  }
  const Request r = request(pa, L.shift, b);
  const int row0 = (tile - slot(b)) * L.bm;
  if (row0 < 0 || row0 >= r.nq * L.G) return;
  const Item it = make_item(a, L, r, b, h, row0);
  run_tile<E, HD>(pa, L, it, lds, 0, Steps<att_bn<HD>()>(it).n, nullptr);
}

// Who makes a workgroup's plan: all its threads, PER entries each, or, with up to 64 requests of up to 256 tiles, every wave for
// itself and without a barrier (16 single tokens: 2.5 us to the plan's end when its sums still went through LDS, 4.8 with sums
// over the workgroup).
template <int BLOCK>
struct BlockTeam {
  void* sums;
  int* mine;
  __device__ __forceinline__ int rank() const { return threadIdx.x; }
  template <class T>
  __device__ __forceinline__ T scan(T v, T& total) const { return block_scan<BLOCK>(v, total, (T*)sums); }
  // v of the one member that has `me`, on all of them
  __device__ __forceinline__ void tell(bool me, int (&v)[3]) const {
    if (me)
      for (int i = 0; i < 3; ++i) mine[i] = v[i];
    __syncthreads();
    for (int i = 0; i < 3; ++i) v[i] = __builtin_amdgcn_readfirstlane(mine[i]);
    __syncthreads();
  }
};
struct WaveTeam {
  static __device__ __forceinline__ int last(int x) { return __builtin_amdgcn_readlane(x, 63); }
  static __device__ __forceinline__ long long last(long long x) {
    return (long long)((unsigned long long)(uint32_t)last((int)(x >> 32)) << 32 | (uint32_t)last((int)x));
  }
  __device__ __forceinline__ int rank() const { return threadIdx.x & 63; }
  template <class T>
  __device__ __forceinline__ T scan(T v, T& total) const {
    const T x = wave_sum(v);
    total = last(x);
    return x - v;
  }
  __device__ __forceinline__ void tell(bool me, int (&v)[3]) const {
    const int from = __ffsll(__ballot(me)) - 1;
    for (int i = 0; i < 3; ++i) v[i] = __builtin_amdgcn_readlane(v[i], from);
  }
};

// Where part g starts: an entry, its first unit, and (own) the parts of that entry; the line's end for the part.
struct Place {
  int entry, start, parts, h, share, end;  // share == 0: parts of their own
};
// The entries' steps n and the cost of each step, PER of them on each member: false where part g has nothing to do.
template <int PER, class Team>
__device__ __forceinline__ bool find_place(const Team& team, const int (&n)[PER], const int (&cost)[PER], int per, int NK, int parts, int g, Place& pl) {
  int units = 0, some = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    units += n[i] * cost[i];
    some += n[i] > 0;
  }
  long long sum;
  team.scan((long long)some << 32 | units, sum);
  const int work = __builtin_amdgcn_readfirstlane((int)sum) * NK, tiles = __builtin_amdgcn_readfirstlane((int)(sum >> 32)) * NK;
  if (work == 0) return false;
  // Parts of their own for tiles: as many as the tile's units are shares, and as many as keep joining them below the steps
  // that they save (31 K keys of one request: 34 us with 122 pieces a tile, 29 with 63). Of four shares the smallest is
  // taken whose parts are there; the largest always fits, since sum(ceil(units / share)) <= work / share + tiles.
  const bool own = tiles * 4 <= parts;
  int share = 0;
  auto pieces = [&](int i, int sh) {
    return n[i] == 0 ? 0 : min(udiv(n[i] * cost[i] + sh - 1, sh), (int)(4 * __builtin_sqrtf((float)n[i])) + 1);
  };
  if (own) {
    const int even = udiv(work + parts - 1, parts);
    auto candidate = [&](int c) { return c < 3 ? even + udiv(even * (c + 1), 10) + 1 : udiv(work + parts - tiles - 1, parts - tiles); };
    long long sums = 0;
#pragma unroll
    for (int c = 0; c < 3; ++c)
#pragma unroll
      for (int i = 0; i < PER; ++i) sums += (long long)pieces(i, candidate(c)) << (16 * c);
    team.scan(sums, sum);
    int c = 0;
    while (c < 3 && ((int)(sum >> (16 * c)) & 0xffff) * NK > parts) ++c;
    share = max(__builtin_amdgcn_readfirstlane(candidate(c)), 3);
  }
  int len[PER];
  units = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    len[i] = n[i] == 0 ? 0 : own ? pieces(i, share) : n[i] * cost[i] + ATT_BEGIN;
    units += len[i];
  }
  int W, u = team.scan(units, W);
  W = __builtin_amdgcn_readfirstlane(W);
  const int all = W * NK;
  if (!own) share = max(udiv(all + parts - 1, parts), 4 + ATT_BEGIN);
  const int x = own ? g : g * share;
  pl.end = own ? min(x + 1, all) : min(x + share, all);
  if (x >= pl.end) return false;
  pl.h = udiv(x, W);
  pl.share = own ? 0 : share;
  int v[3] = {0, 0, 0};
  bool me = false;
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (len[i] > 0) {
      if (u <= x - pl.h * W && x - pl.h * W < u + len[i]) {
        me = true;
        v[0] = team.rank() * per + i;
        v[1] = u;
        v[2] = len[i];
      }
      u += len[i];
    }
  team.tell(me, v);
  pl.entry = v[0];
  pl.start = pl.h * W + v[1];
  pl.parts = v[2];
  return true;
}

template <class E, int HD>
__global__ __launch_bounds__(ATT_BLOCK, 2) void attend_kernel(mkx_attend_args, AttendLaunch) {
  const args_ptr pa = (args_ptr)__builtin_amdgcn_kernarg_segment_ptr();
  const AttendLaunch L = launch_args(pa);
  extern __shared__ __align__(1024) char lds[];
  using LD = AttendLds<HD>;
  using St = Steps<att_bn<HD>()>;
  int32_t* s_q0 = (int32_t*)(lds + LD::REQS);         // first token of each request, and the end of the last
  int32_t* s_n = s_q0 + MKX_MAX_SLOTS + 4;            // its keys
  uint16_t* s_first = (uint16_t*)(lds + LD::FIRST);  // tiles ahead of it
  int* s_all = (int*)(s_first + MKX_MAX_SLOTS);
  const int tid = threadIdx.x, B = pa->B, NK = pa->NK;
  // neighbouring parts share keys: they go to one XCD (workgroups are dealt out to the 8 XCDs in turn)
  const int g = (blockIdx.x & 7) * (L.parts >> 3) + (blockIdx.x >> 3);
  auto req_of = [&](int b) {
    Request r;
    r.q0 = s_q0[b];
    r.nq = max(s_q0[b + 1] - r.q0, 0);
    r.n = s_n[b];
    return r;
  };
  auto keep = [&](int b, const Request& r) {
    s_q0[b] = r.q0;
    if (b == B - 1) s_q0[B] = r.q0 + r.nq;
    s_n[b] = r.n;
  };
  auto cost_rows = [&](const Item& it) { return cost_of(form_of(min(it.nrows - it.row0, L.bm))); };
  // entries: the requests where none has more than one tile, otherwise the tiles; a tile whose rows see nothing has a step
  // too: its rows are zeros
  bool many = true, any = false;
  int entries = B;
  Place pl;
  auto tile_cost = [&](int rank, int per, int i, int& n, int& cost) {
    const int t = rank * per + i;
    n = cost = 0;
    if (i < per && t < entries) {
      const int b = many ? last_at_or_below(s_first, B, t) : t;
      const Request r = req_of(b);
      const int row0 = many ? (t - s_first[b]) * L.bm : 0;
      if (row0 >= 0 && row0 < r.nq * L.G) {
        const Item it = make_item(*pa, L, r, b, 0, row0);
        n = max(St(it).n, 1);
        cost = cost_rows(it);
      }
    }
  };
  bool block = B > 64;
  if (!block) {  // every wave writes the same numbers into s_q0, s_n and s_first, and reads its own
    const WaveTeam team;
    const int b = tid & 63;
    Request r = {0, 0, 0};
    if (b < B) {
      r = request(pa, L.shift, b);
      keep(b, r);
    }
    const int nt = (r.nq * L.G + L.bm - 1) / L.bm;
    many = __any(nt > 1);
    if (!many) {
      int n[1] = {0}, cost[1] = {0};
      if (r.nq > 0) {
        const Item it = make_item(*pa, L, r, b, 0, 0);
        n[0] = max(St(it).n, 1);
        cost[0] = cost_rows(it);
      }
      any = find_place<1>(team, n, cost, 1, NK, L.parts, g, pl);
    } else {
      constexpr int PER = 4;
      int total;
      const int at = team.scan(min(nt, ATT_TILES), total);
      entries = __builtin_amdgcn_readfirstlane(min(total, L.tiles));
      block = entries > 64 * PER;
      if (!block) {
        if (b < B) s_first[b] = (uint16_t)min(at, ATT_TILES);
        const int per = (entries + 63) / 64;
        int n[PER], cost[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) tile_cost(tid & 63, per, i, n[i], cost[i]);
        any = find_place<PER>(team, n, cost, per, NK, L.parts, g, pl);
      }
    }
  }
  if (block) {
    constexpr int PER = MKX_MAX_SLOTS / ATT_BLOCK;
    static_assert(ATT_TILES <= MKX_MAX_SLOTS, "as many tiles as requests a thread");
    long long* s_sums = (long long*)lds;  // until the first step
    const int per_b = (B + ATT_BLOCK - 1) / ATT_BLOCK;
    Request req[PER];
    int nt = 0, most = 0, n[PER], cost[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int b = tid * per_b + i;
      req[i] = Request{0, 0, 0};
      if (i < per_b && b < B) {
        req[i] = request(pa, L.shift, b);
        keep(b, req[i]);
        const int tiles = (req[i].nq * L.G + L.bm - 1) / L.bm;
        nt = min(nt + tiles, ATT_TILES);
        most = max(most, tiles);
      }
    }
    many = __syncthreads_or(most > 1);
    if (many) {
      int total, at = block_scan<ATT_BLOCK>(nt, total, (int*)s_sums);
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (i < per_b && tid * per_b + i < B) {
          s_first[tid * per_b + i] = (uint16_t)min(at, ATT_TILES);
          at = min(at + (req[i].nq * L.G + L.bm - 1) / L.bm, INT32_MAX / 2);
        }
      entries = min(total, L.tiles);  // no more where cu rises, as it should
      __syncthreads();
    }
    const int per_t = (entries + ATT_BLOCK - 1) / ATT_BLOCK;
#pragma unroll
    for (int i = 0; i < PER; ++i) tile_cost(tid, per_t, i, n[i], cost[i]);
    any = find_place<PER>(BlockTeam<ATT_BLOCK>{s_sums, (int*)(s_sums + ATT_WAVES)}, n, cost, per_t, NK, L.parts, g, pl);
  }
  if (!any) return;
  int t = pl.entry, h = pl.h, start = pl.start;
  const bool own = pl.share == 0;
  const int share = pl.share, own_parts = pl.parts, x_end = pl.end;
  while (start < x_end) {
    const int b = many ? __builtin_amdgcn_readfirstlane(last_at_or_below(s_first, B, t)) : t;
    const Request r0 = req_of(b);
    const Request r = {__builtin_amdgcn_readfirstlane(r0.q0), __builtin_amdgcn_readfirstlane(r0.nq), __builtin_amdgcn_readfirstlane(r0.n)};
    const int row0 = many ? (t - __builtin_amdgcn_readfirstlane((int)s_first[b])) * L.bm : 0;
    if (row0 >= 0 && row0 < r.nq * L.G) {
      const Item it = make_item(*fresh(pa), L, r, b, h, row0);
      const St st(it);
      Cut cut = {start + ATT_BEGIN, share, max(st.n, 1), cost_rows(it), 0, 0};
      if (own) {
        const int each = udiv(cut.n, own_parts);
        cut = Cut{start, 0, cut.n, own_parts, each, cut.n - each * own_parts};
      }
      const int s0 = __builtin_amdgcn_readfirstlane(cut.lo(g)), s1 = __builtin_amdgcn_readfirstlane(cut.hi(g));
      if (s0 < s1) {
        const bool whole = s0 == 0 && s1 == cut.n;
        const int place = s0 > 0 ? 0 : 1;
        run_tile<E, HD>(pa, L, it, lds, s0, min(s1, st.n), whole ? nullptr : Parts<HD>::data(fresh(pa)->ws, L.parts, L.bm, g, place));
        if (!whole) {
          void* ws = fresh(pa)->ws;
          wait_vm0();  // this wave's part of the piece is at the coherence point
          __syncthreads();
          if (tid < 64) {
            if (tid == 0) __hip_atomic_store(Parts<HD>::stamp(ws, g, place), L.stamp, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            wait_vm0();
            __atomic_signal_fence(__ATOMIC_SEQ_CST);
            bool there = true;
            const int first = cut.first();  // holds the tile's first step
            for (int k = first + tid; k <= cut.last(); k += 64)
              if (cut.lo(k) < cut.hi(k))
                there = there && __hip_atomic_load(Parts<HD>::stamp(ws, k, cut.lo(k) > 0 ? 0 : 1), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == L.stamp;
            const bool all_there = __all(there);
            // of several workgroups that see all of them, the one that takes the first stamp joins
            if (tid == 0)
              *s_all = all_there && __hip_atomic_exchange(Parts<HD>::stamp(ws, first, 1), 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == L.stamp;
          }
          __syncthreads();
          if (*s_all) {
            if (form_of(min(it.nrows - it.row0, L.bm)) == 8) join_large<E, HD>(pa, L, it, cut);
            else join_pieces<E, HD>(pa, L, it, cut, lds);
            // a launch replayed from a graph has the same stamp again
            for (int k = cut.first() + tid; k <= cut.last(); k += ATT_BLOCK)
              if (cut.lo(k) < cut.hi(k)) __hip_atomic_store(Parts<HD>::stamp(ws, k, cut.lo(k) > 0 ? 0 : 1), 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          }
          __syncthreads();
        }
      }
      if (own) return;
      start = cut.start + cut.n * cut.cost;
    }
    if (++t == entries) {
      t = 0;
      ++h;
    }
  }
}

}  // namespace mkx
