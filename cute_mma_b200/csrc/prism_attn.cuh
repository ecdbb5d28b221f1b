// Device-side pieces shared by the attention kernels: which rows a CTA works on, TMEM moves of whole rows, products
// issued from one thread.
//
// A tile is 128 rows of one head of one sequence, 64 features wide in shared memory ([128][64] 16-bit elements with the
// 128-byte swizzle); heads wider than 64 take two such tiles side by side (DH = 128), narrower ones are filled up with
// zeros by TMA, whose tensor map ends at the head's own width.
#pragma once

#include "prism_common.cuh"

namespace prism {

constexpr int kAttnTile = 128;                 // rows of a tile
constexpr uint32_t kAttnSub = 128 * 128;       // bytes of [128][64] 16-bit elements
constexpr float kLog2e = 1.44269504088896340736f;

// The rows of a batch: packed (cu: n + 1 offsets into `rows` rows) or dense (cu null: n sequences of len rows).
struct AttnRows {
  const int* cu;
  int n, len, rows;
  int tiles;   // tiles of the grid: an upper bound for packed rows
};

// What one CTA works on.
struct AttnWork {
  int tile;    // tile of the sequence; -1: none
  int len;     // rows of the sequence
  int row;     // coordinate of its first row in the tensor maps ...
  int batch;   // ... and of its batch
  long long orow;  // its first row in the outputs, which are rows x heads x dim
  int spare, n_spare;  // tile < 0: the CTA's number among those without a tile
};

__device__ __forceinline__ int attn_clamp(int x, int lo, int hi) { return min(max(x, lo), hi); }

// The idx-th tile of `bm` rows, by one whole warp, the costliest first: blocks start in order of idx, and what is long
// must not start last.  A causal row tile costs the more the later it is (late), a key tile the earlier.  Packed: offsets
// are taken into [0, rows] and never run backwards, whatever the tensor holds.  Up to 32 kOwn sequences (a lane keeps
// kOwn tile counts for as long as the CTA lives) are gone through by levels: a sequence of nt tiles has one each of cost
// 1 to nt, the tiles of cost above L number sum max(0, nt - L), and a binary search finds the level of idx.  More
// sequences come in their own order (a search by scanning from where the last one ended; with so many no single one
// weighs much).
constexpr int kOwn = 8;
struct AttnOrder {
  int nt[kOwn];
  int total, most;   // packed: all tiles (by scanning: once they are known), by levels: tiles of the longest sequence
  bool levels;
  int from, before;  // packed, by scanning: where the last search ended, and the tiles before it
};
__device__ __forceinline__ void attn_range(const AttnRows& r, int b, int* s, int* e) {
  *s = attn_clamp(__ldg(r.cu + b), 0, r.rows);
  *e = attn_clamp(__ldg(r.cu + b + 1), *s, r.rows);
}
__device__ __forceinline__ AttnOrder attn_order(const AttnRows& r, int bm) {
  AttnOrder o;
  o.levels = r.cu != nullptr && r.n <= 32 * kOwn;
  o.from = o.before = 0;
  int sum = 0, top = 0;
#pragma unroll
  for (int k = 0; k < kOwn; ++k) {
    const int b = k * 32 + (threadIdx.x & 31);
    o.nt[k] = 0;
    if (o.levels && b < r.n) {
      int s, e;
      attn_range(r, b, &s, &e);
      o.nt[k] = (e - s + bm - 1) / bm;
    }
    sum += o.nt[k];
    top = max(top, o.nt[k]);
  }
  o.total = o.levels ? __reduce_add_sync(0xffffffffu, sum) : 0x7fffffff;
  o.most = __reduce_max_sync(0xffffffffu, top);
  return o;
}
__device__ __forceinline__ AttnWork attn_find(const AttnRows& r, AttnOrder& o, int idx, int bm, bool late) {
  AttnWork w;
  w.spare = w.n_spare = 0;
  if (r.cu == nullptr) {
    const int nt = (r.len + bm - 1) / bm;
    const int t = idx / r.n;
    w.tile = late ? nt - 1 - t : t;
    w.len = r.len;
    w.row = 0;
    w.batch = idx - t * r.n;
    w.orow = (long long)w.batch * r.len;
    return w;
  }
  const int lane = threadIdx.x & 31;
  w.tile = -1;
  w.len = w.row = w.batch = 0;
  int base = o.total;
  if (o.levels) {
    if (idx < o.total) {
      auto above = [&](int level) {
        int c = 0;
#pragma unroll
        for (int k = 0; k < kOwn; ++k) c += max(0, o.nt[k] - level);
        return (int)__reduce_add_sync(0xffffffffu, c);
      };
      int lo = 1, hi = o.most;   // the largest level whose tiles and those above it reach past idx
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (above(mid - 1) > idx) lo = mid;
        else hi = mid - 1;
      }
      int left = idx - above(lo);
#pragma unroll
      for (int k = 0; k < kOwn; ++k) {
        const unsigned has = __ballot_sync(0xffffffffu, o.nt[k] >= lo);
        const int c = __popc(has);
        if (left >= 0 && left < c) {
          const int l = __fns(has, 0, left + 1);
          const int nt = __shfl_sync(0xffffffffu, o.nt[k], l);
          int s, e;
          attn_range(r, k * 32 + l, &s, &e);
          w.tile = late ? lo - 1 : nt - lo;
          w.len = e - s;
          w.row = s;
        }
        left -= c;
      }
    }
  } else if (idx < o.total) {
    if (idx < o.before) o.from = o.before = 0;
    base = o.before;
    for (int b0 = o.from; b0 < r.n; b0 += 32) {
      const int b = b0 + lane;
      int s = 0, e = 0;
      if (b < r.n) attn_range(r, b, &s, &e);
      const int nt = (e - s + bm - 1) / bm;
      int incl = nt;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += v;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, idx < base + incl);
      if (hit) {
        o.from = b0;
        o.before = base;
        const int l = __ffs(hit) - 1;
        const int t = idx - base - (incl - nt);
        w.tile = __shfl_sync(0xffffffffu, late ? nt - 1 - t : t, l);
        w.len = __shfl_sync(0xffffffffu, e - s, l);
        w.row = __shfl_sync(0xffffffffu, s, l);
        break;
      }
      base += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (w.tile < 0) o.total = base;
  }
  w.orow = w.row;
  if (w.tile < 0) {
    w.spare = idx - base;
    w.n_spare = r.tiles - base;
  }
  return w;
}

// Rows of a packed batch that belong to no sequence, [0, cu[0]) and [cu[n], rows), are zeros in every output: written for
// the tiles of the grid that there are none of.  out: rows x heads x dim; one warp, one head, 16-byte pieces.
__device__ __forceinline__ void attn_zero_gap(const AttnRows& r, const AttnWork& w, uint16_t* out, int heads, int head,
                                              int dim) {
  const int front = attn_clamp(__ldg(r.cu), 0, r.rows), end = attn_clamp(__ldg(r.cu + r.n), front, r.rows);
  const int pieces = dim >> 3, lane = threadIdx.x & 31;
  const long long gap = (long long)front + (r.rows - end);
  for (long long i = (long long)w.spare * 32 + lane; i < gap * pieces; i += (long long)w.n_spare * 32) {
    const long long g = i / pieces;
    const long long row = g < front ? g : end + (g - front);
    reinterpret_cast<uint4*>(out + (row * heads + head) * dim)[i - g * pieces] = make_uint4(0u, 0u, 0u, 0u);
  }
}

// A bounded wait by a whole warp, which stays together: false for all lanes if it ran out for one.  It polls instead of
// sleeping in try_wait: the waits of these kernels are links of one chain, and a sleeper wakes some 100 clocks late.
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t"
      ".reg .pred P1;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 P1, [%1], %2;\n\t"
      "selp.b32 %0, 1, 0, P1;\n\t"
      "}\n"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
template <bool POLL, int LIMITS = 1>
__device__ __forceinline__ bool warp_wait_t(uint64_t* bar, uint32_t parity) {
  if (__all_sync(0xffffffffu, mbar_test(bar, parity))) return true;
  const long long t0 = clock64();
  while (true) {
#pragma unroll 1
    for (int i = 0; i < 64; ++i)
      if (__all_sync(0xffffffffu, POLL ? mbar_test(bar, parity) : mbar_try_wait(bar, parity))) return true;
    if (__any_sync(0xffffffffu, clock64() - t0 > LIMITS * PRISM_WAIT_LIMIT_CYCLES)) return false;
  }
}
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) { return warp_wait_t<true>(bar, parity); }
// For warps with time to spare, whose polling would only take issue slots from the arithmetic: asleep in try_wait.
__device__ __forceinline__ bool warp_wait_asleep(uint64_t* bar, uint32_t parity) { return warp_wait_t<false>(bar, parity); }

// The work of a CTA: it begins with the tile of its own block index and then takes over blocks that have not started yet
// (cluster launch control), so that the loads and first products of the next tile run beside the end of this one and no
// CTA is set up twice.  The warp that loads looks for work ahead and hands it to the others through two slots.
struct AttnSched {
  uint64_t full[2], empty[2], answer_full;
  alignas(16) uint64_t answer[2];
  AttnWork work[2];
  int head[2];
};
__device__ __forceinline__ void attn_sched_init(AttnSched& s, uint32_t consumers) {
  for (int i = 0; i < 2; ++i) {
    mbar_init(&s.full[i], 1);
    mbar_init(&s.empty[i], consumers);
  }
  mbar_init(&s.answer_full, 1);
}
__device__ __forceinline__ void clc_try_cancel(uint64_t* answer, uint64_t* bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];"
               :
               : "r"(smem_u32(answer)), "r"(smem_u32(bar))
               : "memory");
}
// The x index of the block taken over, or -1 where there is none left.
__device__ __forceinline__ int clc_answer(const uint64_t* answer) {
  uint32_t took, x;
  asm volatile(
      "{\n\t"
      ".reg .b128 h;\n\t"
      ".reg .pred p;\n\t"
      "mov.b128 h, {%2, %3};\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t"
      "mov.b32 %1, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, h;\n\t"
      "}\n"
      : "=r"(took), "=r"(x)
      : "l"(answer[0]), "l"(answer[1]));
  return took ? (int)x : -1;
}

// The warp that looks for work and brings its tiles in.  load(work, head) returns false if a wait ran out; zero(work, head):
// what to do for a tile that there is none of.
template <typename Load, typename Zero>
__device__ __forceinline__ bool attn_schedule(AttnSched& s, const AttnRows& rows, int heads, int bm, bool late, Load load,
                                              Zero zero) {
  const int lane = threadIdx.x & 31;
  Ring r(2);
  uint32_t phase = 0;
  int idx = blockIdx.x;
  bool ok = true;
  AttnOrder order = attn_order(rows, bm);
  while (ok && idx >= 0) {
    const int head = idx % heads;
    const AttnWork w = attn_find(rows, order, idx / heads, bm, late);
    if (w.tile < 0) {
      zero(w, head);
    } else {
      ok = warp_wait(&s.empty[r.idx], r.phase ^ 1);
      if (ok && lane == 0) {
        s.work[r.idx] = w;
        s.head[r.idx] = head;
        mbar_arrive(&s.full[r.idx]);
      }
      r.next();
      ok = ok && load(w, head);
    }
    // the next block is asked for when this one's last tiles are on their way, not before: a CTA with a long one must not
    // keep a second from the others
    if (lane == 0) {
      mbar_arrive_expect_tx(&s.answer_full, 16);
      clc_try_cancel(s.answer, &s.answer_full);
    }
    // (the answer is waited for in any case: it is on its way into this CTA's memory)
    if (!warp_wait(&s.answer_full, phase)) ok = false;
    phase ^= 1u;
    idx = __shfl_sync(0xffffffffu, clc_answer(s.answer), 0);
    fence_proxy_async_smem();   // the answer is read before the next one may overwrite it
    __syncwarp();
  }
  // (also where a wait has run out: there is no more work for the others either)
  if (!warp_wait(&s.empty[r.idx], r.phase ^ 1)) return false;
  if (lane == 0) {
    s.work[r.idx].tile = -1;
    mbar_arrive(&s.full[r.idx]);
  }
  return ok;
}
// The next piece of work for one of the other warps: false at the end (or if the wait ran out, with ok false).  The limit is 32
// times that of other waits: a CTA may go through millions of tiles that there are none of before it finds the next one that
// there is, 12 ns each over all CTAs, 26 s for the largest grid.  The warp that looks has its own, short waits, and says so when one
// has run out.  (A wait that looks for progress instead cost dk and dv 1 to 6 % of their time.)
__device__ __forceinline__ bool attn_next(AttnSched& s, Ring& r, AttnWork* w, int* head, bool* ok) {
  if (!warp_wait_t<true, 32>(&s.full[r.idx], r.phase)) { *ok = false; return false; }
  // (through shuffles: the compiler then knows that all lanes have the same)
  const AttnWork& o = s.work[r.idx];
  w->tile = __shfl_sync(0xffffffffu, o.tile, 0);
  w->len = __shfl_sync(0xffffffffu, o.len, 0);
  w->row = __shfl_sync(0xffffffffu, o.row, 0);
  w->batch = __shfl_sync(0xffffffffu, o.batch, 0);
  w->orow = __shfl_sync(0xffffffffu, o.orow, 0);
  *head = __shfl_sync(0xffffffffu, s.head[r.idx], 0);
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(&s.empty[r.idx]);
  r.next();
  return w->tile >= 0;
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
// 2^x for two values on the FMA pipe: x = n + f with f in [-1/2, 1/2], a polynomial of degree 5 for 2^f (least largest
// relative error with the constant fixed to 1, by linear programming: 1.9e-7 in fp32) times 2^n.  Below 2^-126 the result
// stays at 2^-126 (of a largest probability of 1); NaN stays NaN.  The special function unit makes 16 of these a clock and
// SM: 1024 clocks for a tile of 128 x 128, as long as two products take with heads of 128.  The backward kernels do a quarter of
// them here (8192 rows, 16 heads: dk and dv 526 -> 508 us with heads of 128, 400 -> 386 us with heads of 64; dq 314 -> 309
// and 253 -> 231 us).  The forward kernel, which issues more beside them, does not: 253 -> 264 and 199 -> 204 us with an eighth.
__device__ __forceinline__ float2 ex2_poly2(float2 x) {
  x = make_float2(max_nan(x.x, -126.f), max_nan(x.y, -126.f));
  const float2 t = add2(x, both(12582912.f));                       // n in the low bits
  const float2 f = fma2(add2(t, both(-12582912.f)), both(-1.f), x);
  float2 p = fma2(f, both(0x1.5bb994p-10f), both(0x1.3cea84p-7f));
  p = fma2(p, f, both(0x1.c6b754p-5f));
  p = fma2(p, f, both(0x1.ebf9bcp-3f));
  p = fma2(p, f, both(0x1.62e42ap-1f));
  p = fma2(p, f, both(1.f));
  const float2 s = make_float2(__uint_as_float(__float_as_uint(t.x) * 0x800000u + 0x3f800000u),
                               __uint_as_float(__float_as_uint(t.y) * 0x800000u + 0x3f800000u));
  return mul2(p, s);
}

// 2^x, the hardware's approximation (2 ulp); -infinity gives 0.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }   // 2^e, -126 <= e <= 127
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Registers -> TMEM: 32 consecutive columns of the thread's own lane.
__device__ __forceinline__ void tmem_st_x32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      :
      : "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
        "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
        "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      :
      : "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// 4-D tiled load: box of 64 features x 128 rows of one head of one batch entry.
__device__ __forceinline__ void tma_load_4d(void* smem_dst, const CUtensorMap* m, uint64_t* bar, int c0, int c1, int c2,
                                            int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];"
      :
      : "r"(smem_u32(smem_dst)), "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
template <int DH>
__device__ __forceinline__ void attn_load_tile(void* dst, const CUtensorMap* m, uint64_t* bar, int row, int head, int batch) {
#pragma unroll
  for (int s = 0; s < DH / 64; ++s)
    tma_load_4d(static_cast<char*>(dst) + s * kAttnSub, m, bar, s * 64, row, head, batch);
}

// A from TMEM (16-bit pairs, 8 columns per 16 elements of the contraction), single CTA.
__device__ __forceinline__ void umma_f16_cta_ts_lh(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t b_hi,
                                                   uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      ".reg .b64 db;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 db, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t"
      "}\n"
      :
      : "r"(d_tmem), "r"(a_tmem), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}

// D[128 x 128] = X . Y^T over the features of two tiles (both feature-contiguous): one thread.
template <int DH>
__device__ __forceinline__ void attn_mma_xyt(uint32_t d, uint32_t x_smem, uint32_t y_smem, uint32_t idesc) {
  const uint64_t dx = desc_kmajor_sw128(x_smem, 1024), dy = desc_kmajor_sw128(y_smem, 1024);
  const uint32_t xl = (uint32_t)dx, xh = (uint32_t)(dx >> 32), yl = (uint32_t)dy, yh = (uint32_t)(dy >> 32);
#pragma unroll
  for (int k = 0; k < DH / 16; ++k) {
    const uint32_t off = ((k >> 2) * kAttnSub + (k & 3) * 32) >> 4;
    umma_f16_cta_lh(d, xl + off, xh, yl + off, yh, idesc, k > 0);
  }
}
// D[128 x DH] (+)= P . Y over the rows of a tile: P from TMEM in 16 bits, its second 64 rows of the contraction
// `half` columns after the first; steps: sixteens of rows that count.  One thread.
template <int DH>
__device__ __forceinline__ void attn_mma_py(uint32_t d, uint32_t p_tmem, uint32_t half, uint32_t y_smem, uint32_t idesc,
                                            bool accumulate, int steps) {
  const uint64_t dy = desc_mnmajor_sw128(y_smem, kAttnSub, 1024);
  const uint32_t yl = (uint32_t)dy, yh = (uint32_t)(dy >> 32);
  if (steps == 8) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      umma_f16_cta_ts_lh(d, p_tmem + (k >> 2) * half + (k & 3) * 8, yl + k * (2048 >> 4), yh, idesc, accumulate || k > 0);
  } else {
    for (int k = 0; k < steps; ++k)
      umma_f16_cta_ts_lh(d, p_tmem + (k >> 2) * half + (k & 3) * 8, yl + k * (2048 >> 4), yh, idesc, accumulate || k > 0);
  }
}

// Rows [valid, next multiple of 16) of a tile become zeros, by one warp, before products that contract over rows read
// them: what stands there belongs to the next sequence, and 0 times its infinities would not be 0.
template <int DH>
__device__ __forceinline__ void attn_zero_tail(char* tile, int valid) {
  const int rows = ((valid + 15) & ~15) - valid;
  const int lane = threadIdx.x & 31;
  for (int i = lane; i < rows * (DH / 64) * 8; i += 32) {
    const int sub = i / (rows * 8), rest = i - sub * rows * 8;
    reinterpret_cast<uint4*>(tile + sub * kAttnSub + (valid + (rest >> 3)) * 128)[rest & 7] = make_uint4(0u, 0u, 0u, 0u);
  }
  fence_proxy_async_smem();
  __syncwarp();
}

// Four fp32 values as e5m2 bytes, and back.
__device__ __forceinline__ uint32_t pack_e5m2(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return (uint32_t)lo | (uint32_t)hi << 16;
}
__device__ __forceinline__ void unpack_e5m2(uint32_t v, float (&f)[4]) {
  uint32_t a, b;
  asm("cvt.rn.f16x2.e5m2x2 %0, %1;" : "=r"(a) : "h"((uint16_t)v));
  asm("cvt.rn.f16x2.e5m2x2 %0, %1;" : "=r"(b) : "h"((uint16_t)(v >> 16)));
  const float2 x = Elem<DT_F16>::unpack(a), y = Elem<DT_F16>::unpack(b);
  f[0] = x.x; f[1] = x.y; f[2] = y.x; f[3] = y.y;
}
// What rounding to 16 bits took from o is kept times this, which puts it near o's own size.
template <int DT>
__device__ __forceinline__ constexpr float low_scale() { return DT == DT_BF16 ? 256.f : 2048.f; }

// Four lanes exchange W-word pieces: lane b of four, which held the pieces 0 to 3 of its row, gets piece b of their rows.
template <int W>
__device__ __forceinline__ void transpose_pieces(uint32_t (&p)[4][W]) {
  const int b = threadIdx.x & 3;
#pragma unroll
  for (int step = 1; step <= 2; step <<= 1) {
    const bool up = b & step;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i & step) continue;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const uint32_t t = __shfl_xor_sync(0xffffffffu, up ? p[i][w] : p[i | step][w], step);
        if (up) p[i][w] = t;
        else p[i | step][w] = t;
      }
    }
  }
}

// The warp's 32 rows of `dim` features from TMEM (a row per lane) times f, rounded once to 16 bits, to global memory: row i
// at dst + i * step, the first `rows` of them; LOW: what the rounding took goes to `low` at the same place.
// A store whose lanes write 16 bytes of 32 rows each takes the L1 cache 32 clocks; four lanes together write 64 bytes of a
// row, 8 rows a store.  (The 128 x 128 results of a backward tile: 3900 clocks one way, 1700 the other.)
template <int DT, int DH, bool LOW>
__device__ __forceinline__ void attn_store_rows(uint32_t taddr, float f, uint16_t* dst, uint8_t* low, long long step, int dim,
                                                int rows) {
  const int lane = threadIdx.x & 31, first = lane & ~3, b = lane & 3;
#pragma unroll
  for (int c = 0; c < DH; c += 32) {
    if (c >= dim) break;
    uint32_t r[32], p[4][4], z[4][2];
    tmem_ld_x32(taddr + c, r);
    tmem_ld_wait();
#pragma unroll
    for (int e = 0; e < 4; ++e) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t& lo = r[e * 8 + 2 * i];
        uint32_t& hi = r[e * 8 + 2 * i + 1];
        const float x = __uint_as_float(lo) * f, y = __uint_as_float(hi) * f;
        p[e][i] = Elem<DT>::pack(x, y);
        if constexpr (LOW) {
          const float2 h = Elem<DT>::unpack(p[e][i]);
          lo = __float_as_uint((x - h.x) * low_scale<DT>());
          hi = __float_as_uint((y - h.y) * low_scale<DT>());
        }
      }
      if constexpr (LOW) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t* q = r + e * 8 + i * 4;
          z[e][i] = pack_e5m2(__uint_as_float(q[0]), __uint_as_float(q[1]), __uint_as_float(q[2]), __uint_as_float(q[3]));
        }
      }
    }
    transpose_pieces<4>(p);
    if constexpr (LOW) transpose_pieces<2>(z);
    if (c + b * 8 < dim) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (first + i >= rows) break;
        const long long at = (first + i) * step + c + b * 8;
        *reinterpret_cast<uint4*>(dst + at) = make_uint4(p[i][0], p[i][1], p[i][2], p[i][3]);
        if constexpr (LOW) *reinterpret_cast<uint2*>(low + at) = make_uint2(z[i][0], z[i][1]);
      }
    }
  }
}

}  // namespace prism
