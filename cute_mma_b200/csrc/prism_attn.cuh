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

// The idx-th tile of `bm` rows, by one whole warp.  last_first: the tiles of a sequence in descending order (a causal
// row tile costs the more the later it is; CTAs start in order of idx, so that the long ones start first).
// Packed: offsets are taken into [0, rows] and never run backwards, whatever the tensor holds.
__device__ __forceinline__ AttnWork attn_find(const AttnRows& r, int idx, int bm, bool last_first) {
  AttnWork w;
  w.spare = w.n_spare = 0;
  if (r.cu == nullptr) {
    const int nt = (r.len + bm - 1) / bm;
    const int t = idx / r.n;
    w.tile = last_first ? nt - 1 - t : t;
    w.len = r.len;
    w.row = 0;
    w.batch = idx - t * r.n;
    w.orow = (long long)w.batch * r.len;
    return w;
  }
  const int lane = threadIdx.x & 31;
  int base = 0;
  for (int b0 = 0; b0 < r.n; b0 += 32) {
    const int b = b0 + lane;
    int s = 0, e = 0;
    if (b < r.n) {
      s = attn_clamp(__ldg(r.cu + b), 0, r.rows);
      e = attn_clamp(__ldg(r.cu + b + 1), s, r.rows);
    }
    const int nt = (e - s + bm - 1) / bm;
    int incl = nt;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += o;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, idx < base + incl);
    if (hit) {
      const int l = __ffs(hit) - 1;
      const int t = idx - base - (incl - nt);
      w.tile = __shfl_sync(0xffffffffu, last_first ? nt - 1 - t : t, l);
      w.len = __shfl_sync(0xffffffffu, e - s, l);
      w.row = __shfl_sync(0xffffffffu, s, l);
      w.batch = 0;
      w.orow = w.row;
      return w;
    }
    base += __shfl_sync(0xffffffffu, incl, 31);
  }
  w.tile = -1;
  w.len = w.row = w.batch = 0;
  w.orow = 0;
  w.spare = idx - base;
  w.n_spare = r.tiles - base;
  return w;
}

// Rows of a packed batch that belong to no sequence, [0, cu[0]) and [cu[n], rows), are zeros in every output: written by
// the CTAs that got no tile.  out: rows x heads x dim, this CTA's head; 16-byte pieces.
__device__ __forceinline__ void attn_zero_gap(const AttnRows& r, const AttnWork& w, uint16_t* out, int heads, int head,
                                              int dim) {
  const int front = attn_clamp(__ldg(r.cu), 0, r.rows), end = attn_clamp(__ldg(r.cu + r.n), 0, r.rows);
  const int pieces = dim >> 3;
  const long long gap = (long long)front + (r.rows - end);
  for (long long i = (long long)w.spare * blockDim.x + threadIdx.x; i < gap * pieces; i += (long long)w.n_spare * blockDim.x) {
    const long long g = i / pieces;
    const long long row = g < front ? g : end + (g - front);
    reinterpret_cast<uint4*>(out + (row * heads + head) * dim)[i - g * pieces] = make_uint4(0u, 0u, 0u, 0u);
  }
}

// A bounded wait by a whole warp, which stays together: false for all lanes if it ran out for one.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity));
}

// 2^x, the hardware's approximation (2 ulp); -infinity gives 0.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }

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

// One row of `cols` features from TMEM (the thread's lane) times f, rounded once to 16 bits, to global memory in
// 16-byte pieces.  All threads of the warp call it; only those with `store` write.
template <int DT, int DH>
__device__ __forceinline__ void attn_store_row(uint32_t taddr, float f, uint16_t* dst, int dim, bool store) {
#pragma unroll
  for (int c = 0; c < DH; c += 32) {
    if (c >= dim) break;
    uint32_t r[32];
    tmem_ld_x32(taddr + c, r);
    tmem_ld_wait();
#pragma unroll
    for (int e = 0; e < 32; e += 8) {
      uint4 v;
      v.x = Elem<DT>::pack(__uint_as_float(r[e]) * f, __uint_as_float(r[e + 1]) * f);
      v.y = Elem<DT>::pack(__uint_as_float(r[e + 2]) * f, __uint_as_float(r[e + 3]) * f);
      v.z = Elem<DT>::pack(__uint_as_float(r[e + 4]) * f, __uint_as_float(r[e + 5]) * f);
      v.w = Elem<DT>::pack(__uint_as_float(r[e + 6]) * f, __uint_as_float(r[e + 7]) * f);
      if (store && c + e < dim) *reinterpret_cast<uint4*>(dst + c + e) = v;
    }
  }
}

}  // namespace prism
