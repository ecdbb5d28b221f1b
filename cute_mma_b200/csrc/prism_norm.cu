// Layer norm, forward and backward, of 16-bit rows:
//   s = x (+ residual, rounded to 16 bits), mu = mean s, rstd = (mean (s - mu)^2 + eps)^-1/2, xh = (s - mu) rstd,
//   y = xh w + b;   g = dy w, dx = rstd (g - mean g - xh mean(g xh)) (+ ds), dw = sum over rows of dy xh, db = sum of dy.
// Bound by HBM: every element is read once and kept in registers (16 to 32 a thread) between the two sums of a row.  The
// squares are taken of deviations from the mean, not as a difference of means, which would lose rows far from zero.
// Measured, bf16, 16384 rows of 4096 with a residual (cold L2): forward 82 us for 537 MB, 6.5 TB/s, as fast as a copy;
// backward 83 us for 537 MB and the weight gradients' second launch.  Rows of 768: 20.5 and 27.6 us for 101 MB.  Without a
// residual 4096 rows of 8192 take 35 and 64 us, of 12288 57 and 158 us, of 16384 64 and 178 us: above 8192 columns a thread of the
// backward has 32 of them and its registers do not hold their weights and sums (512 to 904 bytes of it in local memory).
//
// The threads of a row are 8 to 512, the first that hold its columns; up to 32 they are part of a warp and reduce by
// shuffles, several rows to a CTA.  Rows of full 16-byte pieces move in those, others in pairs or singly.
#include "prism_host.cuh"
#include "prism_norm.cuh"

namespace prism {
namespace {

// VEC consecutive 16-bit values as packed words (VEC 1: one value in the low half).
template <int VEC>
struct Piece {
  static constexpr int kWords = (VEC + 1) / 2;
  uint32_t w[kWords];
};
template <int VEC>
__device__ __forceinline__ Piece<VEC> load_piece(const uint16_t* p) {
  Piece<VEC> v;
  if constexpr (VEC == 8) {
    const uint4 q = *reinterpret_cast<const uint4*>(p);
    v.w[0] = q.x; v.w[1] = q.y; v.w[2] = q.z; v.w[3] = q.w;
  } else if constexpr (VEC == 2) {
    v.w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else {
    v.w[0] = *p;
  }
  return v;
}
template <int VEC>
__device__ __forceinline__ void store_piece(uint16_t* p, const Piece<VEC>& v) {
  if constexpr (VEC == 8) *reinterpret_cast<uint4*>(p) = make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]);
  else if constexpr (VEC == 2) *reinterpret_cast<uint32_t*>(p) = v.w[0];
  else *p = (uint16_t)v.w[0];
}
template <int DT, int VEC>
__device__ __forceinline__ void widen(const Piece<VEC>& v, float (&f)[VEC]) {
  if constexpr (VEC == 1) {
    f[0] = Elem<DT>::unpack(v.w[0]).x;
  } else {
#pragma unroll
    for (int e = 0; e < VEC / 2; ++e) {
      const float2 t = Elem<DT>::unpack(v.w[e]);
      f[2 * e] = t.x;
      f[2 * e + 1] = t.y;
    }
  }
}
template <int DT, int VEC>
__device__ __forceinline__ Piece<VEC> narrow(const float (&f)[VEC]) {
  Piece<VEC> v;
  if constexpr (VEC == 1) {
    v.w[0] = Elem<DT>::pack(f[0], 0.f) & 0xffffu;
  } else {
#pragma unroll
    for (int e = 0; e < VEC / 2; ++e) v.w[e] = Elem<DT>::pack(f[2 * e], f[2 * e + 1]);
  }
  return v;
}
// VEC values of a parameter, fp32 or 16-bit.
template <int DT, int VEC>
__device__ __forceinline__ void load_param(const void* p, bool f32, int col, float (&f)[VEC]) {
  if (f32) {
    const float* q = static_cast<const float*>(p) + col;
    if constexpr (VEC == 8) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(q)), b = __ldg(reinterpret_cast<const float4*>(q) + 1);
      f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[e] = __ldg(q + e);
    }
  } else {
    widen<DT, VEC>(load_piece<VEC>(static_cast<const uint16_t*>(p) + col), f);
  }
}

// Sums of N values over the TPR threads of a row, the same bits in all of them.  Several rows of whole warps may share a
// CTA; `slot` alternates from call to call, so that one barrier a call is enough.
template <int TPR, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float (*red)[N][16], int slot) {
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int d = (TPR < 32 ? TPR : 32) / 2; d > 0; d >>= 1) v[n] += __shfl_xor_sync(0xffffffffu, v[n], d);
  if constexpr (TPR > 32) {
    constexpr int kWarps = TPR / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, first = warp / kWarps * kWarps;
    if (lane == 0)
#pragma unroll
      for (int n = 0; n < N; ++n) red[slot][n][warp] = v[n];
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) {
      float t = red[slot][n][first];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) t += red[slot][n][first + w];
      v[n] = t;
    }
  }
}

// A thread's E columns in fp32, two to a register pair (two operations an instruction).
template <int DT, int VEC, int E>
__device__ __forceinline__ void widen_all(const Piece<VEC> (&v)[E / VEC], float2 (&f)[E / 2]) {
#pragma unroll
  for (int i = 0; i < E / VEC; ++i) {
    float t[VEC];
    widen<DT, VEC>(v[i], t);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int at = i * VEC + e;
      if (at & 1) f[at / 2].y = t[e];
      else f[at / 2].x = t[e];
    }
  }
}
template <int DT, int VEC, int E>
__device__ __forceinline__ Piece<VEC> narrow_at(const float2 (&f)[E / 2], int i) {
  float t[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) t[e] = (i * VEC + e) & 1 ? f[(i * VEC + e) / 2].y : f[(i * VEC + e) / 2].x;
  return narrow<DT, VEC>(t);
}
template <int VEC, int E, int TPR>
__device__ __forceinline__ void load_row(const uint16_t* p, int t, int cols, bool live, Piece<VEC> (&v)[E / VEC]) {
#pragma unroll
  for (int i = 0; i < E / VEC; ++i) {
    const int col = (i * TPR + t) * VEC;
#pragma unroll
    for (int e = 0; e < Piece<VEC>::kWords; ++e) v[i].w[e] = 0u;
    if (live && col < cols) v[i] = load_piece<VEC>(p + col);
  }
}
// A parameter's E columns in fp32, zeros behind the row.
template <int DT, int VEC, int E, int TPR>
__device__ __forceinline__ void load_params(const void* p, bool f32, int t, int cols, float2 (&f)[E / 2]) {
#pragma unroll
  for (int i = 0; i < E / VEC; ++i) {
    const int col = (i * TPR + t) * VEC;
    float v[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = 0.f;
    if (p != nullptr && col < cols) load_param<DT, VEC>(p, f32, col, v);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int at = i * VEC + e;
      if (at & 1) f[at / 2].y = v[e];
      else f[at / 2].x = v[e];
    }
  }
}

// ---------------------------------------------------------------------------------------------------- forward
template <int TPR>
__host__ __device__ constexpr int fwd_threads() { return TPR <= 32 ? 256 : TPR; }   // of a CTA
template <int DT, int VEC, int TPR, int E>
__global__ void __launch_bounds__(fwd_threads<TPR>()) norm_fwd_kernel(const NormArgs a) {
  constexpr int kRows = fwd_threads<TPR>() / TPR;
  __shared__ float red[2][1][16];
  const int t = threadIdx.x % TPR;
  const long long row = (long long)blockIdx.x * kRows + threadIdx.x / TPR;
  const bool live = row < a.rows;   // (all threads stay for the sums)
  Piece<VEC> s[E / VEC];
  float2 f[E / 2];
  load_row<VEC, E, TPR>(static_cast<const uint16_t*>(a.x) + row * a.ldx, t, a.cols, live, s);
  if (a.residual != nullptr) {
    Piece<VEC> q[E / VEC];
    load_row<VEC, E, TPR>(static_cast<const uint16_t*>(a.residual) + row * a.ldr, t, a.cols, live, q);
    uint16_t* so = static_cast<uint16_t*>(a.sum) + row * a.cols;
#pragma unroll
    for (int i = 0; i < E / VEC; ++i) {
      const int col = (i * TPR + t) * VEC;
      float x[VEC], g[VEC];
      widen<DT, VEC>(s[i], x);
      widen<DT, VEC>(q[i], g);
#pragma unroll
      for (int e = 0; e < VEC; ++e) x[e] += g[e];
      s[i] = narrow<DT, VEC>(x);   // what is normalised is the sum as it is returned
      if (live && col < a.cols) store_piece<VEC>(so + col, s[i]);
    }
  }
  widen_all<DT, VEC, E>(s, f);
  float2 acc = both(0.f);
#pragma unroll
  for (int e = 0; e < E / 2; ++e) acc = add2(acc, f[e]);
  float sum[1] = {acc.x + acc.y};
  row_sum<TPR, 1>(sum, red, 0);
  const float mean = sum[0] / (float)a.cols;
  acc = both(0.f);
  const float2 neg = both(-mean);
#pragma unroll
  for (int e = 0; e < E / 2; ++e) {
    f[e] = add2(f[e], neg);
    // (columns behind the row do not count; a pair may hold the row's last one)
    const int col = VEC == 1 ? 2 * e * TPR + t : ((2 * e / VEC) * TPR + t) * VEC + 2 * e % VEC;
    const int next = VEC == 1 ? col + TPR : col + 1;
    float2 d = f[e];
    if (col >= a.cols) d.x = 0.f;
    if (next >= a.cols) d.y = 0.f;
    acc = fma2(d, d, acc);
  }
  float var[1] = {acc.x + acc.y};
  row_sum<TPR, 1>(var, red, 1);
  const float rstd = rsqrtf(var[0] / (float)a.cols + a.eps);
  if (!live) return;
  if (t == 0 && a.mean != nullptr) {
    a.mean[row] = mean;
    a.rstd[row] = rstd;
  }
  uint16_t* y = static_cast<uint16_t*>(a.y) + row * a.cols;
  const float2 r2 = both(rstd);
#pragma unroll
  for (int i = 0; i < E / VEC; ++i) {
    const int col = (i * TPR + t) * VEC;
    if (col >= a.cols) continue;
    float w[VEC], b[VEC], o[VEC];
    load_param<DT, VEC>(a.weight, a.w_f32, col, w);
    if (a.bias != nullptr) load_param<DT, VEC>(a.bias, a.w_f32, col, b);
    else for (int e = 0; e < VEC; ++e) b[e] = 0.f;
    if constexpr (VEC == 1) {
      o[0] = fmaf((i & 1 ? f[i / 2].y : f[i / 2].x) * rstd, w[0], b[0]);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; e += 2) {
        const float2 v = fma2(mul2(f[(i * VEC + e) / 2], r2), make_float2(w[e], w[e + 1]), make_float2(b[e], b[e + 1]));
        o[e] = v.x;
        o[e + 1] = v.y;
      }
    }
    store_piece<VEC>(y + col, narrow<DT, VEC>(o));
  }
}

// ---------------------------------------------------------------------------------------------------- backward
// A fixed number of CTAs walk through the rows, every thread with its E columns' weights and sums for dw and db in
// registers; the CTAs' sums go to `partial` [ctas][2][cols], which a second launch adds up in a fixed order: bit-stable.
// Two operations an instruction where they come in pairs: with one each, and the weights read again for every row, the
// kernel issued 38 instructions a column and was bound by that (16384 x 4096: 130 us).
//
// Rows come through shared memory by cp.async, kStages - 1 of them ahead; every thread copies and reads its own columns
// only, so that the ring needs no barrier.  (2-byte pieces cannot be copied so: rows of odd columns are loaded where they
// are used.)
template <int TPR>
__host__ __device__ constexpr int bwd_threads() { return TPR <= 32 ? 256 : TPR < 256 ? 256 / TPR * TPR : TPR; }
template <int TPR, int E>
struct BwdSmem {
  static constexpr int kStages = E == 32 ? 2 : 3;
  static constexpr int kStage = bwd_threads<TPR>() * E * 2 * 3;   // the row's three tensors
  static constexpr int kSums = bwd_threads<TPR>() > TPR ? bwd_threads<TPR>() * E * 2 * 4 : 0;
  static constexpr int bytes(int vec) { return vec > 1 && kStages * kStage > kSums ? kStages * kStage : kSums; }
};
template <int BYTES>
__device__ __forceinline__ void copy_async(void* dst, const void* src, bool live) {
  const int n = live ? BYTES : 0;
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(n) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(n) : "memory");
}
template <int DT, int VEC, int TPR, int E>
__global__ void __launch_bounds__(bwd_threads<TPR>(), (E == 8 ? 768 : 512) / bwd_threads<TPR>()) norm_bwd_kernel(const NormArgs a) {
  using L = BwdSmem<TPR, E>;
  constexpr int kThreads = bwd_threads<TPR>(), kRows = kThreads / TPR, NV = E / VEC;
  constexpr bool kAhead = VEC > 1;
  extern __shared__ __align__(16) uint8_t smem[];   // ring [stage][tensor][piece][thread]; at the end the rows' sums
  __shared__ float red[2][2][16];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  float2 w[E / 2], dw[E / 2], db[E / 2];
  load_params<DT, VEC, E, TPR>(a.weight, a.w_f32, t, a.cols, w);
#pragma unroll
  for (int e = 0; e < E / 2; ++e) dw[e] = db[e] = both(0.f);
  const float inv = 1.f / (float)a.cols;
  const long long step = (long long)gridDim.x * kRows;
  const bool with_ds = a.dsum != nullptr;
  auto slot_of = [&](int stage, int tensor, int i) {
    return smem + stage * L::kStage + ((tensor * NV + i) * kThreads + threadIdx.x) * (VEC * 2);
  };
  auto issue = [&](long long row, int stage) {
    if constexpr (kAhead) {
      const bool live = row < a.rows;
      const uint16_t* x = static_cast<const uint16_t*>(a.x) + (live ? row * a.ldx : 0);
      const uint16_t* g = static_cast<const uint16_t*>(a.dy) + (live ? row * a.lddy : 0);
      const uint16_t* ds = static_cast<const uint16_t*>(a.dsum) + (live ? row * a.ldds : 0);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = (i * TPR + t) * VEC;
        const bool in = live && col < a.cols;
        copy_async<VEC * 2>(slot_of(stage, 0, i), x + (in ? col : 0), in);
        copy_async<VEC * 2>(slot_of(stage, 1, i), g + (in ? col : 0), in);
        if (with_ds) copy_async<VEC * 2>(slot_of(stage, 2, i), ds + (in ? col : 0), in);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
  };
  int slot = 0, stage = 0;
  const long long first = (long long)blockIdx.x * kRows;
#pragma unroll
  for (int i = 0; i < L::kStages - 1; ++i) issue(first + sub + i * step, i);
  float next_mean = first + sub < a.rows ? a.mean[first + sub] : 0.f, next_rstd = first + sub < a.rows ? a.rstd[first + sub] : 0.f;
  for (long long r0 = first; r0 < a.rows; r0 += step, slot ^= 1) {
    const long long row = r0 + sub;
    const bool live = row < a.rows;
    Piece<VEC> s[NV], d[NV], z[NV];
    if constexpr (kAhead) {
      asm volatile("cp.async.wait_group %0;" ::"n"(L::kStages - 2) : "memory");
      issue(row + (L::kStages - 1) * step, stage == 0 ? L::kStages - 1 : stage - 1);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        s[i] = load_piece<VEC>(reinterpret_cast<const uint16_t*>(slot_of(stage, 0, i)));
        d[i] = load_piece<VEC>(reinterpret_cast<const uint16_t*>(slot_of(stage, 1, i)));
#pragma unroll
        for (int e = 0; e < Piece<VEC>::kWords; ++e) z[i].w[e] = 0u;
        if (with_ds) z[i] = load_piece<VEC>(reinterpret_cast<const uint16_t*>(slot_of(stage, 2, i)));
      }
      if (++stage == L::kStages) stage = 0;
    } else {
      load_row<VEC, E, TPR>(static_cast<const uint16_t*>(a.x) + row * a.ldx, t, a.cols, live, s);
      load_row<VEC, E, TPR>(static_cast<const uint16_t*>(a.dy) + row * a.lddy, t, a.cols, live, d);
      load_row<VEC, E, TPR>(static_cast<const uint16_t*>(a.dsum) + row * a.ldds, t, a.cols, live && with_ds, z);
    }
    const float mean = next_mean, rstd = next_rstd;
    next_mean = row + step < a.rows ? a.mean[row + step] : 0.f;
    next_rstd = row + step < a.rows ? a.rstd[row + step] : 0.f;
    const float2 r2 = both(rstd), neg = both(-mean);
    float2 h[E / 2], q[E / 2], c0 = both(0.f), c1 = both(0.f);
    widen_all<DT, VEC, E>(s, h);
    widen_all<DT, VEC, E>(d, q);
#pragma unroll
    for (int e = 0; e < E / 2; ++e) {
      h[e] = mul2(add2(h[e], neg), r2);
      dw[e] = fma2(q[e], h[e], dw[e]);
      db[e] = add2(db[e], q[e]);
      q[e] = mul2(q[e], w[e]);
      c0 = add2(c0, q[e]);
      c1 = fma2(q[e], h[e], c1);
    }
    float c[2] = {c0.x + c0.y, c1.x + c1.y};
    row_sum<TPR, 2>(c, red, slot);
    if (!live) continue;
    const float2 m0 = both(-c[0] * inv), m1 = both(-c[1] * inv);
    uint16_t* dx = static_cast<uint16_t*>(a.dx) + row * a.cols;
    float2 add[E / 2];
    widen_all<DT, VEC, E>(z, add);
#pragma unroll
    for (int e = 0; e < E / 2; ++e) q[e] = fma2(fma2(h[e], m1, add2(q[e], m0)), r2, add[e]);
#pragma unroll
    for (int i = 0; i < E / VEC; ++i) {
      const int col = (i * TPR + t) * VEC;
      if (col < a.cols) store_piece<VEC>(dx + col, narrow_at<DT, VEC, E>(q, i));
    }
  }
  // the CTA's sums: those of its rows side by side in shared memory, then added in their order
  float* out = a.partial + (long long)blockIdx.x * 2 * a.cols;
  auto column = [&](int e, int tt) { return ((e / VEC) * TPR + tt) * VEC + e % VEC; };
  if constexpr (kRows > 1) {
    // (the ring's last copies are behind the last row: all have landed before their memory is used otherwise)
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    float* acc = reinterpret_cast<float*>(smem);   // [kRows][2][E][TPR]
    float* mine = acc + sub * 2 * TPR * E;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      mine[e * TPR + t] = e & 1 ? dw[e / 2].y : dw[e / 2].x;
      mine[(E + e) * TPR + t] = e & 1 ? db[e / 2].y : db[e / 2].x;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * TPR * E; i += blockDim.x) {
      float v = acc[i];
#pragma unroll
      for (int r = 1; r < kRows; ++r) v += acc[r * 2 * TPR * E + i];
      const int half = i / (TPR * E), col = column(i / TPR - half * E, i % TPR);
      if (col < a.cols) out[half * a.cols + col] = v;
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int col = column(e, t);
      if (col < a.cols) {
        out[col] = e & 1 ? dw[e / 2].y : dw[e / 2].x;
        out[a.cols + col] = e & 1 ? db[e / 2].y : db[e / 2].x;
      }
    }
  }
}

// Column sums of partial [ctas][2 cols] -> dw, db: 32 columns a CTA, 32 rows at a time, added in a fixed order.
template <int DT>
__global__ void __launch_bounds__(1024) norm_reduce_kernel(const float* partial, int ctas, int cols, bool f32, void* dw,
                                                           void* db) {
  __shared__ float red[32][33];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int c = blockIdx.x * 32 + threadIdx.x;
  float t = 0.f;
  if (c < 2 * cols) {
#pragma unroll 8
    for (int r = threadIdx.y; r < ctas; r += 32) t += partial[(long long)r * 2 * cols + c];
  }
  red[threadIdx.y][threadIdx.x] = t;
  __syncthreads();
  float v = red[threadIdx.x][threadIdx.y];
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  const int o = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && o < 2 * cols) {
    void* dst = o < cols ? dw : db;
    const int i = o < cols ? o : o - cols;
    if (dst == nullptr) return;
    if (f32) static_cast<float*>(dst)[i] = v;
    else static_cast<uint16_t*>(dst)[i] = (uint16_t)(Elem<DT>::pack(v, 0.f) & 0xffffu);
  }
}

// Elements per access: all tensors' rows must start and end on it.
int vec_of(const NormArgs& a, const void* const* ptrs, int n, const long long* lds, int n_ld) {
  const int wsize = a.w_f32 ? 4 : 2;
  for (int vec : {8, 2}) {
    bool fits = a.cols % vec == 0;
    for (int i = 0; i < n; ++i) fits = fits && (reinterpret_cast<uintptr_t>(ptrs[i]) % (vec * 2)) == 0;
    for (int i = 0; i < n_ld; ++i) fits = fits && lds[i] % vec == 0;
    for (const void* w : {a.weight, a.bias})
      fits = fits && (reinterpret_cast<uintptr_t>(w) % (vec == 8 ? 16 : 2 * wsize)) == 0;
    if (fits) return vec;
  }
  return 1;
}

template <int DT, int VEC, int TPR, int E>
int launch_fwd_t(const NormArgs& a) {
  constexpr int kRows = fwd_threads<TPR>() / TPR;
  norm_fwd_kernel<DT, VEC, TPR, E><<<(unsigned)((a.rows + kRows - 1) / kRows), fwd_threads<TPR>(), 0, a.stream>>>(a);
  return check_launch("layer norm");
}
template <int DT, int VEC, int TPR, int E>
int launch_bwd_t(const NormArgs& a) {
  auto* kern = norm_bwd_kernel<DT, VEC, TPR, E>;
  constexpr int kBytes = BwdSmem<TPR, E>::bytes(VEC);
  if (int rc = set_max_dynamic_smem(reinterpret_cast<const void*>(kern), kBytes, "layer norm backward")) return rc;
  kern<<<a.ctas, bwd_threads<TPR>(), kBytes, a.stream>>>(a);
  return check_launch("layer norm backward");
}

// The smallest of these (threads of a row) x (columns of a thread) that holds the row.  They go up by powers of two, with one
// step between 512 and 1024, where the library's own decoder is: 65536 rows of 768 with a residual take 68 us forward and 80 us
// backward, with the next instance 74 and 92 us (16384 x 544: 20.5 and 28.7, else 22.5 and 32.8); odd widths, which move two
// bytes at a time, lose forward (16384 x 767: 45, else 41 us) and gain backward (68, else 78 us).
template <int DT, int VEC>
int by_width_fwd(const NormArgs& a) {
  if (a.cols <= 16 * 16) return launch_fwd_t<DT, VEC, 16, 16>(a);
  if (a.cols <= 32 * 16) return launch_fwd_t<DT, VEC, 32, 16>(a);
  if (a.cols <= 32 * 24) return launch_fwd_t<DT, VEC, 32, 24>(a);
  if (a.cols <= 64 * 16) return launch_fwd_t<DT, VEC, 64, 16>(a);
  if (a.cols <= 128 * 16) return launch_fwd_t<DT, VEC, 128, 16>(a);
  if (a.cols <= 256 * 16) return launch_fwd_t<DT, VEC, 256, 16>(a);
  if (a.cols <= 256 * 32) return launch_fwd_t<DT, VEC, 256, 32>(a);
  return launch_fwd_t<DT, VEC, 512, 32>(a);
}
template <int DT, int VEC>
int by_width_bwd(const NormArgs& a) {
  if (a.cols <= 16 * 8) return launch_bwd_t<DT, VEC, 16, 8>(a);
  if (a.cols <= 32 * 8) return launch_bwd_t<DT, VEC, 32, 8>(a);
  if (a.cols <= 32 * 16) return launch_bwd_t<DT, VEC, 32, 16>(a);
  if (a.cols <= 96 * 8) return launch_bwd_t<DT, VEC, 96, 8>(a);
  if (a.cols <= 128 * 8) return launch_bwd_t<DT, VEC, 128, 8>(a);
  if (a.cols <= 256 * 8) return launch_bwd_t<DT, VEC, 256, 8>(a);
  if (a.cols <= 256 * 16) return launch_bwd_t<DT, VEC, 256, 16>(a);
  if (a.cols <= 512 * 16) return launch_bwd_t<DT, VEC, 512, 16>(a);
  return launch_bwd_t<DT, VEC, 512, 32>(a);
}
template <int DT>
int by_vec(const NormArgs& a, int vec, int ctas) {
  if (ctas == 0) return vec == 8 ? by_width_fwd<DT, 8>(a) : vec == 2 ? by_width_fwd<DT, 2>(a) : by_width_fwd<DT, 1>(a);
  return vec == 8 ? by_width_bwd<DT, 8>(a) : vec == 2 ? by_width_bwd<DT, 2>(a) : by_width_bwd<DT, 1>(a);
}

}  // namespace

int norm_max_cols() { return 512 * 32; }

// CTAs of the backward kernel: what an SM holds, fewer where they would have less than four rounds of rows each (their
// sums cost two rows of fp32 to write and to read again).
int norm_bwd_ctas(long long rows, int cols, int num_sms) {
  const int per = cols <= 16 * 8 ? 16 : cols <= 32 * 16 ? 8 : cols <= 128 * 8 ? 2 : 1;   // rows of a round
  const int held = cols <= 32 * 8 ? 3 : cols <= 32 * 16 ? 2 : cols <= 96 * 8 ? 4 : cols <= 256 * 8 ? 3 : cols <= 256 * 16 ? 2 : 1;
  const long long most = (long long)num_sms * held, want = (rows + 4 * per - 1) / (4 * per);
  return (int)(want < most ? (want < 1 ? 1 : want) : most);
}

int launch_norm_fwd(const NormArgs& a) {
  const void* ptrs[] = {a.x, a.residual, a.y, a.sum};
  const long long lds[] = {a.ldx, a.residual ? a.ldr : 8};
  const int vec = vec_of(a, ptrs, 4, lds, 2);
  return a.dtype == DT_BF16 ? by_vec<DT_BF16>(a, vec, 0) : by_vec<DT_F16>(a, vec, 0);
}

int launch_norm_bwd(const NormArgs& a) {
  const void* ptrs[] = {a.x, a.dy, a.dsum, a.dx};
  const long long lds[] = {a.ldx, a.lddy, a.dsum ? a.ldds : 8};
  const int vec = vec_of(a, ptrs, 4, lds, 3);
  if (int rc = a.dtype == DT_BF16 ? by_vec<DT_BF16>(a, vec, a.ctas) : by_vec<DT_F16>(a, vec, a.ctas)) return rc;
  // (launched beside the kernel before it, for whose end it waits)
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((2u * (unsigned)a.cols + 31) / 32);
  cfg.blockDim = dim3(32, 32);
  cfg.stream = a.stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, a.dtype == DT_BF16 ? norm_reduce_kernel<DT_BF16> : norm_reduce_kernel<DT_F16>,
                                           (const float*)a.partial, a.ctas, a.cols, a.w_f32, a.dw, a.db);
  if (e != cudaSuccess) return fail(PRISM_ERR_CUDA, "layer norm weight gradient: launch failed: %s", cudaGetErrorString(e));
  return check_launch("layer norm weight gradient");
}

}  // namespace prism
