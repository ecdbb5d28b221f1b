// Layer norm, forward and backward, of 16-bit rows:
//   s = x (+ residual, rounded to 16 bits), mu = mean s, rstd = (mean (s - mu)^2 + eps)^-1/2, xh = (s - mu) rstd,
//   y = xh w + b;   g = dy w, dx = rstd (g - mean g - xh mean(g xh)) (+ ds), dw = sum over rows of dy xh, db = sum of dy.
// Bound by HBM: every element is read once and kept in registers (32 a thread) between the two sums of a row.  The
// squares are taken of deviations from the mean, not as a difference of means, which would lose rows far from zero.
//
// The threads of a row are 8, 32, 128 or 512, the first that hold the row's columns; up to 32 they are part of a warp
// and reduce by shuffles, several rows to a CTA.  Rows of full 16-byte pieces move in those, others in pairs or singly.
#include "prism_host.cuh"
#include "prism_norm.cuh"

namespace prism {
namespace {

constexpr int kElems = 32;   // columns a thread holds at most

template <int DT>
__device__ __forceinline__ float to_float(uint16_t v) {
  return Elem<DT>::unpack((uint32_t)v).x;
}

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
    f[0] = to_float<DT>((uint16_t)v.w[0]);
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

// Sums of N values over the threads of a row, the same bits in all of them.  `slot` alternates from row to row, so that
// one barrier a call is enough.
template <int TPR, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float (*red)[N][16], int slot) {
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int d = (TPR < 32 ? TPR : 32) / 2; d > 0; d >>= 1) v[n] += __shfl_xor_sync(0xffffffffu, v[n], d);
  if constexpr (TPR > 32) {
    constexpr int kWarps = TPR / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0)
#pragma unroll
      for (int n = 0; n < N; ++n) red[slot][n][warp] = v[n];
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) {
      float t = lane < kWarps ? red[slot][n][lane] : 0.f;
#pragma unroll
      for (int d = kWarps / 2; d > 0; d >>= 1) t += __shfl_xor_sync(0xffffffffu, t, d);
      v[n] = __shfl_sync(0xffffffffu, t, 0);
    }
  }
}

template <int TPR>
__host__ __device__ constexpr int threads_of() { return TPR <= 32 ? 256 : TPR; }

// ---------------------------------------------------------------------------------------------------- forward
template <int DT, int VEC, int TPR>
__global__ void __launch_bounds__(threads_of<TPR>()) norm_fwd_kernel(const NormArgs a) {
  constexpr int NV = kElems / VEC, kRows = threads_of<TPR>() / TPR;
  __shared__ float red[2][1][16];
  const int t = threadIdx.x % TPR;
  const long long row = (long long)blockIdx.x * kRows + threadIdx.x / TPR;
  const bool live = row < a.rows;   // (all threads stay for the sums)
  const uint16_t* x = static_cast<const uint16_t*>(a.x) + row * a.ldx;
  Piece<VEC> s[NV];
  float sum[1] = {0.f};
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int col = (i * TPR + t) * VEC;
    if (live && col < a.cols) s[i] = load_piece<VEC>(x + col);
    else for (int e = 0; e < Piece<VEC>::kWords; ++e) s[i].w[e] = 0u;
  }
  if (a.residual != nullptr) {
    const uint16_t* r = static_cast<const uint16_t*>(a.residual) + row * a.ldr;
    Piece<VEC> q[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * TPR + t) * VEC;
      if (live && col < a.cols) q[i] = load_piece<VEC>(r + col);
      else for (int e = 0; e < Piece<VEC>::kWords; ++e) q[i].w[e] = 0u;
    }
    uint16_t* so = static_cast<uint16_t*>(a.sum) + row * a.cols;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * TPR + t) * VEC;
      float f[VEC], g[VEC];
      widen<DT, VEC>(s[i], f);
      widen<DT, VEC>(q[i], g);
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[e] += g[e];
      s[i] = narrow<DT, VEC>(f);   // what is normalised is the sum as it is returned
      if (live && col < a.cols) store_piece<VEC>(so + col, s[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float f[VEC];
    widen<DT, VEC>(s[i], f);
#pragma unroll
    for (int e = 0; e < VEC; ++e) sum[0] += f[e];
  }
  row_sum<TPR, 1>(sum, red, 0);
  const float mean = sum[0] / (float)a.cols;
  float var[1] = {0.f};
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int col = (i * TPR + t) * VEC;
    float f[VEC];
    widen<DT, VEC>(s[i], f);
    if (col < a.cols)
#pragma unroll
      for (int e = 0; e < VEC; ++e) var[0] = fmaf(f[e] - mean, f[e] - mean, var[0]);
  }
  row_sum<TPR, 1>(var, red, 1);
  const float rstd = rsqrtf(var[0] / (float)a.cols + a.eps);
  if (!live) return;
  if (t == 0 && a.mean != nullptr) {
    a.mean[row] = mean;
    a.rstd[row] = rstd;
  }
  uint16_t* y = static_cast<uint16_t*>(a.y) + row * a.cols;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int col = (i * TPR + t) * VEC;
    if (col >= a.cols) continue;
    float f[VEC], w[VEC], b[VEC];
    widen<DT, VEC>(s[i], f);
    load_param<DT, VEC>(a.weight, a.w_f32, col, w);
    if (a.bias != nullptr) load_param<DT, VEC>(a.bias, a.w_f32, col, b);
    else for (int e = 0; e < VEC; ++e) b[e] = 0.f;
#pragma unroll
    for (int e = 0; e < VEC; ++e) f[e] = fmaf((f[e] - mean) * rstd, w[e], b[e]);
    store_piece<VEC>(y + col, narrow<DT, VEC>(f));
  }
}

// ---------------------------------------------------------------------------------------------------- backward
// A fixed number of CTAs walk through the rows, every thread with its E columns' sums for dw and db in registers; the CTAs'
// sums go to `partial` [ctas][2][cols], which a second launch adds up in a fixed order: bit-stable.  The next row's
// loads are under way while this row is reduced (not with 32 columns at 512 threads: registers); xh and g are formed
// again from the packed row after the reduction, which costs arithmetic that is to spare and frees 2 E registers.
template <int DT, int VEC, int TPR, int E>
__global__ void __launch_bounds__(threads_of<TPR>()) norm_bwd_kernel(const NormArgs a) {
  constexpr int NV = E / VEC, kRows = threads_of<TPR>() / TPR;
  constexpr bool kAhead = TPR * E <= 8192;
  __shared__ float red[2][2][16];
  const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  float dw[E], db[E];
#pragma unroll
  for (int e = 0; e < E; ++e) dw[e] = db[e] = 0.f;
  Piece<VEC> s[NV], d[NV], s1[NV], d1[NV];
  auto fetch = [&](long long row, Piece<VEC> (&fs)[NV], Piece<VEC> (&fd)[NV]) {
    const bool live = row < a.rows;
    const uint16_t* x = static_cast<const uint16_t*>(a.x) + row * a.ldx;
    const uint16_t* g = static_cast<const uint16_t*>(a.dy) + row * a.lddy;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * TPR + t) * VEC;
      if (live && col < a.cols) {
        fs[i] = load_piece<VEC>(x + col);
        fd[i] = load_piece<VEC>(g + col);
      } else {
        for (int e = 0; e < Piece<VEC>::kWords; ++e) fs[i].w[e] = fd[i].w[e] = 0u;
      }
    }
  };
  const float inv = 1.f / (float)a.cols;
  const long long step = (long long)gridDim.x * kRows;
  int slot = 0;
  if (kAhead) fetch((long long)blockIdx.x * kRows + sub, s1, d1);
  for (long long r0 = (long long)blockIdx.x * kRows; r0 < a.rows; r0 += step, slot ^= 1) {
    const long long row = r0 + sub;
    const bool live = row < a.rows;
    const float mean = live ? a.mean[row] : 0.f, rstd = live ? a.rstd[row] : 0.f;
    if (kAhead) {
#pragma unroll
      for (int i = 0; i < NV; ++i) { s[i] = s1[i]; d[i] = d1[i]; }
      fetch(row + step, s1, d1);
    } else {
      fetch(row, s, d);
    }
    float c[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * TPR + t) * VEC;
      float f[VEC], dy[VEC], w[VEC];
      widen<DT, VEC>(s[i], f);
      widen<DT, VEC>(d[i], dy);
      if (col < a.cols) load_param<DT, VEC>(a.weight, a.w_f32, col, w);
      else for (int e = 0; e < VEC; ++e) w[e] = 0.f;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float h = (f[e] - mean) * rstd, q = dy[e] * w[e];
        c[0] += q;
        c[1] = fmaf(q, h, c[1]);
        dw[i * VEC + e] = fmaf(dy[e], h, dw[i * VEC + e]);
        db[i * VEC + e] += dy[e];
      }
    }
    row_sum<TPR, 2>(c, red, slot);
    if (!live) continue;
    const float c0 = c[0] * inv, c1 = c[1] * inv;
    uint16_t* dx = static_cast<uint16_t*>(a.dx) + row * a.cols;
    const uint16_t* ds = static_cast<const uint16_t*>(a.dsum) + row * a.ldds;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * TPR + t) * VEC;
      if (col >= a.cols) continue;
      float f[VEC], dy[VEC], w[VEC], z[VEC];
      widen<DT, VEC>(s[i], f);
      widen<DT, VEC>(d[i], dy);
      load_param<DT, VEC>(a.weight, a.w_f32, col, w);
      if (a.dsum != nullptr) widen<DT, VEC>(load_piece<VEC>(ds + col), z);
      else for (int e = 0; e < VEC; ++e) z[e] = 0.f;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float h = (f[e] - mean) * rstd;
        f[e] = fmaf(rstd, fmaf(dy[e], w[e], -c0) - h * c1, z[e]);
      }
      store_piece<VEC>(dx + col, narrow<DT, VEC>(f));
    }
  }
  // the CTA's sums: rows of a CTA in turn through shared memory
  float* out = a.partial + (long long)blockIdx.x * 2 * a.cols;
  if constexpr (kRows > 1) {
    extern __shared__ float acc[];   // [2][cols]
    for (int r = 0; r < kRows; ++r) {
      if (sub == r) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const int col = (i * TPR + t) * VEC + e;
            if (col < a.cols) {
              acc[col] = (r ? acc[col] : 0.f) + dw[i * VEC + e];
              acc[a.cols + col] = (r ? acc[a.cols + col] : 0.f) + db[i * VEC + e];
            }
          }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < 2 * a.cols; c += blockDim.x) out[c] = acc[c];
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const int col = (i * TPR + t) * VEC + e;
        if (col < a.cols) {
          out[col] = dw[i * VEC + e];
          out[a.cols + col] = db[i * VEC + e];
        }
      }
  }
}

// Column sums of partial [ctas][2 cols] -> dw, db: 32 columns a CTA, 32 rows at a time, added in a fixed order.
template <int DT>
__global__ void __launch_bounds__(1024) norm_reduce_kernel(const float* partial, int ctas, int cols, bool f32, void* dw,
                                                           void* db) {
  __shared__ float red[32][33];
  const int c = blockIdx.x * 32 + threadIdx.x;
  float t = 0.f;
  if (c < 2 * cols)
    for (int r = threadIdx.y; r < ctas; r += 32) t += partial[(long long)r * 2 * cols + c];
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

template <int DT, int VEC, int TPR>
int launch_fwd_t(const NormArgs& a) {
  constexpr int kRows = threads_of<TPR>() / TPR;
  norm_fwd_kernel<DT, VEC, TPR><<<(unsigned)((a.rows + kRows - 1) / kRows), threads_of<TPR>(), 0, a.stream>>>(a);
  return check_launch("layer norm");
}
template <int DT, int VEC, int TPR, int E>
int launch_bwd_t(const NormArgs& a, int ctas) {
  constexpr int kRows = threads_of<TPR>() / TPR;
  norm_bwd_kernel<DT, VEC, TPR, E><<<ctas, threads_of<TPR>(), kRows > 1 ? 8 * a.cols : 0, a.stream>>>(a);
  return check_launch("layer norm backward");
}

template <int DT, int VEC>
int by_width_fwd(const NormArgs& a) {
  if (a.cols <= 8 * kElems) return launch_fwd_t<DT, VEC, 8>(a);
  if (a.cols <= 32 * kElems) return launch_fwd_t<DT, VEC, 32>(a);
  if (a.cols <= 128 * kElems) return launch_fwd_t<DT, VEC, 128>(a);
  return launch_fwd_t<DT, VEC, 512>(a);
}
template <int DT, int VEC>
int by_width_bwd(const NormArgs& a, int ctas) {
  if (a.cols <= 16 * 16) return launch_bwd_t<DT, VEC, 16, 16>(a, ctas);
  if (a.cols <= 32 * 16) return launch_bwd_t<DT, VEC, 32, 16>(a, ctas);
  if (a.cols <= 32 * 24) return launch_bwd_t<DT, VEC, 32, 24>(a, ctas);
  if (a.cols <= 32 * 32) return launch_bwd_t<DT, VEC, 32, 32>(a, ctas);
  if (a.cols <= 256 * 16) return launch_bwd_t<DT, VEC, 256, 16>(a, ctas);
  if (a.cols <= 512 * 16) return launch_bwd_t<DT, VEC, 512, 16>(a, ctas);
  return launch_bwd_t<DT, VEC, 512, 32>(a, ctas);
}
template <int DT>
int by_vec(const NormArgs& a, int vec, int ctas) {
  if (ctas == 0) return vec == 8 ? by_width_fwd<DT, 8>(a) : vec == 2 ? by_width_fwd<DT, 2>(a) : by_width_fwd<DT, 1>(a);
  return vec == 8 ? by_width_bwd<DT, 8>(a, ctas) : vec == 2 ? by_width_bwd<DT, 2>(a, ctas) : by_width_bwd<DT, 1>(a, ctas);
}

}  // namespace

int norm_max_cols() { return 512 * kElems; }

// CTAs of the backward kernel: two to an SM, fewer where the rows do not fill them.
int norm_bwd_ctas(long long rows, int cols, int num_sms) {
  const int per = cols <= 16 * 16 ? 16 : cols <= 32 * 32 ? 8 : 1;
  const long long want = (rows + per - 1) / per;
  return (int)(want < 2 * num_sms ? (want < 1 ? 1 : want) : 2 * num_sms);
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
  const unsigned blocks = (2u * (unsigned)a.cols + 31) / 32;
  const dim3 threads(32, 32);
  if (a.dtype == DT_BF16)
    norm_reduce_kernel<DT_BF16><<<blocks, threads, 0, a.stream>>>(a.partial, a.ctas, a.cols, a.w_f32, a.dw, a.db);
  else
    norm_reduce_kernel<DT_F16><<<blocks, threads, 0, a.stream>>>(a.partial, a.ctas, a.cols, a.w_f32, a.dw, a.db);
  return check_launch("layer norm weight gradient");
}

}  // namespace prism
