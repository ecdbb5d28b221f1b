// Causal attention, backward.  With P_ij = 2^(c q_i.k_j - lse_i), delta_i = do_i . o_i, dP_ij = do_i . v_j and
// dS = P (dP - delta):   dv_j = sum_i P_ij do_i,   dk_j = scale sum_i dS_ij q_i,   dq_i = scale sum_j dS_ij k_j.
//
// Three launches: delta (one pass over o and do), dk + dv by key tiles, dq by query tiles.  S and dP are formed twice
// (seven products of a tile pair instead of five) and in return every sum has one owner: no atomics, no fp32 copy of dq
// to clear and convert, the same bits every run.  A key tile walks through all query heads of its group, so that the
// gradients of shared heads are sums in TMEM as well.
#include "prism_attn.cuh"
#include "prism_attn_host.cuh"
#include "prism_host.cuh"

namespace prism {
namespace {

struct BwdParams {
  AttnRows rows;
  uint16_t *dq, *dk, *dv;
  const float *lse, *delta;   // heads x rows
  int hq, hkv, group, dim;
  float c, scale;             // scale * log2 e, scale
  int* err;
};

constexpr int kThreads = 384;   // two warpgroups of arithmetic, MMA warp, TMA warp, warp of the row statistics

// ---------------------------------------------------------------------------------------------------- delta
// Sixteen lanes a row of a head: 16-byte pieces of o and do.
struct DeltaParams {
  const uint16_t *o, *d_o;
  AttnStrides sdo;
  float* delta;
  int heads, dim, len;   // len: rows per batch entry
  long long rows;
};
template <int DT>
__global__ void __launch_bounds__(256) attn_delta_kernel(const DeltaParams p) {
  const long long unit = (long long)blockIdx.x * 16 + (threadIdx.x >> 4);
  const int piece = threadIdx.x & 15;
  float sum = 0.f;
  const long long row = unit / p.heads;
  const int head = (int)(unit - row * p.heads);
  if (row < p.rows && piece * 8 < p.dim) {
    const long long b = row / p.len;
    const uint4 x = *reinterpret_cast<const uint4*>(p.o + unit * p.dim + piece * 8);
    const uint4 y = *reinterpret_cast<const uint4*>(p.d_o + b * p.sdo.batch + (row - b * p.len) * p.sdo.row +
                                                    head * p.sdo.head + piece * 8);
    const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 a = Elem<DT>::unpack(xs[e]), b2 = Elem<DT>::unpack(ys[e]);
      sum = fmaf(a.x, b2.x, fmaf(a.y, b2.y, sum));
    }
  }
#pragma unroll
  for (int d = 8; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  if (row < p.rows && piece == 0) p.delta[head * p.rows + row] = sum;
}

// ---------------------------------------------------------------------------------------------------- dk, dv
// Transposed scores: S^T = K Q^T and dP^T = V dO^T have a key row per TMEM lane, so that P^T and dS^T, written back over
// them in 16 bits, are the TMEM operands of dv += P^T dO and dk += dS^T Q.  The row statistics lie along the columns and
// are read from shared memory, the same word by all lanes.  Rows behind the sequence get lse = +infinity: P = 0.
template <int DH>
struct DkvSmem {
  static constexpr uint32_t kTile = (DH / 64) * kAttnSub;
  static constexpr int kRing = 2;   // pairs of Q and dO tiles
  static constexpr uint32_t kBytes = (2 + 2 * kRing) * kTile + 1024;
};
struct DkvBars {
  uint64_t kv_full, s_full, p_full, dp_full, ds_full, done;
  uint64_t q_full[2], q_empty[2], st_full[2], st_empty[2];
};

template <int DT, int DH>
__global__ void __launch_bounds__(kThreads, 1)
    attn_bwd_dkv_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                        const __grid_constant__ CUtensorMap mv, const __grid_constant__ CUtensorMap mdo, const BwdParams p) {
  using L = DkvSmem<DH>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ DkvBars bars;
  __shared__ uint32_t tmem_slot;
  __shared__ AttnWork work;
  __shared__ __align__(16) float st_lse[2][kAttnTile], st_delta[2][kAttnTile];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const int kvh = blockIdx.x % p.hkv;

  if (warp == 0) {
    const AttnWork w = attn_find(p.rows, blockIdx.x / p.hkv, kAttnTile, false);
    if (lane == 0) work = w;
  } else if (warp == 8) {
    tmem_alloc_cta(&tmem_slot, 512);
    tmem_relinquish_cta();
  } else if (warp == 9 && lane == 0) {
    mbar_init(&bars.kv_full, 1);
    mbar_init(&bars.s_full, 1);
    mbar_init(&bars.p_full, 8);
    mbar_init(&bars.dp_full, 1);
    mbar_init(&bars.ds_full, 8);
    mbar_init(&bars.done, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bars.q_full[s], 1);
      mbar_init(&bars.q_empty[s], 1);
      mbar_init(&bars.st_full[s], 1);
      mbar_init(&bars.st_empty[s], 8);
    }
    fence_mbar_init();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_slot;
  const AttnWork w = work;
  if (w.tile < 0) {
    attn_zero_gap(p.rows, w, p.dk, p.hkv, kvh, p.dim);
    attn_zero_gap(p.rows, w, p.dv, p.hkv, kvh, p.dim);
  } else {
    const int nq = (w.len + kAttnTile - 1) / kAttnTile - w.tile;   // query tiles from the diagonal on
    const int n = nq * p.group;
    bool ok = true;
    if (warp == 9) {
      if (lane == 0) {
        mbar_arrive_expect_tx(&bars.kv_full, 2 * L::kTile);
        attn_load_tile<DH>(smem, &mk, &bars.kv_full, w.row + w.tile * kAttnTile, kvh, w.batch);
        attn_load_tile<DH>(smem + L::kTile, &mv, &bars.kv_full, w.row + w.tile * kAttnTile, kvh, w.batch);
        Ring r(2);
        int head = kvh * p.group, i = 0;
        for (int it = 0; it < n; ++it, r.next()) {
          if (!mbar_wait(&bars.q_empty[r.idx], r.phase ^ 1)) { ok = false; break; }
          mbar_arrive_expect_tx(&bars.q_full[r.idx], 2 * L::kTile);
          char* dst = smem + (2 + 2 * r.idx) * L::kTile;
          attn_load_tile<DH>(dst, &mq, &bars.q_full[r.idx], w.row + (w.tile + i) * kAttnTile, head, w.batch);
          attn_load_tile<DH>(dst + L::kTile, &mdo, &bars.q_full[r.idx], w.row + (w.tile + i) * kAttnTile, head, w.batch);
          if (++i == nq) { i = 0; ++head; }
        }
      }
    } else if (warp == 10) {
      Ring r(2);
      int head = kvh * p.group, i = 0;
      for (int it = 0; it < n; ++it, r.next()) {
        const long long at = (long long)head * p.rows.rows + w.orow;
        float a[4], b[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int row = (w.tile + i) * kAttnTile + e * 32 + lane;
          a[e] = row < w.len ? __ldg(p.lse + at + row) : INFINITY;
          b[e] = row < w.len ? __ldg(p.delta + at + row) : 0.f;
        }
        if (!warp_wait(&bars.st_empty[r.idx], r.phase ^ 1)) { ok = false; break; }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          st_lse[r.idx][e * 32 + lane] = a[e];
          st_delta[r.idx][e * 32 + lane] = b[e];
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.st_full[r.idx]);
        if (++i == nq) { i = 0; ++head; }
      }
    } else if (warp == 8) {
      const uint32_t id_s = make_idesc(DT, 128, 128, 0, 0), id_o = make_idesc(DT, 128, DH, 0, 1);
      const uint32_t sk = smem_u32(smem), sv = sk + L::kTile, ring = sk + 2 * L::kTile;
      const uint32_t t_s = tmem, t_dp = tmem + 128, t_dv = tmem + 256, t_dk = tmem + 256 + DH;
      int i = 0;   // query tile of the head
      auto steps_of = [&](int tile) {
        const int valid = w.len - (w.tile + tile) * kAttnTile;
        return valid >= kAttnTile ? 8 : (valid + 15) >> 4;
      };
      auto arrived = [&](Ring& r, int tile) {   // the pair of tiles is there, and clean behind the sequence
        if (!warp_wait(&bars.q_full[r.idx], r.phase)) return false;
        const int valid = w.len - (w.tile + tile) * kAttnTile;
        if (valid < kAttnTile) {
          attn_zero_tail<DH>(smem + (2 + 2 * r.idx) * L::kTile, valid);
          attn_zero_tail<DH>(smem + (3 + 2 * r.idx) * L::kTile, valid);
        }
        tc_fence_after_sync();
        return true;
      };
      Ring r(2);
      ok = warp_wait(&bars.kv_full, 0) && arrived(r, 0);
      if (ok && lane == 0) {
        attn_mma_xyt<DH>(t_s, sk, ring, id_s);
        umma_commit_cta(&bars.s_full);
        attn_mma_xyt<DH>(t_dp, sv, ring + L::kTile, id_s);
        umma_commit_cta(&bars.dp_full);
      }
      for (int it = 0; ok && it < n; ++it) {
        const uint32_t q = ring + 2 * r.idx * L::kTile;
        const int steps = steps_of(i);
        Ring nx = r;
        nx.next();
        if (++i == nq) i = 0;
        const bool more = it + 1 < n;
        if (!warp_wait(&bars.p_full, it & 1)) { ok = false; break; }
        tc_fence_after_sync();
        if (lane == 0) attn_mma_py<DH>(t_dv, t_s, 64, q + L::kTile, id_o, it > 0, steps);
        if (more) {
          if (!arrived(nx, i)) { ok = false; break; }
          if (lane == 0) {
            attn_mma_xyt<DH>(t_s, sk, ring + 2 * nx.idx * L::kTile, id_s);
            umma_commit_cta(&bars.s_full);
          }
        }
        if (!warp_wait(&bars.ds_full, it & 1)) { ok = false; break; }
        tc_fence_after_sync();
        if (lane == 0) {
          attn_mma_py<DH>(t_dk, t_dp, 64, q, id_o, it > 0, steps);
          umma_commit_cta(&bars.q_empty[r.idx]);
          if (more) {
            attn_mma_xyt<DH>(t_dp, sv, ring + (2 * nx.idx + 1) * L::kTile, id_s);
            umma_commit_cta(&bars.dp_full);
          } else {
            umma_commit_cta(&bars.done);
          }
        }
        r = nx;
      }
    } else if (warp < 8) {
      const int half = warp >> 2;   // which 64 query columns
      const uint32_t lanes = (uint32_t)(warp & 3) << 21;
      const uint32_t s_addr = tmem + lanes + half * 64, dp_addr = s_addr + 128;
      const int key = (warp & 3) * 32 + lane;
      Ring r(2);
      int i = 0;
      const float2 c2 = make_float2(p.c, p.c);
      for (int it = 0; it < n; ++it, r.next()) {
        const bool diag = i == 0;
        if (++i == nq) i = 0;
        if (!warp_wait(&bars.st_full[r.idx], r.phase) || !warp_wait(&bars.s_full, it & 1)) { ok = false; break; }
        tc_fence_after_sync();
        uint32_t s[64];
        tmem_ld_x32(s_addr, *reinterpret_cast<uint32_t(*)[32]>(s));
        tmem_ld_x32(s_addr + 32, *reinterpret_cast<uint32_t(*)[32]>(s + 32));
        tmem_ld_wait();
        const float4* lse = reinterpret_cast<const float4*>(st_lse[r.idx] + half * 64);
        uint32_t pk[32];
#pragma unroll
        for (int e = 0; e < 64; e += 4) {
          const float4 z = lse[e >> 2];
          const float2 x = fma2(make_float2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), c2, make_float2(-z.x, -z.y));
          const float2 y = fma2(make_float2(__uint_as_float(s[e + 2]), __uint_as_float(s[e + 3])), c2, make_float2(-z.z, -z.w));
          float v[4] = {ex2(x.x), ex2(x.y), ex2(y.x), ex2(y.y)};
          if (diag) {
#pragma unroll
            for (int f = 0; f < 4; ++f)
              if (half * 64 + e + f < key) v[f] = 0.f;
          }
#pragma unroll
          for (int f = 0; f < 4; ++f) s[e + f] = __float_as_uint(v[f]);
          pk[e >> 1] = Elem<DT>::pack(v[0], v[1]);
          pk[(e >> 1) + 1] = Elem<DT>::pack(v[2], v[3]);
        }
        tmem_st_x32(s_addr, pk);
        tmem_st_wait();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.p_full);
        if (!warp_wait(&bars.dp_full, it & 1)) { ok = false; break; }
        tc_fence_after_sync();
        const float4* del = reinterpret_cast<const float4*>(st_delta[r.idx] + half * 64);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t dp[32];
          tmem_ld_x32(dp_addr + h * 32, dp);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            const float4 z = del[(h * 32 + e) >> 2];
            const float zz[4] = {z.x, z.y, z.z, z.w};
            float v[4];
#pragma unroll
            for (int f = 0; f < 4; ++f) {
              v[f] = __uint_as_float(s[h * 32 + e + f]) * (__uint_as_float(dp[e + f]) - zz[f]);
              if (diag && half * 64 + h * 32 + e + f < key) v[f] = 0.f;
            }
            pk[(h * 32 + e) >> 1] = Elem<DT>::pack(v[0], v[1]);
            pk[((h * 32 + e) >> 1) + 1] = Elem<DT>::pack(v[2], v[3]);
          }
        }
        tmem_st_x32(dp_addr, pk);
        tmem_st_wait();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&bars.st_empty[r.idx]);
          mbar_arrive(&bars.ds_full);
        }
      }
      if (ok) {
        if (warp_wait(&bars.done, 0)) {
          tc_fence_after_sync();
          const int row = w.tile * kAttnTile + key;
          const bool mine = row < w.len;
          const long long at = ((w.orow + row) * p.hkv + kvh) * p.dim;
          if (half == 0) attn_store_row<DT, DH>(tmem + lanes + 256, 1.f, p.dv + at, p.dim, mine);
          else attn_store_row<DT, DH>(tmem + lanes + 256 + DH, p.scale, p.dk + at, p.dim, mine);
        } else {
          ok = false;
        }
      }
    }
    if (!ok && lane == 0) atomicExch(p.err, PRISM_ERR_DEVICE_WAIT);
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 8) tmem_dealloc_cta(tmem, 512);
}

// ---------------------------------------------------------------------------------------------------- dq
// A query tile stays, key and value tiles stream by; two S buffers, so that the next scores are formed while the
// warpgroups (64 key columns each) are in their exponentials.
template <int DH>
struct DqSmem {
  static constexpr uint32_t kTile = (DH / 64) * kAttnSub;
  static constexpr int kRing = 2;   // pairs of K and V tiles
  static constexpr uint32_t kBytes = (2 + 2 * kRing) * kTile + 1024;
};
struct DqBars {
  uint64_t q_full, s_full[2], dp_full, ds_full, done;
  uint64_t k_full[2], v_full[2], kv_empty[2];
};

template <int DT, int DH>
__global__ void __launch_bounds__(kThreads, 1)
    attn_bwd_dq_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                       const __grid_constant__ CUtensorMap mv, const __grid_constant__ CUtensorMap mdo, const BwdParams p) {
  using L = DqSmem<DH>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ DqBars bars;
  __shared__ uint32_t tmem_slot;
  __shared__ AttnWork work;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const int head = blockIdx.x % p.hq, kvh = head / p.group;

  if (warp == 0) {
    const AttnWork w = attn_find(p.rows, blockIdx.x / p.hq, kAttnTile, true);
    if (lane == 0) work = w;
  } else if (warp == 8) {
    tmem_alloc_cta(&tmem_slot, 512);
    tmem_relinquish_cta();
  } else if (warp == 9 && lane == 0) {
    mbar_init(&bars.q_full, 1);
    mbar_init(&bars.dp_full, 1);
    mbar_init(&bars.ds_full, 8);
    mbar_init(&bars.done, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bars.s_full[s], 1);
      mbar_init(&bars.k_full[s], 1);
      mbar_init(&bars.v_full[s], 1);
      mbar_init(&bars.kv_empty[s], 1);
    }
    fence_mbar_init();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_slot;
  const AttnWork w = work;
  if (w.tile < 0) {
    attn_zero_gap(p.rows, w, p.dq, p.hq, head, p.dim);
  } else {
    const int n = w.tile + 1;   // key tiles up to the diagonal
    bool ok = true;
    if (warp == 9) {
      if (lane == 0) {
        mbar_arrive_expect_tx(&bars.q_full, 2 * L::kTile);
        attn_load_tile<DH>(smem, &mq, &bars.q_full, w.row + w.tile * kAttnTile, head, w.batch);
        attn_load_tile<DH>(smem + L::kTile, &mdo, &bars.q_full, w.row + w.tile * kAttnTile, head, w.batch);
        Ring r(2);
        for (int j = 0; j < n; ++j, r.next()) {
          if (!mbar_wait(&bars.kv_empty[r.idx], r.phase ^ 1)) { ok = false; break; }
          char* dst = smem + (2 + 2 * r.idx) * L::kTile;
          mbar_arrive_expect_tx(&bars.k_full[r.idx], L::kTile);
          attn_load_tile<DH>(dst, &mk, &bars.k_full[r.idx], w.row + j * kAttnTile, kvh, w.batch);
          mbar_arrive_expect_tx(&bars.v_full[r.idx], L::kTile);
          attn_load_tile<DH>(dst + L::kTile, &mv, &bars.v_full[r.idx], w.row + j * kAttnTile, kvh, w.batch);
        }
      }
    } else if (warp == 8) {
      const uint32_t id_s = make_idesc(DT, 128, 128, 0, 0), id_o = make_idesc(DT, 128, DH, 0, 1);
      const uint32_t sq = smem_u32(smem), sdo = sq + L::kTile, ring = sq + 2 * L::kTile;
      const uint32_t t_dp = tmem + 256, t_dq = tmem + 384;
      Ring r(2);
      auto scores = [&](Ring& rr, int j) {
        if (!warp_wait(&bars.k_full[rr.idx], rr.phase)) return false;
        const int valid = w.len - j * kAttnTile;
        if (valid < kAttnTile) attn_zero_tail<DH>(smem + (2 + 2 * rr.idx) * L::kTile, valid);
        tc_fence_after_sync();
        if (lane == 0) {
          attn_mma_xyt<DH>(tmem + (j & 1) * 128, sq, ring + 2 * rr.idx * L::kTile, id_s);
          umma_commit_cta(&bars.s_full[j & 1]);
        }
        return true;
      };
      auto dprobs = [&](Ring& rr) {
        if (!warp_wait(&bars.v_full[rr.idx], rr.phase)) return false;
        tc_fence_after_sync();
        if (lane == 0) {
          attn_mma_xyt<DH>(t_dp, sdo, ring + (2 * rr.idx + 1) * L::kTile, id_s);
          umma_commit_cta(&bars.dp_full);
        }
        return true;
      };
      ok = warp_wait(&bars.q_full, 0) && scores(r, 0) && dprobs(r);
      for (int j = 0; ok && j < n; ++j) {
        Ring nx = r;
        nx.next();
        const bool more = j + 1 < n;
        if (more && !scores(nx, j + 1)) { ok = false; break; }
        if (!warp_wait(&bars.ds_full, j & 1)) { ok = false; break; }
        tc_fence_after_sync();
        const int valid = w.len - j * kAttnTile;
        if (lane == 0) {
          attn_mma_py<DH>(t_dq, t_dp, 64, ring + 2 * r.idx * L::kTile, id_o, j > 0, valid >= kAttnTile ? 8 : (valid + 15) >> 4);
          umma_commit_cta(&bars.kv_empty[r.idx]);
          if (!more) umma_commit_cta(&bars.done);
        }
        if (more && !dprobs(nx)) { ok = false; break; }
        r = nx;
      }
    } else if (warp < 8) {
      const int half = warp >> 2;   // which 64 key columns
      const uint32_t lanes = (uint32_t)(warp & 3) << 21;
      const uint32_t dp_addr = tmem + lanes + 256 + half * 64;
      const int r = (warp & 3) * 32 + lane;
      const int row = w.tile * kAttnTile + r;
      const bool mine = row < w.len;
      const long long at = (long long)head * p.rows.rows + w.orow + row;
      const float neg = mine ? -__ldg(p.lse + at) : -INFINITY, delta = mine ? __ldg(p.delta + at) : 0.f;
      const float2 c2 = make_float2(p.c, p.c), n2 = make_float2(neg, neg);
      for (int j = 0; j < n; ++j) {
        const bool diag = j + 1 == n;
        if (!warp_wait(&bars.s_full[j & 1], (j >> 1) & 1)) { ok = false; break; }
        tc_fence_after_sync();
        const uint32_t s_addr = tmem + lanes + (j & 1) * 128 + half * 64;
        uint32_t s[64];
        tmem_ld_x32(s_addr, *reinterpret_cast<uint32_t(*)[32]>(s));
        tmem_ld_x32(s_addr + 32, *reinterpret_cast<uint32_t(*)[32]>(s + 32));
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 64; e += 2) {
          const float2 x = fma2(make_float2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), c2, n2);
          s[e] = __float_as_uint(ex2(x.x));
          s[e + 1] = __float_as_uint(ex2(x.y));
        }
        if (!warp_wait(&bars.dp_full, j & 1)) { ok = false; break; }
        tc_fence_after_sync();
        uint32_t pk[32];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t dp[32];
          tmem_ld_x32(dp_addr + h * 32, dp);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            float a = __uint_as_float(s[h * 32 + e]) * (__uint_as_float(dp[e]) - delta);
            float b = __uint_as_float(s[h * 32 + e + 1]) * (__uint_as_float(dp[e + 1]) - delta);
            if (diag) {
              if (half * 64 + h * 32 + e > r) a = 0.f;
              if (half * 64 + h * 32 + e + 1 > r) b = 0.f;
            }
            pk[(h * 32 + e) >> 1] = Elem<DT>::pack(a, b);
          }
        }
        tmem_st_x32(dp_addr, pk);
        tmem_st_wait();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.ds_full);
      }
      if (ok) {
        if (warp_wait(&bars.done, 0)) {
          tc_fence_after_sync();
          if (half == 0)
            attn_store_row<DT, DH>(tmem + lanes + 384, p.scale, p.dq + ((w.orow + row) * p.hq + head) * p.dim, p.dim, mine);
        } else {
          ok = false;
        }
      }
    }
    if (!ok && lane == 0) atomicExch(p.err, PRISM_ERR_DEVICE_WAIT);
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 8) tmem_dealloc_cta(tmem, 512);
}

template <int DT, int DH>
int launch_t(const AttnArgs& a, const CUtensorMap* m, BwdParams p) {
  if (p.dk != nullptr) {
    if (int rc = attn_rows(a, kAttnTile, a.hkv, &p.rows)) return rc;
    auto* dkv = attn_bwd_dkv_kernel<DT, DH>;
    if (int rc = set_max_dynamic_smem(reinterpret_cast<const void*>(dkv), DkvSmem<DH>::kBytes, "causal attention dk, dv")) return rc;
    dkv<<<(unsigned)p.rows.tiles * (unsigned)a.hkv, kThreads, DkvSmem<DH>::kBytes, a.stream>>>(m[0], m[1], m[2], m[3], p);
    if (int rc = check_launch("causal attention dk, dv")) return rc;
  }
  if (p.dq == nullptr) return PRISM_OK;
  if (int rc = attn_rows(a, kAttnTile, a.hq, &p.rows)) return rc;
  auto* dq = attn_bwd_dq_kernel<DT, DH>;
  if (int rc = set_max_dynamic_smem(reinterpret_cast<const void*>(dq), DqSmem<DH>::kBytes, "causal attention dq")) return rc;
  dq<<<(unsigned)p.rows.tiles * (unsigned)a.hq, kThreads, DqSmem<DH>::kBytes, a.stream>>>(m[0], m[1], m[2], m[3], p);
  return check_launch("causal attention dq");
}

}  // namespace

int launch_attn_bwd(const AttnArgs& a) {
  if (a.rows == 0) return PRISM_OK;
  DeltaParams d;
  d.o = static_cast<const uint16_t*>(a.o);
  d.d_o = static_cast<const uint16_t*>(a.d_o);
  d.sdo = a.sdo;
  d.delta = a.delta;
  d.heads = a.hq; d.dim = a.dim; d.rows = a.rows;
  d.len = a.cu == nullptr ? a.len : a.rows;
  const long long blocks = ((long long)a.rows * a.hq + 15) / 16;
  if (blocks > 0x7fffffffll) return fail(PRISM_ERR_UNSUPPORTED, "attention: more than 2^35 rows");
  if (a.dtype == DT_BF16) attn_delta_kernel<DT_BF16><<<(unsigned)blocks, 256, 0, a.stream>>>(d);
  else attn_delta_kernel<DT_F16><<<(unsigned)blocks, 256, 0, a.stream>>>(d);
  if (int rc = check_launch("causal attention delta")) return rc;
  BwdParams p;
  p.dq = static_cast<uint16_t*>(a.dq); p.dk = static_cast<uint16_t*>(a.dk); p.dv = static_cast<uint16_t*>(a.dv);
  p.lse = a.lse; p.delta = a.delta;
  p.hq = a.hq; p.hkv = a.hkv; p.group = a.hq / a.hkv; p.dim = a.dim;
  p.c = a.scale * kLog2e; p.scale = a.scale;
  p.err = a.err;
  CUtensorMap m[4];
  if (int rc = attn_tmap(&m[0], a, a.q, a.hq, a.sq)) return rc;
  if (int rc = attn_tmap(&m[1], a, a.k, a.hkv, a.sk)) return rc;
  if (int rc = attn_tmap(&m[2], a, a.v, a.hkv, a.sv)) return rc;
  if (int rc = attn_tmap(&m[3], a, a.d_o, a.hq, a.sdo)) return rc;
  const bool wide = a.dim > 64;
  if (a.dtype == DT_BF16) return wide ? launch_t<DT_BF16, 128>(a, m, p) : launch_t<DT_BF16, 64>(a, m, p);
  return wide ? launch_t<DT_F16, 128>(a, m, p) : launch_t<DT_F16, 64>(a, m, p);
}

}  // namespace prism
