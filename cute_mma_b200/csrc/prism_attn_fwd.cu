// Causal attention, forward: o_i = sum_{j <= i} softmax_j(scale q_i . k_j) v_j for every head of every sequence.
//
// One pass over the keys with a running maximum m and sum l per row (exponents in base 2, c = scale log2 e):
//   S = Q K^T (tcgen05, fp32 in TMEM) -> p = 2^(c s - c m) (registers, one row a thread) -> 16 bits, into TMEM over S
//   -> O += P V (tcgen05, P from TMEM);  O and l are rescaled only when a row's maximum has grown by more than 2^8
// (every p stays below 2^8, exactly representable headroom in both 16-bit types); the end divides by l.
// A CTA owns 256 rows of a head as two 128-row tiles with a warpgroup each: while one warpgroup is in its
// exponentials, the tensor core works on the other's products.  Keys and values pass through one ring of shared tiles.
#include "prism_attn.cuh"
#include "prism_host.cuh"
#include "prism_attn_host.cuh"

namespace prism {
namespace {

struct FwdParams {
  AttnRows rows;
  uint16_t* o;     // rows x heads x dim
  float* lse;      // heads x rows, c m + log2 l per row, or null
  int hq, group, dim;
  float c;         // scale * log2 e
  int* err;
};

constexpr int kThreads = 320;   // two softmax warpgroups, the MMA warp, the TMA warp

template <int DH>
struct FwdSmem {
  static constexpr uint32_t kTile = (DH / 64) * kAttnSub;
  static constexpr int kRing = DH == 128 ? 5 : 10;
  static constexpr uint32_t kBytes = (2 + kRing) * kTile + 1024;
};

struct FwdBars {
  uint64_t q_full[2], s_full[2], p_full[2], o_full[2];
  uint64_t kv_full[10], kv_empty[10];
};

template <int DT, int DH>
__global__ void __launch_bounds__(kThreads, 1)
    attn_fwd_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                    const __grid_constant__ CUtensorMap mv, const FwdParams p) {
  using L = FwdSmem<DH>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ FwdBars bars;
  __shared__ uint32_t tmem_slot;
  __shared__ AttnWork work;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const int head = blockIdx.x % p.hq, kvh = head / p.group;

  if (warp == 0) {
    const AttnWork w = attn_find(p.rows, blockIdx.x / p.hq, 2 * kAttnTile, true);
    if (lane == 0) work = w;
  } else if (warp == 8) {
    tmem_alloc_cta(&tmem_slot, 512);
    tmem_relinquish_cta();
  } else if (warp == 9 && lane == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(&bars.q_full[t], 1);
      mbar_init(&bars.s_full[t], 1);
      mbar_init(&bars.p_full[t], 4);
      mbar_init(&bars.o_full[t], 1);
    }
    for (int s = 0; s < L::kRing; ++s) {
      mbar_init(&bars.kv_full[s], 1);
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
    attn_zero_gap(p.rows, w, p.o, p.hq, head, p.dim);
  } else {
    const int m0 = w.tile * 2 * kAttnTile;
    const int n0 = 2 * w.tile + 1;                                   // key blocks of the first tile ...
    const int n1 = w.len > m0 + kAttnTile ? n0 + 1 : 0;              // ... and of the second, which may be empty
    const int n = max(n0, n1);
    bool ok = true;
    if (warp == 9) {
      if (lane == 0) {
        char* ring = smem + 2 * L::kTile;
        for (int t = 0; t < (n1 ? 2 : 1); ++t) {
          mbar_arrive_expect_tx(&bars.q_full[t], L::kTile);
          attn_load_tile<DH>(smem + t * L::kTile, &mq, &bars.q_full[t], w.row + m0 + t * kAttnTile, head, w.batch);
        }
        Ring r(L::kRing);
        for (int i = 0; i < 2 * n; ++i, r.next()) {
          if (!mbar_wait(&bars.kv_empty[r.idx], r.phase ^ 1)) { ok = false; break; }
          mbar_arrive_expect_tx(&bars.kv_full[r.idx], L::kTile);
          attn_load_tile<DH>(ring + r.idx * L::kTile, (i & 1) ? &mv : &mk, &bars.kv_full[r.idx],
                             w.row + (i >> 1) * kAttnTile, kvh, w.batch);
        }
      }
    } else if (warp == 8) {
      const uint32_t id_s = make_idesc(DT, 128, 128, 0, 0), id_o = make_idesc(DT, 128, DH, 0, 1);
      const uint32_t ring = smem_u32(smem) + 2 * L::kTile;
      Ring rk(L::kRing), rv(L::kRing);
      rv.next();
      auto next2 = [](Ring& r) { r.next(); r.next(); };
      // every lane waits (the warp stays together for the zeros of a last tile), one issues
      if (!warp_wait(&bars.kv_full[0], 0)) ok = false;
      for (int t = 0; ok && t < (n1 ? 2 : 1); ++t) {
        if (!warp_wait(&bars.q_full[t], 0)) { ok = false; break; }
        tc_fence_after_sync();
        if (lane == 0) {
          attn_mma_xyt<DH>(tmem + t * 128, smem_u32(smem) + t * L::kTile, ring, id_s);
          umma_commit_cta(&bars.s_full[t]);
        }
      }
      if (ok && lane == 0) umma_commit_cta(&bars.kv_empty[0]);
      next2(rk);
      for (int j = 0; ok && j < n; ++j) {
        if (!warp_wait(&bars.kv_full[rv.idx], rv.phase)) { ok = false; break; }
        const int valid = w.len - j * kAttnTile;
        if (valid < kAttnTile) attn_zero_tail<DH>(smem + (2 + rv.idx) * L::kTile, valid);
        const int steps = valid >= kAttnTile ? 8 : (valid + 15) >> 4;
        const bool more = j + 1 < n;
        if (more && !warp_wait(&bars.kv_full[rk.idx], rk.phase)) { ok = false; break; }
        for (int t = 0; t < 2; ++t) {
          const int nt = t ? n1 : n0;
          if (j >= nt) continue;
          if (!warp_wait(&bars.p_full[t], j & 1)) { ok = false; break; }
          tc_fence_after_sync();
          if (lane == 0) {
            attn_mma_py<DH>(tmem + 256 + t * DH, tmem + t * 128, 32, ring + rv.idx * L::kTile, id_o, j > 0, steps);
            if (j + 1 == nt) umma_commit_cta(&bars.o_full[t]);
            if (j + 1 < nt) {
              attn_mma_xyt<DH>(tmem + t * 128, smem_u32(smem) + t * L::kTile, ring + rk.idx * L::kTile, id_s);
              umma_commit_cta(&bars.s_full[t]);
            }
          }
        }
        if (!ok) break;
        if (lane == 0) {
          umma_commit_cta(&bars.kv_empty[rv.idx]);
          if (more) umma_commit_cta(&bars.kv_empty[rk.idx]);
        }
        next2(rv);
        next2(rk);
      }
    } else {
      const int t = warp >> 2;
      const int nt = t ? n1 : n0;
      const uint32_t lanes = (uint32_t)(warp & 3) << 21;
      const uint32_t s_addr = tmem + lanes + t * 128, o_addr = tmem + lanes + 256 + t * DH;
      const int r = (warp & 3) * 32 + lane;
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < nt; ++j) {
        if (!warp_wait(&bars.s_full[t], j & 1)) { ok = false; break; }
        tc_fence_after_sync();
        uint32_t s[128];
#pragma unroll
        for (int q = 0; q < 4; ++q) tmem_ld_x32(s_addr + q * 32, *reinterpret_cast<uint32_t(*)[32]>(s + q * 32));
        tmem_ld_wait();
        if (j + 1 == nt) {   // the tile's own rows: keys up to the row itself
#pragma unroll
          for (int e = 0; e < 128; ++e)
            if (e > r) s[e] = 0xff800000u;
        }
        float mx0 = __uint_as_float(s[0]), mx1 = __uint_as_float(s[1]);
#pragma unroll
        for (int e = 2; e < 128; e += 4) {
          mx0 = max3(mx0, __uint_as_float(s[e]), __uint_as_float(s[e + 1]));
          if (e + 3 < 128) mx1 = max3(mx1, __uint_as_float(s[e + 2]), __uint_as_float(s[e + 3]));
        }
        const float mx = max3(m, mx0, mx1);
        // (two rows at -infinity: the difference is NaN and nothing is rescaled, there is nothing yet)
        if (__any_sync(0xffffffffu, (mx - m) * p.c > 8.f)) {
          const float f = ex2((m - (mx == -INFINITY ? 0.f : mx)) * p.c);
          m = mx;
          l *= f;
          if (j > 0) {
#pragma unroll
            for (int q = 0; q < DH / 32; ++q) {
              uint32_t o[32];
              tmem_ld_x32(o_addr + q * 32, o);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st_x32(o_addr + q * 32, o);
            }
          }
        }
        const float2 c2 = make_float2(p.c, p.c);
        const float neg = m == -INFINITY ? 0.f : -m * p.c;
        const float2 n2 = make_float2(neg, neg);
        float l0 = 0.f, l1 = 0.f;
        uint32_t* pk = s;   // pairs land in the first half of the registers
#pragma unroll
        for (int e = 0; e < 128; e += 2) {
          const float2 x = fma2(make_float2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), c2, n2);
          const float a = ex2(x.x), b = ex2(x.y);
          l0 += a;
          l1 += b;
          pk[e >> 1] = Elem<DT>::pack(a, b);
        }
        l += l0 + l1;
        tmem_st_x32(s_addr, pk);
        tmem_st_x32(s_addr + 32, pk + 32);
        tmem_st_wait();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.p_full[t]);
      }
      if (ok && nt > 0) {
        if (warp_wait(&bars.o_full[t], 0)) {
          tc_fence_after_sync();
          const int row = m0 + t * kAttnTile + r;
          const bool mine = row < w.len;
          attn_store_row<DT, DH>(o_addr, 1.f / l, p.o + ((w.orow + row) * p.hq + head) * p.dim, p.dim, mine);
          if (mine && p.lse != nullptr) p.lse[(long long)head * p.rows.rows + w.orow + row] = m * p.c + lg2(l);
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
int launch_t(const AttnArgs& a, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const FwdParams& p) {
  auto* kern = attn_fwd_kernel<DT, DH>;
  if (int rc = set_max_dynamic_smem(reinterpret_cast<const void*>(kern), FwdSmem<DH>::kBytes, "causal attention")) return rc;
  kern<<<(unsigned)p.rows.tiles * (unsigned)a.hq, kThreads, FwdSmem<DH>::kBytes, a.stream>>>(mq, mk, mv, p);
  return check_launch("causal attention");
}

}  // namespace

int launch_attn_fwd(const AttnArgs& a) {
  FwdParams p;
  if (int rc = attn_rows(a, 2 * kAttnTile, a.hq, &p.rows)) return rc;
  if (p.rows.tiles == 0) return PRISM_OK;
  p.o = static_cast<uint16_t*>(a.o);
  p.lse = a.lse;
  p.hq = a.hq; p.group = a.hq / a.hkv; p.dim = a.dim;
  p.c = a.scale * kLog2e;
  p.err = a.err;
  CUtensorMap mq, mk, mv;
  if (int rc = attn_tmap(&mq, a, a.q, a.hq, a.sq)) return rc;
  if (int rc = attn_tmap(&mk, a, a.k, a.hkv, a.sk)) return rc;
  if (int rc = attn_tmap(&mv, a, a.v, a.hkv, a.sv)) return rc;
  const bool wide = a.dim > 64;
  if (a.dtype == DT_BF16)
    return wide ? launch_t<DT_BF16, 128>(a, mq, mk, mv, p) : launch_t<DT_BF16, 64>(a, mq, mk, mv, p);
  return wide ? launch_t<DT_F16, 128>(a, mq, mk, mv, p) : launch_t<DT_F16, 64>(a, mq, mk, mv, p);
}

}  // namespace prism
