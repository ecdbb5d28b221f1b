// Causal attention, backward.  With P_ij = 2^(c q_i.k_j - lse_i), delta_i = do_i . o_i, dP_ij = do_i . v_j and
// dS = P (dP - delta):   dv_j = sum_i P_ij do_i,   dk_j = scale sum_i dS_ij q_i,   dq_i = scale sum_j dS_ij k_j.
//
// Three launches: delta (one pass over o and do), dk + dv by key tiles, dq by query tiles.  S and dP are formed twice
// (seven products of a tile pair instead of five) and in return every sum has one owner: no atomics, no fp32 copy of dq
// to clear and convert, the same bits every run.  A key tile walks through all query heads of its group, so that the
// gradients of shared heads are sums in TMEM as well.
//
// fp16 ends at 2^-24, and P of a row of n keys is about 1/n: P^T carries a factor of 2^15 there (bwd_lift), which dv's store
// takes out again and dS does not get.  dS has a factor of its own, 2^e with |dS| 2^e <= 2^15: |dS_ij| <= |do_i| |v_j - o_i|
// <= 2 max |do| max |v| (o_i lies among the values), and the delta pass, which reads do anyway, takes both maxima.  Unscaled,
// 8192 keys and do of 1e-3 gave dq and dk 1 % off, and do of 1e4 gave infinities.
//
// Measured, bf16, one sequence of 8192 rows, 16 heads: of 128, dk and dv 460 us (tensor pipe 57 % busy: bound by the chain
// S -> P -> dS -> dk of a tile, whose two accumulators leave no TMEM for a second tile), dq 280 us (86 %: bound by the
// tensor pipe); of 64, 335 and 208 us (38 and 46 %: bound by the arithmetic between the products).  delta takes 14 and
// 7 us (fp16, with norms: 27 and 14 us; dk and dv 478 and 355 us).
// Together 742 us, 926 TFLOP/s of the five products that the mathematics needs, and 553 us, 621 TFLOP/s; replayed without a pause,
// under the power cap, 845 and 565 us.
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
  const float* norms;         // fp16: largest squares of the norms of do's and of v's rows (null: dS as it is)
  int* err;
};

// Two warpgroups of arithmetic, and one of the loading warp, the issuing warps and (dk, dv) the warp of the row statistics.
//  256 x 208 + 128 x 88 registers = 384 x 168, what the block is launched with.
constexpr int kThreads = 384, kMathRegs = 208, kOtherRegs = 88;

template <int DT>
__device__ __forceinline__ constexpr float bwd_lift() { return DT == DT_F16 ? 15.f : 0.f; }

// e of dS's factor 2^e.  Norms of zero leave nothing to scale; 40 is as good as any.
template <int DT>
__device__ __forceinline__ int ds_exponent(const float* norms) {
  if (DT != DT_F16 || norms == nullptr) return 0;
  const float e = floorf(13.99f - 0.5f * (lg2(__ldg(norms)) + lg2(__ldg(norms + 1))));
  return (int)fminf(fmaxf(e, -40.f), 40.f);
}

// ---------------------------------------------------------------------------------------------------- delta
// LANES lanes (8 for heads of up to 64, 16 for wider ones) have 16-byte pieces of a row's o and do, and 8 bytes of what o's
// rounding took, for kDeltaHeads heads one after the other.  An error of delta is one of every dS of its row with the same sign,
// which no sum over the keys averages out: with o as rounded alone dq was 0.0025 off (relative norm, 1024 rows, heads of 64,
// bf16), with the rest 0.0024, of which 0.0023 is the rounding of dS.  16 x 1024 rows, 12 heads of 64: 25 us with a division for
// every 16 bytes; now, with norms, 19 us (and one of the clearing before it).
constexpr int kDeltaHeads = 4;
struct DeltaParams {
  const uint16_t *o, *d_o;
  const uint8_t* low;
  AttnStrides sdo;
  float* delta;
  int heads, dim, len, rows;   // len: rows per batch entry
  unsigned groups, all_groups;   // of heads: of o, and of o and (NORMS) v behind them
  const uint16_t* v;             // NORMS
  AttnStrides sv;
  const int* cu;
  int n, kv_heads;
  float* norms;
};

// The largest of a block's squared norms to *most.
__device__ __forceinline__ void attn_largest(float sq, float* most) {
  __shared__ float red[8];
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) sq = fmaxf(sq, __shfl_xor_sync(0xffffffffu, sq, d));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = sq;
  __syncthreads();
  if (threadIdx.x != 0) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) sq = fmaxf(sq, red[i]);
  // (bits of floats that are not negative are in their order; a maximum does not depend on the order that it is taken in)
  if (sq > __ldcg(most)) atomicMax(reinterpret_cast<int*>(most), __float_as_int(sq));
}

template <int DT, bool NORMS, int LANES>
__global__ void __launch_bounds__(256) attn_delta_kernel(const DeltaParams p) {
  const int piece = threadIdx.x & (LANES - 1);
  const unsigned block = blockIdx.x / p.all_groups;
  unsigned group = blockIdx.x - block * p.all_groups;
  const int row = (int)(block * (256 / LANES) + threadIdx.x / LANES);
  const bool values = NORMS && group >= p.groups;
  if (values) group -= p.groups;
  const int heads = values ? p.kv_heads : p.heads, head0 = (int)group * kDeltaHeads;
  const bool there = row < p.rows, inside = there && piece * 8 < p.dim;
  const int b = there ? row / p.len : 0;
  const AttnStrides& st = values ? p.sv : p.sdo;
  const uint16_t* y0 = (values ? p.v : p.d_o) + b * st.batch + (long long)(row - b * p.len) * st.row + piece * 8;
  const long long at0 = (long long)row * p.heads * p.dim + piece * 8;
  uint4 x[kDeltaHeads], y[kDeltaHeads];
  uint2 z[kDeltaHeads];
#pragma unroll
  for (int h = 0; h < kDeltaHeads; ++h) {
    const bool live = inside && head0 + h < heads;
    x[h] = y[h] = make_uint4(0u, 0u, 0u, 0u);
    z[h] = make_uint2(0u, 0u);
    if (!live) continue;
    y[h] = *reinterpret_cast<const uint4*>(y0 + (head0 + h) * st.head);
    if (values) continue;
    const long long at = at0 + (long long)(head0 + h) * p.dim;
    x[h] = *reinterpret_cast<const uint4*>(p.o + at);
    if (p.low != nullptr) z[h] = *reinterpret_cast<const uint2*>(p.low + at);
  }
  float most = 0.f;
#pragma unroll
  for (int h = 0; h < kDeltaHeads; ++h) {
    const uint32_t xs[4] = {x[h].x, x[h].y, x[h].z, x[h].w}, ys[4] = {y[h].x, y[h].y, y[h].z, y[h].w};
    float sum = 0.f, sq = 0.f, rest = 0.f, f[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 a = Elem<DT>::unpack(xs[e]), g = Elem<DT>::unpack(ys[e]);
      sum = fmaf(a.x, g.x, fmaf(a.y, g.y, sum));
      if ((e & 1) == 0) unpack_e5m2(e == 0 ? z[h].x : z[h].y, f);
      rest = fmaf(f[(e & 1) * 2], g.x, fmaf(f[(e & 1) * 2 + 1], g.y, rest));
      if (NORMS) sq = fmaf(g.x, g.x, fmaf(g.y, g.y, sq));
    }
    if (p.low != nullptr) sum = fmaf(rest, 1.f / low_scale<DT>(), sum);
#pragma unroll
    for (int d = LANES / 2; d > 0; d >>= 1) {
      sum += __shfl_xor_sync(0xffffffffu, sum, d);
      if (NORMS) sq += __shfl_xor_sync(0xffffffffu, sq, d);
    }
    if (!values && there && piece == 0 && head0 + h < heads) p.delta[(long long)(head0 + h) * p.rows + row] = sum;
    // (a row that is not finite does not count: what it gives is not either)
    if (NORMS && isfinite(sq)) most = fmaxf(most, sq);
  }
  if constexpr (NORMS) {
    // rows of no sequence do not count
    const int front = p.cu == nullptr ? 0 : attn_clamp(__ldg(p.cu), 0, p.rows);
    const int end = p.cu == nullptr ? p.rows : attn_clamp(__ldg(p.cu + p.n), front, p.rows);
    attn_largest(row >= front && row < end ? most : 0.f, p.norms + values);
  }
}

template <int DT, bool NORMS>
int launch_delta(DeltaParams d, cudaStream_t stream) {
  const int lanes = d.dim <= 64 ? 8 : 16;
  d.groups = ((unsigned)d.heads + kDeltaHeads - 1) / kDeltaHeads;
  d.all_groups = d.groups + (NORMS ? ((unsigned)d.kv_heads + kDeltaHeads - 1) / kDeltaHeads : 0u);
  const long long blocks = ((long long)d.rows + 256 / lanes - 1) / (256 / lanes) * d.all_groups;
  if (blocks > 0x7fffffffll) return fail(PRISM_ERR_UNSUPPORTED, "attention: more than 2^31 blocks of rows and heads");
  if (NORMS) {
    const cudaError_t e = cudaMemsetAsync(d.norms, 0, 2 * sizeof(float), stream);
    if (e != cudaSuccess) return fail(PRISM_ERR_CUDA, "causal attention delta: %s", cudaGetErrorString(e));
  }
  if (lanes == 8) attn_delta_kernel<DT, NORMS, 8><<<(unsigned)blocks, 256, 0, stream>>>(d);
  else attn_delta_kernel<DT, NORMS, 16><<<(unsigned)blocks, 256, 0, stream>>>(d);
  return check_launch("causal attention delta");
}

// ---------------------------------------------------------------------------------------------------- dk, dv
// Transposed scores: S^T = K Q^T and dP^T = V dO^T have a key row per TMEM lane, so that P^T and dS^T, written back over
// them in 16 bits, are the TMEM operands of dv += P^T dO and dk += dS^T Q.  The row statistics lie along the columns and
// are read from shared memory, the same word by all lanes.  Rows behind the sequence get lse = +infinity: P = 0.
// Each warpgroup has 64 of the 128 query columns.  P goes over in two pieces of 32 columns of each, so that dv's product
// starts in the middle of the exponentials.  Heads of up to 64 leave TMEM for a second S buffer: the next scores are then
// formed beside this tile's exponentials; wider heads form them behind dv's product, which frees S.
template <int DH>
struct DkvSmem {
  static constexpr uint32_t kTile = (DH / 64) * kAttnSub;
  static constexpr int kKv = DH == 128 ? 1 : 2;   // pairs of K and V tiles: the next work's beside this one's
  static constexpr int kQ = DH == 128 ? 2 : 4, kDo = DH == 128 ? 3 : 4;   // rings of Q and of dO tiles
  static constexpr uint32_t kBytes = (2 * kKv + kQ + kDo) * kTile + 1024;
};
// (Barriers in pairs, used in turn: where one side may be a whole tile ahead of the other, a single one could complete
// twice before it is looked at.  P of tile i + 2 needs scores that are issued behind the wait for P of tile i.)
struct DkvBars {
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2][2], dp_full, ds_full, acc_full, acc_empty, st_full, st_empty, clean[2];
  uint64_t q_full[4], q_empty[4], do_full[4], do_empty[4];
};

template <int DT, int DH>
__global__ void __launch_bounds__(kThreads, 1)
    attn_bwd_dkv_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                        const __grid_constant__ CUtensorMap mv, const __grid_constant__ CUtensorMap mdo, const BwdParams p) {
  using L = DkvSmem<DH>;
  constexpr bool kEarly = DH == 64;
  constexpr uint32_t kDp = kEarly ? 256 : 128, kDv = kDp + 128, kDk = kDv + DH;
  extern __shared__ uint8_t smem_raw[];
  __shared__ DkvBars bars;
  __shared__ AttnSched sched;
  __shared__ uint32_t tmem_slot;
  __shared__ __align__(16) float st_lse[kAttnTile], st_delta[kAttnTile];   // negated; with P's factor, and with what dS's is beyond it
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);

  if (warp == 8) {
    tmem_alloc_cta(&tmem_slot, 512);
    tmem_relinquish_cta();
  } else if (warp == 9 && lane == 0) {
    attn_sched_init(sched, 11);
    mbar_init(&bars.clean[0], 1);
    mbar_init(&bars.clean[1], 1);
    mbar_init(&bars.dp_full, 1);
    mbar_init(&bars.ds_full, 8);
    mbar_init(&bars.acc_full, 2);
    mbar_init(&bars.acc_empty, 8);
    mbar_init(&bars.st_full, 1);
    mbar_init(&bars.st_empty, 8);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bars.k_full[s], 1);
      mbar_init(&bars.k_empty[s], 1);
      mbar_init(&bars.v_full[s], 1);
      mbar_init(&bars.v_empty[s], 1);
      mbar_init(&bars.s_full[s], 1);
      mbar_init(&bars.p_full[s][0], 8);
      mbar_init(&bars.p_full[s][1], 8);
    }
    for (int s = 0; s < 4; ++s) {
      mbar_init(&bars.q_full[s], 1);
      mbar_init(&bars.q_empty[s], 1);
      mbar_init(&bars.do_full[s], 1);
      mbar_init(&bars.do_empty[s], 2);
    }
    fence_mbar_init();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);   // (known to be the same in all lanes)
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // (dq's CTAs may follow where SMs run out of this work)
  bool ok = true;
  AttnWork w;
  int kvh;
  Ring rw(2);
  auto q_tiles = [](const AttnWork& g) { return (g.len + kAttnTile - 1) / kAttnTile - g.tile; };   // of a head, from the diagonal on

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == 9) {
      char *q_ring = smem + 2 * L::kKv * L::kTile, *do_ring = q_ring + L::kQ * L::kTile;
      Ring rq(L::kQ), rd(L::kDo), rkv(L::kKv);
      ok = attn_schedule(
          sched, p.rows, p.hkv, kAttnTile, false,
          [&](const AttnWork& g, int h) {
            const int nq = q_tiles(g), n = nq * p.group;
            const int krow = g.row + g.tile * kAttnTile;
            if (!warp_wait(&bars.k_empty[rkv.idx], rkv.phase ^ 1)) return false;
            if (lane == 0) {
              mbar_arrive_expect_tx(&bars.k_full[rkv.idx], L::kTile);
              attn_load_tile<DH>(smem + 2 * rkv.idx * L::kTile, &mk, &bars.k_full[rkv.idx], krow, h, g.batch);
            }
            int head = h * p.group, i = 0;
            for (int it = 0; it < n; ++it, rq.next(), rd.next()) {
              const int row = g.row + (g.tile + i) * kAttnTile;
              if (!warp_wait(&bars.q_empty[rq.idx], rq.phase ^ 1)) return false;
              if (lane == 0) {
                mbar_arrive_expect_tx(&bars.q_full[rq.idx], L::kTile);
                attn_load_tile<DH>(q_ring + rq.idx * L::kTile, &mq, &bars.q_full[rq.idx], row, head, g.batch);
              }
              if (it == 0) {   // (V is given back later than K, and wanted later)
                if (!warp_wait(&bars.v_empty[rkv.idx], rkv.phase ^ 1)) return false;
                if (lane == 0) {
                  mbar_arrive_expect_tx(&bars.v_full[rkv.idx], L::kTile);
                  attn_load_tile<DH>(smem + (2 * rkv.idx + 1) * L::kTile, &mv, &bars.v_full[rkv.idx], krow, h, g.batch);
                }
              }
              if (!warp_wait(&bars.do_empty[rd.idx], rd.phase ^ 1)) return false;
              if (lane == 0) {
                mbar_arrive_expect_tx(&bars.do_full[rd.idx], L::kTile);
                attn_load_tile<DH>(do_ring + rd.idx * L::kTile, &mdo, &bars.do_full[rd.idx], row, head, g.batch);
              }
              if (++i == nq) { i = 0; ++head; }
            }
            rkv.next();
            return true;
          },
          [&](const AttnWork& g, int h) {
            attn_zero_gap(p.rows, g, p.dk, p.hkv, h, p.dim);
            attn_zero_gap(p.rows, g, p.dv, p.hkv, h, p.dim);
          });
    } else if (warp == 10) {
      // the row statistics; and a sequence's last tiles are cleaned behind its end before any product reads them
      Ring rq(L::kQ), rd(L::kDo);
      uint32_t cnt = 0, cleaned = 0;
      const float drop = pow2i(ds_exponent<DT>(p.norms) - (int)bwd_lift<DT>());
      while (ok && attn_next(sched, rw, &w, &kvh, &ok)) {
        const int nq = q_tiles(w), n = nq * p.group;
        int head = kvh * p.group, i = 0;
        for (int it = 0; it < n; ++it, ++cnt, rq.next(), rd.next()) {
          const long long at = (long long)head * p.rows.rows + w.orow;
          float a[4], b[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int row = (w.tile + i) * kAttnTile + e * 32 + lane;
            a[e] = row < w.len ? bwd_lift<DT>() - __ldg(p.lse + at + row) : -INFINITY;
            b[e] = row < w.len ? -__ldg(p.delta + at + row) * drop : 0.f;
          }
          const int valid = w.len - (w.tile + i) * kAttnTile;
          if (valid < kAttnTile) {
            if (!warp_wait(&bars.q_full[rq.idx], rq.phase) || !warp_wait(&bars.do_full[rd.idx], rd.phase)) { ok = false; break; }
            attn_zero_tail<DH>(smem + (2 * L::kKv + rq.idx) * L::kTile, valid);
            attn_zero_tail<DH>(smem + (2 * L::kKv + L::kQ + rd.idx) * L::kTile, valid);
            if (lane == 0) mbar_arrive(&bars.clean[cleaned & 1]);   // (two: this warp may be a tile ahead of those that wait)
            ++cleaned;
          }
          if (!warp_wait(&bars.st_empty, (cnt & 1) ^ 1)) { ok = false; break; }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            st_lse[e * 32 + lane] = a[e];
            st_delta[e * 32 + lane] = b[e];
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars.st_full);
          if (++i == nq) { i = 0; ++head; }
        }
      }
    } else {
      // two issuing warps, because a product costs its issuer about as long as the tensor core and every barrier more:
      // warp 8 has S and dv, whose order on one thread protects S and P in the same columns, warp 11 dP and dk likewise
      const bool dk_side = warp == 11;
      const uint32_t id_s = make_idesc(DT, 128, 128, 0, 0), id_o = make_idesc(DT, 128, DH, 0, 1);
      const uint32_t kv = smem_u32(smem), q_ring = kv + 2 * L::kKv * L::kTile, do_ring = q_ring + L::kQ * L::kTile;
      Ring rq(L::kQ), rd(L::kDo), rkv(L::kKv);
      uint32_t used = 0, cnt = 0, cleaned = 0;   // pieces of work; query tiles of all of them, and those that were cleaned
      // a tile of one of the rings is there, and clean behind the sequence
      auto arrived = [&](uint64_t* full, uint32_t phase, int i) {
        if (!warp_wait(full, phase)) return false;
        if (w.len - (w.tile + i) * kAttnTile < kAttnTile) {
          if (!warp_wait(&bars.clean[cleaned & 1], (cleaned >> 1) & 1)) return false;
          ++cleaned;
        }
        tc_fence_after_sync();
        return true;
      };
      auto scores = [&](Ring& r, int i, uint32_t c, bool first, bool last) {
        if ((kEarly || first) && !arrived(&bars.q_full[r.idx], r.phase, i)) return false;
        if (elect_one()) {
          const uint32_t b = kEarly ? (c & 1) : 0;
          attn_mma_xyt<DH>(tmem + b * 128, kv + 2 * rkv.idx * L::kTile, q_ring + r.idx * L::kTile, id_s);
          umma_commit_cta(&bars.s_full[b]);
          if (last) umma_commit_cta(&bars.k_empty[rkv.idx]);
        }
        return true;
      };
      auto dprobs = [&](Ring& r, int i, bool last) {
        if (!arrived(&bars.do_full[r.idx], r.phase, i)) return false;
        if (elect_one()) {
          attn_mma_xyt<DH>(tmem + kDp, kv + (2 * rkv.idx + 1) * L::kTile, do_ring + r.idx * L::kTile, id_s);
          umma_commit_cta(&bars.dp_full);
          umma_commit_cta(&bars.do_empty[r.idx]);
          if (last) umma_commit_cta(&bars.v_empty[rkv.idx]);
        }
        return true;
      };
      while (ok && attn_next(sched, rw, &w, &kvh, &ok)) {
        const int nq = q_tiles(w), n = nq * p.group;
        int i = 0;
        ok = dk_side ? warp_wait(&bars.v_full[rkv.idx], rkv.phase) && dprobs(rd, 0, n == 1)
                     : warp_wait(&bars.k_full[rkv.idx], rkv.phase) && scores(rq, 0, cnt, true, n == 1);
        for (int it = 0; ok && it < n; ++it, ++cnt) {
          const int valid = w.len - (w.tile + i) * kAttnTile;
          const int steps = valid >= kAttnTile ? 8 : (valid + 15) >> 4;
          Ring nrq = rq, nrd = rd;
          nrq.next();
          nrd.next();
          if (++i == nq) i = 0;
          const bool more = it + 1 < n;
          if (dk_side) {
            if (it == 0 && !warp_wait(&bars.acc_empty, (used & 1) ^ 1)) { ok = false; break; }
            if (!warp_wait(&bars.ds_full, cnt & 1)) { ok = false; break; }
            tc_fence_after_sync();
            if (elect_one()) {
              attn_mma_py<DH>(tmem + kDk, tmem + kDp, 64, q_ring + rq.idx * L::kTile, id_o, it > 0, steps);
              umma_commit_cta(&bars.q_empty[rq.idx]);
              if (!more) umma_commit_cta(&bars.acc_full);
            }
            if (more && !dprobs(nrd, i, it + 2 == n)) { ok = false; break; }
          } else {
            if (kEarly && more && !scores(nrq, i, cnt + 1, false, it + 2 == n)) { ok = false; break; }
            const uint32_t dot = do_ring + rd.idx * L::kTile, pt = tmem + (kEarly ? (cnt & 1) * 128 : 0);
            if (it == 0 && !warp_wait(&bars.acc_empty, (used & 1) ^ 1)) { ok = false; break; }
            if (!warp_wait(&bars.do_full[rd.idx], rd.phase)) { ok = false; break; }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              // (the next scores' operands are looked for while the second piece is on its way)
              if (c == 1 && !kEarly && more && !arrived(&bars.q_full[nrq.idx], nrq.phase, i)) { ok = false; break; }
              if (!warp_wait(&bars.p_full[cnt & 1][c], (cnt >> 1) & 1)) { ok = false; break; }
              tc_fence_after_sync();
              if (elect_one())
#pragma unroll
                for (int h = 0; h < 2; ++h)
                  if (h * 4 + c * 2 < steps)
                    attn_mma_py<DH>(tmem + kDv, pt + h * 64 + c * 16, 0, dot + (h * 4 + c * 2) * 2048, id_o,
                                    it > 0 || c > 0 || h > 0, min(2, steps - h * 4 - c * 2));
            }
            if (!ok) break;
            if (elect_one()) {
              umma_commit_cta(&bars.do_empty[rd.idx]);
              if (!more) umma_commit_cta(&bars.acc_full);
            }
            if (!kEarly && more && !scores(nrq, i, cnt + 1, false, it + 2 == n)) { ok = false; break; }
          }
          rq = nrq;
          rd = nrd;
        }
        rkv.next();
        ++used;
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kMathRegs));
    const int half = warp >> 2;   // which 64 query columns
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;
    const uint32_t dp_addr = tmem + lanes + kDp + half * 64;
    const int key = (warp & 3) * 32 + lane;
    const int raised = ds_exponent<DT>(p.norms);
    const float2 c2 = both(p.c), drop2 = both(pow2i(raised - (int)bwd_lift<DT>()));
    const float4* lse = reinterpret_cast<const float4*>(st_lse + half * 64);
    const float4* del = reinterpret_cast<const float4*>(st_delta + half * 64);
    uint32_t cnt = 0, used = 0;
    while (ok && attn_next(sched, rw, &w, &kvh, &ok)) {
      const int nq = q_tiles(w), n = nq * p.group;
      int i = 0;
      for (int it = 0; it < n; ++it, ++cnt) {
        const bool diag = i == 0;
        if (++i == nq) i = 0;
        const uint32_t b = kEarly ? (cnt & 1) : 0;
        const uint32_t s_addr = tmem + lanes + b * 128 + half * 64;
        if (!warp_wait(&bars.st_full, cnt & 1) || !warp_wait(&bars.s_full[b], kEarly ? (cnt >> 1) & 1 : cnt & 1)) { ok = false; break; }
        tc_fence_after_sync();
        uint32_t s[64], pk[32];
        tmem_ld_x32(s_addr, *reinterpret_cast<uint32_t(*)[32]>(s));
        tmem_ld_x32(s_addr + 32, *reinterpret_cast<uint32_t(*)[32]>(s + 32));
        tmem_ld_wait();
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int e = c * 32; e < c * 32 + 32; e += 4) {
            const float4 z = lse[e >> 2];
            const float2 x = fma2(make_float2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), c2, make_float2(z.x, z.y));
            const float2 y = fma2(make_float2(__uint_as_float(s[e + 2]), __uint_as_float(s[e + 3])), c2, make_float2(z.z, z.w));
            s[e] = __float_as_uint(ex2(x.x));
            s[e + 1] = __float_as_uint(ex2(x.y));
            float2 q;
            if (e & 4) q = ex2_poly2(y);
            else q = make_float2(ex2(y.x), ex2(y.y));
            s[e + 2] = __float_as_uint(q.x);
            s[e + 3] = __float_as_uint(q.y);
          }
          if (diag) {
#pragma unroll
            for (int e = c * 32; e < c * 32 + 32; ++e)
              if (half * 64 + e < key) s[e] = 0u;
          }
#pragma unroll
          for (int e = c * 32; e < c * 32 + 32; e += 2)
            pk[e >> 1] = Elem<DT>::pack(__uint_as_float(s[e]), __uint_as_float(s[e + 1]));
          tmem_st_x16(s_addr + c * 16, pk + c * 16);
          tmem_st_wait();
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars.p_full[cnt & 1][c]);
        }
        if (!warp_wait(&bars.dp_full, cnt & 1)) { ok = false; break; }
        tc_fence_after_sync();
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t dp[32];
          tmem_ld_x32(dp_addr + c * 32, dp);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            const float4 z = del[(c * 32 + e) >> 2];
            float2 x = make_float2(__uint_as_float(dp[e]), __uint_as_float(dp[e + 1]));
            float2 y = make_float2(__uint_as_float(dp[e + 2]), __uint_as_float(dp[e + 3]));
            x = DT == DT_F16 ? fma2(x, drop2, make_float2(z.x, z.y)) : add2(x, make_float2(z.x, z.y));
            y = DT == DT_F16 ? fma2(y, drop2, make_float2(z.z, z.w)) : add2(y, make_float2(z.z, z.w));
            x = mul2(x, make_float2(__uint_as_float(s[c * 32 + e]), __uint_as_float(s[c * 32 + e + 1])));
            y = mul2(y, make_float2(__uint_as_float(s[c * 32 + e + 2]), __uint_as_float(s[c * 32 + e + 3])));
            dp[e] = __float_as_uint(x.x); dp[e + 1] = __float_as_uint(x.y);
            dp[e + 2] = __float_as_uint(y.x); dp[e + 3] = __float_as_uint(y.y);
          }
          if (diag) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (half * 64 + c * 32 + e < key) dp[e] = 0u;
          }
#pragma unroll
          for (int e = 0; e < 32; e += 2)
            pk[(c * 32 + e) >> 1] = Elem<DT>::pack(__uint_as_float(dp[e]), __uint_as_float(dp[e + 1]));
        }
        tmem_st_x32(dp_addr, pk);
        tmem_st_wait();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&bars.st_empty);
          mbar_arrive(&bars.ds_full);
        }
      }
      if (!ok) break;
      if (!warp_wait(&bars.acc_full, used & 1)) { ok = false; break; }
      ++used;
      tc_fence_after_sync();
      const int row0 = w.tile * kAttnTile + key - lane;
      const long long at = ((w.orow + row0) * p.hkv + kvh) * p.dim, step = (long long)p.hkv * p.dim;
      if (half == 0) attn_store_rows<DT, DH, false>(tmem + lanes + kDv, pow2i(-(int)bwd_lift<DT>()), p.dv + at, nullptr, step, p.dim, w.len - row0);
      else attn_store_rows<DT, DH, false>(tmem + lanes + kDk, p.scale * pow2i(-raised), p.dk + at, nullptr, step, p.dim, w.len - row0);
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.acc_empty);
    }
  }
  if (!ok && lane == 0) atomicExch(p.err, PRISM_ERR_DEVICE_WAIT);
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 8) tmem_dealloc_cta(tmem, 512);
}

// ---------------------------------------------------------------------------------------------------- dq
// A query tile stays, key and value tiles stream by.  S has one buffer, free again as soon as it is in registers; dP, over
// which dS is written for dq += dS K, has two: the next tile's scores and dP are formed while the warpgroups (64 key
// columns each) work on this one's.
template <int DH>
struct DqSmem {
  static constexpr uint32_t kTile = (DH / 64) * kAttnSub;
  static constexpr int kK = DH == 128 ? 3 : 4, kV = DH == 128 ? 2 : 4;   // rings of K and of V tiles
  static constexpr int kQ = DH == 128 ? 1 : 2;   // pairs of Q and dO tiles: the next work's beside this one's
  static constexpr uint32_t kBytes = (2 * kQ + kK + kV) * kTile + 1024;
};
struct DqBars {
  uint64_t q_full[2], q_empty[2], do_full[2], do_empty[2], s_full, s_read, dp_full[2], ds_full[2], ds_empty[2], acc_full, acc_empty;
  uint64_t k_full[4], k_empty[4], v_full[4], v_empty[4];
};

template <int DT, int DH>
__global__ void __launch_bounds__(kThreads, 1)
    attn_bwd_dq_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                       const __grid_constant__ CUtensorMap mv, const __grid_constant__ CUtensorMap mdo, const BwdParams p) {
  using L = DqSmem<DH>;
  constexpr uint32_t kDp = 128, kDq = 384;
  extern __shared__ uint8_t smem_raw[];
  __shared__ DqBars bars;
  __shared__ AttnSched sched;
  __shared__ uint32_t tmem_slot;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);

  if (warp == 8) {
    tmem_alloc_cta(&tmem_slot, 512);
    tmem_relinquish_cta();
  } else if (warp == 9 && lane == 0) {
    attn_sched_init(sched, 11);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bars.q_full[s], 1);
      mbar_init(&bars.q_empty[s], 1);
      mbar_init(&bars.do_full[s], 1);
      mbar_init(&bars.do_empty[s], 1);
    }
    mbar_init(&bars.ds_empty[0], 1);
    mbar_init(&bars.ds_empty[1], 1);
    mbar_init(&bars.s_full, 1);
    mbar_init(&bars.s_read, 8);
    mbar_init(&bars.ds_full[0], 8);
    mbar_init(&bars.ds_full[1], 8);
    mbar_init(&bars.acc_full, 1);
    mbar_init(&bars.acc_empty, 8);
    mbar_init(&bars.dp_full[0], 1);
    mbar_init(&bars.dp_full[1], 1);
    for (int s = 0; s < 4; ++s) {
      mbar_init(&bars.k_full[s], 1);
      mbar_init(&bars.k_empty[s], 1);
      mbar_init(&bars.v_full[s], 1);
      mbar_init(&bars.v_empty[s], 1);
    }
    fence_mbar_init();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);   // (known to be the same in all lanes)
  bool ok = true;
  AttnWork w;
  int head;
  Ring rw(2);

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    const uint32_t id_s = make_idesc(DT, 128, 128, 0, 0), id_o = make_idesc(DT, 128, DH, 0, 1);
    const uint32_t sq = smem_u32(smem), k_ring = sq + 2 * L::kQ * L::kTile, v_ring = k_ring + L::kK * L::kTile;
    uint32_t used = 0, cnt = 0;   // pieces of work, key tiles of all of them
    Ring rq(L::kQ);
    if (warp == 9) {
      Ring rk(L::kK), rv(L::kV);
      ok = attn_schedule(
          sched, p.rows, p.hq, kAttnTile, true,
          [&](const AttnWork& g, int h) {
            const int kvh = h / p.group;
            const int row = g.row + g.tile * kAttnTile;
            if (!warp_wait(&bars.q_empty[rq.idx], rq.phase ^ 1)) return false;
            if (lane == 0) {
              mbar_arrive_expect_tx(&bars.q_full[rq.idx], L::kTile);
              attn_load_tile<DH>(smem + 2 * rq.idx * L::kTile, &mq, &bars.q_full[rq.idx], row, h, g.batch);
            }
            for (int j = 0; j <= g.tile; ++j, rk.next(), rv.next()) {
              if (!warp_wait(&bars.k_empty[rk.idx], rk.phase ^ 1)) return false;
              if (lane == 0) {
                mbar_arrive_expect_tx(&bars.k_full[rk.idx], L::kTile);
                attn_load_tile<DH>(smem + (2 * L::kQ + rk.idx) * L::kTile, &mk, &bars.k_full[rk.idx], g.row + j * kAttnTile, kvh, g.batch);
              }
              if (j == 0) {
                if (!warp_wait(&bars.do_empty[rq.idx], rq.phase ^ 1)) return false;
                if (lane == 0) {
                  mbar_arrive_expect_tx(&bars.do_full[rq.idx], L::kTile);
                  attn_load_tile<DH>(smem + (2 * rq.idx + 1) * L::kTile, &mdo, &bars.do_full[rq.idx], row, h, g.batch);
                }
              }
              if (!warp_wait(&bars.v_empty[rv.idx], rv.phase ^ 1)) return false;
              if (lane == 0) {
                mbar_arrive_expect_tx(&bars.v_full[rv.idx], L::kTile);
                attn_load_tile<DH>(smem + (2 * L::kQ + L::kK + rv.idx) * L::kTile, &mv, &bars.v_full[rv.idx], g.row + j * kAttnTile,
                                   kvh, g.batch);
              }
            }
            rq.next();
            return true;
          },
          [&](const AttnWork& g, int h) { attn_zero_gap(p.rows, g, p.dq, p.hq, h, p.dim); });
    } else if (warp == 8) {   // S (three issuing warps: a product costs its issuer about as long as the tensor core)
      Ring r(L::kK);
      while (ok && attn_next(sched, rw, &w, &head, &ok)) {
        ok = warp_wait(&bars.q_full[rq.idx], rq.phase);
        for (int j = 0; ok && j <= w.tile; ++j, ++cnt, r.next()) {
          if (!warp_wait(&bars.k_full[r.idx], r.phase)) { ok = false; break; }
          const int valid = w.len - j * kAttnTile;
          if (valid < kAttnTile) attn_zero_tail<DH>(smem + (2 * L::kQ + r.idx) * L::kTile, valid);   // for dq's product
          if (!warp_wait(&bars.s_read, (cnt & 1) ^ 1)) { ok = false; break; }
          tc_fence_after_sync();
          if (elect_one()) {
            attn_mma_xyt<DH>(tmem, sq + 2 * rq.idx * L::kTile, k_ring + r.idx * L::kTile, id_s);
            umma_commit_cta(&bars.s_full);
            if (j == w.tile) umma_commit_cta(&bars.q_empty[rq.idx]);
          }
        }
        rq.next();
      }
    } else if (warp == 10) {   // dP
      Ring r(L::kV);
      while (ok && attn_next(sched, rw, &w, &head, &ok)) {
        ok = warp_wait(&bars.do_full[rq.idx], rq.phase);
        for (int j = 0; ok && j <= w.tile; ++j, ++cnt, r.next()) {
          if (!warp_wait(&bars.v_full[r.idx], r.phase)) { ok = false; break; }
          // dS of two tiles ago, in the same columns, has gone into dq
          if (!warp_wait(&bars.ds_empty[cnt & 1], ((cnt >> 1) & 1) ^ 1)) { ok = false; break; }
          tc_fence_after_sync();
          if (elect_one()) {
            attn_mma_xyt<DH>(tmem + kDp + (cnt & 1) * 128, sq + (2 * rq.idx + 1) * L::kTile, v_ring + r.idx * L::kTile, id_s);
            umma_commit_cta(&bars.dp_full[cnt & 1]);
            umma_commit_cta(&bars.v_empty[r.idx]);
            if (j == w.tile) umma_commit_cta(&bars.do_empty[rq.idx]);
          }
        }
        rq.next();
      }
    } else {   // dq
      Ring r(L::kK);
      while (ok && attn_next(sched, rw, &w, &head, &ok)) {
        ok = warp_wait(&bars.acc_empty, (used & 1) ^ 1);
        ++used;
        for (int j = 0; ok && j <= w.tile; ++j, ++cnt, r.next()) {
          if (!warp_wait(&bars.ds_full[cnt & 1], (cnt >> 1) & 1)) { ok = false; break; }
          tc_fence_after_sync();
          const int valid = w.len - j * kAttnTile;
          if (elect_one()) {
            attn_mma_py<DH>(tmem + kDq, tmem + kDp + (cnt & 1) * 128, 64, k_ring + r.idx * L::kTile, id_o, j > 0,
                            valid >= kAttnTile ? 8 : (valid + 15) >> 4);
            umma_commit_cta(&bars.k_empty[r.idx]);
            umma_commit_cta(&bars.ds_empty[cnt & 1]);
            if (j == w.tile) umma_commit_cta(&bars.acc_full);
          }
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kMathRegs));
    const int half = warp >> 2;   // which 64 key columns
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;
    const uint32_t s_addr = tmem + lanes + half * 64;
    const int r = (warp & 3) * 32 + lane;
    const float2 c2 = both(p.c);
    const int raised = ds_exponent<DT>(p.norms);
    uint32_t cnt = 0, used = 0;
    while (ok && attn_next(sched, rw, &w, &head, &ok)) {
      const int n = w.tile + 1, row = w.tile * kAttnTile + r;
      const bool mine = row < w.len;
      const long long at = (long long)head * p.rows.rows + w.orow + row;
      const float2 n2 = both(mine ? (float)raised - __ldg(p.lse + at) : -INFINITY), d2 = both(mine ? -__ldg(p.delta + at) : 0.f);
      for (int j = 0; j < n; ++j, ++cnt) {
        if (!warp_wait(&bars.s_full, cnt & 1)) { ok = false; break; }
        tc_fence_after_sync();
        uint32_t s[64];
        tmem_ld_x32(s_addr, *reinterpret_cast<uint32_t(*)[32]>(s));
        tmem_ld_x32(s_addr + 32, *reinterpret_cast<uint32_t(*)[32]>(s + 32));
        tmem_ld_wait();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.s_read);
#pragma unroll
        for (int e = 0; e < 64; e += 2) {
          const float2 x = fma2(make_float2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), c2, n2);
          float2 q;
          if ((e / 2) % 4 == 3) q = ex2_poly2(x);
          else q = make_float2(ex2(x.x), ex2(x.y));
          s[e] = __float_as_uint(q.x);
          s[e + 1] = __float_as_uint(q.y);
        }
        if (!warp_wait(&bars.dp_full[cnt & 1], (cnt >> 1) & 1)) { ok = false; break; }
        tc_fence_after_sync();
        const uint32_t dp_addr = tmem + lanes + kDp + (cnt & 1) * 128 + half * 64;
        uint32_t pk[32];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t dp[32];
          tmem_ld_x32(dp_addr + h * 32, dp);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float2 x = mul2(add2(make_float2(__uint_as_float(dp[e]), __uint_as_float(dp[e + 1])), d2),
                                  make_float2(__uint_as_float(s[h * 32 + e]), __uint_as_float(s[h * 32 + e + 1])));
            dp[e] = __float_as_uint(x.x);
            dp[e + 1] = __float_as_uint(x.y);
          }
          if (j + 1 == n) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (half * 64 + h * 32 + e > r) dp[e] = 0u;
          }
#pragma unroll
          for (int e = 0; e < 32; e += 2)
            pk[(h * 32 + e) >> 1] = Elem<DT>::pack(__uint_as_float(dp[e]), __uint_as_float(dp[e + 1]));
        }
        tmem_st_x32(dp_addr, pk);
        tmem_st_wait();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.ds_full[cnt & 1]);
      }
      if (!ok) break;
      if (!warp_wait(&bars.acc_full, used & 1)) { ok = false; break; }
      ++used;
      tc_fence_after_sync();
      const int row0 = row - lane, part = half * (DH / 2);   // (each warpgroup half of the features)
      if (part < p.dim)
        attn_store_rows<DT, DH / 2, false>(tmem + lanes + kDq + part, p.scale * pow2i(-raised), p.dq + ((w.orow + row0) * p.hq + head) * p.dim + part,
                                           nullptr, (long long)p.hq * p.dim, p.dim - part, w.len - row0);
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.acc_empty);
    }
  }
  if (!ok && lane == 0) atomicExch(p.err, PRISM_ERR_DEVICE_WAIT);
  // nothing here needs dk and dv, but the launch must not count as done before theirs is
  asm volatile("griddepcontrol.wait;" ::: "memory");
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
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)p.rows.tiles * (unsigned)a.hq);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = DqSmem<DH>::kBytes;
  cfg.stream = a.stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.dk != nullptr;   // behind dk and dv's launch only: that one started when delta was there
  const cudaError_t e = cudaLaunchKernelEx(&cfg, dq, m[0], m[1], m[2], m[3], p);
  if (e != cudaSuccess) return fail(PRISM_ERR_CUDA, "causal attention dq: launch failed: %s", cudaGetErrorString(e));
  return check_launch("causal attention dq");
}

}  // namespace

int launch_attn_bwd(const AttnArgs& a) {
  if (a.rows == 0) return PRISM_OK;
  DeltaParams d;
  d.o = static_cast<const uint16_t*>(a.o);
  d.d_o = static_cast<const uint16_t*>(a.d_o);
  d.low = a.low;
  d.sdo = a.sdo;
  d.delta = a.delta;
  d.heads = a.hq; d.dim = a.dim; d.rows = a.rows;
  d.len = a.cu == nullptr ? a.len : a.rows;
  d.v = static_cast<const uint16_t*>(a.v); d.sv = a.sv;
  d.cu = a.cu; d.n = a.n; d.kv_heads = a.hkv;
  d.norms = a.dtype == DT_F16 ? a.norms : nullptr;
  int rc;
  if (a.dtype == DT_BF16) rc = launch_delta<DT_BF16, false>(d, a.stream);
  else if (d.norms == nullptr) rc = launch_delta<DT_F16, false>(d, a.stream);
  else rc = launch_delta<DT_F16, true>(d, a.stream);
  if (rc) return rc;
  BwdParams p;
  p.dq = static_cast<uint16_t*>(a.dq); p.dk = static_cast<uint16_t*>(a.dk); p.dv = static_cast<uint16_t*>(a.dv);
  p.lse = a.lse; p.delta = a.delta;
  p.hq = a.hq; p.hkv = a.hkv; p.group = a.hq / a.hkv; p.dim = a.dim;
  p.c = a.scale * kLog2e; p.scale = a.scale;
  p.norms = d.norms;
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
