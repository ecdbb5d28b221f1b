// Causal attention, forward: o_i = sum_{j <= i} softmax_j(scale q_i . k_j) v_j for every head of every sequence.
//
// One pass over the keys with a running maximum m and sum l per row (exponents in base 2, c = scale log2 e):
//   S = Q K^T (tcgen05, fp32 in TMEM) -> p = 2^(c s - c m) (registers, one row a thread) -> 16 bits, into TMEM
//   -> O += P V (tcgen05, P from TMEM);  O and l are rescaled only when a row's maximum has grown by more than 2^8
// (every p stays below 2^8, which costs neither 16-bit type any of its digits); the end divides by l.
// fp16 ends at 2^-24, where many keys that weigh little would be lost from P V but not from l: there every p, and so l and O,
// carries a factor of 2^7 more (fwd_lift), up to 2^15 of the type's 2^16.
// A CTA works on two 128-row tiles at a time with a warpgroup each (two heads of a group, whose keys are the same, or 256
// rows of one head), so that the tensor core has the other tile's products while a warpgroup is in its exponentials.
// P is handed over in two pieces: the first one's product runs beside the second one's exponentials.  Keys and values pass
// through one ring of shared tiles.  TMEM, heads of up to 64: S of both tiles, P of both, O of both, so that the next
// scores are formed as soon as these have been read; wider heads: P takes the place of S, which waits for P V.
//
// Measured, bf16, one sequence of 8192 rows, 16 heads: of 128, 253 us, 1086 TFLOP/s of the causal half's products (of a
// measured 1655), tensor pipe 53 % and special function unit 53 % busy: bound by the chain S -> P -> O of a tile, which
// two tiles of a CTA overlap in part; of 64, 190 us, 723 TFLOP/s, special function unit 66 %: bound by the exponentials,
// which take the unit twice as long as both products take the tensor core.
#include "prism_attn.cuh"
#include "prism_host.cuh"
#include "prism_attn_host.cuh"

namespace prism {
namespace {

struct FwdParams {
  AttnRows rows;
  uint16_t* o;     // rows x heads x dim
  float* lse;      // heads x rows, c m + log2 of the sum per row, or null
  uint8_t* low;    // rows x heads x dim, what o's rounding took (e5m2), or null
  const uint16_t* v;   // as the tensor map has it, for the rows of infinities and NaN
  AttnStrides sv;
  int hq, group, dim;
  int pair;        // 1: the two tiles are the same rows of two heads; 0: 256 rows of one head
  float c;         // scale * log2 e
  int* err;
};

// Two softmax warpgroups, and one of the two issuing warps, the loading warp and one that looks through values: a softmax
// thread holds a row of 128 scores.  256 x 208 + 128 x 88 registers = 384 x 168, what the block is
// launched with.
constexpr int kThreads = 384, kSoftmaxRegs = 208, kOtherRegs = 88;

// Blocks of keys that are looked through before their product (the tiles' own rows) in turn: at most as many are under way
// as the ring holds value tiles.
constexpr int kChecks = 8;

template <int DT>
__device__ __forceinline__ constexpr float fwd_lift() { return DT == DT_F16 ? 7.f : 0.f; }

template <int DH>
struct FwdSmem {
  static constexpr uint32_t kTile = (DH / 64) * kAttnSub;
  static constexpr int kQ = DH == 128 ? 1 : 2;   // pairs of Q tiles: the next work's beside this one's
  static constexpr int kRing = DH == 128 ? 5 : 9;
  static constexpr uint32_t kBytes = (2 * kQ + kRing) * kTile + 1024;
};

struct FwdBars {
  uint64_t q_full[2][2], q_empty[2][2], s_full[2], s_read[2], p_full[2][2], pv_done[2], o_full[2], o_empty[2];
  uint64_t turn[2][4];
  uint64_t kv_full[10], kv_empty[10];
  uint64_t checked[kChecks];
  int found[4];   // of a piece of work: infinities or NaN among the values of its first (1) and second (2) block of those
};
// A piece's place in it: two pieces can be under way behind the one that a warp is at.
__device__ __forceinline__ int piece_of(const Ring& r) { return (int)(r.phase * 2 + r.idx); }

// The two tiles of a piece of work: row offset, head and number of key blocks.  From block n[0] - 1 on keys stand beside
// rows that must not see them.
struct FwdTiles {
  int row[2], head[2], n[2];
  __device__ __forceinline__ FwdTiles(const FwdParams& p, const AttnWork& w, int slot_head) {
    if (p.pair) {
      row[0] = row[1] = w.tile * kAttnTile;
      head[0] = 2 * slot_head;
      head[1] = 2 * slot_head + 1;
      n[0] = n[1] = w.tile + 1;
    } else {
      row[0] = 2 * w.tile * kAttnTile;
      row[1] = row[0] + kAttnTile;
      head[0] = head[1] = slot_head;
      n[0] = 2 * w.tile + 1;
      n[1] = w.len > row[1] ? n[0] + 1 : 0;
    }
  }
  __device__ __forceinline__ int most() const { return max(n[0], n[1]); }
};

// Looks through the first `valid` rows of a value tile, by one warp.  A masked key has the probability 0, but 0 times its
// infinities and NaN would not be 0: those become zeros here (true: there were any), and the rows that do see them get
// them at the end (attn_add_unbounded).  (Inlined, like all that runs behind a change of the register share: a called
// function is compiled without regard to it.)  Rows behind the sequence become zeros up to the next sixteen.
template <int DT, int DH>
__device__ __forceinline__ bool attn_check_values(char* tile, int valid) {
  constexpr uint32_t kExp = DT == DT_BF16 ? 0x7f807f80u : 0x7c007c00u, kOne = DT == DT_BF16 ? 0x00800080u : 0x04000400u;
  const int lane = threadIdx.x & 31;
  if (valid < kAttnTile) attn_zero_tail<DH>(tile, valid);
  const int pieces = min(valid, kAttnTile) * 8;   // of 16 bytes, of one 64-feature half
  uint32_t sum[4] = {0u, 0u, 0u, 0u};   // of zero times every value: zero, or NaN
#pragma unroll 1
  for (int s = 0; s < DH / 64; ++s) {
    const uint4* t = reinterpret_cast<const uint4*>(tile + s * kAttnSub);
#pragma unroll 8
    for (int i = lane; i < pieces; i += 32) {
      const uint4 x = t[i];
      sum[0] = Pk<DT>::fma(x.x, 0u, sum[0]);
      sum[1] = Pk<DT>::fma(x.y, 0u, sum[1]);
      sum[2] = Pk<DT>::fma(x.z, 0u, sum[2]);
      sum[3] = Pk<DT>::fma(x.w, 0u, sum[3]);
    }
  }
  uint32_t any = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) any |= (sum[i] & kExp) + kOne;   // (an exponent of ones overflows into the bit above)
  if (!__any_sync(0xffffffffu, any & 0x80008000u)) return false;
  for (int s = 0; s < DH / 64; ++s) {
    uint32_t* t = reinterpret_cast<uint32_t*>(tile + s * kAttnSub);
    for (int i = lane; i < pieces * 4; i += 32) {
      const uint32_t c = (t[i] & kExp) + kOne;
      if (c & 0x8000u) t[i] &= 0xffff0000u;
      if (c & 0x80000000u) t[i] &= 0x0000ffffu;
    }
  }
  fence_proxy_async_smem();
  __syncwarp();
  return true;
}

// o += the infinities and NaN among the values that row `row` of the sequence sees, from row `first` on; by a whole warp, whose
// rows end at `last`.  All lanes look at the same 16 bytes of a value row at a time, and take what they see of it where it has
// any.  16 x 1024 rows, 12 heads of 64 (67 us without any): one NaN in all 170 us, all values from row 600 on NaN 560 us; 4.2 and
// 17.6 ms when each thread went through its row's values one by one, and through those of all pieces behind the first that had any.
template <int DT>
__device__ __forceinline__ void attn_add_unbounded(const FwdParams& p, const AttnWork& w, int first, int row, int last, int kvh,
                                                   uint16_t* o) {
  constexpr uint32_t kExp = DT == DT_BF16 ? 0x7f807f80u : 0x7c007c00u, kOne = DT == DT_BF16 ? 0x00800080u : 0x04000400u;
  const uint16_t* v = p.v + w.batch * p.sv.batch + (long long)(w.row + first) * p.sv.row + kvh * p.sv.head;
#pragma unroll 1
  for (int d = 0; d < p.dim; d += 8) {
    float sum[8] = {};
    bool any = false;
    const uint16_t* vj = v + d;
#pragma unroll 8
    for (int j = first; j <= last; ++j, vj += p.sv.row) {
      const uint4 x = __ldg(reinterpret_cast<const uint4*>(vj));
      const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
      uint32_t c = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) c |= (xs[e] & kExp) + kOne;   // (an exponent of ones overflows into the bit above)
      if ((c & 0x80008000u) == 0 || j > row) continue;
      any = true;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = Elem<DT>::unpack(xs[e]);
        if (!isfinite(f.x)) sum[2 * e] += f.x;
        if (!isfinite(f.y)) sum[2 * e + 1] += f.y;
      }
    }
    if (!any) continue;
    uint4* at = reinterpret_cast<uint4*>(o + d);
    uint4 y = *at;
    uint32_t* ys = &y.x;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = Elem<DT>::unpack(ys[e]);
      ys[e] = Elem<DT>::pack(f.x + sum[2 * e], f.y + sum[2 * e + 1]);
    }
    *at = y;
  }
}

template <int DT, int DH, bool LOW>
__global__ void __launch_bounds__(kThreads, 1)
    attn_fwd_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                    const __grid_constant__ CUtensorMap mv, const FwdParams p) {
  using L = FwdSmem<DH>;
  constexpr bool kEarly = DH == 64;   // S does not share its columns with P
  constexpr uint32_t kO = kEarly ? 384 : 256;
  // keys of P's first piece (8192 rows, 16 heads: of 64, 201 / 199 / 190 us with 32 / 64 / 96; of 128, 262 / 253 / 262)
  constexpr int kFirst = kEarly ? 96 : 64;
  extern __shared__ uint8_t smem_raw[];
  __shared__ FwdBars bars;
  __shared__ AttnSched sched;
  __shared__ uint32_t tmem_slot;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);

  if (warp == 8) {
    tmem_alloc_cta(&tmem_slot, 512);
    tmem_relinquish_cta();
  } else if (warp == 9 && lane == 0) {
    attn_sched_init(sched, 11);
    for (int i = 0; i < kChecks; ++i) mbar_init(&bars.checked[i], 1);
    for (int t = 0; t < 2; ++t) {
      for (int i = 0; i < 4; ++i) mbar_init(&bars.turn[t][i], 1);
      for (int i = 0; i < 2; ++i) {
        mbar_init(&bars.q_full[t][i], 1);
        mbar_init(&bars.q_empty[t][i], 1);
      }
      mbar_init(&bars.s_full[t], 1);
      mbar_init(&bars.s_read[t], 4);
      mbar_init(&bars.p_full[t][0], 4);
      mbar_init(&bars.p_full[t][1], 4);
      mbar_init(&bars.pv_done[t], 1);
      mbar_init(&bars.o_full[t], 1);
      mbar_init(&bars.o_empty[t], 4);
    }
    for (int s = 0; s < L::kRing; ++s) {
      mbar_init(&bars.kv_full[s], 1);
      mbar_init(&bars.kv_empty[s], 3);
    }
    fence_mbar_init();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);   // (known to be the same in all lanes)
  bool ok = true;
  AttnWork w;
  int slot_head;
  Ring rw(2);

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == 9) {
      char* ring = smem + 2 * L::kQ * L::kTile;
      Ring r(L::kRing), rq(L::kQ);
      ok = attn_schedule(
          sched, p.rows, p.pair ? p.hq / 2 : p.hq, p.pair ? kAttnTile : 2 * kAttnTile, true,
          [&](const AttnWork& g, int h) {
            const FwdTiles tl(p, g, h);
            for (int t = 0; t < 2; ++t) {
              if (!warp_wait(&bars.q_empty[t][rq.idx], rq.phase ^ 1)) return false;
              if (lane == 0) {
                if (tl.n[t] == 0) {   // no such tile: its warps pass the buffer on
                  mbar_arrive(&bars.q_full[t][rq.idx]);
                } else {
                  mbar_arrive_expect_tx(&bars.q_full[t][rq.idx], L::kTile);
                  attn_load_tile<DH>(smem + (2 * rq.idx + t) * L::kTile, &mq, &bars.q_full[t][rq.idx], g.row + tl.row[t],
                                     tl.head[t], g.batch);
                }
              }
            }
            rq.next();
            const int n = tl.most(), kvh = tl.head[0] / p.group;
            for (int i = 0; i < 2 * n; ++i, r.next()) {
              if (!warp_wait(&bars.kv_empty[r.idx], r.phase ^ 1)) return false;
              if (lane == 0) {
                mbar_arrive_expect_tx(&bars.kv_full[r.idx], L::kTile);
                attn_load_tile<DH>(ring + r.idx * L::kTile, (i & 1) ? &mv : &mk, &bars.kv_full[r.idx],
                                   g.row + (i >> 1) * kAttnTile, kvh, g.batch);
              }
            }
            return true;
          },
          [&](const AttnWork& g, int h) {
            for (int t = 0; t <= p.pair; ++t) attn_zero_gap(p.rows, g, p.o, p.hq, p.pair ? 2 * h + t : h, p.dim);
          });
    } else if (warp == 8 || warp == 10) {
      // one issuing warp per tile: a product costs its issuer about as long as the tensor core, every barrier more
      const int t = warp == 10;
      const uint32_t id_s = make_idesc(DT, 128, 128, 0, 0), id_o = make_idesc(DT, 128, DH, 0, 1);
      const uint32_t q_tile = smem_u32(smem) + t * L::kTile, ring = smem_u32(smem) + 2 * L::kQ * L::kTile;
      const uint32_t st = tmem + t * 128, ot = tmem + kO + t * DH, pt = kEarly ? tmem + 256 + t * 64 : st;
      Ring rk(L::kRing), rq(L::kQ);
      uint32_t used = 0, made = 0, blocks = 0, checks = 0;   // pieces of work, scores, key blocks and checked ones so far
      auto scores = [&](bool last) {
        tc_fence_after_sync();
        if (elect_one()) {
          attn_mma_xyt<DH>(st, q_tile + 2 * rq.idx * L::kTile, ring + rk.idx * L::kTile, id_s);
          umma_commit_cta(&bars.s_full[t]);
          umma_commit_cta(&bars.kv_empty[rk.idx]);
          if (last) umma_commit_cta(&bars.q_empty[t][rq.idx]);
        }
        ++made;
      };
      while (ok && attn_next(sched, rw, &w, &slot_head, &ok)) {
        const FwdTiles tl(p, w, slot_head);
        const int n = tl.most(), nt = tl.n[t];
        ok = warp_wait(&bars.q_full[t][rq.idx], rq.phase);
        if (ok && nt == 0 && elect_one()) mbar_arrive(&bars.q_empty[t][rq.idx]);
        // every lane waits, one issues
        for (int j = -1; ok && j < n; ++j) {
          // scores of block j + 1, where they need not wait for block j's product
          Ring rv = rk;   // (for j >= 0: stands on K of block j + 1, V of block j before it)
          if (j >= 0) {
            if (rv.idx == 0) { rv.idx = L::kRing; rv.phase ^= 1u; }
            --rv.idx;
          }
          const bool more = j + 1 < n, mine = j + 1 < nt;
          if (more && !warp_wait(&bars.kv_full[rk.idx], rk.phase)) { ok = false; break; }
          if (more && !mine) {
            if (elect_one()) mbar_arrive(&bars.kv_empty[rk.idx]);
          } else if (mine && (kEarly || j < 0)) {
            if (kEarly && !warp_wait(&bars.s_read[t], (made & 1) ^ 1)) { ok = false; break; }
            scores(j + 2 == nt);
          }
          if (j >= 0) {
            if (!warp_wait(&bars.kv_full[rv.idx], rv.phase)) { ok = false; break; }
            if (j >= tl.n[0] - 1) {
              if (!warp_wait(&bars.checked[checks % kChecks], (checks / kChecks) & 1)) { ok = false; break; }
              ++checks;
            }
            if (j >= nt) {
              if (elect_one()) mbar_arrive(&bars.kv_empty[rv.idx]);
            } else {
              const int valid = w.len - j * kAttnTile;
              const int steps = valid >= kAttnTile ? 8 : (valid + 15) >> 4;
              const uint32_t v_tile = ring + rv.idx * L::kTile;
              if (j == 0 && !warp_wait(&bars.o_empty[t], (used & 1) ^ 1)) { ok = false; break; }
              if (!warp_wait(&bars.p_full[t][0], blocks & 1)) { ok = false; break; }
              tc_fence_after_sync();
              if (elect_one()) attn_mma_py<DH>(ot, pt, 32, v_tile, id_o, j > 0, min(steps, kFirst / 16));
              if (!warp_wait(&bars.p_full[t][1], blocks & 1)) { ok = false; break; }
              tc_fence_after_sync();
              if (elect_one()) {
                if (steps > kFirst / 16)
                  attn_mma_py<DH>(ot, pt + kFirst / 2, 32, v_tile + kFirst / 16 * 2048, id_o, true, steps - kFirst / 16);
                if (j + 1 == nt) umma_commit_cta(&bars.o_full[t]);
                else if (kEarly) umma_commit_cta(&bars.pv_done[t]);
                umma_commit_cta(&bars.kv_empty[rv.idx]);
              }
              ++blocks;
              if (!kEarly && mine) scores(j + 2 == nt);
            }
          }
          // on to the next K: behind V(j + 1), or at the end to the next work's first
          if (more) {
            rk.next();
            rk.next();
          }
        }
        used += nt > 0;
        rq.next();
      }
    } else {
      // the warp that looks through the values of the tiles' own rows
      Ring r(L::kRing);
      uint32_t checks = 0;
      while (ok && attn_next(sched, rw, &w, &slot_head, &ok)) {
        const FwdTiles tl(p, w, slot_head);
        const int n = tl.most();
        int some = 0;
        // (it sees every tile of the ring and gives it back like the issuing warps: a barrier's parity says nothing to one
        // that has left out a phase)
        for (int i = 0; i < 2 * n; ++i, r.next()) {
          const int j = i >> 1;
          if (!warp_wait_asleep(&bars.kv_full[r.idx], r.phase)) { ok = false; break; }
          if ((i & 1) && j >= tl.n[0] - 1) {
            const bool found = attn_check_values<DT, DH>(smem + (2 * L::kQ + r.idx) * L::kTile, w.len - j * kAttnTile);
            if (lane == 0) {
              some |= found << (j - tl.n[0] + 1);
              bars.found[piece_of(rw)] = some;
              mbar_arrive(&bars.checked[checks % kChecks]);
            }
            ++checks;
          }
          if (lane == 0) mbar_arrive(&bars.kv_empty[r.idx]);
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const int t = warp >> 2;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;
    const uint32_t s_addr = tmem + lanes + t * 128, o_addr = tmem + lanes + kO + t * DH;
    const uint32_t p_addr = kEarly ? tmem + lanes + 256 + t * 64 : s_addr;
    const int r = (warp & 3) * 32 + lane;
    uint32_t phase = 0, used = 0, pv = 0, turns = 0;
    while (ok && attn_next(sched, rw, &w, &slot_head, &ok)) {
      const FwdTiles tl(p, w, slot_head);
      const int nt = tl.n[t], n = tl.most();
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < n; ++j) {
        if (j >= nt) {   // nothing of this tile: the turn passes on
          if (kEarly) break;
          if (!warp_wait(&bars.turn[t][warp & 3], (turns & 1) ^ (t ^ 1))) { ok = false; break; }
          ++turns;
          if (lane == 0) mbar_arrive(&bars.turn[t ^ 1][warp & 3]);
          continue;
        }
        if (!warp_wait(&bars.s_full[t], phase)) { ok = false; break; }
        phase ^= 1u;
        tc_fence_after_sync();
        uint32_t s[128];
#pragma unroll
        for (int q = 0; q < 4; ++q) tmem_ld_x32(s_addr + q * 32, *reinterpret_cast<uint32_t(*)[32]>(s + q * 32));
        tmem_ld_wait();
        if (kEarly) {
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars.s_read[t]);
        }
        if (j + 1 == nt) {   // the tile's own rows: keys up to the row itself
#pragma unroll
          for (int e = 0; e < 128; ++e)
            if (e > r) s[e] = 0xff800000u;
        }
        float mx[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) mx[e] = max_nan(__uint_as_float(s[e]), __uint_as_float(s[e + 8]));
#pragma unroll
        for (int e = 16; e < 128; e += 16)
#pragma unroll
          for (int f = 0; f < 8; ++f)
            mx[f] = max3_nan(mx[f], __uint_as_float(s[e + f]), __uint_as_float(s[e + 8 + f]));
        const float mnew = max3_nan(max3_nan(m, mx[0], mx[1]), max3_nan(mx[2], mx[3], mx[4]), max3_nan(mx[5], mx[6], mx[7]));
        // P V of the block before is done: its P may be written over and O rescaled.  (Where S waits for that product, the
        // scores' arrival says so.)
        if (kEarly && j > 0) {
          if (!warp_wait(&bars.pv_done[t], pv & 1)) { ok = false; break; }
          ++pv;
          tc_fence_after_sync();
        }
        // (a NaN among the scores makes the comparison fail and m NaN: the whole row is NaN then.  A row at -infinity
        // has NaN on its left side as well, and nothing to rescale.)
        const bool grown = !((mnew - m) * p.c <= 8.f);
        if (__any_sync(0xffffffffu, grown)) {
          // (each row by its own maximum alone: its bits do not depend on its neighbours)
          const float f = grown ? ex2((m - (mnew == -INFINITY ? 0.f : mnew)) * p.c) : 1.f;
          if (grown) m = mnew;
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
        const float2 c2 = both(p.c), n2 = both(fmaf(m == -INFINITY ? 0.f : -m, p.c, fwd_lift<DT>()));
        float2 sum0 = both(0.f), sum1 = both(0.f);
        // Wide heads: the exponentials of the two warps of a quarter SM take turns, so that one tile's run beside the
        // other's products (8192 rows, 16 heads of 128: 288 -> 244 us).  Where S does not wait for P V there is nothing to
        // wait for between them, and turns only cost (heads of 64: 196 -> 216 us).
        if (!kEarly && !warp_wait(&bars.turn[t][warp & 3], (turns & 1) ^ (t ^ 1))) { ok = false; break; }
        ++turns;
#pragma unroll
        for (int e = 0; e < 128; e += 2) {
          const float2 x = fma2(make_float2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), c2, n2);
          const float2 y = make_float2(ex2(x.x), ex2(x.y));
          if (e & 2) sum1 = add2(sum1, y);
          else sum0 = add2(sum0, y);
          s[e >> 1] = Elem<DT>::pack(y.x, y.y);   // pairs land in the first half of the registers
          if (e % 32 == 30) tmem_st_x16(p_addr + (e - 30) / 2, s + (e - 30) / 2);
          if (e + 2 == kFirst || e + 2 == 128) {
            tmem_st_wait();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.p_full[t][e + 2 == 128]);
          }
        }
        if (!kEarly && lane == 0) mbar_arrive(&bars.turn[t ^ 1][warp & 3]);
        sum0 = add2(sum0, sum1);
        l += sum0.x + sum0.y;
      }
      if (!ok) break;
      if (nt == 0) continue;
      if (!warp_wait(&bars.o_full[t], used & 1)) { ok = false; break; }
      ++used;
      tc_fence_after_sync();
      const int found = *static_cast<volatile int*>(&bars.found[piece_of(rw)]) & (nt > tl.n[0] ? 3 : 1);
      const int row = tl.row[t] + r, head = tl.head[t];
      const bool mine = row < w.len;
      const int row0 = row - lane;
      const long long at = ((w.orow + row0) * p.hq + head) * p.dim, step = (long long)p.hq * p.dim;
      attn_store_rows<DT, DH, LOW>(o_addr, 1.f / l, p.o + at, LOW ? p.low + at : nullptr, step, p.dim, w.len - row0);
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.o_empty[t]);
      __syncwarp();   // (its row was stored by the lanes beside it)
      if (mine && p.lse != nullptr) p.lse[(long long)head * p.rows.rows + w.orow + row] = m * p.c + (lg2(l) - fwd_lift<DT>());
      // (tile 0 sees the first of the blocks only)
      if (found && mine)
        attn_add_unbounded<DT>(p, w, (tl.n[0] - 1) * kAttnTile, row, min(row0 + 31, w.len - 1), head / p.group, p.o + at + lane * step);
    }
  }
  if (!ok && lane == 0) atomicExch(p.err, PRISM_ERR_DEVICE_WAIT);
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 8) tmem_dealloc_cta(tmem, 512);
}

template <int DT, int DH>
int launch_t(const AttnArgs& a, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const FwdParams& p) {
  auto* kern = p.low != nullptr ? attn_fwd_kernel<DT, DH, true> : attn_fwd_kernel<DT, DH, false>;
  if (int rc = set_max_dynamic_smem(reinterpret_cast<const void*>(kern), FwdSmem<DH>::kBytes, "causal attention")) return rc;
  const unsigned heads = (unsigned)(p.pair ? a.hq / 2 : a.hq);
  kern<<<(unsigned)p.rows.tiles * heads, kThreads, FwdSmem<DH>::kBytes, a.stream>>>(mq, mk, mv, p);
  return check_launch("causal attention");
}

}  // namespace

int launch_attn_fwd(const AttnArgs& a) {
  FwdParams p;
  p.hq = a.hq; p.group = a.hq / a.hkv; p.dim = a.dim;
  p.pair = p.group % 2 == 0;
  if (int rc = attn_rows(a, p.pair ? kAttnTile : 2 * kAttnTile, a.hq, &p.rows)) return rc;
  if (p.rows.tiles == 0) return PRISM_OK;
  p.o = static_cast<uint16_t*>(a.o);
  p.lse = a.lse;
  p.low = a.low;
  p.v = static_cast<const uint16_t*>(a.v);
  p.sv = a.sv;
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
