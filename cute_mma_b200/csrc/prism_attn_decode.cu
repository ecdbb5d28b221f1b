// Attention of one query row a sequence over the keys and values that the sequence has so far:
//   o = sum_{j < length} softmax_j(scale q . k_j) v_j   for every head.
//
// Bound by HBM: every key and value is read once for all query heads that share it (up to 16, the rows of one
// mma.sync product; the matrix work is a fraction of the time its bytes take).  The tiles of 64 keys of all sequences
// and key heads stand in one line, and every CTA takes an equal stretch of it, whatever the lengths are: no CTA waits for
// the longest sequence, and a single long one is spread over the whole GPU.  A stretch may begin or end inside a
// sequence; what a CTA has of such a sequence (maximum, sum, weighted values, fp32) goes to scratch, and a second
// launch joins the pieces in order: bit-stable.  The lengths are read on the GPU only.  The join's CTAs stand for stretches,
// not sequences, which each would look through all lengths (1024 sequences of 256 keys: 311 -> 204 us, 4096 of 128: 2.09 ->
// 0.59 ms, 64 of 8192: 134 -> 132 us).
// Measured, bf16, 32 sequences of 4000 keys, 8 key heads of 128 for 32 query heads (525 MB): 87 us, 6.0 TB/s, and 8 us for
// the join (92 % of the measured copy rate without it).
//
// Inside a CTA each of 4 warps owns 16 keys of every tile, with a cp.async ring, a running maximum and sum, and values
// of its own: no barrier but at the end of a sequence, where the warps join through shared memory.
#include "prism_attn_host.cuh"
#include "prism_host.cuh"

namespace prism {
namespace {

constexpr int kWarps = 4, kKeys = 16, kTileKeys = kWarps * kKeys, kStages = 3, kHeads = 16;

struct DecodeParams {
  const uint16_t *q, *k, *v;
  AttnStrides sq, sk, sv;   // q: batch and head; k, v: batch, row, head
  const int* lengths;
  int n, room;              // sequences; rows of the caches
  int hq, hkv, group, chunks, dim;   // chunks: of kHeads query heads of a group
  float c;                  // scale * log2 e
  uint16_t* o;              // n x hq x dim
  float* part;              // scratch [2 ctas][kHeads][padded dim + 2]: values, then maximum and sum
  int ctas;
};

__device__ __forceinline__ int decode_len(const DecodeParams& p, int b) {
  return attn_clamp(__ldg(p.lengths + b), 0, p.room);
}
__device__ __forceinline__ int decode_tiles(const DecodeParams& p, int b) {
  return (decode_len(p, b) + kTileKeys - 1) / kTileKeys;
}
// Tiles of all sequences, for one key head; by one warp.
__device__ __forceinline__ long long decode_total(const DecodeParams& p) {
  long long t = 0;
  for (int b = threadIdx.x & 31; b < p.n; b += 32) t += decode_tiles(p, b);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) t += __shfl_xor_sync(0xffffffffu, t, d);
  return t;
}

// A position in the line of tiles.
struct Cursor {
  int b, hc, t, nt, len;
  __device__ __forceinline__ void open(const DecodeParams& p) {
    len = decode_len(p, b);
    nt = (len + kTileKeys - 1) / kTileKeys;
  }
  __device__ __forceinline__ void next(const DecodeParams& p) {
    if (++t < nt) return;
    t = 0;
    if (++hc < p.hkv * p.chunks) return;
    hc = 0;
    do {
      if (++b >= p.n) return;
      open(p);
    } while (nt == 0);
  }
};

// Where tile `first` of the line is (there is such a tile); by one warp.
__device__ __forceinline__ Cursor decode_find(const DecodeParams& p, long long first) {
  const int lane = threadIdx.x & 31, hcs = p.hkv * p.chunks;
  long long at = 0;
  Cursor c;
  c.b = 0;
  for (int b0 = 0; b0 < p.n; b0 += 32) {
    const int nt = b0 + lane < p.n ? decode_tiles(p, b0 + lane) : 0;
    long long incl = nt;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long o = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += o;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, first < (at + incl) * hcs);
    if (hit) {
      const int l = __ffs(hit) - 1;
      c.b = b0 + l;
      at += __shfl_sync(0xffffffffu, incl - nt, l);
      break;
    }
    at += __shfl_sync(0xffffffffu, incl, 31);
  }
  c.open(p);
  const long long off = first - at * hcs;
  c.hc = (int)(off / c.nt);
  c.t = (int)(off - (long long)c.hc * c.nt);
  return c;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <int DT>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (DT == DT_BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int KD>   // 16-feature steps
struct DecodeSmem {
  // Rows of 16-byte pieces without bank conflicts for ldmatrix: an odd number of pieces to a row; at the widest, where the
  // padding would leave room for one CTA to an SM only, the pieces of a row in an order of its own instead.
  static constexpr bool kSwizzle = KD == 8;
  static constexpr int kPitch = KD * 32 + (kSwizzle ? 0 : 16);
  __device__ static __forceinline__ uint32_t at(int row, int piece) {
    return row * kPitch + ((kSwizzle ? piece ^ (row & 7) : piece) << 4);
  }
  static constexpr int kSlice = kKeys * kPitch;               // 16 rows of K or of V
  static constexpr int kRing = kStages * 2 * kSlice;          // of one warp
  static constexpr int kJoin = 2 * kHeads * (KD * 16 + 2) * 4;   // two warps' results
  static constexpr int kBytes = kWarps * kRing + kJoin;
};

// Exponents of P are raised by this, which the sums carry as well, so that it is gone from the quotient.  fp16 ends at 2^-24:
// with a largest P of 1 many keys that weigh little are lost from the values' product but not from the sum (4099 keys, one of
// them 17 nats above the others: what the others add up to was 1.5 % off); with 2^15 its whole range is used.  bf16 has fp32's
// exponents.
template <int DT>
__device__ __forceinline__ constexpr float decode_lift() { return DT == DT_F16 ? 15.f : 0.f; }

template <int DT, int KD>
__global__ void __launch_bounds__(kWarps * 32, KD <= 4 ? 3 : 2) attn_decode_kernel(const DecodeParams p) {
  using L = DecodeSmem<KD>;
  extern __shared__ __align__(16) uint8_t dsmem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const long long total = decode_total(p) * p.hkv * p.chunks;
  const long long share = (total + p.ctas - 1) / p.ctas;
  const long long first = share * blockIdx.x, last = min(first + share, total);
  if (first >= last) return;
  Cursor ld = decode_find(p, first);   // (every warp finds it for itself)
  Cursor cur = ld;
  const int n = (int)(last - first);
  const uint32_t ring = smem_u32(dsmem) + warp * L::kRing;
  // a lane copies the same piece of every kPer-th row
  constexpr int kPer = 32 / (2 * KD), kRounds = (kKeys + kPer - 1) / kPer;
  const int lr = lane / (2 * KD), piece = lane - lr * 2 * KD;
  const bool active = lr < kPer, inside = active && piece < (p.dim >> 3);   // (features behind the head: zeros)
  uint32_t at[kRounds];
#pragma unroll
  for (int e = 0; e < kRounds; ++e) at[e] = L::at(min(e * kPer + lr, kKeys - 1), piece);
  const uint16_t *kp = nullptr, *vp = nullptr;   // this lane's piece of the head's first row
  bool moved = true;                             // the head has changed
  auto issue = [&](int i) {
    if (i < n) {
      const uint32_t dst = ring + (i % kStages) * 2 * L::kSlice;
      if (moved) {
        const int kvh = ld.hc / p.chunks;
        kp = p.k + ld.b * p.sk.batch + kvh * p.sk.head + (inside ? piece * 8 : 0);
        vp = p.v + ld.b * p.sv.batch + kvh * p.sv.head + (inside ? piece * 8 : 0);
      }
      const int row0 = ld.t * kTileKeys + warp * kKeys + lr;
      const uint16_t *kr = kp + row0 * p.sk.row, *vr = vp + row0 * p.sv.row;
      const bool whole = ld.t + 1 < ld.nt;
#pragma unroll
      for (int e = 0; e < kRounds; ++e) {
        if (active && e * kPer + lr < kKeys) {
          const bool live = inside && (whole || row0 + e * kPer < ld.len);   // rows behind the length: zeros, nothing read
          cp_async16(dst + at[e], live ? kr + e * kPer * p.sk.row : p.k, live);
          cp_async16(dst + L::kSlice + at[e], live ? vr + e * kPer * p.sv.row : p.v, live);
        }
      }
      const int hc = ld.hc, b = ld.b;
      ld.next(p);
      moved = hc != ld.hc || b != ld.b;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) issue(i);

  const int r0 = lane >> 2, cq = (lane & 3) * 2;
  uint32_t qf[KD][4];
  float o[2 * KD][4], m[2], l[2];
  bool fresh = true;       // the sequence's head begins here or the stretch does
  bool from_start = false; // this CTA has its first tile
  for (int i = 0; i < n; ++i) {
    if (fresh) {
      fresh = false;
      from_start = cur.t == 0;
      const int kvh = cur.hc / p.chunks, h0 = (cur.hc - kvh * p.chunks) * kHeads;
      const uint16_t* q = p.q + cur.b * p.sq.batch + (long long)(kvh * p.group + h0) * p.sq.head;
      const int heads = min(kHeads, p.group - h0);
#pragma unroll
      for (int s = 0; s < KD; ++s)
#pragma unroll
        for (int f = 0; f < 4; ++f) {
          const int row = r0 + (f & 1) * 8, col = s * 16 + (f >> 1) * 8 + cq;
          qf[s][f] = row < heads && col < p.dim ? __ldg(reinterpret_cast<const uint32_t*>(q + row * p.sq.head + col)) : 0u;
        }
#pragma unroll
      for (int s = 0; s < 2 * KD; ++s)
#pragma unroll
        for (int f = 0; f < 4; ++f) o[s][f] = 0.f;
      m[0] = m[1] = -INFINITY;
      l[0] = l[1] = 0.f;
    }
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
    __syncwarp();
    issue(i + kStages - 1);
    const uint32_t kt = ring + (i % kStages) * 2 * L::kSlice, vt = kt + L::kSlice;
    float s[2][4] = {}, s1[2][4] = {};   // (two chains each: a product waits for the one before on its accumulator)
    {
      const int row = (lane & 7) + (lane >> 4) * 8, piece = (lane >> 3) & 1;
#pragma unroll
      for (int d = 0; d < KD; ++d) {
        uint32_t b[4];
        ldsm4(kt + L::at(row, d * 2 + piece), b);
        mma16816<DT>(d & 1 ? s1[0] : s[0], qf[d], b[0], b[1]);
        mma16816<DT>(d & 1 ? s1[1] : s[1], qf[d], b[2], b[3]);
      }
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int f = 0; f < 4; ++f) s[x][f] += s1[x][f];
    }
    if (cur.t + 1 == cur.nt) {
      const int key = cur.t * kTileKeys + warp * kKeys + cq;
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int f = 0; f < 4; ++f)
          if (key + x * 8 + (f & 1) >= cur.len) s[x][f] = -INFINITY;
    }
    uint32_t pf[4];
    float f2[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {   // rows r0 and r0 + 8
      float mx = fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      mx = fmaxf(mx, m[h]);
      const float base = mx == -INFINITY ? 0.f : mx;
      const float f = f2[h] = ex2((m[h] - base) * p.c);
      m[h] = mx;
      const float neg = fmaf(-base, p.c, decode_lift<DT>());
      const float e0 = ex2(fmaf(s[0][2 * h], p.c, neg)), e1 = ex2(fmaf(s[0][2 * h + 1], p.c, neg));
      const float e2 = ex2(fmaf(s[1][2 * h], p.c, neg)), e3 = ex2(fmaf(s[1][2 * h + 1], p.c, neg));
      l[h] = l[h] * f + ((e0 + e1) + (e2 + e3));
      pf[h] = Elem<DT>::pack(e0, e1);
      pf[2 + h] = Elem<DT>::pack(e2, e3);
    }
    if (__any_sync(0xffffffffu, f2[0] != 1.f || f2[1] != 1.f)) {   // (a maximum has grown: rare behind the first keys)
#pragma unroll
      for (int d = 0; d < 2 * KD; ++d)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          o[d][2 * h] *= f2[h];
          o[d][2 * h + 1] *= f2[h];
        }
    }
    {
#pragma unroll
      for (int d = 0; d < KD; ++d) {
        uint32_t b[4];
        ldsm4_t(vt + L::at(lane & 15, d * 2 + (lane >> 4)), b);
        mma16816<DT>(o[2 * d], pf, b[0], b[1]);
        mma16816<DT>(o[2 * d + 1], pf, b[2], b[3]);
      }
    }
    const bool ends = cur.t + 1 == cur.nt;
    if (!ends && i + 1 < n) {
      ++cur.t;
      continue;
    }
    // the head's keys, or the stretch, end: the four warps join (3 and 2 into 1 and 0, then 1 into 0)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    }
    float* join = reinterpret_cast<float*>(dsmem + kWarps * L::kRing);
    constexpr int kRow = KD * 16 + 2;
#pragma unroll
    for (int step = 2; step >= 1; step >>= 1) {
      float* slot = join + (warp & (step - 1)) * kHeads * kRow;
      if (warp >= step && warp < 2 * step) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float* row = slot + (r0 + h * 8) * kRow;
#pragma unroll
          for (int d = 0; d < 2 * KD; ++d) {
            row[d * 8 + cq] = o[d][2 * h];
            row[d * 8 + cq + 1] = o[d][2 * h + 1];
          }
          if ((lane & 3) == 0) {
            row[KD * 16] = m[h];
            row[KD * 16 + 1] = l[h];
          }
        }
      }
      __syncthreads();
      if (warp < step) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float* row = slot + (r0 + h * 8) * kRow;
          const float m1 = row[KD * 16], mx = fmaxf(m[h], m1), base = mx == -INFINITY ? 0.f : mx;
          const float f0 = ex2((m[h] - base) * p.c), f1 = ex2((m1 - base) * p.c);
          m[h] = mx;
          l[h] = l[h] * f0 + row[KD * 16 + 1] * f1;
#pragma unroll
          for (int d = 0; d < 2 * KD; ++d) {
            o[d][2 * h] = o[d][2 * h] * f0 + row[d * 8 + cq] * f1;
            o[d][2 * h + 1] = o[d][2 * h + 1] * f0 + row[d * 8 + cq + 1] * f1;
          }
        }
      }
      __syncthreads();
    }
    if (warp == 0) {
      if (from_start && ends) {
        const int kvh = cur.hc / p.chunks, h0 = (cur.hc - kvh * p.chunks) * kHeads;
        const int heads = min(kHeads, p.group - h0);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int row = r0 + h * 8;
          if (row < heads) {
            const float f = 1.f / l[h];
            uint16_t* dst = p.o + ((long long)cur.b * p.hq + kvh * p.group + h0 + row) * p.dim;
#pragma unroll
            for (int d = 0; d < 2 * KD; ++d)
              if (d * 8 + cq < p.dim)
                *reinterpret_cast<uint32_t*>(dst + d * 8 + cq) = Elem<DT>::pack(o[d][2 * h] * f, o[d][2 * h + 1] * f);
          }
        }
      } else {
        // slot 0: the head began before this CTA; slot 1: it begins here and goes on
        float* slot = p.part + ((long long)blockIdx.x * 2 + (from_start ? 1 : 0)) * kHeads * kRow;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float* row = slot + (r0 + h * 8) * kRow;
#pragma unroll
          for (int d = 0; d < 2 * KD; ++d)
            *reinterpret_cast<float2*>(row + d * 8 + cq) = make_float2(o[d][2 * h], o[d][2 * h + 1]);
          if ((lane & 3) == 0) *reinterpret_cast<float2*>(row + KD * 16) = make_float2(m[h], l[h]);
        }
      }
    }
    fresh = true;
    cur.next(p);
  }
}

// Joins the pieces of the heads that more than one CTA worked on, and writes zeros for sequences without keys.  A CTA for
// every query head of every stretch, which has work where a head begins in that stretch and does not end in it: however
// many sequences there are, there are no more of those than stretches.  First all pieces' maxima and sums, a thread each,
// which gives their weights; then the weighted values, a quarter of the pieces to a warp.
constexpr int kMostPieces = 1024;   // CTAs of a launch at most
template <int DT, int KD>
__global__ void __launch_bounds__(128) attn_decode_join_kernel(const DecodeParams p, int rows) {
  constexpr int kRow = KD * 16 + 2;
  __shared__ float acc[4][KD * 16], weight[kMostPieces], part_m[4], part_l[4];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int b = blockIdx.x; b < p.n; b += gridDim.x)
    if (decode_len(p, b) == 0)
      for (int d = threadIdx.x; d < p.hq * p.dim / 8; d += 128)
        reinterpret_cast<uint4*>(p.o + (long long)b * p.hq * p.dim)[d] = make_uint4(0u, 0u, 0u, 0u);
  const int c0 = blockIdx.x / rows, row = blockIdx.x - c0 * rows;
  const long long total = decode_total(p) * p.hkv * p.chunks;
  const long long share = (total + p.ctas - 1) / p.ctas, first = share * c0, last = first + share;
  Cursor at;
  at.t = at.nt = 0;
  if (last < total) at = decode_find(p, last - 1);
  asm volatile("griddepcontrol.wait;" ::: "memory");   // (every CTA: the launch must not count as done before the first one)
  const long long begin = last - 1 - at.t;
  if (last >= total || at.t + 1 == at.nt || begin < first) return;
  const int kvh = at.hc / p.chunks, h0 = (at.hc - kvh * p.chunks) * kHeads;
  if (h0 + row >= p.group) return;
  uint16_t* dst = p.o + ((long long)at.b * p.hq + kvh * p.group + h0 + row) * p.dim;
  const int pieces = (int)((begin + at.nt - 1) / share) - c0 + 1;
  auto piece = [&](int c) { return p.part + (((long long)(c0 + c) * 2 + (c == 0 ? 1 : 0)) * kHeads + row) * kRow; };
  float m = -INFINITY;
  for (int c = threadIdx.x; c < pieces; c += 128) {
    weight[c] = piece(c)[KD * 16];
    m = max_nan(m, weight[c]);
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, d));
  if (lane == 0) part_m[warp] = m;
  __syncthreads();
  m = max_nan(max_nan(part_m[0], part_m[1]), max_nan(part_m[2], part_m[3]));
  if (m == -INFINITY) m = 0.f;
  float l = 0.f;
  for (int c = threadIdx.x; c < pieces; c += 128) {
    const float f = ex2((weight[c] - m) * p.c);
    weight[c] = f;
    l += piece(c)[KD * 16 + 1] * f;
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
  if (lane == 0) part_l[warp] = l;
  __syncthreads();
  constexpr int kPer = (KD * 16 + 31) / 32;
  float o[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) o[e] = 0.f;
#pragma unroll 4
  for (int c = warp; c < pieces; c += 4) {
    const float* src = piece(c);
    const float f = weight[c];
#pragma unroll
    for (int e = 0; e < kPer; ++e)
      if (e * 32 + lane < KD * 16) o[e] = fmaf(src[e * 32 + lane], f, o[e]);
  }
#pragma unroll
  for (int e = 0; e < kPer; ++e)
    if (e * 32 + lane < KD * 16) acc[warp][e * 32 + lane] = o[e];
  __syncthreads();
  const float inv = 1.f / ((part_l[0] + part_l[1]) + (part_l[2] + part_l[3]));
  for (int d = threadIdx.x; d < p.dim; d += 128) {
    const float x = (acc[0][d] + acc[1][d]) + (acc[2][d] + acc[3][d]);
    dst[d] = (uint16_t)(Elem<DT>::pack(x * inv, 0.f) & 0xffffu);
  }
}

template <int DT, int KD>
int launch_t(const DecodeParams& p, cudaStream_t stream) {
  auto* kern = attn_decode_kernel<DT, KD>;
  if (int rc = set_max_dynamic_smem(reinterpret_cast<const void*>(kern), DecodeSmem<KD>::kBytes, "decode attention")) return rc;
  kern<<<p.ctas, kWarps * 32, DecodeSmem<KD>::kBytes, stream>>>(p);
  if (int rc = check_launch("decode attention")) return rc;
  cudaLaunchConfig_t cfg = {};
  const int rows = p.group < kHeads ? p.group : kHeads;
  cfg.gridDim = dim3((unsigned)(p.ctas * rows));
  cfg.blockDim = dim3(128);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, attn_decode_join_kernel<DT, KD>, p, rows);
  if (e != cudaSuccess) return fail(PRISM_ERR_CUDA, "decode attention: launch failed: %s", cudaGetErrorString(e));
  return check_launch("decode attention join");
}
template <int DT>
int launch_d(const DecodeParams& p, cudaStream_t stream) {
  switch ((p.dim + 15) / 16) {
    case 1: return launch_t<DT, 1>(p, stream);
    case 2: return launch_t<DT, 2>(p, stream);
    case 3: return launch_t<DT, 3>(p, stream);
    case 4: return launch_t<DT, 4>(p, stream);
    case 5: return launch_t<DT, 5>(p, stream);
    case 6: return launch_t<DT, 6>(p, stream);
    case 7: return launch_t<DT, 7>(p, stream);
    default: return launch_t<DT, 8>(p, stream);
  }
}

}  // namespace

// As many CTAs as are resident together: three to an SM for heads of up to 64, two for wider ones (shared memory).
static int decode_ctas(int dim, int num_sms) {
  const int n = (dim <= 64 ? 3 : 2) * num_sms;
  return n < kMostPieces ? n : kMostPieces;
}

size_t attn_decode_scratch_bytes(int dim, int num_sms) {
  return (size_t)2 * decode_ctas(dim, num_sms) * kHeads * ((dim + 15) / 16 * 16 + 2) * sizeof(float);
}

int launch_attn_decode(const AttnArgs& a, const int* lengths, float* scratch, int num_sms) {
  DecodeParams p;
  p.q = static_cast<const uint16_t*>(a.q);
  p.k = static_cast<const uint16_t*>(a.k);
  p.v = static_cast<const uint16_t*>(a.v);
  p.sq = a.sq; p.sk = a.sk; p.sv = a.sv;
  p.lengths = lengths;
  p.n = a.n; p.room = a.len;
  p.hq = a.hq; p.hkv = a.hkv; p.group = a.hq / a.hkv; p.dim = a.dim;
  p.chunks = (p.group + kHeads - 1) / kHeads;
  p.c = a.scale * kLog2e;
  p.o = static_cast<uint16_t*>(a.o);
  p.part = scratch;
  p.ctas = decode_ctas(a.dim, num_sms);
  if ((long long)p.n * p.hq > 0x7fffffffll) return fail(PRISM_ERR_UNSUPPORTED, "decode attention: more than 2^31 rows");
  return a.dtype == DT_BF16 ? launch_d<DT_BF16>(p, a.stream) : launch_d<DT_F16>(p, a.stream);
}

}  // namespace prism
