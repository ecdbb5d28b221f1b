// Host side of the attention kernels: their arguments, tensor maps and grids.
#pragma once

#include <algorithm>

#include <cuda_runtime.h>

#include "prism_attn.cuh"
#include "prism_host.cuh"

namespace prism {

struct AttnStrides { long long batch, row, head; };   // elements; features are contiguous

struct AttnArgs {
  const void *q, *k, *v;      // rows x heads x dim with the strides below
  AttnStrides sq, sk, sv;
  const int* cu;              // packed: n + 1 offsets; null: dense, n sequences of len rows
  int n, len, rows;           // rows: of the whole batch
  int hq, hkv, dim, dtype;
  float scale;
  void* o;                    // rows x hq x dim, contiguous (backward: the forward's)
  float* lse;                 // hq x rows, or null (backward: the forward's)
  uint8_t* low;               // rows x hq x dim, what o's rounding took, or null (backward: the forward's)
  const void* d_o;            // backward: gradient of o with strides sdo
  AttnStrides sdo;
  float* delta;               // backward: scratch hq x rows
  float* norms;               // backward in fp16: scratch of 2, or null
  void *dq, *dk, *dv;         // backward: rows x heads x dim, contiguous
  int* err;
  cudaStream_t stream;
};

int launch_attn_fwd(const AttnArgs& a);
int launch_attn_bwd(const AttnArgs& a);
// q: n rows (strides batch and head), k and v: n x len rows, lengths [n]; scratch: attn_decode_scratch_bytes.
int launch_attn_decode(const AttnArgs& a, const int* lengths, float* scratch, int num_sms);
size_t attn_decode_scratch_bytes(int dim, int num_sms);

// Tiles of bm rows over all sequences.  Packed: the lengths stand on the GPU; n sequences of `rows` rows have at most
// (rows + n (bm - 1)) / bm tiles, nor more than they have rows, and one more CTA row sees to the rows of no sequence.
inline int attn_rows(const AttnArgs& a, int bm, int heads, AttnRows* r) {
  r->cu = a.cu; r->n = a.n; r->len = a.len; r->rows = a.rows;
  long long tiles;
  if (a.rows == 0) tiles = 0;
  else if (a.cu == nullptr) tiles = (long long)a.n * ((a.len + bm - 1) / bm);
  else tiles = std::min(((long long)a.rows + (long long)a.n * (bm - 1)) / bm, (long long)a.rows) + 1;
  if (tiles * heads > 0x7fffffffll) return fail(PRISM_ERR_UNSUPPORTED, "attention: more than 2^31 tiles");
  r->tiles = (int)tiles;
  return PRISM_OK;
}

// [batch][head][row][feature] view of a tensor, boxes of 64 features x 128 rows.
inline int attn_tmap(CUtensorMap* out, const AttnArgs& a, const void* base, int heads, const AttnStrides& s) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return fail(PRISM_ERR_NO_DRIVER, "cuTensorMapEncodeTiled is not available");
  const int batches = a.cu == nullptr ? a.n : 1, rows = a.cu == nullptr ? a.len : a.rows;
  cuuint64_t gdim[4] = {(cuuint64_t)a.dim, (cuuint64_t)rows, (cuuint64_t)heads, (cuuint64_t)batches};
  cuuint64_t gstride[3] = {(cuuint64_t)s.row * 2, (cuuint64_t)s.head * 2, (cuuint64_t)s.batch * 2};
  cuuint32_t box[4] = {64, (cuuint32_t)kAttnTile, 1, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUtensorMapDataType t = a.dtype == DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const CUresult r = fn(out, t, 4, const_cast<void*>(base), gdim, gstride, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(PRISM_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d): base=%p dim=%d rows=%d heads=%d batches=%d strides %lld %lld %lld",
                (int)r, base, a.dim, rows, heads, batches, s.row, s.head, s.batch);
  return PRISM_OK;
}

}  // namespace prism
