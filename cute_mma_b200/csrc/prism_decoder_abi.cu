// extern "C" entry points of the operators between the linears of a decoder: argument checks, dispatch to the launchers.
#include "../../include/prism_b200.h"
#include "prism_attn_host.cuh"
#include "prism_host.cuh"
#include "prism_norm.cuh"

#include <initializer_list>

using namespace prism;

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool aligned_to(size_t size, std::initializer_list<const void*> ptrs) {   // to their own elements
  for (const void* p : ptrs)
    if (reinterpret_cast<uintptr_t>(p) % size != 0) return false;
  return true;
}

int check_workspace(const char* what, void* workspace, size_t bytes) {
  if (workspace == nullptr || bytes < PRISM_WORKSPACE_HEADER_BYTES)
    return fail(PRISM_ERR_WORKSPACE, "%s: the workspace must hold its status header (%d bytes)", what, PRISM_WORKSPACE_HEADER_BYTES);
  if ((reinterpret_cast<uintptr_t>(workspace) & 255) != 0)
    return fail(PRISM_ERR_BAD_ARG, "%s: the workspace must be 256-byte aligned", what);
  return PRISM_OK;
}

int num_sms() {   // of the current device; 148 without one
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) {
    (void)cudaGetLastError();
    return 148;
  }
  return n;
}

constexpr int kMostRows = 0x7fffffff - 256;   // (row numbers rounded up to whole tiles are ints)
constexpr int kMostSeqs = 1 << 20;   // packed (looked through while others wait, whose limit is about a second)

AttnStrides strides_at(const long long* s, int i) { return AttnStrides{s[3 * i], s[3 * i + 1], s[3 * i + 2]}; }

int check_attn(const char* what, const AttnArgs& a, const long long* strides, int n_strides) {
  if (a.rows > kMostRows) return fail(PRISM_ERR_UNSUPPORTED, "%s: more than %d rows", what, kMostRows);
  if (a.cu != nullptr && a.n > kMostSeqs) return fail(PRISM_ERR_UNSUPPORTED, "%s: more than %d packed sequences", what, kMostSeqs);
  if (a.n < 1 || a.len < 0 || a.rows < 0) return fail(PRISM_ERR_BAD_ARG, "%s: n_seqs must be positive, seq_len and rows not negative", what);
  if (a.cu == nullptr && (long long)a.n * a.len != a.rows)
    return fail(PRISM_ERR_BAD_ARG, "%s: rows must be n_seqs * seq_len without cu_seqlens", what);
  if (a.hq < 1 || a.hkv < 1 || a.hq % a.hkv != 0)
    return fail(PRISM_ERR_BAD_ARG, "%s: heads (%d) must be a multiple of kv_heads (%d)", what, a.hq, a.hkv);
  if (a.dim < 8 || a.dim > 128 || a.dim % 8 != 0)
    return fail(PRISM_ERR_UNSUPPORTED, "%s: head_dim must be a multiple of 8 up to 128, got %d", what, a.dim);
  if (a.dtype != DT_F16 && a.dtype != DT_BF16) return fail(PRISM_ERR_BAD_ARG, "%s: dtype must be fp16 or bf16", what);
  if (!(a.scale > 0.f) || !isfinite(a.scale)) return fail(PRISM_ERR_BAD_ARG, "%s: the scale must be positive and finite", what);
  if (strides == nullptr) return fail(PRISM_ERR_BAD_ARG, "%s: strides is null", what);
  for (int i = 0; i < n_strides; ++i)
    if (strides[i] <= 0 || strides[i] % 8 != 0 || strides[i] >= (1ll << 39))
      return fail(PRISM_ERR_BAD_ARG, "%s: strides must be positive multiples of 8 elements", what);
  if (a.rows > 0 && (a.q == nullptr || a.k == nullptr || a.v == nullptr || a.o == nullptr))
    return fail(PRISM_ERR_BAD_ARG, "%s: null tensor", what);
  if (!aligned16(a.q) || !aligned16(a.k) || !aligned16(a.v) || !aligned16(a.o) || !aligned16(a.d_o) || !aligned16(a.dq) ||
      !aligned16(a.dk) || !aligned16(a.dv) || !aligned16(a.low))
    return fail(PRISM_ERR_BAD_ARG, "%s: tensors must be 16-byte aligned", what);
  if (!aligned_to(4, {a.lse, a.delta, a.norms, a.cu}))
    return fail(PRISM_ERR_BAD_ARG, "%s: lse, delta, norms and cu_seqlens must be 4-byte aligned", what);
  return PRISM_OK;
}

}  // namespace

extern "C" int prism_attn_fwd(const void* q, const void* k, const void* v, void* o, float* lse, void* o_low,
                              const int* cu_seqlens, int n_seqs, int seq_len, int rows, int heads, int kv_heads, int head_dim, int dtype, float scale,
                              const long long* strides, void* workspace, size_t workspace_bytes, void* stream) {
  AttnArgs a{};
  a.q = q; a.k = k; a.v = v; a.o = o; a.lse = lse; a.low = static_cast<uint8_t*>(o_low);
  a.cu = cu_seqlens; a.n = n_seqs; a.len = seq_len; a.rows = rows;
  a.hq = heads; a.hkv = kv_heads; a.dim = head_dim; a.dtype = dtype; a.scale = scale;
  if (int rc = check_attn("prism_attn_fwd", a, strides, 9)) return rc;
  a.sq = strides_at(strides, 0); a.sk = strides_at(strides, 1); a.sv = strides_at(strides, 2);
  if (int rc = check_workspace("prism_attn_fwd", workspace, workspace_bytes)) return rc;
  a.err = static_cast<int*>(workspace);
  a.stream = static_cast<cudaStream_t>(stream);
  return launch_attn_fwd(a);
}

extern "C" int prism_attn_bwd_scaled(const void* d_o, const void* q, const void* k, const void* v, const void* o, const float* lse,
                                     const void* o_low, void* dq, void* dk, void* dv, float* delta, float* norms, const int* cu_seqlens,
                                     int n_seqs, int seq_len, int rows, int heads, int kv_heads, int head_dim, int dtype, float scale,
                                     const long long* strides, void* workspace, size_t workspace_bytes, void* stream) {
  AttnArgs a{};
  a.q = q; a.k = k; a.v = v; a.o = const_cast<void*>(o); a.lse = const_cast<float*>(lse); a.d_o = d_o;
  a.low = const_cast<uint8_t*>(static_cast<const uint8_t*>(o_low));
  a.dq = dq; a.dk = dk; a.dv = dv; a.delta = delta; a.norms = norms;
  a.cu = cu_seqlens; a.n = n_seqs; a.len = seq_len; a.rows = rows;
  a.hq = heads; a.hkv = kv_heads; a.dim = head_dim; a.dtype = dtype; a.scale = scale;
  if (int rc = check_attn("prism_attn_bwd", a, strides, 12)) return rc;
  a.sq = strides_at(strides, 0); a.sk = strides_at(strides, 1); a.sv = strides_at(strides, 2); a.sdo = strides_at(strides, 3);
  if (rows > 0 && (d_o == nullptr || lse == nullptr || delta == nullptr))
    return fail(PRISM_ERR_BAD_ARG, "prism_attn_bwd: null tensor");
  if ((dk == nullptr) != (dv == nullptr)) return fail(PRISM_ERR_BAD_ARG, "prism_attn_bwd: dk and dv go together");
  if (int rc = check_workspace("prism_attn_bwd", workspace, workspace_bytes)) return rc;
  a.err = static_cast<int*>(workspace);
  a.stream = static_cast<cudaStream_t>(stream);
  return launch_attn_bwd(a);
}

extern "C" int prism_attn_bwd(const void* d_o, const void* q, const void* k, const void* v, const void* o, const float* lse,
                              const void* o_low, void* dq, void* dk, void* dv, float* delta, const int* cu_seqlens, int n_seqs, int seq_len,
                              int rows, int heads, int kv_heads, int head_dim, int dtype, float scale,
                              const long long* strides, void* workspace, size_t workspace_bytes, void* stream) {
  return prism_attn_bwd_scaled(d_o, q, k, v, o, lse, o_low, dq, dk, dv, delta, nullptr, cu_seqlens, n_seqs, seq_len, rows, heads, kv_heads,
                               head_dim, dtype, scale, strides, workspace, workspace_bytes, stream);
}

extern "C" size_t prism_attn_decode_scratch_bytes(int head_dim) {
  return head_dim < 8 || head_dim > 128 ? 0 : attn_decode_scratch_bytes(head_dim, num_sms());
}

extern "C" int prism_attn_decode(const void* q, const void* k, const void* v, void* o, const int* lengths, int n_seqs, int room,
                                 int heads, int kv_heads, int head_dim, int dtype, float scale, const long long* strides,
                                 void* scratch, size_t scratch_bytes, void* stream) {
  const char* what = "prism_attn_decode";
  if (n_seqs < 0 || room < 0) return fail(PRISM_ERR_BAD_ARG, "%s: n_seqs and room must not be negative", what);
  if (room > kMostRows) return fail(PRISM_ERR_UNSUPPORTED, "%s: room for more than %d rows", what, kMostRows);
  if (heads < 1 || kv_heads < 1 || heads % kv_heads != 0)
    return fail(PRISM_ERR_BAD_ARG, "%s: heads (%d) must be a multiple of kv_heads (%d)", what, heads, kv_heads);
  if (head_dim < 8 || head_dim > 128 || head_dim % 8 != 0)
    return fail(PRISM_ERR_UNSUPPORTED, "%s: head_dim must be a multiple of 8 up to 128, got %d", what, head_dim);
  if (dtype != DT_F16 && dtype != DT_BF16) return fail(PRISM_ERR_BAD_ARG, "%s: dtype must be fp16 or bf16", what);
  if (!(scale > 0.f) || !isfinite(scale)) return fail(PRISM_ERR_BAD_ARG, "%s: the scale must be positive and finite", what);
  if (strides == nullptr) return fail(PRISM_ERR_BAD_ARG, "%s: strides is null", what);
  for (int i = 0; i < 8; ++i)
    if (strides[i] < 0 || strides[i] % 8 != 0)
      return fail(PRISM_ERR_BAD_ARG, "%s: strides must be multiples of 8 elements, not negative", what);
  if (n_seqs == 0) return PRISM_OK;
  if (q == nullptr || o == nullptr || lengths == nullptr || (room > 0 && (k == nullptr || v == nullptr)))
    return fail(PRISM_ERR_BAD_ARG, "%s: null tensor", what);
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o) || !aligned16(scratch))
    return fail(PRISM_ERR_BAD_ARG, "%s: tensors must be 16-byte aligned", what);
  if (!aligned_to(4, {lengths})) return fail(PRISM_ERR_BAD_ARG, "%s: lengths must be 4-byte aligned", what);
  AttnArgs a{};
  a.q = q; a.k = k; a.v = v; a.o = o;
  a.n = n_seqs; a.len = room;
  a.hq = heads; a.hkv = kv_heads; a.dim = head_dim; a.dtype = dtype; a.scale = scale;
  a.sq = AttnStrides{strides[0], 0, strides[1]};
  a.sk = AttnStrides{strides[2], strides[3], strides[4]};
  a.sv = AttnStrides{strides[5], strides[6], strides[7]};
  a.stream = static_cast<cudaStream_t>(stream);
  const int sms = num_sms();
  if (scratch == nullptr || scratch_bytes < attn_decode_scratch_bytes(head_dim, sms))
    return fail(PRISM_ERR_WORKSPACE, "%s: scratch of %zu bytes, needs %zu", what, scratch_bytes, attn_decode_scratch_bytes(head_dim, sms));
  return launch_attn_decode(a, lengths, static_cast<float*>(scratch), sms);
}

namespace {

int check_norm(const char* what, const NormArgs& a, int w_dtype) {
  if (a.rows < 0 || a.rows > 0x7fffffffll) return fail(PRISM_ERR_BAD_ARG, "%s: rows must be in [0, 2^31)", what);
  if (a.cols < 1 || a.cols > norm_max_cols())
    return fail(PRISM_ERR_UNSUPPORTED, "%s: cols must be in [1, %d], got %d", what, norm_max_cols(), a.cols);
  if (a.dtype != DT_F16 && a.dtype != DT_BF16) return fail(PRISM_ERR_BAD_ARG, "%s: dtype must be fp16 or bf16", what);
  if (w_dtype != PRISM_DTYPE_F32 && w_dtype != a.dtype)
    return fail(PRISM_ERR_BAD_ARG, "%s: the parameters must be fp32 or of the rows' type", what);
  if (!(a.eps >= 0.f)) return fail(PRISM_ERR_BAD_ARG, "%s: eps must not be negative", what);
  if (a.weight == nullptr || (a.rows > 0 && a.x == nullptr)) return fail(PRISM_ERR_BAD_ARG, "%s: null tensor", what);
  if (!aligned_to(2, {a.x, a.residual, a.y, a.sum, a.dy, a.dsum, a.dx}) || !aligned_to(4, {a.mean, a.rstd}) ||
      !aligned_to(a.w_f32 ? 4 : 2, {a.weight, a.bias, a.dw, a.db}))
    return fail(PRISM_ERR_BAD_ARG, "%s: tensors must be aligned to their elements", what);
  if (a.ldx < 0 || a.ldr < 0 || a.lddy < 0 || a.ldds < 0) return fail(PRISM_ERR_BAD_ARG, "%s: negative row stride", what);
  return PRISM_OK;
}

}  // namespace

extern "C" int prism_layer_norm(const void* x, const void* residual, const void* weight, const void* bias, void* y, void* sum,
                                float* mean, float* rstd, long long rows, int cols, int dtype, int w_dtype, float eps,
                                long long ldx, long long ldr, void* stream) {
  NormArgs a{};
  a.x = x; a.residual = residual; a.weight = weight; a.bias = bias; a.y = y; a.sum = sum; a.mean = mean; a.rstd = rstd;
  a.rows = rows; a.cols = cols; a.dtype = dtype; a.w_f32 = w_dtype == PRISM_DTYPE_F32; a.eps = eps;
  a.ldx = ldx; a.ldr = ldr;
  a.stream = static_cast<cudaStream_t>(stream);
  if (int rc = check_norm("prism_layer_norm", a, w_dtype)) return rc;
  if ((residual == nullptr) != (sum == nullptr)) return fail(PRISM_ERR_BAD_ARG, "prism_layer_norm: residual and sum go together");
  if ((mean == nullptr) != (rstd == nullptr)) return fail(PRISM_ERR_BAD_ARG, "prism_layer_norm: mean and rstd go together");
  if (rows == 0) return PRISM_OK;
  if (y == nullptr) return fail(PRISM_ERR_BAD_ARG, "prism_layer_norm: null tensor");
  return launch_norm_fwd(a);
}

extern "C" size_t prism_layer_norm_scratch_bytes(long long rows, int cols) {
  if (rows < 0 || cols < 1 || cols > norm_max_cols()) return 0;
  return (size_t)norm_bwd_ctas(rows, cols, num_sms()) * 2 * cols * sizeof(float);
}

extern "C" int prism_layer_norm_bwd(const void* dy, const void* dsum, const void* s, const void* weight, const float* mean,
                                    const float* rstd, void* dx, void* dweight, void* dbias, long long rows, int cols, int dtype,
                                    int w_dtype, long long lddy, long long ldds, long long lds, void* scratch,
                                    size_t scratch_bytes, void* stream) {
  NormArgs a{};
  a.x = s; a.weight = weight; a.mean = const_cast<float*>(mean); a.rstd = const_cast<float*>(rstd);
  a.dy = dy; a.dsum = dsum; a.dx = dx; a.dw = dweight; a.db = dbias;
  a.rows = rows; a.cols = cols; a.dtype = dtype; a.w_f32 = w_dtype == PRISM_DTYPE_F32;
  a.ldx = lds; a.lddy = lddy; a.ldds = ldds;
  a.stream = static_cast<cudaStream_t>(stream);
  if (int rc = check_norm("prism_layer_norm_bwd", a, w_dtype)) return rc;
  if (rows > 0 && (dy == nullptr || dx == nullptr || mean == nullptr || rstd == nullptr))
    return fail(PRISM_ERR_BAD_ARG, "prism_layer_norm_bwd: null tensor");
  a.ctas = norm_bwd_ctas(rows, cols, num_sms());
  const size_t need = (size_t)a.ctas * 2 * cols * sizeof(float);
  if (scratch == nullptr || scratch_bytes < need)
    return fail(PRISM_ERR_WORKSPACE, "prism_layer_norm_bwd: scratch of %zu bytes, needs %zu", scratch_bytes, need);
  if (!aligned16(scratch)) return fail(PRISM_ERR_BAD_ARG, "prism_layer_norm_bwd: scratch must be 16-byte aligned");
  a.partial = static_cast<float*>(scratch);
  return launch_norm_bwd(a);
}
