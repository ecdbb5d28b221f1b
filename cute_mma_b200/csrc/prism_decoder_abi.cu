// extern "C" entry points of the operators between the linears of a decoder: argument checks, dispatch to the launchers.
#include "../../include/prism_b200.h"
#include "prism_attn_host.cuh"
#include "prism_host.cuh"

using namespace prism;

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int check_workspace(const char* what, void* workspace, size_t bytes) {
  if (workspace == nullptr || bytes < PRISM_WORKSPACE_HEADER_BYTES)
    return fail(PRISM_ERR_WORKSPACE, "%s: the workspace must hold its status header (%d bytes)", what, PRISM_WORKSPACE_HEADER_BYTES);
  if ((reinterpret_cast<uintptr_t>(workspace) & 255) != 0)
    return fail(PRISM_ERR_BAD_ARG, "%s: the workspace must be 256-byte aligned", what);
  return PRISM_OK;
}

AttnStrides strides_at(const long long* s, int i) { return AttnStrides{s[3 * i], s[3 * i + 1], s[3 * i + 2]}; }

int check_attn(const char* what, const AttnArgs& a, const long long* strides, int n_strides) {
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
      !aligned16(a.dk) || !aligned16(a.dv))
    return fail(PRISM_ERR_BAD_ARG, "%s: tensors must be 16-byte aligned", what);
  return PRISM_OK;
}

}  // namespace

extern "C" int prism_attn_fwd(const void* q, const void* k, const void* v, void* o, float* lse, const int* cu_seqlens,
                              int n_seqs, int seq_len, int rows, int heads, int kv_heads, int head_dim, int dtype, float scale,
                              const long long* strides, void* workspace, size_t workspace_bytes, void* stream) {
  AttnArgs a{};
  a.q = q; a.k = k; a.v = v; a.o = o; a.lse = lse;
  a.cu = cu_seqlens; a.n = n_seqs; a.len = seq_len; a.rows = rows;
  a.hq = heads; a.hkv = kv_heads; a.dim = head_dim; a.dtype = dtype; a.scale = scale;
  if (int rc = check_attn("prism_attn_fwd", a, strides, 9)) return rc;
  a.sq = strides_at(strides, 0); a.sk = strides_at(strides, 1); a.sv = strides_at(strides, 2);
  if (int rc = check_workspace("prism_attn_fwd", workspace, workspace_bytes)) return rc;
  a.err = static_cast<int*>(workspace);
  a.stream = static_cast<cudaStream_t>(stream);
  return launch_attn_fwd(a);
}

extern "C" int prism_attn_bwd(const void* d_o, const void* q, const void* k, const void* v, const void* o, const float* lse,
                              void* dq, void* dk, void* dv, float* delta, const int* cu_seqlens, int n_seqs, int seq_len,
                              int rows, int heads, int kv_heads, int head_dim, int dtype, float scale,
                              const long long* strides, void* workspace, size_t workspace_bytes, void* stream) {
  AttnArgs a{};
  a.q = q; a.k = k; a.v = v; a.o = const_cast<void*>(o); a.lse = const_cast<float*>(lse); a.d_o = d_o;
  a.dq = dq; a.dk = dk; a.dv = dv; a.delta = delta;
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
