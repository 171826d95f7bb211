// prefix.cu -- dense attention over the paged latent cache for a batch whose
// requests share one prefix: token t attends to the prefix's rows and then to
// the first token_lens[t] rows of its request's own pages,
//   o = sum_k p_k ckv_k / sum_k p_k,  p_k = exp(sm_scale (q_nope.ckv_k + q_pe.kpe_k)),
//   lse = log2 sum_k p_k.
// One pass over the rows with the running maximum and sum of the softmax.
#include "../../../include/dsa_b200.h"
#include "../common.cuh"

namespace dsa {
namespace {

constexpr int kPreThreads = 256;
constexpr int kRowPitch = 584;  // 576 values and 16 bytes: rows start in different banks

struct PrefixParams {
  const __nv_bfloat16 *qn, *qp, *ckv, *kpe;
  int64_t qn_st, qn_sh, qp_st, qp_sh, ckv_sp, ckv_sr, kpe_sp, kpe_sr;
  const int32_t *prefix_pages, *prefix_len, *block_table, *token_request, *token_lens;
  int64_t max_prefix, bt_stride, batch, max_pages, tokens, num_pages;
  int heads;
  float scale_log2;
  __nv_bfloat16* out;
  int64_t out_st, out_sh;
  float* lse;
  int64_t lse_st, lse_sh;
  int* err;
};

struct PreSmem {
  __nv_bfloat16 kv[64][kRowPitch];
  __nv_bfloat16 q[16][kRowPitch];
  float s[16][64];
  float m[16], l[16], alpha[16];
};

__global__ void __launch_bounds__(kPreThreads) dsa_prefix_attention_kernel(const PrefixParams p) {
  extern __shared__ uint8_t raw[];
  PreSmem& S = *reinterpret_cast<PreSmem*>(raw);
  const int64_t t = blockIdx.x;
  const int h0 = blockIdx.y * 16, tid = threadIdx.x;
  for (int e = tid; e < 16 * 576; e += kPreThreads) {
    const int h = e / 576, d = e % 576;
    S.q[h][d] = d < 512 ? p.qn[t * p.qn_st + (h0 + h) * p.qn_sh + d] : p.qp[t * p.qp_st + (h0 + h) * p.qp_sh + d - 512];
  }
  if (tid < 16) {
    S.m[tid] = -INFINITY;
    S.l[tid] = 0.f;
  }
  int64_t prefix = p.max_prefix;
  if (p.prefix_len) prefix = min(prefix, (int64_t)max(*p.prefix_len, 0));
  int64_t own = max(p.token_lens[t], 0), req = p.token_request ? p.token_request[t] : t;
  if (own > 0 && (req < 0 || req >= p.batch || own > p.max_pages * 64)) {
    if (tid == 0) set_error(p.err, kErrBadIndex);
    own = (req < 0 || req >= p.batch) ? 0 : p.max_pages * 64;
  }
  const int64_t pre_pages = (prefix + 63) / 64, pages = pre_pages + (own + 63) / 64;
  float o[16][2] = {};
  for (int64_t k = 0; k < pages; ++k) {
    const bool is_own = k >= pre_pages;
    const int64_t kk = is_own ? k - pre_pages : k;
    const int32_t page = is_own ? p.block_table[req * p.bt_stride + kk] : p.prefix_pages[kk];
    int valid = (int)min((int64_t)64, (is_own ? own : prefix) - kk * 64);
    if (page < 0 || page >= p.num_pages) {
      if (tid == 0) set_error(p.err, kErrBadIndex);
      valid = 0;
    }
    __syncthreads();
    for (int e = tid; e < 64 * 72; e += kPreThreads) {
      const int r = e / 72, c = e % 72;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (r < valid)
        v = c < 64 ? *reinterpret_cast<const uint4*>(p.ckv + page * p.ckv_sp + r * p.ckv_sr + c * 8)
                   : *reinterpret_cast<const uint4*>(p.kpe + page * p.kpe_sp + r * p.kpe_sr + (c - 64) * 8);
      *reinterpret_cast<uint4*>(&S.kv[r][c * 8]) = v;
    }
    __syncthreads();
    {
      const int r = tid & 63, hb = (tid >> 6) * 4;
      float acc[4] = {};
      for (int d = 0; d < 576; ++d) {
        const float kv = __bfloat162float(S.kv[r][d]);
#pragma unroll
        for (int h = 0; h < 4; ++h) acc[h] += __bfloat162float(S.q[hb + h][d]) * kv;
      }
#pragma unroll
      for (int h = 0; h < 4; ++h) S.s[hb + h][r] = r < valid ? acc[h] * p.scale_log2 : -INFINITY;
    }
    __syncthreads();
    if (tid < 16) {
      float top = S.m[tid];
      for (int r = 0; r < 64; ++r) top = fmaxf(top, S.s[tid][r]);
      const float a = top == -INFINITY ? 1.f : exp2f(S.m[tid] - top);
      float l = S.l[tid] * a;
      for (int r = 0; r < 64; ++r) {
        const float e = r < valid ? exp2f(S.s[tid][r] - top) : 0.f;
        S.s[tid][r] = e;
        l += e;
      }
      S.m[tid] = top;
      S.l[tid] = l;
      S.alpha[tid] = a;
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 16; ++h) {
      o[h][0] *= S.alpha[h];
      o[h][1] *= S.alpha[h];
    }
    for (int r = 0; r < valid; ++r) {
      const float v0 = __bfloat162float(S.kv[r][2 * tid]), v1 = __bfloat162float(S.kv[r][2 * tid + 1]);
#pragma unroll
      for (int h = 0; h < 16; ++h) {
        o[h][0] += S.s[h][r] * v0;
        o[h][1] += S.s[h][r] * v1;
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int h = 0; h < 16; ++h) {
    const float inv = S.l[h] == 0.f ? 0.f : 1.f / S.l[h];
    *reinterpret_cast<uint32_t*>(p.out + t * p.out_st + (h0 + h) * p.out_sh + 2 * tid) =
        pack_bf16(o[h][0] * inv, o[h][1] * inv);
  }
  if (tid < 16) p.lse[t * p.lse_st + (h0 + tid) * p.lse_sh] = S.l[tid] == 0.f ? -INFINITY : S.m[tid] + log2f(S.l[tid]);
}

}  // namespace
}  // namespace dsa

using namespace dsa;

extern "C" int dsa_shared_prefix_attention_workspace_size(int64_t num_tokens, int64_t num_heads, size_t* bytes) {
  if (!bytes) return report_error(DSA_ERR_INVALID_ARG, "NULL pointer argument");
  if (num_tokens < 0) return report_error(DSA_ERR_INVALID_ARG, "negative size");
  if (num_heads <= 0 || num_heads % 16) return report_error(DSA_ERR_INVALID_ARG, "heads must be a positive multiple of 16");
  *bytes = 256;
  return DSA_OK;
}

extern "C" int dsa_shared_prefix_attention(
    const void* q_nope, int64_t q_nope_stride_token, int64_t q_nope_stride_head, const void* q_pe,
    int64_t q_pe_stride_token, int64_t q_pe_stride_head, const void* ckv_cache, int64_t ckv_stride_page,
    int64_t ckv_stride_row, const void* kpe_cache, int64_t kpe_stride_page, int64_t kpe_stride_row,
    const int32_t* prefix_pages, int64_t max_prefix_len, const int32_t* prefix_len, const int32_t* block_table,
    int64_t block_table_stride, int64_t batch, int64_t max_pages, const int32_t* token_request,
    const int32_t* token_lens, int64_t num_tokens, int64_t num_heads, int64_t num_pages, float sm_scale,
    void* output, int64_t out_stride_token, int64_t out_stride_head, float* lse, int64_t lse_stride_token,
    int64_t lse_stride_head, void* workspace, size_t workspace_bytes, void* stream) {
  size_t need = 0;
  const int rc = dsa_shared_prefix_attention_workspace_size(num_tokens, num_heads, &need);
  if (rc != DSA_OK) return rc;
  if (max_prefix_len < 0 || batch < 0 || max_pages < 0 || num_pages < 0)
    return report_error(DSA_ERR_INVALID_ARG, "negative size");
  if (num_tokens == 0) return DSA_OK;
  if (!q_nope || !q_pe || !ckv_cache || !kpe_cache || !token_lens || !output || !lse || !workspace ||
      (max_prefix_len > 0 && !prefix_pages) || (batch > 0 && max_pages > 0 && !block_table))
    return report_error(DSA_ERR_INVALID_ARG, "NULL pointer argument");
  if (!token_request && batch < num_tokens)
    return report_error(DSA_ERR_INVALID_ARG, "without token_request the block table needs a row for every token");
  for (const void* q : {q_nope, q_pe, ckv_cache, kpe_cache})
    if (reinterpret_cast<uintptr_t>(q) & 15) return report_error(DSA_ERR_INVALID_ARG, "queries and caches must be 16-byte aligned");
  for (int64_t s : {q_nope_stride_token, q_nope_stride_head, q_pe_stride_token, q_pe_stride_head, ckv_stride_page,
                    ckv_stride_row, kpe_stride_page, kpe_stride_row})
    if (s < 0 || s % 8) return report_error(DSA_ERR_INVALID_ARG, "query and cache strides must be multiples of 8 elements");
  if ((reinterpret_cast<uintptr_t>(output) & 15) || out_stride_token % 8 || out_stride_head % 8)
    return report_error(DSA_ERR_INVALID_ARG, "output rows must be 16-byte aligned");
  if (workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255))
    return report_error(DSA_ERR_WORKSPACE, "workspace too small or not 256-byte aligned");
  PrefixParams p;
  p.qn = static_cast<const __nv_bfloat16*>(q_nope);
  p.qp = static_cast<const __nv_bfloat16*>(q_pe);
  p.ckv = static_cast<const __nv_bfloat16*>(ckv_cache);
  p.kpe = static_cast<const __nv_bfloat16*>(kpe_cache);
  p.qn_st = q_nope_stride_token;
  p.qn_sh = q_nope_stride_head;
  p.qp_st = q_pe_stride_token;
  p.qp_sh = q_pe_stride_head;
  p.ckv_sp = ckv_stride_page;
  p.ckv_sr = ckv_stride_row;
  p.kpe_sp = kpe_stride_page;
  p.kpe_sr = kpe_stride_row;
  p.prefix_pages = prefix_pages;
  p.prefix_len = prefix_len;
  p.block_table = block_table;
  p.token_request = token_request;
  p.token_lens = token_lens;
  p.max_prefix = max_prefix_len;
  p.bt_stride = block_table_stride;
  p.batch = batch;
  p.max_pages = max_pages;
  p.tokens = num_tokens;
  p.num_pages = num_pages;
  p.heads = (int)num_heads;
  p.scale_log2 = sm_scale * 1.44269504088896340736f;
  p.out = static_cast<__nv_bfloat16*>(output);
  p.out_st = out_stride_token;
  p.out_sh = out_stride_head;
  p.lse = lse;
  p.lse_st = lse_stride_token;
  p.lse_sh = lse_stride_head;
  p.err = static_cast<int*>(workspace);
  cudaError_t e = cudaFuncSetAttribute(dsa_prefix_attention_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       (int)sizeof(PreSmem));
  if (e != cudaSuccess) return report_error(DSA_ERR_CUDA, cudaGetErrorString(e));
  dsa_prefix_attention_kernel<<<dim3((unsigned)num_tokens, (unsigned)(num_heads / 16)), kPreThreads, sizeof(PreSmem),
                                static_cast<cudaStream_t>(stream)>>>(p);
  e = cudaGetLastError();
  if (e != cudaSuccess) return report_error(DSA_ERR_CUDA, cudaGetErrorString(e));
  return DSA_OK;
}
