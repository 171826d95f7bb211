// rope.cu -- rotary positions on a slice of every head:
//   (a, b) -> (a cos - b sin, b cos + a sin),  angle = position * inv_freq[i],
// for the pairs (2i, 2i+1) or (i, i + rot/2) of the slice; the rest of the head
// is copied.  The inverse turns by the negative angle, which is also the
// gradient (the rotation's transpose).
//
// A CTA takes whole tokens, so that a token's rot/2 angles are computed once
// and serve all its heads.  Bound by HBM for many rows (each value is read and
// written once) and by latency for a decode step.
#include "../../../include/dsa_b200.h"
#include "rotate.cuh"

namespace dsa {
namespace {

constexpr int kRopeThreads = 256;
constexpr int kRopeMaxHalf = 256;  // angles per token (rot <= 512)

struct RopeParams {
  const void* x;
  void* out;
  int64_t x_st, x_sh, o_st, o_sh;
  int64_t tokens;
  int heads, dim, offset, rot;
  const void* positions;
  int pos64;
  const double* inv_freq;
  int inverse, tokens_per_cta;
  float scale;
};

template <typename T, bool kHalf>
__global__ void __launch_bounds__(kRopeThreads) dsa_rope_kernel(const RopeParams p) {
  __shared__ float cs[kRopeMaxHalf], sn[kRopeMaxHalf];
  const int half = p.rot / 2;
  for (int k = 0; k < p.tokens_per_cta; ++k) {
    const int64_t tok = (int64_t)blockIdx.x * p.tokens_per_cta + k;
    if (tok >= p.tokens) return;
    const int64_t pos = load_position(p.positions, p.pos64, tok);
    __syncthreads();
    for (int i = threadIdx.x; i < half; i += kRopeThreads) {
      float c, s;
      rotation(pos, p.inv_freq[i], p.scale, &c, &s);
      cs[i] = c;
      sn[i] = p.inverse ? -s : s;
    }
    __syncthreads();
    const T* x = static_cast<const T*>(p.x) + tok * p.x_st;
    T* o = static_cast<T*>(p.out) + tok * p.o_st;
    for (int e = threadIdx.x; e < p.heads * half; e += kRopeThreads) {
      const int h = e / half, i = e - h * half;
      const int ia = p.offset + (kHalf ? i : 2 * i), ib = kHalf ? ia + half : ia + 1;
      const float a = to_f32(x[h * p.x_sh + ia]), b = to_f32(x[h * p.x_sh + ib]);
      o[h * p.o_sh + ia] = from_f32<T>(a * cs[i] - b * sn[i]);
      o[h * p.o_sh + ib] = from_f32<T>(b * cs[i] + a * sn[i]);
    }
    if (p.x != p.out) {
      const int rest = p.dim - p.rot;
      for (int e = threadIdx.x; e < p.heads * rest; e += kRopeThreads) {
        const int h = e / rest, r = e - h * rest, d = r < p.offset ? r : r + p.rot;
        o[h * p.o_sh + d] = x[h * p.x_sh + d];
      }
    }
  }
}

template <typename T>
void launch(const RopeParams& p, int layout, cudaStream_t stream) {
  const unsigned grid = (unsigned)((p.tokens + p.tokens_per_cta - 1) / p.tokens_per_cta);
  if (layout == DSA_ROPE_HALF)
    dsa_rope_kernel<T, true><<<grid, kRopeThreads, 0, stream>>>(p);
  else
    dsa_rope_kernel<T, false><<<grid, kRopeThreads, 0, stream>>>(p);
}

}  // namespace
}  // namespace dsa

using namespace dsa;

extern "C" int dsa_apply_rope(const void* x, int64_t x_stride_token, int64_t x_stride_head, void* out,
                              int64_t out_stride_token, int64_t out_stride_head, int dtype,
                              int64_t num_tokens, int64_t num_heads, int64_t head_dim, int64_t rot_offset,
                              int64_t rot_dim, const void* positions, int positions_are_64_bit,
                              const double* inv_freq, int layout, int inverse, float scale, void* stream) {
  if (num_tokens < 0 || num_heads < 0 || head_dim < 0 || rot_offset < 0)
    return report_error(DSA_ERR_INVALID_ARG, "negative size");
  if (rot_dim < 2 || rot_dim % 2 || rot_dim > 2 * kRopeMaxHalf)
    return report_error(DSA_ERR_UNSUPPORTED, "rotated width must be even, 2 to 512");
  if (rot_offset + rot_dim > head_dim)
    return report_error(DSA_ERR_INVALID_ARG, "rotated slice reaches past the head");
  if (num_heads > 65535 || head_dim > 65535)
    return report_error(DSA_ERR_UNSUPPORTED, "at most 65535 heads of at most 65535 values");
  if (layout != DSA_ROPE_INTERLEAVED && layout != DSA_ROPE_HALF)
    return report_error(DSA_ERR_INVALID_ARG, "unknown rotary layout");
  if (dtype != DSA_BF16 && dtype != DSA_FP16 && dtype != DSA_FP32)
    return report_error(DSA_ERR_INVALID_ARG, "unknown element type");
  if (num_tokens == 0 || num_heads == 0) return DSA_OK;
  if (!x || !out || !positions || !inv_freq) return report_error(DSA_ERR_INVALID_ARG, "NULL pointer argument");
  RopeParams p;
  p.x = x;
  p.out = out;
  p.x_st = x_stride_token;
  p.x_sh = x_stride_head;
  p.o_st = out_stride_token;
  p.o_sh = out_stride_head;
  p.tokens = num_tokens;
  p.heads = (int)num_heads;
  p.dim = (int)head_dim;
  p.offset = (int)rot_offset;
  p.rot = (int)rot_dim;
  p.positions = positions;
  p.pos64 = positions_are_64_bit != 0;
  p.inv_freq = inv_freq;
  p.inverse = inverse != 0;
  p.scale = scale;
  p.tokens_per_cta = 1;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == DSA_BF16)
    launch<__nv_bfloat16>(p, layout, s);
  else if (dtype == DSA_FP16)
    launch<__half>(p, layout, s);
  else
    launch<float>(p, layout, s);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return report_error(DSA_ERR_CUDA, cudaGetErrorString(e));
  return DSA_OK;
}
