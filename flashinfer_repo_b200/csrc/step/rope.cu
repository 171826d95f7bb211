// rope.cu -- rotary positions on a slice of every head:
//   (a, b) -> (a cos - b sin, b cos + a sin),  angle = position * inv_freq[i],
// for the pairs (2i, 2i+1) or (i, i + rot/2) of the slice; the rest of the head
// is copied.  The inverse turns by the negative angle, which is also the
// gradient (the rotation's transpose).
//
// A CTA takes whole tokens, so that a token's rot/2 angles are computed once
// and serve all its heads.  Bound by HBM for many rows (each value is read and
// written once) and by latency for a decode step.  Aligned tensors go by 16
// bytes a thread and access, four of them in flight while the angles are
// computed; others value by value.
#include "../../../include/dsa_b200.h"
#include "rotate.cuh"

namespace dsa {
namespace {

constexpr int kRopeThreads = 256;
constexpr int kRopeMaxHalf = 256;  // angles per token (rot <= 512)
constexpr int kRopeAngles = 1024;  // angles in shared memory

struct RopeParams {
  const void* x;
  void* out;
  int64_t x_st, x_sh, o_st, o_sh;
  int64_t tokens;
  int heads, dim, offset, rot;
  const void* positions;
  int pos64;
  const double* inv_freq;
  int inverse, tokens_per_cta, per_head;  // per_head: units of a head
  uint32_t inv_per_head, inv_heads;        // 2^32 / divisor, rounded up
  float scale;
};

__device__ __forceinline__ void angles(const RopeParams& p, int64_t first, int tokens, float* cs, float* sn) {
  const int half = p.rot / 2;
  for (int i = threadIdx.x; i < tokens * half; i += kRopeThreads) {
    const int k = i / half;
    float c, s;
    rotation(load_position(p.positions, p.pos64, first + k), p.inv_freq[i - k * half], p.scale, &c, &s);
    cs[i] = c;
    sn[i] = p.inverse ? -s : s;
  }
}

// A unit is one access of a head: a 16-byte vector of the rotated slice (kHalf:
// one of its first half and its partner), or one of the rest, which is copied.
template <typename T, bool kHalf>
__global__ void __launch_bounds__(kRopeThreads) dsa_rope_vec_kernel(const RopeParams p) {
  constexpr int kN = Vec<T>::kN, kUnroll = 4;
  __shared__ float cs[kRopeAngles], sn[kRopeAngles];
  const int64_t first = (int64_t)blockIdx.x * p.tokens_per_cta;
  const int tokens = (int)min((int64_t)p.tokens_per_cta, p.tokens - first);
  const int half = p.rot / 2, turned = (kHalf ? half : p.rot) / kN;
  const int units = p.heads * p.per_head, total = tokens * units;
  const T* x = static_cast<const T*>(p.x) + first * p.x_st;
  T* o = static_cast<T*>(p.out) + first * p.o_st;
  for (int e0 = threadIdx.x; e0 - (int)threadIdx.x < total; e0 += kUnroll * kRopeThreads) {
    Vec<T> a[kUnroll], b[kUnroll];
    int at[kUnroll], slot[kUnroll], tok[kUnroll], head[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int e = e0 + u * kRopeThreads;
      slot[u] = -1;
      if (e < total) {
        const int hh = __umulhi(e, p.inv_per_head);  // e / per_head
        slot[u] = e - hh * p.per_head;
        tok[u] = __umulhi(hh, p.inv_heads);  // hh / heads
        head[u] = hh - tok[u] * p.heads;
        if (slot[u] < turned) {
          at[u] = p.offset + slot[u] * kN;
        } else {
          at[u] = (slot[u] - turned) * kN;
          if (at[u] >= p.offset) at[u] += p.rot;
        }
        const T* src = x + tok[u] * p.x_st + head[u] * p.x_sh + at[u];
        a[u] = *reinterpret_cast<const Vec<T>*>(src);
        if (kHalf && slot[u] < turned) b[u] = *reinterpret_cast<const Vec<T>*>(src + half);
      }
    }
    if (e0 == (int)threadIdx.x) {  // the first loads are on their way meanwhile
      angles(p, first, tokens, cs, sn);
      __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (slot[u] < 0) continue;
      T* dst = o + tok[u] * p.o_st + head[u] * p.o_sh + at[u];
      if (slot[u] < turned) {
        const int i0 = tok[u] * half + slot[u] * (kHalf ? kN : kN / 2);
        if (kHalf) {
          Vec<T> r;
#pragma unroll
          for (int i = 0; i < kN; ++i) {
            const float c = cs[i0 + i], s = sn[i0 + i], va = to_f32(a[u].v[i]), vb = to_f32(b[u].v[i]);
            a[u].v[i] = from_f32<T>(va * c - vb * s);
            r.v[i] = from_f32<T>(vb * c + va * s);
          }
          *reinterpret_cast<Vec<T>*>(dst + half) = r;
        } else {
#pragma unroll
          for (int i = 0; i < kN / 2; ++i) {
            const float c = cs[i0 + i], s = sn[i0 + i], va = to_f32(a[u].v[2 * i]), vb = to_f32(a[u].v[2 * i + 1]);
            a[u].v[2 * i] = from_f32<T>(va * c - vb * s);
            a[u].v[2 * i + 1] = from_f32<T>(vb * c + va * s);
          }
        }
      }
      *reinterpret_cast<Vec<T>*>(dst) = a[u];
    }
  }
}

// Any alignment: a pair of values, or a value of the rest, at a time.
template <typename T, bool kHalf>
__global__ void __launch_bounds__(kRopeThreads) dsa_rope_kernel(const RopeParams p) {
  __shared__ float cs[kRopeAngles], sn[kRopeAngles];
  const int64_t first = (int64_t)blockIdx.x * p.tokens_per_cta;
  const int tokens = (int)min((int64_t)p.tokens_per_cta, p.tokens - first);
  const int half = p.rot / 2;
  angles(p, first, tokens, cs, sn);
  __syncthreads();
  for (int k = 0; k < tokens; ++k) {
    const T* x = static_cast<const T*>(p.x) + (first + k) * p.x_st;
    T* o = static_cast<T*>(p.out) + (first + k) * p.o_st;
    for (int e = threadIdx.x; e < p.heads * half; e += kRopeThreads) {
      const int h = e / half, i = e - h * half;
      const int ia = p.offset + (kHalf ? i : 2 * i), ib = kHalf ? ia + half : ia + 1;
      const float a = to_f32(x[h * p.x_sh + ia]), b = to_f32(x[h * p.x_sh + ib]);
      const float c = cs[k * half + i], s = sn[k * half + i];
      o[h * p.o_sh + ia] = from_f32<T>(a * c - b * s);
      o[h * p.o_sh + ib] = from_f32<T>(b * c + a * s);
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
void launch(RopeParams p, int layout, cudaStream_t stream) {
  constexpr int kN = Vec<T>::kN;
  const bool half = layout == DSA_ROPE_HALF;
  const int turned = half ? p.rot / 2 : p.rot;
  bool vec = turned % kN == 0 && p.offset % kN == 0 && p.dim % kN == 0;
  for (int64_t s : {p.x_st, p.x_sh, p.o_st, p.o_sh}) vec = vec && s % kN == 0;
  for (const void* q : {p.x, (const void*)p.out}) vec = vec && (reinterpret_cast<uintptr_t>(q) & 15) == 0;
  p.per_head = turned / kN + (p.x == p.out ? 0 : (p.dim - p.rot) / kN);
  // tokens of a CTA: four units a thread, but one CTA at least for every SM, and
  // the angles in shared memory
  const int64_t units = (int64_t)p.heads * (p.per_head < 1 ? 1 : p.per_head), angles = kRopeAngles / (p.rot / 2);
  int64_t per_cta = 4 * kRopeThreads / units;
  per_cta = per_cta < p.tokens / 148 ? per_cta : p.tokens / 148;
  per_cta = per_cta < angles ? per_cta : angles;
  p.tokens_per_cta = (int)(per_cta < 1 ? 1 : per_cta);
  // the divisions by multiplication are exact while numerator * divisor < 2^32
  const int64_t top = units * p.tokens_per_cta;
  vec = vec && top * p.per_head < (1LL << 32) && top / (p.per_head < 1 ? 1 : p.per_head) * p.heads < (1LL << 32);
  const unsigned grid = (unsigned)((p.tokens + p.tokens_per_cta - 1) / p.tokens_per_cta);
  if (vec) {
    p.inv_per_head = (uint32_t)(((1ULL << 32) + p.per_head - 1) / p.per_head);
    p.inv_heads = (uint32_t)(((1ULL << 32) + p.heads - 1) / p.heads);
    if (half)
      dsa_rope_vec_kernel<T, true><<<grid, kRopeThreads, 0, stream>>>(p);
    else
      dsa_rope_vec_kernel<T, false><<<grid, kRopeThreads, 0, stream>>>(p);
  } else if (half) {
    dsa_rope_kernel<T, true><<<grid, kRopeThreads, 0, stream>>>(p);
  } else {
    dsa_rope_kernel<T, false><<<grid, kRopeThreads, 0, stream>>>(p);
  }
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
  if (num_tokens > INT32_MAX) return report_error(DSA_ERR_UNSUPPORTED, "tokens are counted in 32 bits");
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
