// rope.cu -- rotary positions on a slice of every head:
//   (a, b) -> (a cos - b sin, b cos + a sin),  angle = position * inv_freq[i],
// for the pairs (2i, 2i+1) or (i, i + rot/2) of the slice; the rest of the head
// is copied.  The inverse turns by the negative angle, which is also the
// gradient (the rotation's transpose).
//
// A warp takes a token and a stretch of its heads: its lanes compute the token's
// rot/2 angles (one each for the usual 64-wide slice) into shared memory, and no
// barrier of a CTA is in the way.  Bound by HBM for many rows, each value read and
// written once (134 MB of half-layout bf16 25.0 us, 197 MB of interleaved fp32 31.8
// us: 82% and 95% of the copy rate), and by latency for a decode step (2.0 us).  Aligned tensors go by 16
// bytes a lane and access, all of them loaded before the angles are computed;
// others value by value.
#include "../../../include/dsa_b200.h"
#include "rotate.cuh"

namespace dsa {
namespace {

constexpr int kRopeWarps = 4;
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
  int inverse, turned, rest, units, chunks;  // units of a head that turn and that do not, of a token; warps a token
  uint32_t inv_turned, inv_rest;             // 2^32 / turned, 2^32 / rest, rounded up
  float scale;
};

// cos and sin of a token's angles, by the lanes of a warp.
__device__ __forceinline__ void angles(const RopeParams& p, int64_t token, float* cs, float* sn) {
  const int64_t position = load_position(p.positions, p.pos64, token);
  for (int i = threadIdx.x & 31; i < p.rot / 2; i += 32) {
    float c, s;
    rotation(position, p.inv_freq[i], p.scale, &c, &s);
    cs[i] = c;
    sn[i] = p.inverse ? -s : s;
  }
  __syncwarp();
}

// A unit is 16 bytes of a head.  The units that turn come first, of all heads:
// mixed in a warp with the others, which are copied, they would keep its lanes
// waiting.  In the half layout the partner of a unit is rot/2 values away, in
// another lane: the lanes of a head swap their units by shuffles, so that loads
// and stores stay whole lines (a lane that loads both its halves itself moves
// half lines: 33-46 instead of 26 us for 134 MB of bf16, half of it turned).
template <typename T, bool kHalf, int kUnits>
__global__ void __launch_bounds__(32 * kRopeWarps) dsa_rope_vec_kernel(const RopeParams p) {
  constexpr int kN = Vec<T>::kN;
  __shared__ __align__(16) float cs_all[kRopeWarps][kRopeMaxHalf], sn_all[kRopeWarps][kRopeMaxHalf];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t task = (int64_t)blockIdx.x * kRopeWarps + warp, token = task / p.chunks;
  if (token >= p.tokens) return;
  float *cs = cs_all[warp], *sn = sn_all[warp];
  const int turning = p.heads * p.turned;
  const int first = (int)(task - token * p.chunks) * (32 * kUnits) + lane;
  const T* x = static_cast<const T*>(p.x) + token * p.x_st;
  T* o = static_cast<T*>(p.out) + token * p.o_st;
  Vec<T> a[kUnits];
  auto place = [&](int e, int* head, int* slot) -> int {  // first value of the unit in its head
    if (e < turning) {
      *head = p.turned == 1 ? e : __umulhi(e, p.inv_turned);
      *slot = e - *head * p.turned;
      return p.offset + *slot * kN;
    }
    e -= turning;
    *head = p.rest == 1 ? e : __umulhi(e, p.inv_rest);
    const int at = (e - *head * p.rest) * kN;
    return at < p.offset ? at : at + p.rot;
  };
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const int e = first + 32 * u;
    if (e < p.units) {
      int head, slot;
      const int at = place(e, &head, &slot);
      a[u] = *reinterpret_cast<const Vec<T>*>(x + head * p.x_sh + at);
    }
  }
  angles(p, token, cs, sn);
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const int e = first + 32 * u;
    Vec<T> other;
    if (kHalf) {  // a head's lanes lie side by side: turned is a power of two up to 32
#pragma unroll
      for (int i = 0; i < 4; ++i)
        reinterpret_cast<uint32_t*>(&other)[i] =
            __shfl_xor_sync(0xffffffffu, reinterpret_cast<const uint32_t*>(&a[u])[i], p.turned >> 1);
    }
    if (e >= p.units) continue;
    int head, slot;
    const int at = place(e, &head, &slot);
    if (e < turning) {
      constexpr int kA = kHalf ? kN : kN / 2, kQ = kA < 4 ? kA : 4;  // angles of the unit, of a shared load
      struct __align__(4 * kQ) Angles {
        float v[kQ];
      };
      const bool second = kHalf && slot >= p.turned / 2;
      const int i0 = (second ? slot - p.turned / 2 : slot) * kA;
#pragma unroll
      for (int q = 0; q < kA; q += kQ) {
        const Angles c = *reinterpret_cast<const Angles*>(cs + i0 + q);
        const Angles s = *reinterpret_cast<const Angles*>(sn + i0 + q);
#pragma unroll
        for (int i = 0; i < kQ; ++i) {
          if (kHalf) {
            const float mine = to_f32(a[u].v[q + i]), its = to_f32(other.v[q + i]);
            a[u].v[q + i] = from_f32<T>(mine * c.v[i] + its * (second ? s.v[i] : -s.v[i]));
          } else {
            const float va = to_f32(a[u].v[2 * (q + i)]), vb = to_f32(a[u].v[2 * (q + i) + 1]);
            a[u].v[2 * (q + i)] = from_f32<T>(va * c.v[i] - vb * s.v[i]);
            a[u].v[2 * (q + i) + 1] = from_f32<T>(vb * c.v[i] + va * s.v[i]);
          }
        }
      }
    }
    *reinterpret_cast<Vec<T>*>(o + head * p.o_sh + at) = a[u];
  }
}

// Any alignment: a warp per token, a pair of values or a value of the rest at a time.
template <typename T, bool kHalf>
__global__ void __launch_bounds__(32 * kRopeWarps) dsa_rope_kernel(const RopeParams p) {
  __shared__ float cs_all[kRopeWarps][kRopeMaxHalf], sn_all[kRopeWarps][kRopeMaxHalf];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t token = (int64_t)blockIdx.x * kRopeWarps + warp;
  if (token >= p.tokens) return;
  float *cs = cs_all[warp], *sn = sn_all[warp];
  const int half = p.rot / 2;
  angles(p, token, cs, sn);
  const T* x = static_cast<const T*>(p.x) + token * p.x_st;
  T* o = static_cast<T*>(p.out) + token * p.o_st;
  for (int e = lane; e < p.heads * half; e += 32) {
    const int h = e / half, i = e - h * half;
    const int ia = p.offset + (kHalf ? i : 2 * i), ib = kHalf ? ia + half : ia + 1;
    const float a = to_f32(x[h * p.x_sh + ia]), b = to_f32(x[h * p.x_sh + ib]);
    o[h * p.o_sh + ia] = from_f32<T>(a * cs[i] - b * sn[i]);
    o[h * p.o_sh + ib] = from_f32<T>(b * cs[i] + a * sn[i]);
  }
  if (p.x != p.out) {
    const int rest = p.dim - p.rot;
    for (int e = lane; e < p.heads * rest; e += 32) {
      const int h = e / rest, r = e - h * rest, d = r < p.offset ? r : r + p.rot;
      o[h * p.o_sh + d] = x[h * p.x_sh + d];
    }
  }
}

template <typename T, bool kHalf>
void launch(RopeParams p, cudaStream_t stream) {
  constexpr int kN = Vec<T>::kN, kMany = 4;
  p.turned = p.rot / kN;
  p.rest = p.x == p.out ? 0 : (p.dim - p.rot) / kN;
  const int64_t units = (int64_t)p.heads * (p.turned + p.rest), widest = p.turned > p.rest ? p.turned : p.rest;
  // the divisions by multiplication are exact while numerator * divisor < 2^32
  bool vec = p.rot % kN == 0 && p.offset % kN == 0 && p.dim % kN == 0 && units * widest < (1LL << 32);
  if (kHalf) vec = vec && p.turned >= 2 && p.turned <= 32 && (p.turned & (p.turned - 1)) == 0;
  for (int64_t s : {p.x_st, p.x_sh, p.o_st, p.o_sh}) vec = vec && s % kN == 0;
  for (const void* q : {p.x, (const void*)p.out}) vec = vec && (reinterpret_cast<uintptr_t>(q) & 15) == 0;
  if (vec) {
    p.units = (int)units;
    p.inv_turned = (uint32_t)(((1ULL << 32) + p.turned - 1) / p.turned);
    p.inv_rest = p.rest ? (uint32_t)(((1ULL << 32) + p.rest - 1) / p.rest) : 0;
    // four units a lane keep enough bytes in flight (197 MB of fp32: 32 us, 44
    // with one); where that leaves SMs without a CTA, one unit a lane is sooner
    // done (64 tokens of 16 heads: 2.1 us, 3.2 with four)
    auto grid = [&](int per_lane) {
      p.chunks = (p.units + 32 * per_lane - 1) / (32 * per_lane);
      return (unsigned)((p.tokens * p.chunks + kRopeWarps - 1) / kRopeWarps);
    };
    const unsigned ctas = grid(kMany);
    if (ctas >= 148)
      dsa_rope_vec_kernel<T, kHalf, kMany><<<ctas, 32 * kRopeWarps, 0, stream>>>(p);
    else
      dsa_rope_vec_kernel<T, kHalf, 1><<<grid(1), 32 * kRopeWarps, 0, stream>>>(p);
  } else {
    dsa_rope_kernel<T, kHalf><<<(unsigned)((p.tokens + kRopeWarps - 1) / kRopeWarps), 32 * kRopeWarps, 0, stream>>>(p);
  }
}
template <typename T>
void launch(const RopeParams& p, int layout, cudaStream_t stream) {
  if (layout == DSA_ROPE_HALF)
    launch<T, true>(p, stream);
  else
    launch<T, false>(p, stream);
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
  if (num_heads > 65535 || head_dim > 65535 || num_heads * head_dim > (1 << 28))
    return report_error(DSA_ERR_UNSUPPORTED, "at most 65535 heads of at most 65535 values, and 2^28 values a token");
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
