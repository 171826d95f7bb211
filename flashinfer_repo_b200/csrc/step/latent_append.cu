// latent_append.cu -- writes new rows of the paged latent cache: the 512-wide
// latent normalised and weighted, the 64-wide rotary key turned to its position,
//   ckv[slot] = bf16(x * rsqrt(mean(x^2) + eps) * w),  kpe[slot] = bf16(turn(x[512:576])).
// Sums and products in 32 bits, one rounding at the store.
//
// One warp per row: 16 latent values and one rotary pair a lane, the sum of
// squares by shuffles, one angle a lane.  1152 bytes in and out a row: 16384 rows,
// 38 MB, take 6.8 us where inputs and cache are in L2, as behind the projection
// that made them, and 9.8 us from HBM (12 sets of them in turn): 3.9 TB/s, 59% of
// the copy rate.  That grid is over after three rounds of CTAs, so the first loads
// and the last round weigh.  A decode step is latency (64 rows 1.7-2.0 us).
#include "../../../include/dsa_b200.h"
#include "rotate.cuh"

namespace dsa {
namespace {

constexpr int kLatent = 512;

struct AppendParams {
  const void* kv;
  int64_t kv_st;
  const void* w;
  int64_t rows;
  const void* positions;
  int pos64;
  const int32_t* slots;
  const double* inv_freq;
  __nv_bfloat16 *ckv, *kpe;
  int64_t ckv_sp, ckv_sr, kpe_sp, kpe_sr, num_pages;
  float eps, scale;
  int half_layout;
  int* err;
};

// 8 values from `from` on as they are wanted in the sum: 32 bits.  kOnce: nobody
// reads them again, so they leave L2 first and push out less that has to be written
// back: 16384 rows behind 512 MB of other writes 12.3 instead of 14.3 us (timed by
// events around the call); 2-4% slower where L2 holds all or nothing of them (6.8
// against 6.5 us, 9.8 against 9.6).
template <typename T, bool kVec, bool kOnce>
__device__ __forceinline__ void load8(const T* from, float* v) {
  if (kVec) {
#pragma unroll
    for (int k = 0; k < 8 / Vec<T>::kN; ++k) {
      const uint4* at = reinterpret_cast<const uint4*>(from) + k;
      const uint4 raw = kOnce ? __ldcs(at) : *at;
      const Vec<T>& x = reinterpret_cast<const Vec<T>&>(raw);
#pragma unroll
      for (int i = 0; i < Vec<T>::kN; ++i) v[k * Vec<T>::kN + i] = to_f32(x.v[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f32(from[i]);
  }
}

// 4 rows a CTA: with 8 a decode step takes 1.88 instead of 1.70 us, 16384 rows 7.15
// instead of 6.8 (from L2) and 10.7 instead of 9.8.
constexpr int kAppendThreads = 128;

template <typename T, typename W, bool kVec>
__global__ void __launch_bounds__(kAppendThreads) dsa_latent_append_kernel(const AppendParams p) {
  const int64_t row = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (row >= p.rows) return;
  // every load of the row is issued before the first is needed
  const int32_t slot = p.slots[row];
  const T* x = static_cast<const T*>(p.kv) + row * p.kv_st;
  const W* w = static_cast<const W*>(p.w);
  const int ia = p.half_layout ? lane : 2 * lane, ib = p.half_layout ? lane + 32 : 2 * lane + 1;
  float v[2][8], g[2][8];
  load8<T, kVec, true>(x + lane * 8, v[0]);
  load8<T, kVec, true>(x + 256 + lane * 8, v[1]);
  const float a = to_f32(x[kLatent + ia]), b = to_f32(x[kLatent + ib]);
  const int64_t position = load_position(p.positions, p.pos64, row);
  load8<W, kVec, false>(w + lane * 8, g[0]);
  load8<W, kVec, false>(w + 256 + lane * 8, g[1]);
  const double freq = p.inv_freq[lane];
  if (slot < 0) {  // a padded row; anything below -1 is a wrong id
    if (slot < -1 && lane == 0) set_error(p.err, kErrBadIndex);
    return;
  }
  const int64_t page = slot >> 6, at = slot & 63;
  if (page >= p.num_pages) {
    if (lane == 0) set_error(p.err, kErrBadIndex);
    return;
  }
  float sum = 0.f;
#pragma unroll
  for (int k = 0; k < 16; ++k) sum += v[k >> 3][k & 7] * v[k >> 3][k & 7];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const float r = 1.f / sqrtf(sum * (1.f / kLatent) + p.eps);
  __nv_bfloat16* c = p.ckv + page * p.ckv_sp + at * p.ckv_sr;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    Vec<__nv_bfloat16> y;
#pragma unroll
    for (int i = 0; i < 8; ++i) y.v[i] = __float2bfloat16_rn(v[k][i] * r * g[k][i]);
    if (kVec) {
      *reinterpret_cast<Vec<__nv_bfloat16>*>(c + k * 256 + lane * 8) = y;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) c[k * 256 + lane * 8 + i] = y.v[i];
    }
  }
  float cs, sn;
  rotation(position, freq, p.scale, &cs, &sn);
  __nv_bfloat16* e = p.kpe + page * p.kpe_sp + at * p.kpe_sr;
  e[ia] = __float2bfloat16_rn(a * cs - b * sn);
  e[ib] = __float2bfloat16_rn(b * cs + a * sn);
}

template <typename T, typename W>
void launch(const AppendParams& p, cudaStream_t stream) {
  const unsigned grid = (unsigned)((p.rows * 32 + kAppendThreads - 1) / kAppendThreads);
  // 16-byte accesses where every row, the weights and the latent cache allow them
  bool vec = p.kv_st % Vec<T>::kN == 0 && p.ckv_sp % 8 == 0 && p.ckv_sr % 8 == 0;
  for (const void* q : {p.kv, p.w, (const void*)p.ckv}) vec = vec && (reinterpret_cast<uintptr_t>(q) & 15) == 0;
  if (vec)
    dsa_latent_append_kernel<T, W, true><<<grid, kAppendThreads, 0, stream>>>(p);
  else
    dsa_latent_append_kernel<T, W, false><<<grid, kAppendThreads, 0, stream>>>(p);
}
template <typename T>
void launch(const AppendParams& p, int w_dtype, cudaStream_t stream) {
  if (w_dtype == DSA_BF16)
    launch<T, __nv_bfloat16>(p, stream);
  else if (w_dtype == DSA_FP16)
    launch<T, __half>(p, stream);
  else
    launch<T, float>(p, stream);
}

}  // namespace
}  // namespace dsa

using namespace dsa;

extern "C" int dsa_latent_cache_append(const void* kv, int64_t kv_stride, int kv_dtype, const void* norm_weight,
                                       int norm_dtype, int64_t num_tokens, const void* positions,
                                       int positions_are_64_bit, const int32_t* slots, const double* inv_freq,
                                       void* ckv_cache, int64_t ckv_stride_page, int64_t ckv_stride_row,
                                       void* kpe_cache, int64_t kpe_stride_page, int64_t kpe_stride_row,
                                       int64_t num_pages, float eps, int layout, float rope_scale,
                                       int* device_error, void* stream) {
  if (num_tokens < 0 || num_pages < 0) return report_error(DSA_ERR_INVALID_ARG, "negative size");
  if (layout != DSA_ROPE_INTERLEAVED && layout != DSA_ROPE_HALF)
    return report_error(DSA_ERR_INVALID_ARG, "unknown rotary layout");
  for (int t : {kv_dtype, norm_dtype})
    if (t != DSA_BF16 && t != DSA_FP16 && t != DSA_FP32)
      return report_error(DSA_ERR_INVALID_ARG, "unknown element type");
  if (num_tokens == 0) return DSA_OK;
  if (num_tokens > INT32_MAX) return report_error(DSA_ERR_UNSUPPORTED, "tokens are counted in 32 bits");
  if (!kv || !norm_weight || !positions || !slots || !inv_freq || !ckv_cache || !kpe_cache)
    return report_error(DSA_ERR_INVALID_ARG, "NULL pointer argument");
  AppendParams p;
  p.kv = kv;
  p.kv_st = kv_stride;
  p.w = norm_weight;
  p.rows = num_tokens;
  p.positions = positions;
  p.pos64 = positions_are_64_bit != 0;
  p.slots = slots;
  p.inv_freq = inv_freq;
  p.ckv = static_cast<__nv_bfloat16*>(ckv_cache);
  p.kpe = static_cast<__nv_bfloat16*>(kpe_cache);
  p.ckv_sp = ckv_stride_page;
  p.ckv_sr = ckv_stride_row;
  p.kpe_sp = kpe_stride_page;
  p.kpe_sr = kpe_stride_row;
  p.num_pages = num_pages;
  p.eps = eps;
  p.scale = rope_scale;
  p.half_layout = layout == DSA_ROPE_HALF;
  p.err = device_error;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (kv_dtype == DSA_BF16)
    launch<__nv_bfloat16>(p, norm_dtype, s);
  else if (kv_dtype == DSA_FP16)
    launch<__half>(p, norm_dtype, s);
  else
    launch<float>(p, norm_dtype, s);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return report_error(DSA_ERR_CUDA, cudaGetErrorString(e));
  return DSA_OK;
}
