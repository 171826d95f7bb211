// umma_chain.cu -- issue cost of thin tcgen05.mma (kind::f16) on this GPU, as a
// function of the MMA shape and of how many independent accumulators the
// stream of MMAs rotates over.  A measurement probe for the attention
// kernels (no counterpart in the reference): with 16 heads the attention
// MMAs have N=16, so each one is short and a chain of MMAs that accumulate
// into the same TMEM columns may be paced by the accumulate dependency
// rather than by the tensor pipe.
//
// One CTA per SM; one thread issues R MMAs (operands: one 128-byte-swizzled
// K-major panel of A [M x 64] and of B [N x 64] in shared memory, K=16 per
// MMA, stepping through the panel), MMA r accumulating into accumulator
// r % C (C TMEM regions of N columns), then one commit; the clock64 interval
// from the first issue to the commit's arrival, divided by R, is the cost per
// MMA.  Operand values are zero: timing does not depend on them.
//
// That thread is picked by its index, and the operands of its MMAs go through
// lane registers: about 132 cycles an MMA is what this costs, whatever the
// shape.  The second table issues 1024 MMAs, unrolled, from one elected lane of
// a converged warp, alone and for a pair of CTAs (cta_group::2): the tensor
// pipe's own pace.
//
//   python -m flashinfer_repo_b200.build --probes
//   flashinfer_repo_b200/probes/umma_chain
#include <cuda_runtime.h>
#include <cstdio>
#include <cstdlib>
#include <vector>
#include <algorithm>
#include "../csrc/step/pair.cuh"
using namespace dsa;

#define CK(x) do { cudaError_t e_ = (x); if (e_ != cudaSuccess) { printf("CUDA %s at %d\n", cudaGetErrorString(e_), __LINE__); exit(1);} } while (0)

constexpr int kR = 288;          // MMAs per measurement
constexpr int kSmem = 160 * 1024; // forces one CTA per SM

struct __align__(1024) ProbeSmem {
  uint8_t a[128 * 128];  // A panel: up to 128 rows x 128 B
  uint8_t b[256 * 128];  // B panel: up to 256 rows x 128 B
  uint64_t bar;
  uint32_t tmem;
};

__global__ void __launch_bounds__(128, 1) umma_chain_kernel(int m, int n, int chains, long long* cycles,
                                                            int* err) {
  extern __shared__ uint8_t raw[];
  ProbeSmem& S = *reinterpret_cast<ProbeSmem*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < (int)sizeof(S.a) / 16; i += blockDim.x)
    reinterpret_cast<uint4*>(S.a)[i] = make_uint4(0, 0, 0, 0);
  for (int i = threadIdx.x; i < (int)sizeof(S.b) / 16; i += blockDim.x)
    reinterpret_cast<uint4*>(S.b)[i] = make_uint4(0, 0, 0, 0);
  if (threadIdx.x == 0) {
    mbar_init(&S.bar, 1);
    fence_mbar_init();
  }
  fence_proxy_async_smem();
  if (warp == 0) tmem_alloc(&S.tmem, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = S.tmem;
  if (threadIdx.x == 0) {
    const uint32_t idesc = umma_idesc(1, 1, 0, 0, (uint32_t)m, (uint32_t)n);
    const uint32_t ab = smem_u32(S.a), bb = smem_u32(S.b);
    const long long t0 = clock64();
    for (int r = 0; r < kR; ++r) {
      const int j = r & 3;  // K16 step inside the 64-wide panel
      umma_f16(tmem + (uint32_t)((r % chains) * n), umma_desc(ab + j * 32, 16, 1024, kSwizzle128B),
               umma_desc(bb + j * 32, 16, 1024, kSwizzle128B), idesc, r >= chains ? 1u : 0u);
    }
    umma_commit(&S.bar);
    if (!mbar_wait(&S.bar, 0)) atomicOr(err, 1);
    cycles[blockIdx.x] = clock64() - t0;
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ------------------------------------------- issue by an elected lane of a warp
constexpr int kPanels = 4, kRateReps = 64;
constexpr int kRateSmem = kPanels * (128 + 256) * 128 + 1024;  // A and B panels: up to 128 and 256 rows a CTA

template <int kPair, int kM, int kN>
__global__ void __launch_bounds__(128, 1) umma_rate_kernel(long long* cycles, int* err) {
  static_assert(kM / kPair <= 128 && kN <= 256 && kN % 16 == 0, "panels of the probe");
  extern __shared__ uint8_t raw[];
  uint8_t* a = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  uint8_t* b = a + kPanels * 128 * 128;
  __shared__ uint64_t bar;
  __shared__ uint32_t tmem_at;
  const int warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < kPanels * (128 + 256) * 128 / 16; i += blockDim.x)
    reinterpret_cast<uint4*>(a)[i] = make_uint4(0, 0, 0, 0);
  if (threadIdx.x == 0) {
    mbar_init(&bar, 1);
    fence_mbar_init();
  }
  fence_proxy_async_smem();
  if (warp == 0) {
    if (kPair == 1)
      tmem_alloc(&tmem_at, 512);
    else
      tmem_alloc_pair(&tmem_at, 512);
  }
  tc_fence_before();
  __syncthreads();
  if (kPair == 2) cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem = tmem_at;
  if (warp == 1 && (kPair == 1 || cluster_ctarank() == 0)) {
    constexpr uint32_t idesc = umma_idesc(1, 1, 0, 0, kM, kN);
    const uint64_t da = umma_desc(smem_u32(a), 16, 1024, kSwizzle128B);
    const uint64_t db = umma_desc(smem_u32(b), 16, 1024, kSwizzle128B);
    const long long t0 = clock64();
    if (elect_one()) {
      for (int r = 0; r < kRateReps; ++r) {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const uint64_t aj = da + (uint64_t)(((j >> 2) * 128 * 128 + (j & 3) * 32) >> 4);
          const uint64_t bj = db + (uint64_t)(((j >> 2) * 256 * 128 + (j & 3) * 32) >> 4);
          if (kPair == 1)
            umma_f16(tmem, aj, bj, idesc, 1u);
          else
            umma_f16_pair(tmem, aj, bj, idesc, 1u);
        }
      }
      if (kPair == 1)
        umma_commit(&bar);
      else
        umma_commit_pair(&bar);
      if (!mbar_wait(&bar, 0)) atomicOr(err, 1);
      cycles[blockIdx.x] = clock64() - t0;
    }
    __syncwarp();
  } else if (kPair == 2 && warp == 1) {
    if (elect_one() && !mbar_wait(&bar, 0)) atomicOr(err, 1);  // the commit arrives here too
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (kPair == 2) cluster_sync_all();
  if (warp == 0) {
    tc_fence_after();
    if (kPair == 1)
      tmem_dealloc(tmem, 512);
    else
      tmem_dealloc_pair(tmem, 512);
  }
}

template <int kPair, int kM, int kN>
void rate(int sms, long long* d_cyc, int* d_err) {
  CK(cudaFuncSetAttribute(umma_rate_kernel<kPair, kM, kN>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRateSmem));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(sms / 2 * 2);
  cfg.blockDim = dim3(128);
  cfg.dynamicSmemBytes = kRateSmem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kPair;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  for (int rep = 0; rep < 3; ++rep) {  // the last repetition is reported
    CK(cudaLaunchKernelEx(&cfg, umma_rate_kernel<kPair, kM, kN>, d_cyc, d_err));
    CK(cudaDeviceSynchronize());
  }
  long long first = 0;  // of the first CTA, a leader
  CK(cudaMemcpy(&first, d_cyc, sizeof(first), cudaMemcpyDeviceToHost));
  const double cyc = (double)first / (kRateReps * 16);
  printf("%-4d %-4d %-6d %-14.1f %-14.0f\n", kM, kN, kPair, cyc, (double)kM * kN * 16 / cyc / kPair);
}

int main() {
  int sms = 0;
  CK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, 0));
  CK(cudaFuncSetAttribute(umma_chain_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
  long long* d_cyc;
  int* d_err;
  CK(cudaMalloc(&d_cyc, sms * sizeof(long long)));
  CK(cudaMalloc(&d_err, sizeof(int)));
  CK(cudaMemset(d_err, 0, sizeof(int)));
  struct Cfg { int m, n; };
  const Cfg cfgs[] = {{64, 16}, {128, 16}, {128, 32}, {128, 64}, {128, 128}, {128, 256}};
  const int chain_opts[] = {1, 2, 4, 8};
  printf("%-4s %-4s %-6s %-14s %-14s %-12s\n", "M", "N", "chains", "cycles/MMA", "MAC/clk/SM", "grid");
  for (const Cfg& c : cfgs) {
    for (int ch : chain_opts) {
      if (ch * c.n > 512) continue;
      for (int grid : {1, sms}) {
        std::vector<long long> h(grid);
        for (int rep = 0; rep < 3; ++rep) {  // the last repetition is reported
          umma_chain_kernel<<<grid, 128, kSmem>>>(c.m, c.n, ch, d_cyc, d_err);
          CK(cudaGetLastError());
          CK(cudaDeviceSynchronize());
        }
        CK(cudaMemcpy(h.data(), d_cyc, grid * sizeof(long long), cudaMemcpyDeviceToHost));
        std::sort(h.begin(), h.end());
        const double cyc = (double)h[grid / 2] / kR;
        printf("%-4d %-4d %-6d %-14.1f %-14.0f %-12d\n", c.m, c.n, ch, cyc, (double)c.m * c.n * 16 / cyc,
               grid);
      }
    }
  }
  printf("\nelected lane of a converged warp\n%-4s %-4s %-6s %-14s %-14s\n", "M", "N", "CTAs", "cycles/MMA", "MAC/clk/SM");
  rate<1, 64, 16>(sms, d_cyc, d_err);
  rate<1, 64, 64>(sms, d_cyc, d_err);
  rate<1, 64, 128>(sms, d_cyc, d_err);
  rate<1, 64, 256>(sms, d_cyc, d_err);
  rate<1, 128, 16>(sms, d_cyc, d_err);
  rate<1, 128, 32>(sms, d_cyc, d_err);
  rate<1, 128, 64>(sms, d_cyc, d_err);
  rate<1, 128, 128>(sms, d_cyc, d_err);
  rate<1, 128, 256>(sms, d_cyc, d_err);
  rate<2, 128, 64>(sms, d_cyc, d_err);
  rate<2, 128, 128>(sms, d_cyc, d_err);
  rate<2, 128, 256>(sms, d_cyc, d_err);
  int err = 0;
  CK(cudaMemcpy(&err, d_err, sizeof(int), cudaMemcpyDeviceToHost));
  printf("wait timeouts: %d\n", err);
  return 0;
}
