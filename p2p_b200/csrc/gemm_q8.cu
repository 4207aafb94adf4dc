// gemm_q8.cu -- products of 8-bit integer rows with a scale each (a projection, or the gate and up
// projections of a feed-forward block with their activation and product).
//
// The plain form: 64 x 64 outputs a block, 64 codes of k at a time in shared memory, dp4a.
#include "common.cuh"
#include "kernels.h"

namespace p2p {
namespace {

constexpr int kTile = 64, kStep = 64, kPitch = kStep + 4;

__device__ __forceinline__ float act_mul(float g, float u, int act) {
  const float t = act == kActSilu ? g : 1.5957691216057308f * (g + 0.044715f * g * g * g);
  return g / (1.f + expf(-t)) * u;
}

// Rows [r0, r0 + 64) x codes [k0, k0 + 64), zeros outside.
__device__ __forceinline__ void fill(int8_t* dst, const Q8Rows& src, int r0, int k0) {
  for (int i = threadIdx.x; i < kTile * (kStep / 4); i += 256) {
    const int r = i / (kStep / 4), c = i % (kStep / 4) * 4;
    uint32_t w = 0;
    if (r0 + r < src.rows) {
      const int8_t* p = src.q + int64_t(r0 + r) * src.ld + k0 + c;
      if (k0 + c + 4 <= src.cols) {
        w = *reinterpret_cast<const uint32_t*>(p);
      } else {
        for (int j = 0; j < 4; ++j)
          if (k0 + c + j < src.cols) w |= uint32_t(uint8_t(p[j])) << (8 * j);
      }
    }
    *reinterpret_cast<uint32_t*>(dst + r * kPitch + c) = w;
  }
}

template <class T, bool GATE>
__global__ void __launch_bounds__(256) gemm_q8_kernel(const __grid_constant__ GemmQ8Args a) {
  __shared__ __align__(16) int8_t sx[kTile * kPitch], sw[GATE ? 2 : 1][kTile * kPitch];
  const int m0 = blockIdx.y * kTile, n0 = blockIdx.x * kTile;
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  int acc[GATE ? 2 : 1][4][4] = {};
  for (int k0 = 0; k0 < a.x.cols; k0 += kStep) {
    fill(sx, a.x, m0, k0);
    fill(sw[0], a.w, n0, k0);
    if constexpr (GATE) fill(sw[1], a.up, n0, k0);
    __syncthreads();
    for (int k = 0; k < kStep; k += 4) {
      int x[4], w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<int*>(sx + (ty + 16 * i) * kPitch + k);
#pragma unroll
      for (int g = 0; g < (GATE ? 2 : 1); ++g) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          w[j] = *reinterpret_cast<int*>(sw[g] + (tx + 16 * j) * kPitch + k);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[g][i][j] = __dp4a(x[i], w[j], acc[g][i][j]);
      }
    }
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i) {
    const int m = m0 + ty + 16 * i;
    if (m >= a.x.rows) continue;
    const float xs = a.x.scale[m];
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + tx + 16 * j;
      if (n >= a.w.rows) continue;
      float y = __fmul_rn(__fmul_rn(float(acc[0][i][j]), xs), a.w.scale[n]);
      if constexpr (GATE) {
        y = act_mul(y, __fmul_rn(__fmul_rn(float(acc[1][i][j]), xs), a.up.scale[n]), a.act);
      } else {
        if (a.bias) y = __fadd_rn(y, a.bias[n]);
        if (a.res)
          y = __fadd_rn(y, to_f32(static_cast<const T*>(a.res)[int64_t(m) * a.ld_res + n]));
      }
      static_cast<T*>(a.y)[int64_t(m) * a.ld_y + n] = from_f32<T>(y);
    }
  }
}

}  // namespace

cudaError_t launch_gemm_q8(const GemmQ8Args& a, int dtype, int, cudaStream_t s) {
  const dim3 grid((a.w.rows + kTile - 1) / kTile, (a.x.rows + kTile - 1) / kTile);
  if (a.up.q) gemm_q8_kernel<__half, true><<<grid, 256, 0, s>>>(a);
  else if (dtype == 0) gemm_q8_kernel<__half, false><<<grid, 256, 0, s>>>(a);
  else gemm_q8_kernel<float, false><<<grid, 256, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace p2p
