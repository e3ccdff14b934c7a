// Entry points of the linear products (linear.h), the operand packing and the bias gradient.
#include "linear.h"

int lin_fprop(const LinParams& p, int tile, hipStream_t s);
int lin_dgrad(const LinParams& p, int tile, hipStream_t s);
int lin_wgrad(const LinParams& p, int tile, hipStream_t s);

// ---- operands that the DMA cannot take as they are -----------------------------------------------------------------------
// fp32 matrices become their three bf16 parts, bf16 matrices with odd rows or addresses a copy with rows of a multiple of 8;
// the columns behind the last one are zeros.
template <typename T>
__global__ void __launch_bounds__(256) lin_pack_kernel(const T* __restrict__ src, long long ld, int rows, int cols, int ldd, int vec,
                                                       bf16_t* __restrict__ dst) {
  const int groups = ldd / 8;
  const long long total = (long long)rows * groups, part = (long long)rows * ldd;
  for (long long t = blockIdx.x * 256LL + threadIdx.x; t < total; t += gridDim.x * 256LL) {
    const int i = (int)(t / groups), j = (int)(t - (long long)i * groups) * 8;
    Lin8<T> v;
    if (vec && j + 8 <= cols) v.template load<true>(src + i * ld + j, 8); else v.template load<false>(src + i * ld + j, cols - j);
    uint32_t o[3][4];
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      uint32_t w[3] = {0, 0, 0};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float x = v.get(e + h);
        bf16_t b0 = f2bf(x);
        if (sizeof(T) == 4) {
          if ((b0 & 0x7FFF) == 0x7F80 && fabsf(x) < INFINITY) b0 = (bf16_t)(__float_as_uint(x) >> 16);      // no overflow by rounding
          const bool fin = fabsf(x) < INFINITY;
          const float r1 = fin ? x - bf2f(b0) : 0.f;
          const bf16_t b1 = f2bf(r1), b2 = f2bf(r1 - bf2f(b1));
          w[1] |= (uint32_t)b1 << (16 * h); w[2] |= (uint32_t)b2 << (16 * h);
        }
        w[0] |= (uint32_t)b0 << (16 * h);
      }
      o[0][e / 2] = w[0]; o[1][e / 2] = w[1]; o[2][e / 2] = w[2];
    }
#pragma unroll
    for (int q = 0; q < (sizeof(T) == 4 ? 3 : 1); ++q)
      *(uint4*)(dst + q * part + (long long)i * ldd + j) = make_uint4(o[q][0], o[q][1], o[q][2], o[q][3]);
  }
}

// column sums of dy [M, N] in two steps: S row ranges into a slab [S, N], then the slab in a fixed order
template <typename T>
__global__ void __launch_bounds__(256) lin_colsum_kernel(const T* __restrict__ x, long long ld, int rows, int cols, int per, float* __restrict__ slab) {
  __shared__ float sh[4][64];
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6, c = blockIdx.x * 64 + tx;
  const int r0 = blockIdx.y * per, r1 = min(r0 + per, rows);
  float s = 0.f;
  if (c < cols)
    for (int r = r0 + ty; r < r1; r += 4) s += Elem<T>::ld(x + r * ld + c);
  sh[ty][tx] = s;
  __syncthreads();
  if (ty == 0 && c < cols) slab[(long long)blockIdx.y * cols + c] = (sh[0][tx] + sh[1][tx]) + (sh[2][tx] + sh[3][tx]);
}
__global__ void __launch_bounds__(256) lin_colsum_join_kernel(const float* __restrict__ slab, int splits, int cols, int accumulate, float* __restrict__ out) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= cols) return;
  float s = 0.f;
  for (int k = 0; k < splits; ++k) s += slab[(long long)k * cols + c];
  out[c] = accumulate ? out[c] + s : s;
}


DPA_API int dpa_lin_params_size() { return (int)sizeof(LinParams); }
DPA_API int dpa_linear(const LinParams* p, int epi, int tile, hipStream_t s) {
  switch (epi) {
    case EPI_FPROP: return lin_fprop(*p, tile, s);
    case EPI_DGRAD: return lin_dgrad(*p, tile, s);
    case EPI_WGRAD: return lin_wgrad(*p, tile, s);
  }
  return (int)hipErrorInvalidValue;
}
DPA_API int dpa_linear_pack(const void* src, long long ld, int rows, int cols, int ldd, int vec, void* dst, int dtype, hipStream_t s) {
  const int grid = dpa_grid((long long)rows * (ldd / 8), 256);
  if (dtype == 0) lin_pack_kernel<float><<<grid, 256, 0, s>>>((const float*)src, ld, rows, cols, ldd, vec, (bf16_t*)dst);
  else lin_pack_kernel<bf16_t><<<grid, 256, 0, s>>>((const bf16_t*)src, ld, rows, cols, ldd, vec, (bf16_t*)dst);
  return dpa_launch_rc();
}
DPA_API int dpa_linear_colsum(const void* x, long long ld, int rows, int cols, int splits, int per, float* slab, int accumulate, float* out,
                              int dtype, hipStream_t s) {
  const dim3 grid((cols + 63) / 64, splits);
  if (dtype == 0) lin_colsum_kernel<float><<<grid, 256, 0, s>>>((const float*)x, ld, rows, cols, per, slab);
  else lin_colsum_kernel<bf16_t><<<grid, 256, 0, s>>>((const bf16_t*)x, ld, rows, cols, per, slab);
  lin_colsum_join_kernel<<<(cols + 255) / 256, 256, 0, s>>>(slab, splits, cols, accumulate, out);
  return dpa_launch_rc();
}
