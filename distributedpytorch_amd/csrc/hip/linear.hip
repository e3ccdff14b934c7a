// Products of a linear layer with what surrounds them fused into the epilogue.
//
//   fprop   z = x W^T + bias (+ addend),  y = act(z)                x [M, K], W [N, K]; z is kept for the backward pass
//   dgrad   dx = (dy W + addend) * act'(z)                          the derivative of the layer in FRONT, at its z [M, K]
//   wgrad   dW = dy^T x,  db = column sums of dy
#include "act.h"

struct LinParams {
  const void *a, *b;                    // C[i, j] = sum_k A(i, k) B(j, k)
  long long a_i, a_k, b_j, b_k;         // element strides
  const float* bias;                    // [cols]
  const void *addend, *pre;             // pre: z of the activation whose derivative is multiplied in
  void *out, *preact;
  long long ld_add, ld_pre, ld_out, ld_z;
  int rows, cols, K, accumulate;
};

enum : int { EPI_FPROP = 0, EPI_DGRAD = 1, EPI_WGRAD = 2 };

template <typename T, int EPI, int ACT>
__device__ __forceinline__ void lin_store(const LinParams& p, int i, int j, float v) {
  if (EPI == EPI_WGRAD) {
    float* o = (float*)p.out + i * p.ld_out + j;
    *o = p.accumulate ? *o + v : v;
    return;
  }
  if (EPI == EPI_FPROP && p.bias) v += p.bias[j];
  if (p.addend) v += Elem<T>::ld((const T*)p.addend + i * p.ld_add + j);
  if (EPI == EPI_FPROP) {
    if (p.preact) Elem<T>::st((T*)p.preact + i * p.ld_z + j, v);
    v = act_fwd<ACT>(v);
  } else if (ACT != ACT_NONE) {
    v *= act_slope<ACT>(Elem<T>::ld((const T*)p.pre + i * p.ld_pre + j));
  }
  Elem<T>::st((T*)p.out + i * p.ld_out + j, v);
}

// 64 x 64 tile, 4 x 4 outputs a thread, any strides
template <typename T, int EPI, int ACT>
__global__ void __launch_bounds__(256) lin_simple_kernel(LinParams p) {
  __shared__ float sa[16][65], sb[16][65];
  const int t = threadIdx.x, tx = t & 15, ty = t >> 4, i0 = blockIdx.x * 64;
  for (int j0 = blockIdx.y * 64; j0 < p.cols; j0 += gridDim.y * 64) {
    float acc[4][4] = {};
    for (int k0 = 0; k0 < p.K; k0 += 16) {
      for (int e = t; e < 1024; e += 256) {
        const int r = e >> 4, k = e & 15;
        sa[k][r] = (i0 + r < p.rows && k0 + k < p.K) ? Elem<T>::ld((const T*)p.a + (i0 + r) * p.a_i + (k0 + k) * p.a_k) : 0.f;
        sb[k][r] = (j0 + r < p.cols && k0 + k < p.K) ? Elem<T>::ld((const T*)p.b + (j0 + r) * p.b_j + (k0 + k) * p.b_k) : 0.f;
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 16; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[r][c] += sa[k][ty * 4 + r] * sb[k][tx * 4 + c];
      __syncthreads();
    }
    for (int r = 0; r < 4; ++r)
      for (int c = 0; c < 4; ++c) {
        const int i = i0 + ty * 4 + r, j = j0 + tx * 4 + c;
        if (i < p.rows && j < p.cols) lin_store<T, EPI, ACT>(p, i, j, acc[r][c]);
      }
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

template <typename T, int EPI, int ACT>
static int lin_launch(const LinParams& p, hipStream_t s) {
  const dim3 grid((p.rows + 63) / 64, min((p.cols + 63) / 64, 65535));
  lin_simple_kernel<T, EPI, ACT><<<grid, 256, 0, s>>>(p);
  return dpa_launch_rc();
}

template <typename T, int EPI>
static int lin_by_act(const LinParams& p, int act, hipStream_t s) {
  switch (act) {
    case ACT_NONE: return lin_launch<T, EPI, ACT_NONE>(p, s);
    case ACT_RELU: return lin_launch<T, EPI, ACT_RELU>(p, s);
    case ACT_SILU: return lin_launch<T, EPI, ACT_SILU>(p, s);
    case ACT_GELU: return lin_launch<T, EPI, ACT_GELU>(p, s);
  }
  return (int)hipErrorInvalidValue;
}

DPA_API int dpa_lin_params_size() { return (int)sizeof(LinParams); }
DPA_API int dpa_linear_fprop(const LinParams* p, int act, int dtype, hipStream_t s) {
  return dtype == 0 ? lin_by_act<float, EPI_FPROP>(*p, act, s) : lin_by_act<bf16_t, EPI_FPROP>(*p, act, s);
}
DPA_API int dpa_linear_dgrad(const LinParams* p, int act, int dtype, hipStream_t s) {
  return dtype == 0 ? lin_by_act<float, EPI_DGRAD>(*p, act, s) : lin_by_act<bf16_t, EPI_DGRAD>(*p, act, s);
}
DPA_API int dpa_linear_wgrad(const LinParams* p, int dtype, hipStream_t s) {
  return dtype == 0 ? lin_launch<float, EPI_WGRAD, ACT_NONE>(*p, s) : lin_launch<bf16_t, EPI_WGRAD, ACT_NONE>(*p, s);
}
DPA_API int dpa_linear_colsum(const void* x, long long ld, int rows, int cols, int splits, int per, float* slab, int accumulate, float* out,
                              int dtype, hipStream_t s) {
  const dim3 grid((cols + 63) / 64, splits);
  if (dtype == 0) lin_colsum_kernel<float><<<grid, 256, 0, s>>>((const float*)x, ld, rows, cols, per, slab);
  else lin_colsum_kernel<bf16_t><<<grid, 256, 0, s>>>((const bf16_t*)x, ld, rows, cols, per, slab);
  lin_colsum_join_kernel<<<(cols + 255) / 256, 256, 0, s>>>(slab, splits, cols, accumulate, out);
  return dpa_launch_rc();
}
