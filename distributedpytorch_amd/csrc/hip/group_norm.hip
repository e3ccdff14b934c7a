// Group normalisation over channels-last activations, with a residual and an activation, forward and backward.
//
//   forward    u = (x - mean) * rstd * gamma + beta (+ res),  y = act(u)          mean, rstd of every (image, group)
//   backward   dz = dy * act'(u)          dbeta = sum dz       dgamma = sum dz * xhat       dres = dz
//              dx = rstd * (gamma dz - c1 - xhat c2),   c1 = mean over the group of gamma dz,  c2 = of gamma dz xhat
//
// Statistics are means and centred second moments held in 32 bits and joined pairwise (Chan, Golub and LeVeque 1979), so a
// mean far from zero costs no digits.  Partial sums go through a slab in memory and are added in a fixed order: no atomics.
#include "act.h"

struct GnParams {
  const void *x, *res, *dy, *yv;        // yv: the stored forward output, the ReLU mask of a block with a residual
  void *y, *dx, *dres;
  const float *gamma, *beta;
  float *mean, *rstd, *slab, *coef, *dgamma, *dbeta;
  long long x_cs, res_cs, dy_cs, yv_cs, y_cs, dx_cs, dres_cs;      // elements from one pixel to the next
  int N, HW, C, G, cg, S, pps;          // S splits of pps pixels (the last one shorter)
  float eps;
};

__device__ __forceinline__ int gn_count(const GnParams& p, int s) { return min(p.pps, p.HW - s * p.pps); }

// (count, mean, m2) += (cb, mb, qb)
__device__ __forceinline__ void gn_join(float& n, float& mean, float& m2, float cb, float mb, float qb) {
  const float t = n + cb;
  if (cb == 0.f) return;
  const float d = mb - mean, f = cb / t;
  mean += d * f;
  m2 += qb + d * d * n * f;
  n = t;
}

// The sign of u decides a whole gradient element, so where 32 bits cannot tell it u is computed in 64.
__device__ __forceinline__ float gn_relu_slope(float u, float mag, float x, float mean, float rstd, float g, float b, float r) {
  if (fabsf(u) > 1e-6f * mag) return u > 0.f ? 1.f : 0.f;
  return ((double)x - (double)mean) * (double)rstd * (double)g + (double)b + (double)r > 0.0 ? 1.f : 0.f;
}

template <typename T>
__global__ void __launch_bounds__(256) gn_stats_kernel(GnParams p) {
  __shared__ float sh[3][4][64];
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6, c = blockIdx.x * 64 + tx, s = blockIdx.y;
  const int p0 = s * p.pps, p1 = min(p0 + p.pps, p.HW);
  for (int n = blockIdx.z; n < p.N; n += gridDim.z) {
    float cnt = 0.f, mean = 0.f, m2 = 0.f;
    if (c < p.C) {
      const T* xp = (const T*)p.x + (long long)n * p.HW * p.x_cs + c;
      for (int i = p0 + ty; i < p1; i += 4) gn_join(cnt, mean, m2, 1.f, Elem<T>::ld(xp + i * p.x_cs), 0.f);
    }
    sh[0][ty][tx] = cnt; sh[1][ty][tx] = mean; sh[2][ty][tx] = m2;
    __syncthreads();
    if (ty == 0 && c < p.C) {
      for (int k = 1; k < 4; ++k) gn_join(cnt, mean, m2, sh[0][k][tx], sh[1][k][tx], sh[2][k][tx]);
      float* o = p.slab + ((long long)n * p.S + s) * 2 * p.C + c;
      o[0] = mean; o[p.C] = m2;
    }
    __syncthreads();
  }
}

// one wave per (image, group): joins S * cg partial moments
__global__ void __launch_bounds__(64) gn_moments_kernel(GnParams p) {
  for (long long q = blockIdx.x; q < (long long)p.N * p.G; q += gridDim.x) {
    const int n = (int)(q / p.G), g = (int)(q % p.G), total = p.S * p.cg;
    const float* o = p.slab + (long long)n * p.S * 2 * p.C + g * p.cg;
    float cnt = 0.f, mean = 0.f, m2 = 0.f;
    for (int i = threadIdx.x; i < total; i += 64) {
      const int s = i / p.cg;
      const float* e = o + (long long)s * 2 * p.C + (i - s * p.cg);
      gn_join(cnt, mean, m2, (float)gn_count(p, s), e[0], e[p.C]);
    }
#pragma unroll
    for (int k = 32; k > 0; k >>= 1) {
      const float cb = __shfl_xor(cnt, k, 64), mb = __shfl_xor(mean, k, 64), qb = __shfl_xor(m2, k, 64);
      gn_join(cnt, mean, m2, cb, mb, qb);
    }
    if (threadIdx.x == 0) { p.mean[q] = mean; p.rstd[q] = 1.f / sqrtf(m2 / cnt + p.eps); }
  }
}

template <typename T, int ACT, bool RES>
__global__ void __launch_bounds__(256) gn_apply_kernel(GnParams p) {
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6, c = blockIdx.x * 64 + tx;
  if (c >= p.C) return;
  const int p0 = blockIdx.y * p.pps, p1 = min(p0 + p.pps, p.HW);
  const float g = p.gamma[c], b = p.beta[c];
  for (int n = blockIdx.z; n < p.N; n += gridDim.z) {
    const float mean = p.mean[(long long)n * p.G + c / p.cg], rg = p.rstd[(long long)n * p.G + c / p.cg] * g;
    const long long base = (long long)n * p.HW;
    for (int i = p0 + ty; i < p1; i += 4) {
      float u = (Elem<T>::ld((const T*)p.x + (base + i) * p.x_cs + c) - mean) * rg + b;
      if (RES) u += Elem<T>::ld((const T*)p.res + (base + i) * p.res_cs + c);
      Elem<T>::st((T*)p.y + (base + i) * p.y_cs + c, act_fwd<ACT>(u));
    }
  }
}

// dz and xhat of one element
template <typename T, int ACT, bool RES>
__device__ __forceinline__ float gn_dz(const GnParams& p, long long pix, int c, float mean, float rstd, float g, float b, float& xhat) {
  const float x = Elem<T>::ld((const T*)p.x + pix * p.x_cs + c), dy = Elem<T>::ld((const T*)p.dy + pix * p.dy_cs + c);
  xhat = (x - mean) * rstd;
  if (ACT == ACT_NONE) return dy;
  if (ACT == ACT_RELU && p.yv) return Elem<T>::ld((const T*)p.yv + pix * p.yv_cs + c) > 0.f ? dy : 0.f;
  const float r = RES ? Elem<T>::ld((const T*)p.res + pix * p.res_cs + c) : 0.f;
  const float a = xhat * g, u = a + b + r;
  if (ACT == ACT_RELU) return dy * gn_relu_slope(u, fabsf(a) + fabsf(b) + fabsf(r), x, mean, rstd, g, b, r);
  return dy * act_slope<ACT>(u);
}

template <typename T, int ACT, bool RES>
__global__ void __launch_bounds__(256) gn_bwd_sums_kernel(GnParams p) {
  __shared__ float sh[2][4][64];
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6, c = blockIdx.x * 64 + tx, s = blockIdx.y;
  const int p0 = s * p.pps, p1 = min(p0 + p.pps, p.HW);
  for (int n = blockIdx.z; n < p.N; n += gridDim.z) {
    float sa = 0.f, sb = 0.f;
    if (c < p.C) {
      const long long q = (long long)n * p.G + c / p.cg, base = (long long)n * p.HW;
      const float mean = p.mean[q], rstd = p.rstd[q], g = p.gamma[c], b = p.beta[c];
      for (int i = p0 + ty; i < p1; i += 4) {
        float xhat;
        const float dz = gn_dz<T, ACT, RES>(p, base + i, c, mean, rstd, g, b, xhat);
        sa += dz; sb += dz * xhat;
      }
    }
    sh[0][ty][tx] = sa; sh[1][ty][tx] = sb;
    __syncthreads();
    if (ty == 0 && c < p.C) {
      for (int k = 1; k < 4; ++k) { sa += sh[0][k][tx]; sb += sh[1][k][tx]; }
      float* o = p.slab + ((long long)n * p.S + s) * 2 * p.C + c;
      o[0] = sa; o[p.C] = sb;
    }
    __syncthreads();
  }
}

// one wave per (image, group): c1, c2
__global__ void __launch_bounds__(64) gn_bwd_coef_kernel(GnParams p) {
  const float inv = 1.f / ((float)p.HW * (float)p.cg);
  for (long long q = blockIdx.x; q < (long long)p.N * p.G; q += gridDim.x) {
    const int n = (int)(q / p.G), g = (int)(q % p.G), total = p.S * p.cg;
    const float* o = p.slab + (long long)n * p.S * 2 * p.C + g * p.cg;
    float sa = 0.f, sb = 0.f;
    for (int i = threadIdx.x; i < total; i += 64) {
      const int s = i / p.cg, k = i - s * p.cg;
      const float* e = o + (long long)s * 2 * p.C + k;
      const float gm = p.gamma[g * p.cg + k];
      sa += e[0] * gm; sb += e[p.C] * gm;
    }
    sa = wave_sum(sa); sb = wave_sum(sb);
    if (threadIdx.x == 0) { p.coef[2 * q] = sa * inv; p.coef[2 * q + 1] = sb * inv; }
  }
}

// dgamma / dbeta: 64 channels x 4 row lanes over the N * S rows of the slab
__global__ void __launch_bounds__(256) gn_bwd_params_kernel(GnParams p) {
  __shared__ float sh[2][4][64];
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6, c = blockIdx.x * 64 + tx;
  const int rows = p.N * p.S;
  float sa = 0.f, sb = 0.f;
  if (c < p.C)
    for (int r = ty; r < rows; r += 4) { const float* e = p.slab + (long long)r * 2 * p.C + c; sa += e[0]; sb += e[p.C]; }
  sh[0][ty][tx] = sa; sh[1][ty][tx] = sb;
  __syncthreads();
  if (ty == 0 && c < p.C) {
    for (int k = 1; k < 4; ++k) { sa += sh[0][k][tx]; sb += sh[1][k][tx]; }
    if (p.dbeta) p.dbeta[c] = sa;
    if (p.dgamma) p.dgamma[c] = sb;
  }
}

template <typename T, int ACT, bool RES>
__global__ void __launch_bounds__(256) gn_bwd_dx_kernel(GnParams p) {
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6, c = blockIdx.x * 64 + tx;
  if (c >= p.C) return;
  const int p0 = blockIdx.y * p.pps, p1 = min(p0 + p.pps, p.HW);
  const float g = p.gamma[c], b = p.beta[c];
  for (int n = blockIdx.z; n < p.N; n += gridDim.z) {
    const long long q = (long long)n * p.G + c / p.cg, base = (long long)n * p.HW;
    const float mean = p.mean[q], rstd = p.rstd[q], c1 = p.coef[2 * q], c2 = p.coef[2 * q + 1];
    for (int i = p0 + ty; i < p1; i += 4) {
      float xhat;
      const float dz = gn_dz<T, ACT, RES>(p, base + i, c, mean, rstd, g, b, xhat);
      if (RES && p.dres) Elem<T>::st((T*)p.dres + (base + i) * p.dres_cs + c, dz);
      Elem<T>::st((T*)p.dx + (base + i) * p.dx_cs + c, rstd * (g * dz - c1 - xhat * c2));
    }
  }
}

template <typename T, int ACT, bool RES>
static int gn_fwd_launch(const GnParams& p, hipStream_t s) {
  const dim3 grid((p.C + 63) / 64, p.S, min(p.N, 16384));
  gn_stats_kernel<T><<<grid, 256, 0, s>>>(p);
  gn_moments_kernel<<<(int)min((long long)p.N * p.G, 65536LL), 64, 0, s>>>(p);
  gn_apply_kernel<T, ACT, RES><<<grid, 256, 0, s>>>(p);
  return dpa_launch_rc();
}

template <typename T, int ACT, bool RES>
static int gn_bwd_launch(const GnParams& p, hipStream_t s) {
  const dim3 grid((p.C + 63) / 64, p.S, min(p.N, 16384));
  gn_bwd_sums_kernel<T, ACT, RES><<<grid, 256, 0, s>>>(p);
  gn_bwd_coef_kernel<<<(int)min((long long)p.N * p.G, 65536LL), 64, 0, s>>>(p);
  if (p.dgamma || p.dbeta) gn_bwd_params_kernel<<<(p.C + 63) / 64, 256, 0, s>>>(p);
  gn_bwd_dx_kernel<T, ACT, RES><<<grid, 256, 0, s>>>(p);
  return dpa_launch_rc();
}

template <bool BWD, typename T, bool RES>
static int gn_by_act(const GnParams& p, int act, hipStream_t s) {
#define GN_CASE(A) case A: return BWD ? gn_bwd_launch<T, A, RES>(p, s) : gn_fwd_launch<T, A, RES>(p, s);
  switch (act) {
    GN_CASE(ACT_NONE) GN_CASE(ACT_RELU) GN_CASE(ACT_SILU) GN_CASE(ACT_GELU)
  }
#undef GN_CASE
  return (int)hipErrorInvalidValue;
}

template <bool BWD>
static int gn_dispatch(const GnParams& p, int act, int dtype, hipStream_t s) {
  const bool res = BWD ? (p.res || p.dres) : p.res != nullptr;
  if (dtype == 0) return res ? gn_by_act<BWD, float, true>(p, act, s) : gn_by_act<BWD, float, false>(p, act, s);
  return res ? gn_by_act<BWD, bf16_t, true>(p, act, s) : gn_by_act<BWD, bf16_t, false>(p, act, s);
}

DPA_API int dpa_gn_params_size() { return (int)sizeof(GnParams); }
DPA_API int dpa_group_norm_fwd(const GnParams* p, int act, int dtype, hipStream_t s) { return gn_dispatch<false>(*p, act, dtype, s); }
DPA_API int dpa_group_norm_bwd(const GnParams* p, int act, int dtype, hipStream_t s) { return gn_dispatch<true>(*p, act, dtype, s); }
