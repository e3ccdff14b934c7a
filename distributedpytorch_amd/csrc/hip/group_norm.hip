// Group normalisation over channels-last activations, with a residual and an activation, forward and backward.
//
//   forward    u = (x - mean) * rstd * gamma + beta (+ res),  y = act(u)          mean, rstd of every (image, group)
//   backward   dz = dy * act'(u)          dbeta = sum dz       dgamma = sum dz * xhat       dres = dz
//              dx = rstd * (gamma dz - c1 - xhat c2),   c1 = mean over the group of gamma dz,  c2 = of gamma dz xhat
//
// Statistics are means and centred second moments held in 32 bits.  The vector kernels sum up to 104 values a thread and then by a
// tree, and take the deviations from that mean; partial moments are joined pairwise (Chan, Golub and LeVeque 1979), in the kernels
// for any layout pixel by pixel.  With means of 300 to 30000 and a spread of 0.1 the mean came out at most 2.7 times 2^-24 of itself
// away in images of 7 x 7 x 64 to 1500 x 700 x 6, and the result at most 3.9 times 2^-24 of mean / spread.  Partial sums go through a slab in memory and are added in a fixed order: no atomics.
#include "act.h"
#include "conv_common.h"

struct GnParams {
  const void *x, *res, *dy, *yv;        // yv: the stored forward output, the ReLU mask of a block with a residual
  void *y, *dx, *dres;
  const float *gamma, *beta;
  float *mean, *rstd, *slab, *coef, *dgamma, *dbeta;
  long long x_cs, res_cs, dy_cs, yv_cs, y_cs, dx_cs, dres_cs;      // elements from one pixel to the next
  int N, HW, C, G, cg, S, pps;          // S splits of pps pixels (the last one shorter)
  int act, W, rows, R, threads, way;    // the vector kernels: vectors of a chunk, pixels of a sweep, sweeps, threads, which kernel
  float eps;
};
enum : int { GN_ANY = 0, GN_ONE = 1, GN_TWO = 2, GN_LONE = 3 };      // GN_LONE: one pass, one channel a lane

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

// ---- any layout: one channel a lane, scalar accesses, 64 channels x 4 pixels a block ---------------------------------------
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

// four waves per (image, group): join S * cg partial moments
__global__ void __launch_bounds__(256) gn_moments_kernel(GnParams p) {
  __shared__ float sh[4][3];
  for (long long q = blockIdx.x; q < (long long)p.N * p.G; q += gridDim.x) {
    const int n = (int)(q / p.G), g = (int)(q % p.G), total = p.S * p.cg;
    const float* o = p.slab + (long long)n * p.S * 2 * p.C + g * p.cg;
    float cnt = 0.f, mean = 0.f, m2 = 0.f;
    for (int i = threadIdx.x; i < total; i += 256) {
      const int s = i / p.cg;
      const float* e = o + (long long)s * 2 * p.C + (i - s * p.cg);
      gn_join(cnt, mean, m2, (float)gn_count(p, s), e[0], e[p.C]);
    }
#pragma unroll
    for (int k = 32; k > 0; k >>= 1) {
      const float cb = __shfl_xor(cnt, k, 64), mb = __shfl_xor(mean, k, 64), qb = __shfl_xor(m2, k, 64);
      gn_join(cnt, mean, m2, cb, mb, qb);
    }
    if ((threadIdx.x & 63) == 0) { float* w = sh[threadIdx.x >> 6]; w[0] = cnt; w[1] = mean; w[2] = m2; }
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int k = 1; k < 4; ++k) gn_join(cnt, mean, m2, sh[k][0], sh[k][1], sh[k][2]);
      p.mean[q] = mean; p.rstd[q] = 1.f / sqrtf(m2 / cnt + p.eps);
    }
    __syncthreads();
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
  const float r = RES && p.res ? Elem<T>::ld((const T*)p.res + pix * p.res_cs + c) : 0.f;      // (RES also where only dres is there)
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

// c1, c2: four waves per (image, group), four of those a block of 1024
__device__ __forceinline__ void gn_bwd_coef(const GnParams& p, int block, int blocks, float (*sh)[2]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, four = wave >> 2;
  const float inv = 1.f / ((float)p.HW * (float)p.cg);
  for (long long q0 = block * 4LL; q0 < (long long)p.N * p.G; q0 += blocks * 4LL) {
    const long long q = q0 + four;
    float sa = 0.f, sb = 0.f;
    if (q < (long long)p.N * p.G) {
      const int n = (int)(q / p.G), g = (int)(q % p.G), total = p.S * p.cg;
      const float* o = p.slab + (long long)n * p.S * 2 * p.C + g * p.cg;
#pragma unroll 2
      for (int i = threadIdx.x & 255; i < total; i += 256) {
        const int s = i / p.cg, k = i - s * p.cg;
        const float* e = o + (long long)s * 2 * p.C + k;
        const float gm = p.gamma[g * p.cg + k];
        sa += e[0] * gm; sb += e[p.C] * gm;
      }
    }
    sa = wave_sum(sa); sb = wave_sum(sb);
    if (lane == 0) { sh[wave][0] = sa; sh[wave][1] = sb; }
    __syncthreads();
    if ((threadIdx.x & 255) == 0 && q < (long long)p.N * p.G) {
      for (int k = 1; k < 4; ++k) { sa += sh[wave + k][0]; sb += sh[wave + k][1]; }
      p.coef[2 * q] = sa * inv; p.coef[2 * q + 1] = sb * inv;
    }
    __syncthreads();
  }
}

// dgamma / dbeta in the first `strips` blocks: 16 channels x 64 row lanes over the N * S rows of the slab, in a fixed order.  The
// blocks behind them make the coefficients of dx where it has a kernel of its own for any layout: one launch for both.
__global__ void __launch_bounds__(1024) gn_bwd_params_kernel(GnParams p, int strips) {
  __shared__ float sh[2][64][17];
  if ((int)blockIdx.x >= strips) {
    gn_bwd_coef(p, blockIdx.x - strips, gridDim.x - strips, (float(*)[2])sh);
    return;
  }
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, c = blockIdx.x * 16 + tx;
  const int rows = p.N * p.S;
  float sa = 0.f, sb = 0.f;
  if (c < p.C) {
#pragma unroll 4
    for (int r = ty; r < rows; r += 64) { const float* e = p.slab + (long long)r * 2 * p.C + c; sa += e[0]; sb += e[p.C]; }
  }
  sh[0][ty][tx] = sa; sh[1][ty][tx] = sb;
  __syncthreads();
  for (int k = 32; k > 0; k >>= 1) {
    if (ty < k) { sh[0][ty][tx] += sh[0][ty + k][tx]; sh[1][ty][tx] += sh[1][ty + k][tx]; }
    __syncthreads();
  }
  if (ty == 0 && c < p.C) {
    if (p.dbeta) p.dbeta[c] = sh[0][0][tx];
    if (p.dgamma) p.dgamma[c] = sh[1][0][tx];
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


// ---- 16-byte accesses: channels, strides and addresses are multiples of a vector -------------------------------------------
// A block owns one image and a chunk of W vectors (whole groups) of its channels; thread t holds vector t % W of the pixels
// t / W, t / W + rows, ... in registers.
//   one pass    the chunk's whole image fits: statistics and result from one read.  The mean is subtracted before squares
//               are summed, both over registers.
//   two passes  the image is cut into S ranges of pixels; the first kernel leaves each range's moments (or gradient sums), the
//               second joins them for its chunk and goes over the pixels again, the newest first: they are still in the
//               last-level cache.
// Both are bound by memory: the floor is one read of every input and one write of every output, and a copy in segments of 128
// bytes, as the chunks have them, runs at 4.5 TB/s here.  With ReLU and residual, bf16: forward 64 x 28 x 28 x 512 37.7 us,
// 4.1 TB/s of the floor's bytes, 64 x 14 x 14 x 1024 17.5 us, 4.4 TB/s, 64 x 56 x 56 x 256 79.7 us, 3.9 TB/s (segments of 64
// bytes); backward 64 x 28 x 28 x 512 67.8 us, 3.8 TB/s: two blocks of 8 waves a CU at 200 registers, and the arithmetic of
// a vector, some 25 instructions an element, is the next bound, so sign and branch decisions are made once a vector.  Sums over
// the lanes of a wave stay in registers (DPP and lane swaps): through LDS 28 x 28 x 512 backward took 84 us.

// What a thread holds of a pixel: 16 bytes, or one channel (Lone<T>) where the layout allows no more.
template <typename T> struct Lone;
template <typename T> struct GnTypes { typedef T E; typedef Vec16<T> X; };
template <typename T> struct GnTypes<Lone<T>> {
  typedef T E;
  struct X {
    static constexpr int N = 1;
    float v;
    __device__ __forceinline__ void load(const T* p) { v = Elem<T>::ld(p); }
    __device__ __forceinline__ void store(T* p) const { Elem<T>::st(p, v); }
    __device__ __forceinline__ float get(int) const { return v; }
  };
};
template <typename T> using GnX = typename GnTypes<T>::X;
template <typename T> using GnE = typename GnTypes<T>::E;

// all elements of a vector at once: two bf16 in one conversion
__device__ __forceinline__ void gn_pack(Vec16<float>& x, const float (&v)[4]) { x.raw = make_float4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ void gn_pack(Vec16<bf16_t>& x, const float (&v)[8]) {
  typedef __attribute__((ext_vector_type(2))) float f2;
  typedef __attribute__((ext_vector_type(2))) __bf16 b2;
#pragma unroll
  for (int e = 0; e < 8; e += 2) ((uint32_t*)&x.raw)[e >> 1] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){v[e], v[e + 1]}, b2));
}
// the same where every value is a bf16 already
__device__ __forceinline__ void gn_pack_exact(Vec16<float>& x, const float (&v)[4]) { gn_pack(x, v); }
__device__ __forceinline__ void gn_pack_exact(Vec16<bf16_t>& x, const float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; e += 2) ((uint32_t*)&x.raw)[e >> 1] = __builtin_amdgcn_perm(__float_as_uint(v[e + 1]), __float_as_uint(v[e]), 0x07060302u);
}
template <typename X> __device__ __forceinline__ void gn_pack(X& x, const float (&v)[1]) { x.v = v[0]; }
template <typename X> __device__ __forceinline__ void gn_pack_exact(X& x, const float (&v)[1]) { x.v = v[0]; }
// activations of a vector: the launch's activation is uniform, so the branch stands outside the elements
template <int V> __device__ __forceinline__ void gn_acts(int act, float (&u)[V]) {
  if (act == ACT_RELU) {
#pragma unroll
    for (int e = 0; e < V; ++e) u[e] = act_fwd<ACT_RELU>(u[e]);
  } else if (act == ACT_SILU) {
#pragma unroll
    for (int e = 0; e < V; ++e) u[e] = act_fwd<ACT_SILU>(u[e]);
  } else if (act == ACT_GELU) {
#pragma unroll
    for (int e = 0; e < V; ++e) u[e] = act_fwd<ACT_GELU>(u[e]);
  }
}

// the block's image, chunk and range of pixels, and the thread's place in them
template <typename T, int NT>
struct GnPlace {
  static constexpr int V = GnX<T>::N;
  int n, c0, s, row, w, p0, p1;
  bool on;
  __device__ __forceinline__ GnPlace(const GnParams& p, int job) {
    const int chunks = p.C / (p.W * V);
    const int chunk = job % chunks, rest = job / chunks;          // (chunks of one image are neighbours: they share cache lines)
    s = rest % p.S; n = rest / p.S;
    row = threadIdx.x / p.W; w = threadIdx.x - row * p.W;
    c0 = chunk * p.W * V;
    p0 = s * p.pps; p1 = min(p0 + p.pps, p.HW);
    on = row < p.rows;
  }
  __device__ __forceinline__ int c() const { return c0 + w * V; }
  // a tensor's vector of the thread's k-th pixel: a uniform address and one 32-bit offset a lane for all k
  struct Ref {
    char* base; unsigned off; long long step;
    __device__ __forceinline__ GnE<T>* at(int k) const { return (GnE<T>*)(base + k * step + off); }
  };
  __device__ __forceinline__ Ref ref(const GnParams& p, const void* t, long long cs) const {
    return Ref{(char*)t + (((long long)n * p.HW + p0) * cs + c0) * (long long)sizeof(GnE<T>), (unsigned)((row * (int)cs + w * V) * (int)sizeof(GnE<T>)),
               (long long)p.rows * cs * (long long)sizeof(GnE<T>)};
  }
  __device__ __forceinline__ int pixel(const GnParams& p, int k) const { return p0 + row + k * p.rows; }
  __device__ __forceinline__ bool has(const GnParams& p, int k) const { return on && pixel(p, k) < p1; }
};

// Sums over the lanes of a wave that hold the same vector (lane % W, W a power of two up to 64), without LDS: rotations within
// 16 lanes, then exchanges of 16 and of 32 lanes with themselves.
template <int D> __device__ __forceinline__ float gn_ror(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 + D, 0xf, 0xf, false));
}
template <int N> __device__ __forceinline__ void gn_sum_rows(float (&v)[N], int W) {
  if (W <= 1) {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] += gn_ror<1>(v[e]);
  }
  if (W <= 2) {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] += gn_ror<2>(v[e]);
  }
  if (W <= 4) {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] += gn_ror<4>(v[e]);
  }
  if (W <= 8) {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] += gn_ror<8>(v[e]);
  }
  if (W <= 16) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const auto t = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[e]), __float_as_uint(v[e]), false, false);
      v[e] = __uint_as_float(t[0]) + __uint_as_float(t[1]);
    }
  }
  if (W <= 32) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[e]), __float_as_uint(v[e]), false, false);
      v[e] = __uint_as_float(t[0]) + __uint_as_float(t[1]);
    }
  }
}
__host__ __device__ __forceinline__ bool gn_even(int W) { return W <= 64 && (W & (W - 1)) == 0; }

// Sums over the pixels of the block and the channels of each group of the chunk: every thread puts in the sum over its own
// pixels for each of its channels (or for its vector, where a vector lies in one group).
template <int V, int NT, bool WHOLE>
__device__ __forceinline__ void gn_group_sum(const GnParams& p, bool on, float (&v)[WHOLE ? 1 : V], float* part, float* out) {
  constexpr int PER = WHOLE ? 1 : V;
  const int len = p.W * PER, of = WHOLE ? p.cg / V : p.cg, groups = len / of, lane = threadIdx.x & 63;
  const bool even = gn_even(p.W);
  if (even) gn_sum_rows(v, p.W);          // (every thread is on; a wave then has one row to put in)
  const int rows = even ? NT / 64 : p.rows;
  __syncthreads();
  if (even ? lane < p.W : on) {
    const int at = even ? (int)(threadIdx.x >> 6) * p.W + lane : (int)threadIdx.x;
#pragma unroll
    for (int e = 0; e < PER; ++e) part[at * PER + e] = v[e];
  }
  __syncthreads();
  const int total = rows * of;
  if (total <= 64) {          // a few entries a group: all groups at once, `n` lanes each
    int n = 1;
    while (n < total) n <<= 1;
    for (int g = threadIdx.x / n; g < groups; g += NT / n) {
      const int i = threadIdx.x & (n - 1), r = i / of;
      float t = i < total ? part[r * len + g * of + (i - r * of)] : 0.f;
      for (int k = n >> 1; k > 0; k >>= 1) t += __shfl_xor(t, k, 64);
      if (i == 0) out[g] = t;
    }
  } else {
    for (int g = threadIdx.x >> 6; g < groups; g += NT / 64) {
      float t = 0.f;
      for (int i = lane; i < total; i += 64) { const int r = i / of; t += part[r * len + g * of + (i - r * of)]; }
      t = wave_sum(t);
      if (lane == 0) out[g] = t;
    }
  }
  __syncthreads();
}

// mean and rstd of the groups of a chunk, from the S ranges of an image (wave per group)
template <int NT>
__device__ __forceinline__ void gn_join_ranges(const GnParams& p, int n, int g0, int groups, float* mean, float* rstd) {
  const int lane = threadIdx.x & 63;
  for (int g = threadIdx.x >> 6; g < groups; g += NT / 64) {
    float cnt = 0.f, m = 0.f, q = 0.f;
    for (int s = lane; s < p.S; s += 64) {
      const float* e = p.slab + (((long long)n * p.S + s) * p.G + g0 + g) * 2;
      gn_join(cnt, m, q, (float)gn_count(p, s) * p.cg, e[0], e[1]);
    }
#pragma unroll
    for (int k = 32; k > 0; k >>= 1) {
      const float cb = __shfl_xor(cnt, k, 64), mb = __shfl_xor(m, k, 64), qb = __shfl_xor(q, k, 64);
      gn_join(cnt, m, q, cb, mb, qb);
    }
    if (lane == 0) { mean[g] = m; rstd[g] = 1.f / sqrtf(q / cnt + p.eps); }
  }
  __syncthreads();
}

constexpr int GN_GROUPS = 1024;          // groups a chunk may hold

// Per-channel values of a vector: one where a vector lies in one group (WHOLE), which leaves registers for more pixels.
template <int V, bool WHOLE>
struct GnVec {
  float v[WHOLE ? 1 : V];
  __device__ __forceinline__ float& operator[](int e) { return v[WHOLE ? 0 : e]; }
  template <typename F> __device__ __forceinline__ void set(F f) {
#pragma unroll
    for (int e = 0; e < (WHOLE ? 1 : V); ++e) v[e] = f(e);
  }
};

constexpr int GN_AHEAD = 4;          // vectors read together where stores stand between reads (an output may be an input)

// WAY GN_ONE: the whole forward pass.  GN_TWO: moments of a range of pixels.
template <typename T, int NT, int R, bool WHOLE, int WAY>
__global__ void __launch_bounds__(NT, 4) gn_fwd_kernel(GnParams p) {
  constexpr int V = GnX<T>::N;
  extern __shared__ float lds[];          // mean, rstd [groups]; partial sums
  const GnPlace<T, NT> me(p, xcd_remap(blockIdx.x, gridDim.x));
  const int g0 = me.c0 / p.cg, groups = p.W * V / p.cg, c = me.c();
  float *mean = lds, *rstd = lds + groups, *part = lds + 2 * groups;
  const auto px = me.ref(p, p.x, p.x_cs), pr = me.ref(p, p.res, p.res_cs), py = me.ref(p, p.y, p.y_cs);
  GnX<T> x[R];
#pragma unroll
  for (int k = 0; k < R; ++k)
    if (me.has(p, k)) x[k].load(px.at(k));
  GnVec<V, WHOLE> a, mu, rs;
  a.set([](int) { return 0.f; });
#pragma unroll
  for (int k = 0; k < R; ++k)
    if (me.has(p, k)) {
#pragma unroll
      for (int e = 0; e < V; ++e) a[e] += x[k].get(e);
    }
  gn_group_sum<V, NT, WHOLE>(p, me.on, a.v, part, mean);
  const float count = (float)(me.p1 - me.p0) * p.cg;
  auto group = [&](int e) { return me.on ? (me.w * V + e) / p.cg : 0; };
  mu.set([&](int e) { return mean[group(e)] / count; });
  a.set([](int) { return 0.f; });
#pragma unroll
  for (int k = 0; k < R; ++k)
    if (me.has(p, k)) {
#pragma unroll
      for (int e = 0; e < V; ++e) { const float d = x[k].get(e) - mu[e]; a[e] += d * d; }
    }
  gn_group_sum<V, NT, WHOLE>(p, me.on, a.v, part, rstd);
  if (WAY == GN_TWO) {
    for (int g = threadIdx.x; g < groups; g += NT) {
      float* o = p.slab + (((long long)me.n * p.S + me.s) * p.G + g0 + g) * 2;
      o[0] = mean[g] / count; o[1] = rstd[g];
    }
    return;
  }
  for (int g = threadIdx.x; g < groups; g += NT) {
    p.mean[(long long)me.n * p.G + g0 + g] = mean[g] / count;
    p.rstd[(long long)me.n * p.G + g0 + g] = 1.f / sqrtf(rstd[g] / count + p.eps);
  }
  if (!me.on) return;
  float rg[V], b[V];
  rs.set([&](int e) { return 1.f / sqrtf(rstd[group(e)] / count + p.eps); });
#pragma unroll
  for (int e = 0; e < V; ++e) { rg[e] = rs[e] * p.gamma[c + e]; b[e] = p.beta[c + e]; }
#pragma unroll
  for (int k0 = 0; k0 < R; k0 += GN_AHEAD) {
    GnX<T> r[GN_AHEAD];
    if (p.res) {
#pragma unroll
      for (int k = k0; k < k0 + GN_AHEAD && k < R; ++k)
        if (me.has(p, k)) r[k - k0].load(pr.at(k));
    }
#pragma unroll
    for (int k = k0; k < k0 + GN_AHEAD && k < R; ++k)
      if (me.has(p, k)) {
        float u[V];
#pragma unroll
        for (int e = 0; e < V; ++e) u[e] = (x[k].get(e) - mu[e]) * rg[e] + b[e];
        if (p.res) {
#pragma unroll
          for (int e = 0; e < V; ++e) u[e] += r[k - k0].get(e);
        }
        gn_acts(p.act, u);
        gn_pack(x[k], u);
        x[k].store(py.at(k));
      }
  }
}

template <typename T, int NT, int R>
__global__ void __launch_bounds__(NT) gn_fwd_apply_kernel(GnParams p) {
  constexpr int V = GnX<T>::N;
  __shared__ float mean[GN_GROUPS], rstd[GN_GROUPS];
  const GnPlace<T, NT> me(p, gridDim.x - 1 - xcd_remap(blockIdx.x, gridDim.x));
  const int g0 = me.c0 / p.cg, groups = p.W * V / p.cg;
  const auto px = me.ref(p, p.x, p.x_cs), pr = me.ref(p, p.res, p.res_cs), py = me.ref(p, p.y, p.y_cs);
  GnX<T> x[R], r[R];
#pragma unroll
  for (int k = 0; k < R; ++k)
    if (me.has(p, k)) {
      x[k].load(px.at(k));
      if (p.res) r[k].load(pr.at(k));
    }
  gn_join_ranges<NT>(p, me.n, g0, groups, mean, rstd);
  if (me.s == 0)
    for (int g = threadIdx.x; g < groups; g += NT) { p.mean[(long long)me.n * p.G + g0 + g] = mean[g]; p.rstd[(long long)me.n * p.G + g0 + g] = rstd[g]; }
  if (!me.on) return;
  float mu[V], rg[V], b[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const int g = (me.w * V + e) / p.cg;
    mu[e] = mean[g]; rg[e] = rstd[g] * p.gamma[me.c() + e]; b[e] = p.beta[me.c() + e];
  }
#pragma unroll
  for (int k = 0; k < R; ++k)
    if (me.has(p, k)) {
      float u[V];
#pragma unroll
      for (int e = 0; e < V; ++e) u[e] = (x[k].get(e) - mu[e]) * rg[e] + b[e];
      if (p.res) {
#pragma unroll
        for (int e = 0; e < V; ++e) u[e] += r[k].get(e);
      }
      gn_acts(p.act, u);
      gn_pack(x[k], u);
      x[k].store(py.at(k));
    }
}

// dy -> dz = dy * act'(u) of a vector, u = (x - mean) * rstd * gamma + beta (+ residual); side: the stored output of a ReLU
// (BY_Y) or the residual.  A ReLU's dz is dy or zero and may stay in dy's registers; a smooth activation's fills no bf16.
enum : int { GN_BY_Y = 4 };          // beside the ids of act.h
template <int MODE, typename T, int V, typename M>
__device__ __forceinline__ void gn_dz_vec(const GnX<T>& x, const GnX<T>& side, bool has_side, M& mu, M& rs, const float (&ga)[V], const float (&be)[V],
                                          float (&dz)[V], const GnParams& p, int n, int c, const GnE<T>* xp, const GnE<T>* sp) {
  if (MODE == GN_BY_Y) {
#pragma unroll
    for (int e = 0; e < V; ++e) dz[e] = side.get(e) > 0.f ? dz[e] : 0.f;
    return;
  }
  bool near = false;          // a ReLU whose sign 32 bits do not tell, in any element: one branch a vector
  unsigned up = 0;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const float rv = has_side ? side.get(e) : 0.f, t = (x.get(e) - mu[e]) * (rs[e] * ga[e]), u = t + be[e] + rv;
    if (MODE == ACT_SILU) dz[e] *= act_slope<ACT_SILU>(u);
    if (MODE == ACT_GELU) dz[e] *= act_slope<ACT_GELU>(u);
    if (MODE == ACT_RELU) {
      near |= fabsf(u) <= 1e-6f * (fabsf(t) + fabsf(be[e]) + fabsf(rv));
      if (u > 0.f) up |= 1u << e;
    }
  }
  if (MODE == ACT_RELU) {
    if (near) {
      up = 0;
#pragma unroll 1
      for (int e = 0; e < V; ++e) {          // (rare: from memory again, so that it holds no registers)
        const long long q = (long long)n * p.G + (c + e) / p.cg;
        const double u = ((double)Elem<GnE<T>>::ld(xp + e) - p.mean[q]) * p.rstd[q] * p.gamma[c + e] + p.beta[c + e] + (has_side ? Elem<GnE<T>>::ld(sp + e) : 0.f);
        if (u > 0.0) up |= 1u << e;
      }
    }
#pragma unroll
    for (int e = 0; e < V; ++e) dz[e] = up >> e & 1 ? dz[e] : 0.f;
  }
}
template <typename T, int V, typename M, typename P, typename R>
__device__ __forceinline__ void gn_dz_vec(int mode, const GnX<T>& x, const GnX<T>& side, bool has_side, M& mu, M& rs, const float (&ga)[V],
                                          const float (&be)[V], float (&dz)[V], const GnParams& p, const P& me, const R& px, const R& ps, int k) {
#define GN_DZ(MODE) gn_dz_vec<MODE, T, V>(x, side, has_side, mu, rs, ga, be, dz, p, me.n, me.c(), px.at(k), ps.at(k))
  if (mode == GN_BY_Y) GN_DZ(GN_BY_Y);
  else if (mode == ACT_RELU) GN_DZ(ACT_RELU);
  else if (mode == ACT_SILU) GN_DZ(ACT_SILU);
  else if (mode == ACT_GELU) GN_DZ(ACT_GELU);
#undef GN_DZ
}

// Gradient sums over a block's pixels for each channel of the chunk: tot [2][W * V].
template <int V, int NT>
__device__ __forceinline__ void gn_channel_sum(const GnParams& p, bool on, int row, int w, float (&a)[V], float (&b)[V], float* part, float* tot) {
  const int cw = p.W * V;
  int rows = p.rows;
  if (gn_even(p.W)) {
    gn_sum_rows(a, p.W); gn_sum_rows(b, p.W);
    rows = NT / 64; row = threadIdx.x >> 6; on = (int)(threadIdx.x & 63) < p.W;
  }
  float* part2 = part + rows * cw;
  __syncthreads();
  if (on) {
#pragma unroll
    for (int e = 0; e < V; ++e) { part[row * cw + w * V + e] = a[e]; part2[row * cw + w * V + e] = b[e]; }
  }
  __syncthreads();
  // `lanes` threads for each of the 2 cw sums, the rows in a fixed order
  int lanes = 1;
  while (lanes < 64 && lanes * 4 * cw <= NT && lanes * 2 <= rows) lanes *= 2;
  for (int i = threadIdx.x / lanes; i < 2 * cw; i += NT / lanes) {
    const float* q = i < cw ? part + i : part2 + (i - cw);
    float t = 0.f;
    for (int r = threadIdx.x % lanes; r < rows; r += lanes) t += q[r * cw];
    for (int k = lanes >> 1; k > 0; k >>= 1) t += __shfl_xor(t, k, 64);
    if (threadIdx.x % lanes == 0) tot[i] = t;
  }
  __syncthreads();
}

// c1, c2 of the groups of a chunk times the group's element count
template <int NT, typename F>
__device__ __forceinline__ void gn_group_grads(const GnParams& p, int c0, int groups, const float* sa, const float* sb, F out) {
  const int lane = threadIdx.x & 63;
  for (int g = threadIdx.x >> 6; g < groups; g += NT / 64) {
    float ta = 0.f, tb = 0.f;
    for (int k = lane; k < p.cg; k += 64) {
      const float gm = p.gamma[c0 + g * p.cg + k];
      ta += sa[g * p.cg + k] * gm; tb += sb[g * p.cg + k] * gm;
    }
    ta = wave_sum(ta); tb = wave_sum(tb);
    if (lane == 0) out(g, ta, tb);
  }
}

// The whole backward pass of a chunk but the join of the parameter gradients over images (slab [N][2][C]).
template <typename T, int NT, int R, bool WHOLE>
__global__ void __launch_bounds__(NT, R * sizeof(GnX<T>) <= 112 ? 4 : 2) gn_bwd_kernel(GnParams p) {
  constexpr int V = GnX<T>::N;
  extern __shared__ float lds[];          // c1, c2 [groups]; sums of the channels [2][cw]; partial sums
  const GnPlace<T, NT> me(p, xcd_remap(blockIdx.x, gridDim.x));
  const int g0 = me.c0 / p.cg, groups = p.W * V / p.cg, c = me.c();
  const int cw = p.W * V;
  float *c1 = lds, *c2 = lds + groups, *tot = lds + 2 * groups, *part = tot + 2 * cw;
  const int mode = p.act == ACT_RELU && p.yv ? GN_BY_Y : p.act;
  const bool smooth = p.act >= ACT_SILU;
  const auto px = me.ref(p, p.x, p.x_cs), pd = me.ref(p, p.dy, p.dy_cs), pdx = me.ref(p, p.dx, p.dx_cs), pdr = me.ref(p, p.dres, p.dres_cs);
  GnX<T> x[R], dy[R];
#pragma unroll
  for (int k = 0; k < R; ++k)
    if (me.has(p, k)) { x[k].load(px.at(k)); dy[k].load(pd.at(k)); }
  // what the activation needs beside x: the stored output, or the residual (zeros without one)
  const void* side = p.act == ACT_NONE ? nullptr : p.yv ? p.yv : p.res;
  const auto ps = me.ref(p, side, p.yv ? p.yv_cs : p.res_cs);
  auto read = [&](int k0, GnX<T> (&r)[GN_AHEAD]) __attribute__((always_inline)) {
    if (!side) return;
#pragma unroll
    for (int k = k0; k < k0 + GN_AHEAD && k < R; ++k)
      if (me.has(p, k)) r[k - k0].load(ps.at(k));
  };
  GnX<T> r[GN_AHEAD];
  read(0, r);
  GnVec<V, WHOLE> mu, rs;
  auto group = [&](int e) { return (long long)me.n * p.G + g0 + (me.on ? (me.w * V + e) / p.cg : 0); };
  mu.set([&](int e) { return p.mean[group(e)]; });
  rs.set([&](int e) { return p.rstd[group(e)]; });
  float ga[V], be[V], a[V], b[V];
#pragma unroll
  for (int e = 0; e < V; ++e) { ga[e] = me.on ? p.gamma[c + e] : 0.f; be[e] = me.on ? p.beta[c + e] : 0.f; a[e] = 0.f; b[e] = 0.f; }
#pragma unroll
  for (int k0 = 0; k0 < R; k0 += GN_AHEAD) {
    if (k0) read(k0, r);
#pragma unroll
    for (int k = k0; k < k0 + GN_AHEAD && k < R; ++k)
      if (me.has(p, k)) {
        float dz[V];
#pragma unroll
        for (int e = 0; e < V; ++e) dz[e] = dy[k].get(e);
        if (mode != ACT_NONE) {
          gn_dz_vec<T>(mode, x[k], r[k - k0], side != nullptr, mu, rs, ga, be, dz, p, me, px, ps, k);
          if (!smooth) gn_pack_exact(dy[k], dz);
        }
#pragma unroll
        for (int e = 0; e < V; ++e) { a[e] += dz[e]; b[e] += dz[e] * (x[k].get(e) - mu[e]); }
      }
  }
#pragma unroll
  for (int e = 0; e < V; ++e) b[e] *= rs[e];
  gn_channel_sum<V, NT>(p, me.on, me.row, me.w, a, b, part, tot);
  if (p.dgamma || p.dbeta) {
    float* o = p.slab + ((long long)me.n * p.S + me.s) * 2 * p.C + me.c0;
    for (int i = threadIdx.x; i < cw; i += NT) { o[i] = tot[i]; o[p.C + i] = tot[cw + i]; }
  }
  const float inv = 1.f / ((float)p.HW * (float)p.cg);
  gn_group_grads<NT>(p, me.c0, groups, tot, tot + cw, [&](int g, float ta, float tb) { c1[g] = ta * inv; c2[g] = tb * inv; });
  __syncthreads();
  if (!me.on) return;
  // dx = rstd gamma dz - (rstd c1 + (x - mean) rstd^2 c2)
  GnVec<V, WHOLE> k1, k2;
  k1.set([&](int e) { return c1[(me.w * V + e) / p.cg] * rs[e]; });
  k2.set([&](int e) { return c2[(me.w * V + e) / p.cg] * rs[e] * rs[e]; });
#pragma unroll
  for (int k0 = 0; k0 < R; k0 += GN_AHEAD) {
    if (smooth) read(k0, r);
#pragma unroll
    for (int k = k0; k < k0 + GN_AHEAD && k < R; ++k)
      if (me.has(p, k)) {
        float dz[V];
#pragma unroll
        for (int e = 0; e < V; ++e) dz[e] = dy[k].get(e);
        if (smooth) {
          gn_dz_vec<T>(mode, x[k], r[k - k0], side != nullptr, mu, rs, ga, be, dz, p, me, px, ps, k);
          if (p.dres) gn_pack(dy[k], dz);
        }
        if (p.dres) dy[k].store(pdr.at(k));
#pragma unroll
        for (int e = 0; e < V; ++e) dz[e] = rs[e] * ga[e] * dz[e] - (k1[e] + (x[k].get(e) - mu[e]) * k2[e]);
        gn_pack(x[k], dz);
        x[k].store(pdx.at(k));
      }
  }
}

// Sums of a range of pixels, for each channel (slab [N][S][2][C]) and each group (coef [N][S][G][2]): R pixels a thread at a time.
template <typename T, int NT, int R, bool WHOLE>
__global__ void __launch_bounds__(NT, 4) gn_bwd_range_kernel(GnParams p) {
  constexpr int V = GnX<T>::N;
  extern __shared__ float lds[];          // sums of the channels [2][cw]; partial sums
  GnPlace<T, NT> me(p, xcd_remap(blockIdx.x, gridDim.x));
  const int g0 = me.c0 / p.cg, groups = p.W * V / p.cg, c = me.c(), cw = p.W * V, mode = p.act == ACT_RELU && p.yv ? GN_BY_Y : p.act;
  const void* side = p.act == ACT_NONE ? nullptr : p.yv ? p.yv : p.res;
  GnVec<V, WHOLE> mu, rs;
  auto group = [&](int e) { return (long long)me.n * p.G + g0 + (me.on ? (me.w * V + e) / p.cg : 0); };
  mu.set([&](int e) { return p.mean[group(e)]; });
  rs.set([&](int e) { return p.rstd[group(e)]; });
  float ga[V], be[V], a[V], b[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    ga[e] = me.on ? p.gamma[c + e] : 0.f; be[e] = me.on ? p.beta[c + e] : 0.f; a[e] = 0.f; b[e] = 0.f;
  }
  for (; me.p0 < me.p1; me.p0 += p.rows * R) {
    const auto px = me.ref(p, p.x, p.x_cs), pd = me.ref(p, p.dy, p.dy_cs), ps = me.ref(p, side, p.yv ? p.yv_cs : p.res_cs);
    GnX<T> x[R], dy[R], r[R];
#pragma unroll
    for (int k = 0; k < R; ++k)
      if (me.has(p, k)) {
        x[k].load(px.at(k)); dy[k].load(pd.at(k));
        if (side) r[k].load(ps.at(k));
      }
#pragma unroll
    for (int k = 0; k < R; ++k)
      if (me.has(p, k)) {
        float dz[V];
#pragma unroll
        for (int e = 0; e < V; ++e) dz[e] = dy[k].get(e);
        if (mode != ACT_NONE) gn_dz_vec<T>(mode, x[k], r[k], side != nullptr, mu, rs, ga, be, dz, p, me, px, ps, k);
#pragma unroll
        for (int e = 0; e < V; ++e) { a[e] += dz[e]; b[e] += dz[e] * (x[k].get(e) - mu[e]); }
      }
  }
#pragma unroll
  for (int e = 0; e < V; ++e) b[e] *= rs[e];
  gn_channel_sum<V, NT>(p, me.on, me.row, me.w, a, b, lds + 2 * cw, lds);
  if (p.dgamma || p.dbeta) {
    float* o = p.slab + ((long long)me.n * p.S + me.s) * 2 * p.C + me.c0;
    for (int i = threadIdx.x; i < cw; i += NT) { o[i] = lds[i]; o[p.C + i] = lds[cw + i]; }
  }
  float* o = p.coef + (((long long)me.n * p.S + me.s) * p.G + g0) * 2;
  gn_group_grads<NT>(p, me.c0, groups, lds, lds + cw, [&](int g, float ta, float tb) { o[2 * g] = ta; o[2 * g + 1] = tb; });
}

template <typename T, int NT, int R, bool WHOLE>
__global__ void __launch_bounds__(NT, 4) gn_bwd_apply_kernel(GnParams p) {
  constexpr int V = GnX<T>::N;
  __shared__ float c1[GN_GROUPS], c2[GN_GROUPS];
  GnPlace<T, NT> me(p, gridDim.x - 1 - xcd_remap(blockIdx.x, gridDim.x));
  const int g0 = me.c0 / p.cg, groups = p.W * V / p.cg, c = me.c();
  const void* side = p.act == ACT_NONE ? nullptr : p.yv ? p.yv : p.res;
  const int lane = threadIdx.x & 63;
  const float inv = 1.f / ((float)p.HW * (float)p.cg);
  for (int g = threadIdx.x >> 6; g < groups; g += NT / 64) {
    float ta = 0.f, tb = 0.f;
    for (int s = lane; s < p.S; s += 64) {
      const float* e = p.coef + (((long long)me.n * p.S + s) * p.G + g0 + g) * 2;
      ta += e[0]; tb += e[1];
    }
    ta = wave_sum(ta); tb = wave_sum(tb);
    if (lane == 0) { c1[g] = ta * inv; c2[g] = tb * inv; }
  }
  __syncthreads();
  if (!me.on) return;
  GnVec<V, WHOLE> mu, rs, k1, k2;
  auto group = [&](int e) { return (me.w * V + e) / p.cg; };
  mu.set([&](int e) { return p.mean[(long long)me.n * p.G + g0 + group(e)]; });
  rs.set([&](int e) { return p.rstd[(long long)me.n * p.G + g0 + group(e)]; });
  k1.set([&](int e) { return c1[group(e)] * rs[e]; });
  k2.set([&](int e) { return c2[group(e)] * rs[e] * rs[e]; });
  float ga[V], be[V];
#pragma unroll
  for (int e = 0; e < V; ++e) { ga[e] = p.gamma[c + e]; be[e] = p.beta[c + e]; }
  const int mode = p.act == ACT_RELU && p.yv ? GN_BY_Y : p.act;
  for (; me.p0 < me.p1; me.p0 += p.rows * R) {
    const auto px = me.ref(p, p.x, p.x_cs), pd = me.ref(p, p.dy, p.dy_cs), pdx = me.ref(p, p.dx, p.dx_cs), pdr = me.ref(p, p.dres, p.dres_cs);
    const auto ps = me.ref(p, side, p.yv ? p.yv_cs : p.res_cs);
    GnX<T> x[R], dy[R], r[R];
#pragma unroll
    for (int k = 0; k < R; ++k)
      if (me.has(p, k)) {
        x[k].load(px.at(k)); dy[k].load(pd.at(k));
        if (side) r[k].load(ps.at(k));
      }
#pragma unroll
    for (int k = 0; k < R; ++k)
      if (me.has(p, k)) {
        float dz[V];
#pragma unroll
        for (int e = 0; e < V; ++e) dz[e] = dy[k].get(e);
        if (mode != ACT_NONE) gn_dz_vec<T>(mode, x[k], r[k], side != nullptr, mu, rs, ga, be, dz, p, me, px, ps, k);
        if (p.dres) { gn_pack(dy[k], dz); dy[k].store(pdr.at(k)); }
#pragma unroll
        for (int e = 0; e < V; ++e) dz[e] = rs[e] * ga[e] * dz[e] - (k1[e] + (x[k].get(e) - mu[e]) * k2[e]);
        gn_pack(x[k], dz);
        x[k].store(pdx.at(k));
      }
  }
}

template <typename T, int ACT, bool RES>
static int gn_any(const GnParams& p, bool bwd, hipStream_t s) {
  const dim3 grid((p.C + 63) / 64, p.S, min(p.N, 16384));
  const int groups = (int)min((long long)p.N * p.G, 65536LL);
  if (!bwd) {
    gn_stats_kernel<T><<<grid, 256, 0, s>>>(p);
    gn_moments_kernel<<<groups, 256, 0, s>>>(p);
    gn_apply_kernel<T, ACT, RES><<<grid, 256, 0, s>>>(p);
  } else {
    gn_bwd_sums_kernel<T, ACT, RES><<<grid, 256, 0, s>>>(p);
    const int strips = p.dgamma || p.dbeta ? (p.C + 15) / 16 : 0;
    gn_bwd_params_kernel<<<strips + (groups + 3) / 4, 1024, 0, s>>>(p, strips);
    gn_bwd_dx_kernel<T, ACT, RES><<<grid, 256, 0, s>>>(p);
  }
  return 0;
}

// The kernel `Fwd` or `Bwd` of whole vectors in groups or not.  LDS: at most 4 * (2 * groups + 2 * 256 * V + 2 * NT * V) bytes
// (W <= 256, rows * W <= NT).
template <typename T, int NT, int R, bool WHOLE, int WAY>
static void gn_fwd(const GnParams& p, int grid, int rows, hipStream_t s) {
  gn_fwd_kernel<T, NT, R, WHOLE, WAY><<<grid, NT, 4 * (2 * (p.W * GnX<T>::N / p.cg) + rows * p.W * (WHOLE ? 1 : GnX<T>::N)), s>>>(p);
}
template <typename T, int NT, int R, bool WHOLE>
static void gn_bwd(const GnParams& p, int grid, int rows, hipStream_t s) {
  gn_bwd_kernel<T, NT, R, WHOLE><<<grid, NT, 4 * (2 * (p.W * GnX<T>::N / p.cg) + 2 * p.W * GnX<T>::N * (1 + rows)), s>>>(p);
}

template <typename T, int NT, int R, bool WHOLE>
static void gn_bwd_two(const GnParams& p, int grid, int rows, hipStream_t s) {
  gn_bwd_range_kernel<T, NT, R, WHOLE><<<grid, NT, 4 * 2 * p.W * GnX<T>::N * (1 + rows), s>>>(p);
  gn_bwd_apply_kernel<T, NT, R, WHOLE><<<grid, NT, 0, s>>>(p);
}

template <typename T>
static int gn_sizes(const GnParams& p, bool bwd, hipStream_t s) {
  constexpr int V = GnX<T>::N;
  const bool whole = p.cg % V == 0;
  const int grid = p.N * p.S * (p.C / (p.W * V)), rows = gn_even(p.W) ? p.threads / 64 : p.rows;          // rows of partial sums
  const int which = p.way * 1000000 + bwd * 500000 + p.threads * 100 + p.R;
#define GN_FWD(WAY, NT, R) case WAY * 1000000 + NT * 100 + R: if (whole) gn_fwd<T, NT, R, true, WAY>(p, grid, rows, s); else gn_fwd<T, NT, R, V == 1, WAY>(p, grid, rows, s); break;
#define GN_BWD(WAY, NT, R) case WAY * 1000000 + 500000 + NT * 100 + R: if (whole) gn_bwd<T, NT, R, true>(p, grid, rows, s); else gn_bwd<T, NT, R, V == 1>(p, grid, rows, s); break;
#define GN_BOTH(WAY, NT, R) GN_FWD(WAY, NT, R) GN_BWD(WAY, NT, R)
  if constexpr (V > 1) {
    switch (which) {
      GN_BOTH(GN_ONE, 256, 1) GN_BOTH(GN_ONE, 256, 2) GN_BOTH(GN_ONE, 512, 4) GN_BOTH(GN_ONE, 512, 7) GN_BOTH(GN_ONE, 512, 13) GN_FWD(GN_ONE, 1024, 13)
      case GN_TWO * 1000000 + 512 * 100 + 8:
        if (whole) gn_fwd<T, 512, 8, true, GN_TWO>(p, grid, rows, s); else gn_fwd<T, 512, 8, false, GN_TWO>(p, grid, rows, s);
        gn_fwd_apply_kernel<T, 512, 8><<<grid, 512, 0, s>>>(p);
        break;
      case GN_TWO * 1000000 + 500000 + 512 * 100 + 2:
        if (whole) gn_bwd_two<T, 512, 2, true>(p, grid, rows, s); else gn_bwd_two<T, 512, 2, false>(p, grid, rows, s);
        break;
      default: return (int)hipErrorInvalidValue;
    }
  } else {
    switch (which) {
      GN_BOTH(GN_LONE, 256, 4) GN_BOTH(GN_LONE, 512, 16)
      default: return (int)hipErrorInvalidValue;
    }
  }
#undef GN_BOTH
#undef GN_FWD
#undef GN_BWD
  return 0;
}

template <typename T>
static int gn_launch(const GnParams& p, bool bwd, hipStream_t s) {
  int rc = 0;
  if (p.way == GN_ANY) {
    const bool res = p.res || p.dres;
#define GN_CASE(A) case A: if (res) gn_any<T, A, true>(p, bwd, s); else gn_any<T, A, false>(p, bwd, s); break;
    switch (p.act) { GN_CASE(ACT_NONE) GN_CASE(ACT_RELU) GN_CASE(ACT_SILU) GN_CASE(ACT_GELU) default: return (int)hipErrorInvalidValue; }
#undef GN_CASE
  } else if (p.way == GN_LONE) {
    rc = gn_sizes<Lone<T>>(p, bwd, s);
  } else {
    rc = gn_sizes<T>(p, bwd, s);
  }
  if (rc) return rc;
  if (bwd && p.way != GN_ANY && (p.dgamma || p.dbeta)) gn_bwd_params_kernel<<<(p.C + 15) / 16, 1024, 0, s>>>(p, (p.C + 15) / 16);
  return dpa_launch_rc();
}

// Vectors that are written touch nothing else, and no activation that is written touches a vector that is read (which activations may
// be one another the caller has checked).  Here because two dozen comparisons take the caller's language a microsecond.
static bool gn_overlap(const GnParams& p, bool bwd, int es) {
  struct Span { const char *a, *b; };
  Span vout[2], vin[4], mout[2], min_[4];
  int nvo = 0, nvi = 0, nmo = 0, nmi = 0;
  const auto vec = [&](Span* to, int& n, const void* q, long long len) { if (q) to[n++] = {(const char*)q, (const char*)q + 4 * len}; };
  const auto map = [&](Span* to, int& n, const void* q, long long cs) {
    if (q) to[n++] = {(const char*)q, (const char*)q + (((long long)p.N * p.HW - 1) * cs + p.C) * es};
  };
  const long long ng = (long long)p.N * p.G;
  vec(vin, nvi, p.gamma, p.C); vec(vin, nvi, p.beta, p.C);
  vec(bwd ? vin : vout, bwd ? nvi : nvo, p.mean, ng); vec(bwd ? vin : vout, bwd ? nvi : nvo, p.rstd, ng);
  if (bwd) { vec(vout, nvo, p.dgamma, p.C); vec(vout, nvo, p.dbeta, p.C); }
  map(mout, nmo, p.y, p.y_cs); map(mout, nmo, p.dx, p.dx_cs); map(mout, nmo, p.dres, p.dres_cs);
  map(min_, nmi, p.x, p.x_cs); map(min_, nmi, p.res, p.res_cs); map(min_, nmi, p.dy, p.dy_cs); map(min_, nmi, p.yv, p.yv_cs);
  const auto any = [](const Span& s, const Span* o, int n) { for (int k = 0; k < n; ++k) if (s.a < o[k].b && o[k].a < s.b) return true; return false; };
  for (int k = 0; k < nvo; ++k)
    if (any(vout[k], vout + k + 1, nvo - k - 1) || any(vout[k], vin, nvi) || any(vout[k], mout, nmo) || any(vout[k], min_, nmi)) return true;
  for (int k = 0; k < nmo; ++k) if (any(mout[k], vin, nvi)) return true;
  return false;
}

DPA_API int dpa_gn_params_size() { return (int)sizeof(GnParams); }
DPA_API int dpa_group_norm(const GnParams* p, int bwd, int f32, hipStream_t s) {
  if (gn_overlap(*p, bwd, f32 ? 4 : 2)) return -1;
  return f32 ? gn_launch<float>(*p, bwd, s) : gn_launch<bf16_t>(*p, bwd, s);
}
