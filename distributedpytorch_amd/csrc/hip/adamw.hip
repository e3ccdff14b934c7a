// AdamW over the tensors of a parameter arena in one launch, with per-tensor learning-rate and decay multipliers, states in
// 32 bits or in 8.
//
//   m' = b1 m + (1 - b1) g      v' = b2 v + (1 - b2) g^2
//   p' = p (1 - lr wd) - lr / (1 - b1^t) * m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// Every tensor of the arena starts at a multiple of 64 elements; group_ids[i] names the row (lr multiplier, decay
// multiplier) of `groups` that the i-th run of 64 elements uses; the last row stands in for rows that are not there.  `hyper`
// is the vector of optim.hip (slots at its top): in device memory, so a captured graph follows lr and step.
//
// Both kernels are bound by memory: one read and one write of every operand, 30 bytes a parameter with 32-bit
// states and 18.25 with 8-bit ones (p 8, g 4, p16 2, states 16, or 4 and 0.25 of scales).  Operands that no kernel reads before the next step, larger together than
// the caches, pass them by (nontemporal), and many short-lived blocks keep more requests in flight than 2048 long ones: 25.6
// million parameters with p16 159 us in 2048 blocks with cached accesses, 147 in 16384, 124 (6.2 TB/s) with nontemporal ones.
// The 8-bit kernel computes some 110 instructions an element beside its bytes: 132.9 million parameters 528 us with
// IEEE square roots, divisions and rounding by ldexp in 2048 blocks, 499 in 16384, 469 (5.2 TB/s) with the forms below; one
// block a vector, or 4 elements a lane, was no faster (458, 487).
#include "common.h"
#include <algorithm>

typedef __attribute__((ext_vector_type(4))) float adamw_f4;
__device__ __forceinline__ float4 adamw_ld(const float* q) { return __builtin_bit_cast(float4, __builtin_nontemporal_load((const adamw_f4*)q)); }
__device__ __forceinline__ void adamw_st(float* q, float4 x) { __builtin_nontemporal_store(__builtin_bit_cast(adamw_f4, x), (adamw_f4*)q); }
static int adamw_grid(long long threads) { return (int)std::min<long long>(16384, (threads + 255) / 256); }

struct AdamwScalars { float lr, wd, b2, eps, gs, omb1, omb2, inv_bc1, bc2s, inv_bc2s; };

__device__ __forceinline__ AdamwScalars adamw_scalars(const float* __restrict__ h) {
  AdamwScalars a;
  a.lr = h[0]; a.wd = h[4]; a.b2 = h[2]; a.eps = h[3]; a.gs = h[7]; a.omb1 = h[8]; a.omb2 = h[9];
  const double t = (double)h[5] + 1.0, b1 = (double)h[1] + (double)h[10], b2 = (double)h[2] + (double)h[11];
  a.inv_bc1 = (float)(1.0 / (1.0 - pow(b1, t)));
  const double bc2s = sqrt(1.0 - pow(b2, t));
  a.bc2s = (float)bc2s;
  a.inv_bc2s = (float)(1.0 / bc2s);
  return a;
}

// FAST: square root and reciprocal of the hardware, one unit in the last place each, of an update that is added to a parameter
template <bool FAST>
__device__ __forceinline__ float adamw_one(const AdamwScalars& a, float lr, float keep, float p, float g, float& m, float& v) {
  {
    // (rounded operation by operation: an 8-bit code follows from the last bits of a moment, and so it is the same wherever this
    // formula is computed in fp32)
#pragma clang fp contract(off)
    g = g * a.gs;
    m = m + a.omb1 * (g - m);
    v = a.b2 * v + a.omb2 * g * g;
  }
  if (FAST) {
    const bool small = v < 0x1p-96f;          // (the hardware's root of a denormal number is 0)
    const float root = __builtin_amdgcn_sqrtf(small ? v * 0x1p64f : v) * (small ? 0x1p-32f : 1.f);
    return p * keep - (lr * a.inv_bc1) * (m * __builtin_amdgcn_rcpf(root * a.inv_bc2s + a.eps));
  }
  return p * keep - (lr * a.inv_bc1) * (m / (sqrtf(v) / a.bc2s + a.eps));
}

__global__ void __launch_bounds__(256) adamw_kernel(float* __restrict__ p, const float* __restrict__ g, float* __restrict__ m,
                                                    float* __restrict__ v, bf16_t* __restrict__ p16,
                                                    const float* __restrict__ hyper, const float2* __restrict__ groups, int rows,
                                                    const unsigned char* __restrict__ ids, long long n) {
  const AdamwScalars a = adamw_scalars(hyper);
  const long long stride = (long long)gridDim.x * blockDim.x * 4;
  for (long long i = ((long long)blockIdx.x * blockDim.x + threadIdx.x) * 4; i < n; i += stride) {      // n % 64 == 0
    const float2 grp = groups[min((int)ids[i >> 6], rows - 1)];
    const float lr = a.lr * grp.x, keep = 1.f - lr * (a.wd * grp.y);
    float4 pp = adamw_ld(p + i), mm = adamw_ld(m + i), vv = adamw_ld(v + i);
    const float4 gg = adamw_ld(g + i);
    float* pa = (float*)&pp; float* ma = (float*)&mm; float* va = (float*)&vv; const float* ga = (const float*)&gg;
#pragma unroll
    for (int k = 0; k < 4; ++k) pa[k] = adamw_one<false>(a, lr, keep, pa[k], ga[k], ma[k], va[k]);
    adamw_st(p + i, pp); adamw_st(m + i, mm); adamw_st(v + i, vv);
    if (p16) {
      uint2 o;
      o.x = (uint32_t)f2bf(pa[0]) | ((uint32_t)f2bf(pa[1]) << 16);
      o.y = (uint32_t)f2bf(pa[2]) | ((uint32_t)f2bf(pa[3]) << 16);
      *(uint2*)(p16 + i) = o;
    }
  }
}

// ---- 8-bit states ------------------------------------------------------------------------------------------------------
// m is e4m3 and v is e5m2, each times one fp32 scale per 64 elements (64 is the arena's alignment: a scale never spans two
// tensors).  The scale maps the block's largest finite magnitude to the format's largest value.  Rounding is stochastic:
// with b2 = 0.999 a step moves v by about 0.1 % while neighbouring codes lie 12 to 25 % apart, so round-to-nearest would
// never let it move; rounded up with the probability of the remainder the expected state follows the 32-bit one.  The
// random numbers are a hash of (seed, step, element), so a step is reproducible and equal on every rank.
// A second moment that is not zero is never rounded to zero (it would turn m / sqrt(v) into m / eps): it keeps the smallest
// code.  Entries that are not finite take the largest code and are left out of the scale, so they spoil no neighbour.
// A block whose largest magnitude is below 2^-100 holds zeros: sqrt(v) of it is far below any eps, and 1 / scale stays finite.
__device__ __forceinline__ uint32_t adamw_mix(uint32_t h) {        // finalizer of MurmurHash3 (Appleby)
  h ^= h >> 16; h *= 0x85EBCA6Bu; h ^= h >> 13; h *= 0xC2B2AE35u;
  return h ^ (h >> 16);
}

// |t| * inv rounded to a multiple of its binade's step, up with the probability of the remainder (u in (0, 1)).  Below 2^LEAST
// the step stays the same.  The step and its inverse are powers of two made from the exponent bits: no product here rounds.
template <int LEAST, int BITS>
__device__ __forceinline__ float adamw_round(float t, float inv, float top, float u) {
  float y = fabsf(t) * inv;
  y = y < top ? y : top;                                   // (also NaN)
  const uint32_t e = max(__float_as_uint(y) & 0x7F800000u, (uint32_t)(LEAST + 127) << 23);
  const float q = floorf(y * __uint_as_float(((uint32_t)(254 + BITS) << 23) - e) + u) * __uint_as_float(e - ((uint32_t)BITS << 23));
  return q < top ? q : top;
}

__device__ __forceinline__ float adamw_block_max(float a) {        // over the 8 lanes that share a block
  a = fmaxf(a, __shfl_xor(a, 1, 64)); a = fmaxf(a, __shfl_xor(a, 2, 64));
  return fmaxf(a, __shfl_xor(a, 4, 64));
}

__global__ void __launch_bounds__(256) adamw8_kernel(float* __restrict__ p, const float* __restrict__ g, unsigned char* __restrict__ m8,
                                                     unsigned char* __restrict__ v8, float* __restrict__ ms, float* __restrict__ vs,
                                                     bf16_t* __restrict__ p16, const float* __restrict__ hyper,
                                                     const float2* __restrict__ groups, int rows,
                                                     const unsigned char* __restrict__ ids, uint32_t seed, long long first, long long n) {
  const AdamwScalars a = adamw_scalars(hyper);
  const uint32_t key = adamw_mix(seed + (uint32_t)(long long)hyper[5] * 0x9E3779B9u);
  const long long stride = (long long)gridDim.x * blockDim.x * 8;
  for (long long i = ((long long)blockIdx.x * blockDim.x + threadIdx.x) * 8; i < n; i += stride) {      // whole blocks of 8 lanes
    const long long b = i >> 6;
    const float2 grp = groups[min((int)ids[b], rows - 1)];
    const float lr = a.lr * grp.x, keep = 1.f - lr * (a.wd * grp.y);
    const float sm = ms[b], sv = vs[b];
    float4 pp[2], gg[2];
    pp[0] = *(float4*)(p + i); pp[1] = *(float4*)(p + i + 4);
    gg[0] = *(const float4*)(g + i); gg[1] = *(const float4*)(g + i + 4);
    const uint2 mc = *(const uint2*)(m8 + i), vc = *(const uint2*)(v8 + i);
    float* pa = (float*)pp; const float* ga = (const float*)gg;
    float mv[8], vv[8], am = 0.f, av = 0.f;
#pragma unroll
    for (int k = 0; k < 8; k += 4) {
      const int mw = k ? mc.y : mc.x, vw = k ? vc.y : vc.x;
      const auto m0 = __builtin_amdgcn_cvt_pk_f32_fp8(mw, false), m1 = __builtin_amdgcn_cvt_pk_f32_fp8(mw, true);
      const auto v0 = __builtin_amdgcn_cvt_pk_f32_bf8(vw, false), v1 = __builtin_amdgcn_cvt_pk_f32_bf8(vw, true);
      mv[k] = m0[0] * sm; mv[k + 1] = m0[1] * sm; mv[k + 2] = m1[0] * sm; mv[k + 3] = m1[1] * sm;
      vv[k] = v0[0] * sv; vv[k + 1] = v0[1] * sv; vv[k + 2] = v1[0] * sv; vv[k + 3] = v1[1] * sv;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      pa[k] = adamw_one<true>(a, lr, keep, pa[k], ga[k], mv[k], vv[k]);
      const float x = fabsf(mv[k]), y = fabsf(vv[k]);
      am = fmaxf(am, x < INFINITY ? x : 0.f);
      av = fmaxf(av, y < INFINITY ? y : 0.f);
    }
    am = adamw_block_max(am); av = adamw_block_max(av);
    const bool some_m = am >= 0x1p-100f, some_v = av >= 0x1p-100f;
    const float im = some_m ? 1.f / am * 448.f : 0.f, iv = some_v ? 1.f / av * 57344.f : 0.f;
    uint32_t mo[2] = {0, 0}, vo[2] = {0, 0};
#pragma unroll
    for (int k = 0; k < 8; k += 2) {
      float qm[2], qv[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const unsigned long long at = (unsigned long long)(first + i + k + j);
        const uint32_t r = adamw_mix((uint32_t)at ^ key ^ ((uint32_t)(at >> 32) * 0x85EBCA6Bu));
        qm[j] = copysignf(adamw_round<-6, 3>(mv[k + j], im, 448.f, ((float)(r & 0xFFFFu) + 0.5f) * 0x1p-16f), mv[k + j]);
        qv[j] = adamw_round<-14, 2>(vv[k + j], iv, 57344.f, ((float)(r >> 16) + 0.5f) * 0x1p-16f);
        if (vv[k + j] > 0.f && some_v) qv[j] = fmaxf(qv[j], 0x1p-16f);
      }
      // (both values are representable: these conversions round nothing)
      if (k & 2) {
        mo[k >> 2] = __builtin_amdgcn_cvt_pk_fp8_f32(qm[0], qm[1], mo[k >> 2], true);
        vo[k >> 2] = __builtin_amdgcn_cvt_pk_bf8_f32(qv[0], qv[1], vo[k >> 2], true);
      } else {
        mo[k >> 2] = __builtin_amdgcn_cvt_pk_fp8_f32(qm[0], qm[1], mo[k >> 2], false);
        vo[k >> 2] = __builtin_amdgcn_cvt_pk_bf8_f32(qv[0], qv[1], vo[k >> 2], false);
      }
    }
    *(float4*)(p + i) = pp[0]; *(float4*)(p + i + 4) = pp[1];
    *(uint2*)(m8 + i) = make_uint2(mo[0], mo[1]);
    *(uint2*)(v8 + i) = make_uint2(vo[0], vo[1]);
    if ((threadIdx.x & 7) == 0) { ms[b] = some_m ? am * (1.f / 448.f) : 0.f; vs[b] = some_v ? av * (1.f / 57344.f) : 0.f; }
    if (p16) {
      uint4 o;
      o.x = (uint32_t)f2bf(pa[0]) | ((uint32_t)f2bf(pa[1]) << 16); o.y = (uint32_t)f2bf(pa[2]) | ((uint32_t)f2bf(pa[3]) << 16);
      o.z = (uint32_t)f2bf(pa[4]) | ((uint32_t)f2bf(pa[5]) << 16); o.w = (uint32_t)f2bf(pa[6]) | ((uint32_t)f2bf(pa[7]) << 16);
      *(uint4*)(p16 + i) = o;
    }
  }
}

DPA_API int dpa_adamw_step(float* p, const float* g, float* m, float* v, bf16_t* p16, const float* hyper, const float* groups, int rows,
                           const unsigned char* ids, long long n, hipStream_t s) {
  if (n <= 0) return 0;
  hipLaunchKernelGGL(adamw_kernel, dim3(adamw_grid(n / 4)), dim3(256), 0, s, p, g, m, v, p16, hyper, (const float2*)groups, rows, ids, n);
  return dpa_launch_rc();
}
DPA_API int dpa_adamw8_step(float* p, const float* g, unsigned char* m8, unsigned char* v8, float* ms, float* vs, bf16_t* p16,
                            const float* hyper, const float* groups, int rows, const unsigned char* ids, unsigned int seed, long long first,
                            long long n, hipStream_t s) {
  if (n <= 0) return 0;
  hipLaunchKernelGGL(adamw8_kernel, dim3(adamw_grid(n / 8)), dim3(256), 0, s, p, g, m8, v8, ms, vs, p16, hyper,
                     (const float2*)groups, rows, ids, seed, first, n);
  return dpa_launch_rc();
}
