// Entry points of the linear products (linear.h), the operand packing and the bias gradient.
#include "linear.h"

int lin_fprop(const LinParams& p, int tile, bool f32, hipStream_t s);
int lin_dgrad(const LinParams& p, int tile, bool f32, hipStream_t s);
int lin_wgrad(const LinParams& p, int tile, bool f32, hipStream_t s);

// ---- operands that the DMA cannot take as they are -----------------------------------------------------------------------
// fp32 matrices become their three bf16 parts, bf16 matrices with odd rows or addresses a copy with rows of a multiple of 8;
// the columns behind the last one are zeros.  (An infinity has no remainder, its other parts are zero: lin_again.)
struct LinPack { const void* src; bf16_t* dst; long long ld; int rows, cols, ldd, vec; };

template <typename T>
__global__ void __launch_bounds__(256) lin_pack_kernel(LinPack one, LinPack two) {
  const LinPack& p = blockIdx.y ? two : one;
  const T* __restrict__ src = (const T*)p.src;
  const int groups = p.ldd / 8;
  const long long total = (long long)p.rows * groups, part = (long long)p.rows * p.ldd;
  for (long long t = blockIdx.x * 256LL + threadIdx.x; t < total; t += gridDim.x * 256LL) {
    const int i = (int)(t / groups), j = (int)(t - (long long)i * groups) * 8;
    Lin8<T> v;
    if (p.vec && j + 8 <= p.cols) v.template load<true>(src + i * p.ld + j, 8); else v.template load<false>(src + i * p.ld + j, p.cols - j);
    uint32_t o[3][4];
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      uint32_t w[3] = {0, 0, 0};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float x = v.get(e + h);
        bf16_t b0 = f2bf(x);
        if (sizeof(T) == 4) {
          const bool fin = fabsf(x) < INFINITY;
          if ((b0 & 0x7FFF) == 0x7F80 && fin) b0 = (bf16_t)(__float_as_uint(x) >> 16);      // (rounding does not overflow)
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
      *(uint4*)(p.dst + q * part + (long long)i * p.ldd + j) = make_uint4(o[q][0], o[q][1], o[q][2], o[q][3]);
  }
}

// ---- bias gradient where the product does not make it (lin_sums): column sums of dy [M, N] in two steps, S row ranges into a slab [S, N], then the slab in a fixed order.
// A lane owns one 16-byte vector of columns (VEC) or one column and keeps eight rows in flight; `lanes` lanes side by side.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) lin_colsum_kernel(const T* __restrict__ x, long long ld, int rows, int cols, int per, int lanes, float* __restrict__ slab) {
  constexpr int V = VEC ? 16 / (int)sizeof(T) : 1;
  __shared__ float sh[256 * V];
  const int tx = threadIdx.x % lanes, ty = threadIdx.x / lanes, nty = 256 / lanes, c = (blockIdx.x * lanes + tx) * V;
  const int r0 = blockIdx.y * per, r1 = min(r0 + per, rows);
  float s[V] = {};
  if (c < cols) {
    const T* q = x + c;
    int r = r0 + ty;
    auto add = [&](auto count) {
      constexpr int N = decltype(count)::value;
      if constexpr (VEC) {
        Vec16<T> t[N];
#pragma unroll
        for (int k = 0; k < N; ++k) t[k].load(q + (long long)(r + k * nty) * ld);
#pragma unroll
        for (int k = 0; k < N; ++k)
#pragma unroll
          for (int e = 0; e < V; ++e) s[e] += t[k].get(e);
      } else {
#pragma unroll
        for (int k = 0; k < N; ++k) s[0] += Elem<T>::ld(q + (long long)(r + k * nty) * ld);
      }
    };
    for (; r + 7 * nty < r1; r += 8 * nty) add(std::integral_constant<int, 8>());
    for (; r < r1; r += nty) add(std::integral_constant<int, 1>());
  }
#pragma unroll
  for (int e = 0; e < V; ++e) sh[(ty * lanes + tx) * V + e] = s[e];
  __syncthreads();
  for (int e = threadIdx.x; e < lanes * V; e += 256) {
    const int col = blockIdx.x * lanes * V + e;
    if (col < cols) {
      float t = 0.f;
      for (int k = 0; k < nty; ++k) t += sh[k * lanes * V + e];
      slab[(long long)blockIdx.y * cols + col] = t;
    }
  }
}
__global__ void __launch_bounds__(256) lin_colsum_join_kernel(const float* slab, int parts, int cols, int accumulate, float* out) {
  for (int b = blockIdx.x; b * 16LL < cols; b += gridDim.x) {
    lin_join_sums(slab, parts, cols, accumulate, out, b);
    __syncthreads();
  }
}
// (a launch has fewer than 2^32 threads)
static int lin_join_grid(int cols) { return (int)min((cols + 15LL) / 16, 65536LL); }

template <typename T>
static void lin_colsum(const LinCall& c, hipStream_t s) {
  const int rows = c.a_rows, cols = c.a_cols, per = (rows + c.db_splits - 1) / c.db_splits;
  const bool vec = c.vec_a && cols % (16 / (int)sizeof(T)) == 0;
  const int v = vec ? 16 / (int)sizeof(T) : 1, wide = (cols + v - 1) / v;
  int lanes = 64;
  while (lanes > 4 && lanes / 2 >= wide) lanes /= 2;
  const dim3 grid((wide + lanes - 1) / lanes, c.db_splits);
  if (vec) lin_colsum_kernel<T, true><<<grid, 256, 0, s>>>((const T*)c.p.src_a, c.p.src_lda, rows, cols, per, lanes, c.db_slab);
  else lin_colsum_kernel<T, false><<<grid, 256, 0, s>>>((const T*)c.p.src_a, c.p.src_lda, rows, cols, per, lanes, c.db_slab);
  lin_colsum_join_kernel<<<lin_join_grid(cols), 256, 0, s>>>(c.db_slab, c.db_splits, cols, c.p.accumulate, c.db);
}

// ---- few rows (fprop, M <= 16 * MT): the weights are read once, straight into registers ------------------------------------
// A block owns 16 output columns, its 8 waves the chunks of the reduction in turn (128 bytes of each weight row), and a
// wave's loads of U chunks are in flight together; the eight partial tiles are added in LDS in a fixed order.  A matrix
// instruction takes any order of k as long as both operands use the same one, so a lane keeps the bytes that it loads:
// 32 consecutive ones of a row.
template <typename T> struct LinRowChunk;
template <> struct LinRowChunk<bf16_t> {
  bf16x8 v[2];
  __device__ __forceinline__ void load(const bf16_t* p, int left) {
#pragma unroll
    for (int h = 0; h < 2; ++h) v[h] = left > 8 * h ? *(const bf16x8*)(p + 8 * h) : (bf16x8)(short)0;
  }
  __device__ __forceinline__ void zero() { v[0] = v[1] = (bf16x8)(short)0; }
  static __device__ __forceinline__ void mma(const LinRowChunk& w, const LinRowChunk& x, f32x4& c) {
#pragma unroll
    for (int h = 0; h < 2; ++h) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.v[h], x.v[h], c, 0, 0, 0);
  }
};
template <> struct LinRowChunk<float> {
  f32x4 v[2];
  __device__ __forceinline__ void load(const float* p, int left) {
#pragma unroll
    for (int h = 0; h < 2; ++h) v[h] = left > 4 * h ? *(const f32x4*)(p + 4 * h) : (f32x4){0.f, 0.f, 0.f, 0.f};
  }
  __device__ __forceinline__ void zero() { v[0] = v[1] = (f32x4){0.f, 0.f, 0.f, 0.f}; }
  static __device__ __forceinline__ void mma(const LinRowChunk& w, const LinRowChunk& x, f32x4& c) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(w.v[h][e], x.v[h][e], c, 0, 0, 0);
  }
};

template <typename T, int MT, int U>
__global__ void __launch_bounds__(512) lin_rows_kernel(LinParams p) {
  constexpr int LANE = 32 / (int)sizeof(T), CHUNK = 4 * LANE;      // elements of a lane and of a row in a chunk
  __shared__ float red[8][MT][16][17];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l15 = lane & 15, q4 = lane >> 4, n0 = blockIdx.x * 16;
  const T* w = (const T*)p.b + (long long)min(n0 + l15, p.cols - 1) * p.ldb + q4 * LANE;
  const T* x[MT];
  f32x4 acc[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    x[m] = (const T*)p.a + (long long)min(m * 16 + l15, p.rows - 1) * p.lda + q4 * LANE;
    acc[m] = (f32x4){0.f, 0.f, 0.f, 0.f};
  }
  for (int k0 = wave * CHUNK; k0 < p.K; k0 += 8 * U * CHUNK) {
    LinRowChunk<T> cw[U], cx[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u * 8 * CHUNK, left = p.K - k - q4 * LANE;
      if (left > 0) cw[u].load(w + k, left); else cw[u].zero();
#pragma unroll
      for (int m = 0; m < MT; ++m) { if (left > 0) cx[u][m].load(x[m] + k, left); else cx[u][m].zero(); }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int m = 0; m < MT; ++m) LinRowChunk<T>::mma(cw[u], cx[u][m], acc[m]);
  }
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int e = 0; e < 4; ++e) red[wave][m][l15][q4 * 4 + e] = acc[m][e];          // [row of x][column]
  __syncthreads();
  for (int t = threadIdx.x; t < MT * 256; t += 512) {
    const int m = t >> 8, r = (t >> 4) & 15, c = t & 15, i = m * 16 + r, j = n0 + c;
    if (i >= p.rows || j >= p.cols) continue;
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) v += red[k][m][r][c];
    if (p.bias) v += p.bias[j];
    if (p.addend) v += Elem<T>::ld((const T*)p.addend + i * p.ld_add + j);
    if (p.preact) Elem<T>::st((T*)p.preact + i * p.ld_z + j, v);
    v = p.act == ACT_NONE ? v : p.act == ACT_RELU ? act_fwd<ACT_RELU>(v) : p.act == ACT_SILU ? act_fwd<ACT_SILU>(v) : act_fwd<ACT_GELU>(v);
    Elem<T>::st((T*)p.out + i * p.ld_out + j, v);
  }
}

template <typename T>
static int lin_rows(const LinParams& p, hipStream_t s) {
  const int grid = (p.cols + 15) / 16;
  if (p.rows <= 16) lin_rows_kernel<T, 1, 8><<<grid, 512, 0, s>>>(p);
  else if (p.rows <= 32) lin_rows_kernel<T, 2, 4><<<grid, 512, 0, s>>>(p);
  else lin_rows_kernel<T, 4, 2><<<grid, 512, 0, s>>>(p);
  return dpa_launch_rc();
}

DPA_API int dpa_lin_params_size() { return (int)sizeof(LinCall); }

// tile: lin_tile's; -1: the kernel for few rows
DPA_API int dpa_linear(const LinCall* call, hipStream_t s) {
  const LinCall& c = *call;
  if (c.ld_a || c.ld_b) {
    LinPack a{c.p.src_a, (bf16_t*)c.pack_a, c.p.src_lda, c.a_rows, c.a_cols, c.ld_a, c.vec_a}, b{c.p.src_b, (bf16_t*)c.pack_b, c.p.src_ldb, c.b_rows, c.b_cols, c.ld_b, c.vec_b};
    if (!c.ld_a) a = b;
    const long long na = (long long)a.rows * (a.ldd / 8), nb = c.ld_a && c.ld_b ? (long long)b.rows * (b.ldd / 8) : 0;
    const dim3 grid(dpa_grid(na > nb ? na : nb, 256), nb ? 2 : 1);
    if (c.f32) lin_pack_kernel<float><<<grid, 256, 0, s>>>(a, b);
    else lin_pack_kernel<bf16_t><<<grid, 256, 0, s>>>(a, b);
    if (const int rc = dpa_launch_rc()) return rc;
  }
  int rc = (int)hipErrorInvalidValue;
  switch (c.epi) {
    case EPI_FPROP: rc = c.tile >= 0 ? lin_fprop(c.p, c.tile, c.f32, s) : c.f32 ? lin_rows<float>(c.p, s) : lin_rows<bf16_t>(c.p, s); break;
    case EPI_DGRAD: rc = lin_dgrad(c.p, c.tile, c.f32, s); break;
    case EPI_WGRAD: rc = lin_wgrad(c.p, c.tile, c.f32, s); break;
  }
  if (rc || !c.db) return rc;
  if (c.p.sums) {
    if (c.p.splits == 1 && c.p.db) lin_colsum_join_kernel<<<lin_join_grid(c.a_cols), 256, 0, s>>>(c.p.sums, c.p.takers, c.a_cols, c.p.accumulate, c.db);
  } else if (c.f32) lin_colsum<float>(c, s); else lin_colsum<bf16_t>(c, s);
  return dpa_launch_rc();
}
