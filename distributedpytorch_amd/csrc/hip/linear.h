// Products of a linear layer with what surrounds them fused into the epilogue.
//
//   fprop   z = x W^T + bias (+ addend),  y = act(z)                x [M, K], W [N, K]; z is kept for the backward pass
//   dgrad   dx = (dy W + addend) * act'(z)                          the derivative of the layer in FRONT, at its z [M, K]
//   wgrad   dW = dy^T x,  db = column sums of dy
//
// All three are C[i, j] = sum_k A(i, k) B(j, k) of bf16 operands with fp32 accumulators; they differ in which index of an
// operand is contiguous in memory: k (fprop: both; dgrad: dy) or i / j (dgrad: W; wgrad: both).
// fp32 operands are taken as three bf16 parts, x = p0 + p1 + p2 exactly, and the product as the six largest part products
// (the dropped ones are below 2^-23 of the term): the same kernel over six times the reduction, smallest terms first.
#pragma once
#include "act.h"
#include "conv_common.h"
#include <atomic>
#include <type_traits>

struct LinParams {
  const void *a, *b;                    // operands: bf16, row stride lda / ldb elements, parts a_part / b_part elements apart
  long long lda, ldb, a_part, b_part;
  const float* bias;                    // [cols]
  const void *addend, *pre;             // pre: z of the activation whose derivative is multiplied in
  void *out, *preact;
  float* ws;                            // [splits][rows][cols] partial products where splits > 1
  float* sums;                          // [splits * takers][rows] partial sums of a's rows (dy's columns), or null
  float* db;                            // [rows] what they are joined into, the bias gradient; null: sums is it
  long long ld_add, ld_pre, ld_out, ld_z;
  const void *src_a, *src_b;            // the operands as the caller has them
  long long src_lda, src_ldb;
  int rows, cols, K, splits, accumulate, act, vec, bias_vec, takers;      // vec: every matrix of the epilogue takes 16-byte access
};

// What a call hands over besides: the operands as they are, what they are packed into first (ld 0: nothing), the bias gradient.
struct LinCall {
  LinParams p;
  void *pack_a, *pack_b;
  float *db, *db_slab;
  int a_rows, a_cols, b_rows, b_cols, ld_a, ld_b, vec_a, vec_b, db_splits, epi, tile, f32;      // (f32: the operands are)
};

enum : int { EPI_FPROP = 0, EPI_DGRAD = 1, EPI_WGRAD = 2 };

__device__ __attribute__((aligned(16))) const unsigned lin_zero[4] = {0, 0, 0, 0};

// eight neighbouring elements of a row (n of them where the matrix ends or is not aligned: VEC = false)
template <typename T> struct Lin8;
template <> struct Lin8<bf16_t> {
  uint4 w;
  __device__ __forceinline__ float get(int e) const { const uint32_t u = ((const uint32_t*)&w)[e >> 1]; return __uint_as_float((e & 1) ? (u & 0xffff0000u) : (u << 16)); }
  template <bool VEC> __device__ __forceinline__ void load(const bf16_t* p, int n) {
    if (VEC) { w = *(const uint4*)p; return; }
    uint32_t o[4] = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e) if (e < n) o[e >> 1] |= (uint32_t)p[e] << (16 * (e & 1));
    w = make_uint4(o[0], o[1], o[2], o[3]);
  }
};
template <> struct Lin8<float> {
  float4 a, b;
  __device__ __forceinline__ float get(int e) const { return e < 4 ? ((const float*)&a)[e] : ((const float*)&b)[e - 4]; }
  template <bool VEC> __device__ __forceinline__ void load(const float* p, int n) {
    if (VEC) { a = *(const float4*)p; b = *(const float4*)(p + 4); return; }
#pragma unroll
    for (int e = 0; e < 8; ++e) { const float v = e < n ? p[e] : 0.f; if (e < 4) ((float*)&a)[e] = v; else ((float*)&b)[e - 4] = v; }
  }
};
template <bool VEC> __device__ __forceinline__ void lin_st8(float* p, int n, const float (&v)[8]) {
  if (VEC) { *(float4*)p = make_float4(v[0], v[1], v[2], v[3]); *(float4*)(p + 4) = make_float4(v[4], v[5], v[6], v[7]); return; }
#pragma unroll
  for (int e = 0; e < 8; ++e) if (e < n) p[e] = v[e];
}
template <bool VEC> __device__ __forceinline__ void lin_st8(bf16_t* p, int n, const float (&v)[8]) {
  if (VEC) {
    uint4 o;
    o.x = (uint32_t)f2bf(v[0]) | ((uint32_t)f2bf(v[1]) << 16); o.y = (uint32_t)f2bf(v[2]) | ((uint32_t)f2bf(v[3]) << 16);
    o.z = (uint32_t)f2bf(v[4]) | ((uint32_t)f2bf(v[5]) << 16); o.w = (uint32_t)f2bf(v[6]) | ((uint32_t)f2bf(v[7]) << 16);
    *(uint4*)p = o;
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) if (e < n) p[e] = f2bf(v[e]);
}

// What is fused behind the product, for columns [j, j + n) of row i.  The reads are apart from the rest: an output may be one
// of the inputs, so the compiler keeps loads behind stores, and a caller with several vectors reads for all of them first.
template <typename T> struct LinExtra { Lin8<T> add, pre; };          // (wgrad: add = what is accumulated to)

template <typename T, int EPI, int ACT, bool VEC>
__device__ __forceinline__ void lin_extra(const LinParams& p, int i, int j, int n, LinExtra<T>& x) {
  if (EPI == EPI_WGRAD) { if (p.accumulate) x.add.template load<VEC>((const T*)p.out + i * p.ld_out + j, n); return; }
  if (p.addend) x.add.template load<VEC>((const T*)p.addend + i * p.ld_add + j, n);
  if (EPI == EPI_DGRAD && ACT != ACT_NONE) x.pre.template load<VEC>((const T*)p.pre + i * p.ld_pre + j, n);
}

// An infinity is one part and two zeros, so its products with the other operand's parts hold infinity times zero, and differences of
// infinities: NaN where fp32 gives an infinity.  Elements that came out as NaN are computed again from the operands themselves,
// which are read where that happens: the kernels have no registers to keep their addresses in.  A call of 8192 x 4096 x 1024 takes
// 0.40 ms, with NaN everywhere 0.58 (a NaN ends its sum), with one infinity 2.3, with one in every row 49.
template <int EPI>
__device__ __forceinline__ float lin_again(bool bad, int i, int j, float v) {
  constexpr bool AT = EPI == EPI_WGRAD, BT = EPI != EPI_FPROP;
  auto p = (const __attribute__((address_space(4))) LinParams*)__builtin_amdgcn_kernarg_segment_ptr();      // (the first argument)
  asm volatile("" : "+s"(p));
  const float* a = (const float*)p->src_a + (AT ? i : i * p->src_lda);
  const float* b = (const float*)p->src_b + (BT ? j : j * p->src_ldb);
  const long long sa = AT ? p->src_lda : 1, sb = BT ? p->src_ldb : 1;
  if (bad) v = 0.f;
  const int last = p->K - 1;
#pragma unroll 1
  for (int k = 0; k <= last && __any(bad); k += 4)
    if (bad) {
      float x[4], y[4];          // (four loads in flight)
#pragma unroll
      for (int u = 0; u < 4; ++u) { x[u] = a[min(k + u, last) * sa]; y[u] = b[min(k + u, last) * sb]; }
#pragma unroll
      for (int u = 0; u < 4; ++u) v = k + u <= last ? fmaf(x[u], y[u], v) : v;
      bad = v == v;
    }
  return v;
}

template <typename T, int EPI, int ACT, bool VEC>
__device__ __forceinline__ void lin_finish(const LinParams& p, int i, int j, int n, const LinExtra<T>& x, const Lin8<float>& bias, float (&v)[8]) {
  if (EPI == EPI_FPROP) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += bias.get(e);
  }
  if (EPI == EPI_WGRAD ? p.accumulate != 0 : p.addend != nullptr) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += x.add.get(e);
  }
  if (EPI == EPI_FPROP) {
    if (p.preact) lin_st8<VEC>((T*)p.preact + i * p.ld_z + j, n, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = act_fwd<ACT>(v[e]);
  } else if (EPI == EPI_DGRAD && ACT != ACT_NONE) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= act_slope<ACT>(x.pre.get(e));
  }
  lin_st8<VEC>((T*)p.out + i * p.ld_out + j, n, v);
}

template <int EPI>
__device__ __forceinline__ Lin8<float> lin_bias(const LinParams& p, int j, bool whole) {
  Lin8<float> b;
  b.a = b.b = make_float4(0.f, 0.f, 0.f, 0.f);
  if (EPI == EPI_FPROP && p.bias && j < p.cols) { if (whole) b.load<true>(p.bias + j, 8); else b.load<false>(p.bias + j, p.cols - j); }
  return b;
}

// calls f(std::integral_constant<int, ACT>, std::bool_constant<VEC>) for the launch's activation and alignment
template <int EPI, typename F>
__device__ __forceinline__ void lin_by_kind(const LinParams& p, F f) {
  using std::integral_constant;
  if (EPI == EPI_WGRAD) { if (p.vec) f(integral_constant<int, 0>(), std::true_type()); else f(integral_constant<int, 0>(), std::false_type()); return; }
#define LIN_KIND(A) if (p.act == A) { if (p.vec) f(integral_constant<int, A>(), std::true_type()); else f(integral_constant<int, A>(), std::false_type()); return; }
  LIN_KIND(ACT_NONE) LIN_KIND(ACT_RELU) LIN_KIND(ACT_SILU) LIN_KIND(ACT_GELU)
#undef LIN_KIND
}

// ---- operand tiles in LDS ------------------------------------------------------------------------------------------------
// A K step is BK = 64 elements of one part, or 32 elements of all three parts of an fp32 operand.  A tile of R rows (i or j)
// holds R x BK bf16 in one of two layouts, both written by the LDS DMA in pieces of 1 KiB (64 lanes x 16 bytes), the swizzle
// applied to the SOURCE address:
//  k contiguous:   [R][BK], 16-byte chunk c of row r at c ^ s(r): 16 rows x one chunk fall on 16 different bank groups.  A
//                  fragment (lane l: row l & 15, 8 elements from k = 8 (l >> 4)) is one ds_read_b128.
//  k strided (T):  [BK][R], rows of R elements; a unit of 16 elements (32 bytes) u of row k at u ^ g(k).  A fragment is two
//                  ds_read_b64_tr_b16: 16 lanes read 4 rows x 16 elements and get them transposed.  g spreads the 8 rows that
//                  32 lanes read over the 64 banks.
template <int R> __device__ __forceinline__ int lin_g(int k) {
  return R >= 128 ? (k & 3) | (((k >> 3) & 1) << 2) : ((k >> 1) & 1) | (((k >> 3) & 1) << 1);
}
template <int BK> __device__ __forceinline__ int lin_s(int r) { return BK == 64 ? (r >> 1) & 7 : -(r >> 2) & 3; }

// source of one 16-byte chunk of a piece in this lane at K step 0 of part 0; k: the chunk's first k in the step
template <int R, bool T, int BK>
__device__ __forceinline__ const bf16_t* lin_source(const void* base, long long ld, int r0, int limit, int piece, int lane, int& k) {
  if (!T) {
    constexpr int CPR = BK / 8;                          // chunks in a row
    const int r = piece * (64 / CPR) + lane / CPR;
    k = ((lane % CPR) ^ lin_s<BK>(r)) * 8;
    return (const bf16_t*)base + (long long)min(r0 + r, limit - 1) * ld + k;
  }
  constexpr int KPP = 512 / R, LPR = R / 8;              // rows of k in a piece, lanes per row
  k = piece * KPP + lane / LPR;
  const int slot = lane % LPR, e = r0 + (((slot >> 1) ^ lin_g<R>(k)) * 2 + (slot & 1)) * 8;
  return (const bf16_t*)base + (long long)k * ld + (e < limit ? e : 0);
}

// One 16-row fragment of K part ks (32 elements).
template <int R, bool T, int BK>
__device__ __forceinline__ bf16x8 lin_fragment(const char* t, int u, int ks, int lane) {
  const int l15 = lane & 15, q4 = lane >> 4;
  if (!T) return *(const bf16x8*)(t + (u * 16 + l15) * (BK * 2) + ((ks * 4 + q4) ^ lin_s<BK>(l15)) * 16);
  const int k = ks * 32 + q4 * 8 + (l15 >> 2);
  const char* a = t + k * (R * 2) + (u ^ lin_g<R>(k)) * 32 + (l15 & 3) * 8;
  const auto lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) bf16x4*)a);
  const auto hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) bf16x4*)(a + 4 * R * 2));
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// all but this wave's newest N pieces have landed and its LDS reads are done; behind the barrier, everyone's
template <int N> __device__ __forceinline__ void lin_sync() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory"); }

// a kernel that can make the row sums on its way (the 256 x 256 tile has no registers for them, and one part a step would count
// the rows of fp32 operands once for each pass)
template <int MT, int EPI> constexpr bool lin_sums() { return EPI == EPI_WGRAD && MT <= 4; }

// The blocks are persistent and see ONE stream of K steps across their tiles, S of them in LDS: while step s is multiplied, the
// steps behind it land, and step s + S is requested as soon as the buffer of step s is free, also when it belongs to the next
// tile, so the epilogue of a tile runs under the first loads of the next.
// PARTS: of the operands, 1 (bf16) or 3 (fp32).  P: the parts of them in a step.
// P = 1: a step has four phases, each the matrix instructions of half the wave's rows and half the step; a phase first reads
// the fragments of the NEXT phase from LDS.  The barrier stands before the last phase: behind it everyone's reads of the
// buffer are done (registers hold what is left to multiply) and everyone's pieces of step s + 1 have landed.
// P = 3: all three parts of both operands, each fragment read once for the six products of fp32 (P = 1 on parts walks over
// them six times).  Half the LDS and DMA traffic, which is what bounds the smaller tiles (1021 x 1000 x 2048: the matrix pipe is busy
// 33 % of the time); the larger tile has no registers for it.  The fragments of step s + 1 are read while step s is multiplied.
template <typename T, int PARTS, int WM, int WN, int MT, int NT, int S, int P, int EPI>
__global__ void __launch_bounds__(WM * WN * 64, P == 3 && MT > 2 ? 1 : 2) lin_mfma_kernel(LinParams p) {
  constexpr bool AT = EPI == EPI_WGRAD, BT = EPI != EPI_FPROP;
  constexpr int BM = WM * MT * 16, BN = WN * NT * 16, NW = WM * WN, H = MT / 2, BK = P == 1 ? 64 : 32;
  constexpr int A_PART = BM * BK * 2, B_PART = BN * BK * 2, A_BYTES = P * A_PART, STAGE = A_BYTES + P * B_PART;
  constexpr int PA = A_BYTES / 1024 / NW, PB = (STAGE - A_BYTES) / 1024 / NW, PP = PA + PB;      // 1 KiB pieces a wave stages per step
  static_assert(PA >= 1 && PB >= 1 && MT % 2 == 0 && MT <= 8 && NT % 2 == 0 && S >= 2 && S <= 4, "tile");
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
  const int tm = (p.rows + BM - 1) / BM, tn = (p.cols + BN - 1) / BN, tiles = tm * tn, jobs = tiles * p.splits;
  constexpr int passes = P < PARTS ? 6 : 1;
  static_assert(P <= PARTS && !(passes > 1 && lin_sums<MT, EPI>()), "parts");
  const int ksteps = (p.K + BK - 1) / BK, total = ksteps * passes, per = (total + p.splits - 1) / p.splits;
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem);

  // blocks of one XCD get neighbouring tiles: panels of 8 tile rows, walked column by column
  auto place = [&](int job, int& i0, int& j0, int& split) {
    const int id = xcd_remap(job, jobs);
    split = id / tiles;
    const int tile = id - split * tiles, panel = tile / (8 * tn), in = tile - panel * 8 * tn, ph = min(8, tm - panel * 8);
    i0 = (panel * 8 + in % ph) * BM; j0 = (in / ph) * BN;
  };

  // ---- the stream of requests
  const bf16_t* ap[PA]; const bf16_t* bp[PB];
  int ak[PA], bk[PB];
  int d_job = blockIdx.x, d_kt = 0, d_end = 0, d_buf = 0;
  auto d_place = [&]() {
    int i0, j0, split;
    place(d_job, i0, j0, split);
    d_kt = split * per; d_end = min(d_kt + per, total);
    auto part = [](const bf16_t* at, int part, long long stride) { return P == 1 ? at : at + part * stride; };
#pragma unroll
    for (int q = 0; q < PA; ++q) {
      const int piece = wave * PA + q, of = P == 1 ? 0 : piece / (A_PART / 1024);
      ap[q] = part(lin_source<BM, AT, BK>(p.a, p.lda, i0, p.rows, piece - of * (A_PART / 1024), lane, ak[q]), of, p.a_part);
    }
#pragma unroll
    for (int q = 0; q < PB; ++q) {
      const int piece = wave * PB + q, of = P == 1 ? 0 : piece / (B_PART / 1024);
      bp[q] = part(lin_source<BN, BT, BK>(p.b, p.ldb, j0, p.cols, piece - of * (B_PART / 1024), lane, bk[q]), of, p.b_part);
    }
  };
  // A request is made piece by piece between matrix instructions: a block of them holds the wave until the address unit has
  // taken each (16 cycles a piece for every wave of the CU), and the matrix pipe idles behind it.  Behind the last step the
  // stream goes on with the last one again, into buffers that nobody reads any more.
  long long oa = 0, ob = 0;
  int left = 0;
  uint32_t stage = 0;
  auto next_step = [&]() __attribute__((always_inline)) {
    const int pass = passes == 1 ? 0 : d_kt / ksteps, ks = d_kt - pass * ksteps;
    // parts of the six products, smallest first: (2,0) (0,2) (1,1) (1,0) (0,1) (0,0)
    const int pa = passes == 1 ? 0 : (0x001102 >> (pass * 4)) & 15, pb = passes == 1 ? 0 : (0x010120 >> (pass * 4)) & 15;
    oa = pa * p.a_part + (AT ? ks * BK * p.lda : (long long)ks * BK);
    ob = pb * p.b_part + (BT ? ks * BK * p.ldb : (long long)ks * BK);
    left = p.K - ks * BK;
    stage = lds0 + d_buf * STAGE;
    d_buf = d_buf + 1 == S ? 0 : d_buf + 1;
  };
  auto request = [&](int q) __attribute__((always_inline)) {          // (zeros behind the end of an odd reduction)
    if (q < PA) dpa_glds16(ak[q] < left ? ap[q] + oa : (const bf16_t*)lin_zero, stage + (wave * PA + q) * 1024);
    else dpa_glds16(bk[q - PA] < left ? bp[q - PA] + ob : (const bf16_t*)lin_zero, stage + A_BYTES + (wave * PB + q - PA) * 1024);
  };
  auto requested = [&]() __attribute__((always_inline)) {
    if (++d_kt == d_end) { if (d_job + (int)gridDim.x < jobs) { d_job += gridDim.x; d_place(); } else --d_kt; }
  };

  f32x4 acc[MT][NT];
  // operands of the matrix instructions in (j, i) order: a lane then holds four neighbouring columns of one output row
  auto mfma = [](bf16x8 b, bf16x8 a, f32x4& c) __attribute__((always_inline)) { c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b, a, c, 0, 0, 0); };
  auto a_at = [&](int buf, int part, int i, int ks) __attribute__((always_inline)) {
    return lin_fragment<BM, AT, BK>(smem + buf * STAGE + part * A_PART, wm * MT + i, ks, lane);
  };
  auto b_at = [&](int buf, int part, int j, int ks) __attribute__((always_inline)) {
    return lin_fragment<BN, BT, BK>(smem + buf * STAGE + A_BYTES + part * B_PART, wn * NT + j, ks, lane);
  };

  d_place();
#pragma unroll 1
  for (int k = 0; k < S; ++k) {
    next_step();
#pragma unroll
    for (int q = 0; q < PP; ++q) request(q);
    requested();
  }
  lin_sync<(S - 1) * PP>();
  int buf = 0;
  for (int job = blockIdx.x; job < jobs; job += gridDim.x) {
    int i0, j0, split;
    place(job, i0, j0, split);
    int steps = min((split + 1) * per, total) - split * per;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
    // Sums of a's rows on the matrix pipe: a times ones, an accumulator for each row tile (one for all, with ones in a column
    // of each tile's own, would carry an infinity of one row, times zero, into others).  The waves that hold the same rows, WN in
    // each of the tiles of a row, take the steps in turn, so each pays in one step of `takers`.  bf16, 8192 x 4096 x 1024 with
    // the bias gradient: 92.2 us, without it 87.7, and a pass of its own over dy is 14; fp32, 2198 x 16 x 72: 14.2 and 13.8.
    constexpr bool SUMS = lin_sums<MT, EPI>();
    f32x4 sums[SUMS ? MT : 1];
#pragma unroll
    for (int i = 0; i < (SUMS ? MT : 1); ++i) sums[i] = (f32x4){0.f, 0.f, 0.f, 0.f};
    const int taker = j0 / BN * WN + wn;
    const bool takes = SUMS && p.sums && taker < p.takers;
    int turn = takes ? taker : 0x7fffffff;
    auto add_rows = [&](auto fragment, int count) __attribute__((always_inline)) {
      if constexpr (SUMS) {
        if (--turn < 0) {          // (one branch a step: the steps without it lose nothing)
          turn = p.takers - 1;
#pragma unroll
          for (int q = 0; q < count; ++q)
#pragma unroll
            for (int i = 0; i < MT; ++i) sums[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fragment(q, i), (bf16x8)(short)0x3F80, sums[i], 0, 0, 0);
        }
      }
    };
    if constexpr (P == 1) {
      bf16x8 fa[MT], fb[2][NT];
      auto read_a = [&](int half, int ks) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < H; ++i) fa[half * H + i] = a_at(buf, 0, half * H + i, ks);
      };
      auto read_b = [&](int ks) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < NT; ++j) fb[ks][j] = b_at(buf, 0, j, ks);
      };
      auto multiply = [&](int half, int ks) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < H; ++i)
#pragma unroll
          for (int j = 0; j < NT; ++j) mfma(fb[ks][j], fa[half * H + i], acc[half * H + i][j]);
      };
      read_b(0);
      read_a(0, 0);
      for (; steps > 0; --steps) {
        read_a(1, 0);
        multiply(0, 0);
        __builtin_amdgcn_sched_barrier(0);
        read_b(1);
        read_a(0, 1);
        multiply(1, 0);
        __builtin_amdgcn_sched_barrier(0);
        read_a(1, 1);
        multiply(0, 1);
        add_rows([&](int ks, int i) { return a_at(buf, 0, i, ks); }, 2);          // (fragments of its own)
        lin_sync<(S - 2) * PP>();
        buf = buf + 1 == S ? 0 : buf + 1;
        if (steps > 1) {
          read_b(0);
          read_a(0, 0);
        }
        next_step();
#pragma unroll
        for (int n = 0; n < H * NT; ++n) {
#pragma unroll
          for (int q = n * PP / (H * NT); q < (n + 1) * PP / (H * NT); ++q) { request(q); __builtin_amdgcn_sched_barrier(0); }
          mfma(fb[1][n % NT], fa[H + n / NT], acc[H + n / NT][n % NT]);
        }
        requested();
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      struct Parts { bf16x8 a[P][MT], b[P][NT]; } even, odd;
      auto read = [&](Parts& f) __attribute__((always_inline)) {
#pragma unroll
        for (int q = P - 1; q >= 0; --q) {          // (in the order of use)
#pragma unroll
          for (int i = 0; i < MT; ++i) f.a[q][i] = a_at(buf, q, i, 0);
#pragma unroll
          for (int j = 0; j < NT; ++j) f.b[P - 1 - q][j] = b_at(buf, P - 1 - q, j, 0);
        }
      };
      auto step = [&](Parts& f, Parts& next, bool more) __attribute__((always_inline)) {
        lin_sync<(S - 2) * PP>();          // (this wave's reads of the step are done: its buffer is free behind the barrier)
        buf = buf + 1 == S ? 0 : buf + 1;
        if (more) read(next);
        next_step();
        constexpr int EACH = 6 * MT * NT / PP;
#pragma unroll
        for (int n = 0; n < 6 * MT * NT; ++n) {          // parts (a, b), smallest products first: (2,0) (0,2) (1,1) (1,0) (0,1) (0,0)
          const int q = n / (MT * NT), i = n / NT % MT, j = n % NT;
          if (n % EACH == 0 && n / EACH < PP) { request(n / EACH); __builtin_amdgcn_sched_barrier(0); }
          mfma(f.b[(0x010120 >> (q * 4)) & 15][j], f.a[(0x001102 >> (q * 4)) & 15][i], acc[i][j]);
        }
        add_rows([&](int q, int i) { return f.a[P - 1 - q][i]; }, P);
        requested();
        __builtin_amdgcn_sched_barrier(0);
      };
      read(even);
      for (; steps > 1; steps -= 2) {
        step(even, odd, true);
        step(odd, even, steps > 2);
      }
      if (steps) step(even, odd, false);
    }

    if constexpr (SUMS) {
      if (takes && (lane & 15) == 0) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int row = i0 + (wm * MT + i) * 16 + (lane >> 4) * 4 + e;
            if (row < p.rows) {
              float* o = p.sums + ((long long)split * p.takers + taker) * p.rows + row;
              *o = !p.db && p.accumulate ? *o + sums[i][e] : sums[i][e];
            }
          }
      }
    }

    if constexpr (PARTS == 3) {
      bool some = false;
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) some |= __builtin_isunordered(acc[i][j][0], acc[i][j][1]) | __builtin_isunordered(acc[i][j][2], acc[i][j][3]);
      if (__any(some) && p.splits == 1) {          // (parts of a sum are joined first)
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          unsigned bad = 0;
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            const f32x4 c = acc[i][j];
            bad |= ((unsigned)(c[0] != c[0]) | (unsigned)(c[1] != c[1]) << 1 | (unsigned)(c[2] != c[2]) << 2 | (unsigned)(c[3] != c[3]) << 3) << (4 * j);
          }
          if (!__any(bad)) continue;
          const int row = i0 + (wm * MT + i) * 16 + (lane & 15);
#pragma unroll 1
          for (int n = 0; n < NT * 4; ++n) {
            const int col = j0 + (wn * NT + n / 4) * 16 + (lane >> 4) * 4 + (n & 3);
            const bool now = (bad >> n & 1) && row < p.rows && col < p.cols;
            if (!__any(now)) continue;
            const float v = lin_again<EPI>(now, row, col, 0.f);
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              const int e = now && n / 4 == j ? n & 3 : 4;
              const f32x4 c = acc[i][j];
              acc[i][j] = (f32x4){e == 0 ? v : c[0], e == 1 ? v : c[1], e == 2 ? v : c[2], e == 3 ? v : c[3]};
            }
          }
        }
      }
    }

    // ---- epilogue, from registers.  Neighbouring 16-column tiles trade quarters, so that a lane holds 8 columns of one row,
    // and the lanes are permuted so that four neighbouring ones hold 32 neighbouring columns: 64-byte requests instead of
    // 16-byte ones, each of which would take the address unit as long.
    // One row tile at a time in a rolled loop (the code of an activation is long); the accumulators are picked by a scalar
    // branch.  What bf16 epilogues read is requested one trip ahead.
    const int from = ((((lane & 1) << 1) | ((lane >> 1) & 1)) * 16 + (lane >> 2)) * 4;
    constexpr int NV = NT / 2;      // vectors of 8 columns a lane finishes in a trip
    auto where = [&](int i, int k, int& gi, int& gj) __attribute__((always_inline)) {
      gi = i0 + (wm * MT + i) * 16 + (lane >> 2);
      gj = j0 + (wn * NT + k * 2) * 16 + (lane & 3) * 8;
      return gi < p.rows && gj < p.cols;
    };
    auto trips = [&](auto before, auto finish) __attribute__((always_inline)) {
      before(0);
#pragma unroll 1
      for (int i = 0; i < MT; ++i) {
        f32x4 t[NT];
        switch (i) {
#define LIN_PICK(I) case I: for (int j = 0; j < NT; ++j) t[j] = acc[I < MT ? I : 0][j]; break;
          LIN_PICK(0) LIN_PICK(1) LIN_PICK(2) LIN_PICK(3) LIN_PICK(4) LIN_PICK(5) LIN_PICK(6) LIN_PICK(7)
#undef LIN_PICK
        }
        float v[NV][8];
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const auto w = __builtin_amdgcn_permlane16_swap(__float_as_uint(t[2 * k][e]), __float_as_uint(t[2 * k + 1][e]), false, false);
            v[k][e] = __int_as_float(__builtin_amdgcn_ds_bpermute(from, w[0]));
            v[k][e + 4] = __int_as_float(__builtin_amdgcn_ds_bpermute(from, w[1]));
          }
        finish(i, v);
      }
    };
    int gi, gj;
    if (p.splits > 1) {
      float* ws = p.ws + (long long)split * p.rows * p.cols;
      const bool vec = (p.cols & 7) == 0;
      trips([](int) {}, [&](int i, float (&v)[NV][8]) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
          if (where(i, k, gi, gj)) {
            float* o = ws + (long long)gi * p.cols + gj;
            if (vec) lin_st8<true>(o, 8, v[k]); else lin_st8<false>(o, min(8, p.cols - gj), v[k]);
          }
      });
    } else {
      lin_by_kind<EPI>(p, [&](auto act, auto vec) __attribute__((always_inline)) {
        constexpr int ACT = decltype(act)::value;
        constexpr bool VEC = decltype(vec)::value, AHEAD = sizeof(T) == 2 && VEC;
        LinExtra<T> x[NV], y[NV];
        Lin8<float> bias[NV];
#pragma unroll
        for (int k = 0; k < NV; ++k) { where(0, k, gi, gj); bias[k] = lin_bias<EPI>(p, gj, p.bias_vec); }
        auto load = [&](int i, LinExtra<T> (&to)[NV]) __attribute__((always_inline)) {
#pragma unroll
          for (int k = 0; k < NV; ++k)
            if (where(i, k, gi, gj)) lin_extra<T, EPI, ACT, VEC>(p, gi, gj, VEC ? 8 : min(8, p.cols - gj), to[k]);
        };
        trips([&](int i) __attribute__((always_inline)) { if (AHEAD) load(i, y); },
              [&](int i, float (&v)[NV][8]) __attribute__((always_inline)) {
                if (AHEAD) {
#pragma unroll
                  for (int k = 0; k < NV; ++k) x[k] = y[k];
                  if (i + 1 < MT) load(i + 1, y);
                } else {
                  load(i, x);
                }
#pragma unroll
                for (int k = 0; k < NV; ++k)
                  if (where(i, k, gi, gj)) lin_finish<T, EPI, ACT, VEC>(p, gi, gj, VEC ? 8 : min(8, p.cols - gj), x[k], bias[k], v[k]);
              });
      });
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");          // no piece is on its way to LDS that is no longer this block's
}

// joins partial sums [parts][cols] in a fixed order: 16 columns a block of 256, 16 threads over the parts of each
__device__ __forceinline__ void lin_join_sums(const float* __restrict__ slab, int parts, int cols, int accumulate, float* __restrict__ out, int block) {
  __shared__ float sh[16][17];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, c = block * 16 + tx;
  float s = 0.f;
  if (c < cols) {
#pragma unroll 4
    for (int k = ty; k < parts; k += 16) s += slab[(long long)k * cols + c];
  }
  sh[ty][tx] = s;
  __syncthreads();
  if (ty == 0 && c < cols) {
    for (int k = 1; k < 16; ++k) s += sh[k][tx];
    out[c] = accumulate ? out[c] + s : s;
  }
}

// joins the partial products of a split reduction in a fixed order and applies the epilogue; the blocks behind the first `main`
// ones join the bias gradient
template <typename T, int PARTS, int EPI>
__global__ void __launch_bounds__(256) lin_join_kernel(LinParams p, int main) {
  if ((int)blockIdx.x >= main) return lin_join_sums(p.sums, p.splits * p.takers, p.rows, p.accumulate, p.db, blockIdx.x - main);
  const int groups = (p.cols + 7) / 8;
  const long long total = (long long)p.rows * groups, part = (long long)p.rows * p.cols;
  const bool whole = (p.cols & 7) == 0;
  for (long long t = blockIdx.x * 256LL + threadIdx.x; t < total; t += main * 256LL) {
    const int i = (int)(t / groups), j = (int)(t - (long long)i * groups) * 8, n = min(8, p.cols - j);
    float v[8] = {};
#pragma unroll 4
    for (int k = 0; k < p.splits; ++k) {
      Lin8<float> s;
      const float* w = p.ws + k * part + (long long)i * p.cols + j;
      if (whole) s.load<true>(w, 8); else s.load<false>(w, n);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += s.get(e);
    }
    if constexpr (PARTS == 3) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool bad = e < n && v[e] != v[e];
        if (__any(bad)) v[e] = lin_again<EPI>(bad, i, j + e, v[e]);
      }
    }
    lin_by_kind<EPI>(p, [&](auto act, auto vec) {
      LinExtra<T> x;
      lin_extra<T, EPI, decltype(act)::value, decltype(vec)::value>(p, i, j, n, x);
      lin_finish<T, EPI, decltype(act)::value, decltype(vec)::value>(p, i, j, n, x, lin_bias<EPI>(p, j, p.bias_vec), v);
    });
  }
}

// Blocks on the chip at a time: a multiple of 8 where a launch has several rounds (xcd_remap).
template <typename T, int PARTS, int WM, int WN, int MT, int NT, int S, int P, int EPI>
static int lin_run(const LinParams& p, hipStream_t s) {
  constexpr int BM = WM * MT * 16, BN = WN * NT * 16;
  constexpr int lds = S * (BM + BN) * (P == 1 ? 128 : 192), residents = 160 * 1024 / lds;
  const long long jobs = (long long)((p.rows + BM - 1) / BM) * ((p.cols + BN - 1) / BN) * p.splits;
  if (jobs > 0x7FFFFFFF) return (int)hipErrorInvalidConfiguration;
  if (lds > 64 * 1024) {          // once for each device; a lost race sets it twice
    static std::atomic<unsigned> done[64];
    int dev = 0;
    if (const hipError_t e = hipGetDevice(&dev)) return (int)e;
    if (dev >= 64 || !done[dev].load(std::memory_order_relaxed)) {
      const hipError_t e = hipFuncSetAttribute((const void*)lin_mfma_kernel<T, PARTS, WM, WN, MT, NT, S, P, EPI>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
      if (e) return (int)e;
      if (dev < 64) done[dev].store(1, std::memory_order_relaxed);
    }
  }
  const int grid = (int)(jobs < 256 * residents ? jobs : 256 * residents);
  lin_mfma_kernel<T, PARTS, WM, WN, MT, NT, S, P, EPI><<<grid, WM * WN * 64, lds, s>>>(p);
  if (p.splits > 1) {
    const int main = dpa_grid((long long)p.rows * ((p.cols + 7) / 8), 256);
    lin_join_kernel<T, PARTS, EPI><<<main + (p.sums ? (p.rows + 15) / 16 : 0), 256, 0, s>>>(p, main);
  }
  return dpa_launch_rc();
}

template <typename T, int PARTS, int EPI>
static int lin_tile(const LinParams& p, int tile, hipStream_t s) {
  if (tile == 0) return lin_run<T, PARTS, 2, 4, 8, 4, 2, 1, EPI>(p, s);      // 256 x 256, 8 waves
  if constexpr (PARTS == 1) {
    switch (tile) {
      case 1: return lin_run<T, 1, 2, 2, 4, 4, 2, 1, EPI>(p, s);      // 128 x 128, 4 waves, two blocks a CU
      case 2: return lin_run<T, 1, 2, 2, 4, 4, 4, 1, EPI>(p, s);      // 128 x 128, four steps in LDS
      case 3: return lin_run<T, 1, 2, 2, 2, 2, 4, 1, EPI>(p, s);      // 64 x 64, two blocks a CU
    }
  } else {
    switch (tile) {
      case 4: return lin_run<T, 3, 2, 2, 4, 4, 3, 3, EPI>(p, s);      // 128 x 128, three parts at once, one block a CU
      case 5: return lin_run<T, 3, 2, 2, 2, 2, 3, 3, EPI>(p, s);      // 64 x 64, three parts at once, two blocks a CU
    }
  }
  return (int)hipErrorInvalidValue;
}
