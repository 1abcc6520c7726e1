// Row-wise kernels of the 8-bit formats (rows8.h): row codes for the int8 product, checkpoints, and the LayerNorm and GELU that write a checkpoint in
// their forward and read it in their backward.  All are bound by HBM (a 1 GiB copy runs at 5.1 TB/s, one of 64 MiB, which the Infinity Cache holds, at 8.1); each input
// is read once and each output written once.  Measured in a kernel trace, 16-bit data unless said: row codes 12288 x 3072 19 - 21 us (5.4 - 5.9 TB/s; before the loads of a
// row went out together 29), 12288 x 768 8.0 us (3.5 TB/s: 8-byte loads and 4-byte stores a lane, where a checkpoint has 16 and 8); LayerNorm 12288 x 768 forward 13.4 us (5.0 TB/s),
// backward 20.6 us (5.1); GELU 12288 x 3072 forward 32 us (5.8), backward with the activation 47 us (5.6); a checkpoint of 12288 x 768 6.3 us.  Calls in a graph: rows over 3072 columns,
// read twice, 8192 x 4096 22 us (4.6), 4096 x 8192 in fp32 43 (3.9); GELU 12288 x 3072 in fp32 61 (5.6) and 93 (5.3); a checkpoint of 12288 x 768 read back 5.6.
#include "rows8.h"

// the launcher of a row_mode
#define BY_MODE(mode, F, ...) ((mode) == 1 ? F(1, __VA_ARGS__) : (mode) == 0 ? F(0, __VA_ARGS__) : F(2, __VA_ARGS__))
static inline bool al(const void* p, long ld, int elems_per_16b) { return !((uintptr_t)p & 15) && ld % elems_per_16b == 0; }

// ------------------------------------------------------------------------------------------------ row codes
// One wave owns a row of C <= 256 NV and keeps it in registers; columns [C, Kp) of the code row are written as zeros (the product runs over whole
// 128-byte pieces).
template <typename T, int MODE, int NV>
__global__ __launch_bounds__(256) void rows8_quant_kernel(const T* __restrict__ x, long ldx, signed char* __restrict__ q, long ldq, float* __restrict__ s,
                                                          int M, int C, int Kp) {
  const int lane = threadIdx.x & 63;
  const long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= M) return;
  float v[NV][4];
  unsigned mx = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * 64 + lane) * 4;
    row_ld<MODE, 4>(x + row * ldx, c, C, v[i]);
  }
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) mx = max(mx, abs_bits(v[i][j]));
  mx = lanes_umax<64>(mx);
  const float sc = row_scale(mx), rs = 1.f / sc;
  if (lane == 0) s[row] = sc;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * 64 + lane) * 4;
    if (c < Kp) *reinterpret_cast<unsigned*>(q + row * ldq + c) = rowq4(v[i], sc, rs, mx >= 0x7f800000u);
  }
}
// rows too long for one wave's registers: a workgroup a row, read twice (the second time from the caches)
template <typename T, int MODE>
__global__ __launch_bounds__(256) void rows8_quant_long_kernel(const T* __restrict__ x, long ldx, signed char* __restrict__ q, long ldq, float* __restrict__ s,
                                                               int C, int Kp) {
  __shared__ unsigned red[4];
  const long row = blockIdx.x;
  unsigned mx = 0;
  float v[4];
  for (int c = threadIdx.x * 4; c < C; c += 1024) {
    row_ld<MODE, 4>(x + row * ldx, c, C, v);
#pragma unroll
    for (int j = 0; j < 4; ++j) mx = max(mx, abs_bits(v[j]));
  }
  mx = lanes_umax<64>(mx);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = mx;
  __syncthreads();
  mx = max(max(red[0], red[1]), max(red[2], red[3]));
  const float sc = row_scale(mx), rs = 1.f / sc;
  if (threadIdx.x == 0) s[row] = sc;
  for (int c = threadIdx.x * 4; c < Kp; c += 1024) {
    row_ld<MODE, 4>(x + row * ldx, c, C, v);
    *reinterpret_cast<unsigned*>(q + row * ldq + c) = rowq4(v, sc, rs, mx >= 0x7f800000u);
  }
}
template <typename T, int MODE>
static int rows8_quant_launch(const T* x, long ldx, signed char* q, long ldq, float* s, int M, int C, hipStream_t st) {
  const int Kp = (C + 127) / 128 * 128;
  if ((Kp > 12 * 256 ? M : M / 4 + 1L) * 256L >= (1L << 32)) return CLIMB_EUNSUPPORTED;          // (a launch holds less than 2^32 threads)
  const dim3 grid((M + 3) / 4), blk(256);
#define RQ(NV_) hipLaunchKernelGGL((rows8_quant_kernel<T, MODE, NV_>), grid, blk, 0, st, x, ldx, q, ldq, s, M, C, Kp)
  if constexpr (MODE == 2) RQ(1);
  else if (Kp <= 256) RQ(1);
  else if (Kp <= 768) RQ(3);
  else if (Kp <= 1536) RQ(6);
  else if (Kp <= 12 * 256) RQ(12);
  else hipLaunchKernelGGL((rows8_quant_long_kernel<T, MODE>), dim3(M), blk, 0, st, x, ldx, q, ldq, s, C, Kp);
#undef RQ
  LAUNCH_CHECK();
  return CLIMB_OK;
}
extern "C" int climb_rows8_quant(const void* x, long ldx, int dtype, void* q, long ldq, float* s, int M, int C, void* stream) {
  if (M < 0 || M > (1 << 30) || C <= 0 || C > (1 << 30) || ldx < C || ldq < (C + 127) / 128 * 128 || ldq % 16 || ((uintptr_t)q & 15)) return CLIMB_EINVAL;
  if (M == 0) return CLIMB_OK;
  if (!x || !q || !s) return CLIMB_EINVAL;
  hipStream_t st = (hipStream_t)stream;
  signed char* qc = (signed char*)q;
  const int mode = row_mode(al(x, ldx, 4), C, 4);
#define RQL(MODE_, T_) rows8_quant_launch<T_, MODE_>((const T_*)x, ldx, qc, ldq, s, M, C, st)
  if (dtype == CLIMB_DT_F32) return BY_MODE(mode, RQL, float);
  if (dtype == CLIMB_DT_BF16) return BY_MODE(mode, RQL, bf16_t);
#undef RQL
  return CLIMB_EINVAL;
}

// ------------------------------------------------------------------------------------------------ checkpoints, and GELU on them
// Eight lanes hold a group of 64 columns (8 each: 16-byte loads in 16 bits); a thread's unit is (row, group).
//   OP 0  codes <- x                    OP 1  codes <- x, y = gelu(x)
//   OP 2  y <- codes                    OP 3  y = x gelu'(codes), y2 = gelu(codes) if y2
template <typename T, int MODE, int OP>
__global__ __launch_bounds__(256) void act8_kernel(const T* __restrict__ x, long ldx, T* __restrict__ y, long ldy, T* __restrict__ y2, long ldy2,
                                                   signed char* __restrict__ q, long ldq, unsigned char* __restrict__ e, long lde, unsigned units, int C, unsigned G) {
  constexpr int DEG = GeluDeg<T>::v;
  const unsigned u = blockIdx.x * 32u + (threadIdx.x >> 3);
  const unsigned uu = u < units ? u : units - 1;      // (every lane takes part in the group maxima)
  const long row = uu / G;
  const unsigned g = uu - (unsigned)row * G;
  const int c = (int)(g * ACT8_GROUP + (threadIdx.x & 7) * 8), left = u < units ? C - c : 0;
  float v[8], o[8];
  if constexpr (OP == 0 || OP == 1) {
    row_ld<MODE, 8>(x + row * ldx, c, C, v);
    unsigned mx = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) mx = max(mx, abs_bits(v[i]));
    const unsigned ex = act8_exp(lanes_umax<8>(mx));
    if (left > 0)      // (a piece of 8 that starts inside the row lies inside ldq, a multiple of 16)
      *reinterpret_cast<uint2*>(q + row * ldq + c) = make_uint2(act8_pack4(v[0], v[1], v[2], v[3], ex), act8_pack4(v[4], v[5], v[6], v[7], ex));
    if ((threadIdx.x & 7) == 0 && u < units) e[row * lde + g] = (unsigned char)ex;
    if constexpr (OP == 1) {
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = gelu_phi<T>(v[i]);
      row_st<MODE, 8>(y + row * ldy + c, left, o);
    }
  } else {
    if (left <= 0) return;          // (so that every load below is unconditional)
    const uint2 w = *reinterpret_cast<const uint2*>(q + row * ldq + c);
    const unsigned ex = e[row * lde + g];
    if constexpr (OP == 3) row_ld<MODE, 8>(x + row * ldx, c, C, v);
    const float step = act8_step(ex);
    const float4 a = act8_values4<T>(w.x, ex, step), b = act8_values4<T>(w.y, ex, step);
    const float d[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    if constexpr (OP == 2) {
      row_st<MODE, 8>(y + row * ldy + c, left, d);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float dg;
        o[i] = gelu_phi_pair<DEG>(d[i], dg);
        v[i] *= dg;
      }
      row_st<MODE, 8>(y + row * ldy + c, left, v);
      if (y2) row_st<MODE, 8>(y2 + row * ldy2 + c, left, o);
    }
  }
}
static bool ck_ok(const void* q, long ldq, const void* e, long lde, int M, int C) {
  return M >= 0 && M <= (1 << 30) && C > 0 && C <= (1 << 30) && ldq >= C && ldq % 16 == 0 && !((uintptr_t)q & 15) && lde >= (C + ACT8_GROUP - 1) / ACT8_GROUP && (M == 0 || (q && e));
}
template <int OP>
static int act8_launch(const void* x, long ldx, int dtype, void* y, long ldy, void* y2, long ldy2, void* q, long ldq, void* e, long lde, int M, int C, void* stream) {
  if (dtype != CLIMB_DT_F32 && dtype != CLIMB_DT_BF16) return CLIMB_EINVAL;
  if (!ck_ok(q, ldq, e, lde, M, C) || (OP != 2 && ldx < C) || (OP != 0 && ldy < C) || (y2 && ldy2 < C)) return CLIMB_EINVAL;
  if (M == 0) return CLIMB_OK;
  if ((OP != 2 && !x) || (OP != 0 && !y)) return CLIMB_EINVAL;
  const unsigned G = (C + ACT8_GROUP - 1) / ACT8_GROUP;
  const long units = (long)M * G;
  if (units * 8 >= (1L << 32)) return CLIMB_EUNSUPPORTED;      // a launch holds less than 2^32 threads (34 G elements)
  const int pe = dtype == CLIMB_DT_F32 ? 4 : 8;
  const bool aligned = (OP == 2 || al(x, ldx, pe)) && (OP == 0 || al(y, ldy, pe)) && (!y2 || al(y2, ldy2, pe));
  const dim3 grid((unsigned)((units + 31) / 32)), blk(256);
  hipStream_t st = (hipStream_t)stream;
  const int mode = row_mode(aligned, C, 8);
#define AL_(MODE_, T_)                                                                                                                                              \
  hipLaunchKernelGGL((act8_kernel<T_, MODE_, OP>), grid, blk, 0, st, (const T_*)x, ldx, (T_*)y, ldy, (T_*)y2, ldy2, (signed char*)q, ldq, (unsigned char*)e, lde, \
                     (unsigned)units, C, G)
  if (dtype == CLIMB_DT_F32) { if (mode == 1) AL_(1, float); else if (mode == 0) AL_(0, float); else AL_(2, float); }
  else { if (mode == 1) AL_(1, bf16_t); else if (mode == 0) AL_(0, bf16_t); else AL_(2, bf16_t); }
#undef AL_
  LAUNCH_CHECK();
  return CLIMB_OK;
}
extern "C" int climb_act8_group(void) { return ACT8_GROUP; }
extern "C" int climb_act8_save(const void* x, long ldx, int dtype, void* q, long ldq, void* e, long lde, int M, int C, void* stream) {
  return act8_launch<0>(x, ldx, dtype, nullptr, 0, nullptr, 0, q, ldq, e, lde, M, C, stream);
}
extern "C" int climb_act8_load(const void* q, long ldq, const void* e, long lde, void* y, long ldy, int dtype, int M, int C, void* stream) {
  return act8_launch<2>(nullptr, 0, dtype, y, ldy, nullptr, 0, (void*)q, ldq, (void*)e, lde, M, C, stream);
}
extern "C" int climb_act8_gelu_fwd(const void* u, long ldu, int dtype, void* a, long lda, void* q, long ldq, void* e, long lde, int M, int C, void* stream) {
  return act8_launch<1>(u, ldu, dtype, a, lda, nullptr, 0, q, ldq, e, lde, M, C, stream);
}
extern "C" int climb_act8_gelu_bwd(const void* da, long ldda, int dtype, const void* q, long ldq, const void* e, long lde, void* du, long lddu, void* a, long lda, int M,
                                   int C, void* stream) {
  return act8_launch<3>(da, ldda, dtype, du, lddu, a, lda, (void*)q, ldq, (void*)e, lde, M, C, stream);
}

// ------------------------------------------------------------------------------------------------ LayerNorm
// One wave owns a row (4 columns a lane, 256 a step); 16 lanes hold a checkpoint group.
template <typename TO, int MODE, int NV>
__global__ __launch_bounds__(256) void act8_ln_fwd_kernel(const float* __restrict__ x, long ldx, const float* __restrict__ gamma, const float* __restrict__ beta,
                                                          float eps, TO* __restrict__ y, long ldy, float* __restrict__ mean_out, float* __restrict__ rstd_out,
                                                          signed char* __restrict__ q, long ldq, unsigned char* __restrict__ e, long lde, int M, int C) {
  const int lane = threadIdx.x & 63;
  const long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= M) return;
  float v[NV][4];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * 64 + lane) * 4;
    row_ld<MODE, 4>(x + row * ldx, c, C, v[i]);
  }
  float g[NV][4], b[NV][4];          // (fetched under the row's statistics)
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    row_ld<MODE, 4>(gamma, (i * 64 + lane) * 4, C, g[i]);
    row_ld<MODE, 4>(beta, (i * 64 + lane) * 4, C, b[i]);
  }
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) s += (v[i][0] + v[i][1]) + (v[i][2] + v[i][3]);
  const float mean = lanes_sum(s) / (float)C;
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int left = C - (i * 64 + lane) * 4;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float d = v[i][j] - mean;
      if (j < left) ss += d * d;
    }
  }
  const float rstd = rsqrtf(lanes_sum(ss) / (float)C + eps);
  if (lane == 0) {
    mean_out[row] = mean;
    rstd_out[row] = rstd;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) asm volatile("" : "+v"(g[i][j]), "+v"(b[i][j]));          // (hipcc would move the loads to their use)
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * 64 + lane) * 4, left = C - c;
    unsigned mx = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) mx = max(mx, abs_bits(v[i][j]));
    const unsigned ex = act8_exp(lanes_umax<16>(mx));
    if (left > 0) {
      *reinterpret_cast<unsigned*>(q + row * ldq + c) = act8_pack4(v[i][0], v[i][1], v[i][2], v[i][3], ex);
      if ((lane & 15) == 0) e[row * lde + i * 4 + (lane >> 4)] = (unsigned char)ex;
      float o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = fmaf((v[i][j] - mean) * rstd, g[i][j], b[i][j]);
      row_st<MODE, 4>(y + row * ldy + c, left, o);
    }
  }
}
template <typename TO, int MODE>
static int act8_ln_fwd_launch(const float* x, long ldx, const float* gamma, const float* beta, float eps, TO* y, long ldy, float* mean, float* rstd, signed char* q, long ldq,
                              unsigned char* e, long lde, int M, int C, hipStream_t st) {
  const dim3 grid((M + 3) / 4), blk(256);
#define LF(NV_) hipLaunchKernelGGL((act8_ln_fwd_kernel<TO, MODE, NV_>), grid, blk, 0, st, x, ldx, gamma, beta, eps, y, ldy, mean, rstd, q, ldq, e, lde, M, C)
  if constexpr (MODE == 2) LF(1);
  else if (C <= 256) LF(1);
  else if (C <= 768) LF(3);
  else LF(6);
#undef LF
  LAUNCH_CHECK();
  return CLIMB_OK;
}
extern "C" int climb_act8_layernorm_fwd(const float* x, long ldx, const float* gamma, const float* beta, float eps, void* y, long ldy, int y_dtype, float* mean, float* rstd,
                                        void* q, long ldq, void* e, long lde, int M, int C, void* stream) {
  if ((y_dtype != CLIMB_DT_F32 && y_dtype != CLIMB_DT_BF16) || !ck_ok(q, ldq, e, lde, M, C) || ldx < C || ldy < C) return CLIMB_EINVAL;
  if (C > 1536 || M > (1 << 25)) return CLIMB_EUNSUPPORTED;          // (registers of a wave; threads of a launch)
  if (M == 0) return CLIMB_OK;
  if (!x || !gamma || !beta || !y || !mean || !rstd) return CLIMB_EINVAL;
  // 4 elements a lane: 16-byte pieces of fp32, 8-byte pieces of the 16-bit type
  const int mode = row_mode(al(x, ldx, 4) && al(y, ldy, 4) && al(gamma, 0, 4) && al(beta, 0, 4), C, 4);
  hipStream_t st = (hipStream_t)stream;
  signed char* qc = (signed char*)q;
  unsigned char* ec = (unsigned char*)e;
#define LFL(MODE_, TO_) act8_ln_fwd_launch<TO_, MODE_>(x, ldx, gamma, beta, eps, (TO_*)y, ldy, mean, rstd, qc, ldq, ec, lde, M, C, st)
  return y_dtype == CLIMB_DT_F32 ? BY_MODE(mode, LFL, float) : BY_MODE(mode, LFL, bf16_t);
#undef LFL
}

// dx = dres + rstd (g - mean_c(g) - xh mean_c(g xh)),  g = dy gamma,  xh = (codes - mean) rstd;  partial column sums {dgamma, dbeta, colsum(dx)} of the
// workgroup's rows in part[workgroup][3][C], summed in a fixed order by the column reduction that follows.
#define A8LN_WAVES 8
// rows a wave: three from 8192 rows on (342 workgroups on 256 CUs there, 512 at 12288), else one -- fewer partial rows against more waves on a short launch.  768 columns in 16
// bits with the reduction, calls in a graph: 8191 rows 26.5 us with one, 8192 rows 20.2 with three
static inline int a8ln_rpw(int M) { return M >= 8192 ? 3 : 1; }
template <typename T> struct A8LnArgs {
  const T* dy; long lddy;
  const signed char* q; long ldq;
  const unsigned char* e; long lde;
  const float *mean, *rstd, *gamma, *dres; long ldr;
  float* dx; long ldo;
  T* dcast; long ldc;
};
template <int NV> struct A8LnRow { float d[NV][4], r[NV][4], mu, rs; unsigned w[NV], ex[NV]; };
template <int MODE, bool RES, typename T, int NV>
__device__ __forceinline__ void a8ln_load(A8LnRow<NV>& R, const A8LnArgs<T>& p, long row, int C) {
  const int lane = threadIdx.x & 63;
  R.mu = p.mean[row];
  R.rs = p.rstd[row];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * 64 + lane) * 4, left = C - c;
    row_ld<MODE, 4>(p.dy + row * p.lddy, c, C, R.d[i]);
    R.w[i] = *reinterpret_cast<const unsigned*>(p.q + row * p.ldq + (left > 0 ? c : 0));          // (unconditional, as row_ld)
    R.ex[i] = p.e[row * p.lde + (left > 0 ? i * 4 + (lane >> 4) : 0)];
    if constexpr (RES) row_ld<MODE, 4>(p.dres + row * p.ldr, c, C, R.r[i]);
    else
#pragma unroll
      for (int j = 0; j < 4; ++j) R.r[i][j] = 0.f;
  }
}
// dx of a row; each(i, j, dy, xh, dx) for what the caller sums.  KEEP: gm is gamma, kept in registers; longer rows (24 columns a lane) have none left and read it
// twice a row, from L1
template <int MODE, bool KEEP, typename T, int NV, typename F>
__device__ __forceinline__ void a8ln_finish(const A8LnRow<NV>& R, const A8LnArgs<T>& p, const float* __restrict__ gamma, long row, int C, float (&gm)[KEEP ? NV : 1][4],
                                            F each) {
  const int lane = threadIdx.x & 63;
  float s1 = 0.f, s2 = 0.f, xh[NV][4];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const bool in = (i * 64 + lane) * 4 < C;
    const float4 xv = act8_unpack4(in ? R.w[i] : 0u, in ? act8_step(R.ex[i]) : 0.f);
    const float xx[4] = {xv.x, xv.y, xv.z, xv.w};
    if constexpr (!KEEP) row_ld<MODE, 4>(gamma, (i * 64 + lane) * 4, C, gm[0]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {          // (columns past C have d = gamma = 0: no contribution)
      xh[i][j] = (xx[j] - R.mu) * R.rs;
      s1 = fmaf(R.d[i][j], gm[KEEP ? i : 0][j], s1);          // (every fma written out: the kernels that share this give the same bits)
      s2 = fmaf(R.d[i][j] * gm[KEEP ? i : 0][j], xh[i][j], s2);
    }
  }
  const float m1 = lanes_sum(s1) / (float)C, m2 = lanes_sum(s2) / (float)C;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * 64 + lane) * 4, left = C - c;
    float o[4];
    if constexpr (!KEEP) row_ld<MODE, 4>(gamma, c, C, gm[0]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      o[j] = fmaf(R.rs, fmaf(-m2, xh[i][j], fmaf(R.d[i][j], gm[KEEP ? i : 0][j], -m1)), R.r[i][j]);
      each(i, j, R.d[i][j], xh[i][j], o[j]);
    }
    row_st<MODE, 4>(p.dx + row * p.ldo + c, left, o);
    if (p.dcast) row_st<MODE, 4>(p.dcast + row * p.ldc + c, left, o);
  }
}
template <typename T, int MODE, int NV, bool RES>
__global__ __launch_bounds__(64 * A8LN_WAVES) void act8_ln_bwd_kernel(A8LnArgs<T> p, float* __restrict__ part, int M, int C, int rpw) {
  __shared__ __attribute__((aligned(16))) float red[A8LN_WAVES][NV * 256];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  constexpr bool KEEP = NV <= 3;
  float ag[NV][4], ab[NV][4], as[NV][4], gm[KEEP ? NV : 1][4];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if constexpr (KEEP) row_ld<MODE, 4>(p.gamma, (i * 64 + lane) * 4, C, gm[i]);
#pragma unroll
    for (int j = 0; j < 4; ++j) ag[i][j] = ab[i][j] = as[i][j] = 0.f;
  }
  using Row = A8LnRow<NV>;
  auto load = [&](Row& R, long row) { a8ln_load<MODE, RES>(R, p, row, C); };
  auto finish = [&](const Row& R, long row) {
    a8ln_finish<MODE, KEEP>(R, p, p.gamma, row, C, gm, [&](int i, int j, float d, float xh, float o) {
      ag[i][j] += d * xh;
      ab[i][j] += d;
      as[i][j] += o;
    });
  };
  // a row's loads go out before the row in front of it is finished (dx may be dres: rows are disjoint, and a wave reads its row before it writes it); rows of
  // more than 768 columns would need more registers than two waves a SIMD have
  const long row0 = (long)blockIdx.x * rpw * A8LN_WAVES + wid;
  if constexpr (!KEEP) {
    for (int rr = 0; rr < rpw && row0 + rr * A8LN_WAVES < M; ++rr) {
      Row A;
      load(A, row0 + rr * A8LN_WAVES);
      finish(A, row0 + rr * A8LN_WAVES);
    }
  } else if (row0 < M) {
    Row A;
    load(A, row0);
    int rr = 1;
    for (; rr < rpw && row0 + rr * A8LN_WAVES < M; ++rr) {
      Row B;
      load(B, row0 + rr * A8LN_WAVES);
      finish(A, row0 + (rr - 1) * A8LN_WAVES);
      A = B;
    }
    finish(A, row0 + (rr - 1) * A8LN_WAVES);
  }
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    if (k) __syncthreads();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * 64 + lane) * 4;
      const float* a = k == 0 ? ag[i] : (k == 1 ? ab[i] : as[i]);
      *reinterpret_cast<float4*>(&red[wid][c]) = make_float4(a[0], a[1], a[2], a[3]);
    }
    __syncthreads();
    for (int c = threadIdx.x; c < C; c += 64 * A8LN_WAVES) {
      float t = red[0][c];
#pragma unroll
      for (int w = 1; w < A8LN_WAVES; ++w) t += red[w][c];
      part[((long)blockIdx.x * 3 + k) * C + c] = t;
    }
  }
}
// Few rows, and no column sums of dx wanted: everything in one launch.  dgamma = sum dy xh and dbeta = sum dy need the saved statistics only, not the rows' means
// that dx is waiting for, so the first ceil(C / 64) workgroups sum a group's columns over all rows (32 rows side by side, added in a fixed order), the others make
// dx, a row a wave; dy and the codes are read twice, from L2.
#define A8LN_COLS 64
template <typename T, int MODE, int NV, bool RES>
__global__ __launch_bounds__(64 * A8LN_WAVES) void act8_ln_bwd_few_kernel(A8LnArgs<T> p, float* __restrict__ dgamma, float* __restrict__ dbeta, float beta, int M, int C, int ncol) {
  if ((int)blockIdx.x >= ncol) {
    constexpr bool KEEP = NV <= 3;
    const long row = (long)(blockIdx.x - ncol) * A8LN_WAVES + (threadIdx.x >> 6);
    if (row >= M) return;
    float gm[KEEP ? NV : 1][4];
    if constexpr (KEEP)
#pragma unroll
      for (int i = 0; i < NV; ++i) row_ld<MODE, 4>(p.gamma, (i * 64 + (threadIdx.x & 63)) * 4, C, gm[i]);
    A8LnRow<NV> R;
    a8ln_load<MODE, RES>(R, p, row, C);
    a8ln_finish<MODE, KEEP>(R, p, p.gamma, row, C, gm, [](int, int, float, float, float) {});
    return;
  }
  constexpr int SLOTS = 4 * A8LN_WAVES, U = 6;
  __shared__ __attribute__((aligned(16))) float red[2][SLOTS][A8LN_COLS];
  const int sub = threadIdx.x & 15, slot = threadIdx.x >> 4, c = blockIdx.x * A8LN_COLS + sub * 4;
  float ag[4] = {0.f, 0.f, 0.f, 0.f}, ab[4] = {0.f, 0.f, 0.f, 0.f};
  for (int m0 = slot; m0 < M; m0 += SLOTS * U) {
    float d[U][4], mu[U], rs[U];
    unsigned w[U], ex[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long m = min(m0 + u * SLOTS, M - 1);
      row_ld<MODE, 4>(p.dy + m * p.lddy, c, C, d[u]);
      w[u] = *reinterpret_cast<const unsigned*>(p.q + m * p.ldq + (c < C ? c : 0));
      ex[u] = p.e[m * p.lde + blockIdx.x];
      mu[u] = p.mean[m];
      rs[u] = p.rstd[m];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (m0 + u * SLOTS >= M) break;
      const float4 xv = act8_unpack4(w[u], act8_step(ex[u]));
      const float xx[4] = {xv.x, xv.y, xv.z, xv.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        ag[j] += d[u][j] * ((xx[j] - mu[u]) * rs[u]);
        ab[j] += d[u][j];
      }
    }
  }
  *reinterpret_cast<float4*>(&red[0][slot][sub * 4]) = make_float4(ag[0], ag[1], ag[2], ag[3]);
  *reinterpret_cast<float4*>(&red[1][slot][sub * 4]) = make_float4(ab[0], ab[1], ab[2], ab[3]);
  __syncthreads();
  const int k = threadIdx.x >> 6, col = threadIdx.x & 63, n = blockIdx.x * A8LN_COLS + col;
  float* out = k == 0 ? dgamma : dbeta;
  if (k > 1 || !out || n >= C) return;
  float t = red[k][0][col];
#pragma unroll
  for (int i = 1; i < SLOTS; ++i) t += red[k][i][col];
  out[n] = beta != 0.f ? fmaf(beta, out[n], t) : t;
}
// Where that one launch is taken.  us a call of twenty in a graph (a trace, which counts each launch from its start to its end, has 1.4 to 2.4 more), one / two launches, 768
// columns in 16 bits: 1 row 2.6 / 5.7, 185 3.7 / 7.1, 500 6.0 / 8.4, 768 8.1 / 8.1, 1024 10 / 7.4; 1536 in fp32: 333 4.7 / 10.4, 768 8.3 / 10.9, 1024 15 / 10; 96 columns: 185
// 3.5 / 5.6, 768 7.8 / 6.3 -- and the second launch costs the host 3 us.
static inline bool a8ln_few(int M, bool colsum) { return !colsum && M <= 768; }
template <typename T, int MODE>
static int act8_ln_bwd_launch(const A8LnArgs<T>& p, float* part, float* dgamma, float* dbeta, float beta, bool few, int M, int C, hipStream_t st) {
  const int rpw = few ? 1 : a8ln_rpw(M), ncol = few && (dgamma || dbeta) ? (C + A8LN_COLS - 1) / A8LN_COLS : 0;
  const dim3 grid((M + A8LN_WAVES * rpw - 1) / (A8LN_WAVES * rpw) + ncol), blk(64 * A8LN_WAVES);
#define LBK(NV_, RES_)                                                                                                                        \
  do {                                                                                                                                        \
    if (few) hipLaunchKernelGGL((act8_ln_bwd_few_kernel<T, MODE, NV_, RES_>), grid, blk, 0, st, p, dgamma, dbeta, beta, M, C, ncol);           \
    else hipLaunchKernelGGL((act8_ln_bwd_kernel<T, MODE, NV_, RES_>), grid, blk, 0, st, p, part, M, C, rpw);                                   \
  } while (0)
#define LB(NV_) do { if (p.dres) LBK(NV_, true); else LBK(NV_, false); } while (0)
  if constexpr (MODE == 2) LB(1);
  else if (C <= 256) LB(1);
  else if (C <= 768) LB(3);
  else LB(6);
#undef LB
#undef LBK
  LAUNCH_CHECK();
  return CLIMB_OK;
}
extern "C" int climb_colreduce3(const float* part, long stride, int nblk, float* out0, float* out1, float* out2, int ncols, float beta, void* stream);      // rowwise.hip
extern "C" int climb_act8_layernorm_bwd_blocks(int M) { return M <= 0 ? 0 : (int)(((long)M + A8LN_WAVES * a8ln_rpw(M) - 1) / (A8LN_WAVES * a8ln_rpw(M))); }
extern "C" long climb_act8_layernorm_bwd_workspace(int M, int C, int colsum) {
  if (M < 0 || C <= 0) return CLIMB_EINVAL;
  return a8ln_few(M, colsum != 0) ? 0 : (long)climb_act8_layernorm_bwd_blocks(M) * 3 * C * 4;
}
extern "C" int climb_act8_layernorm_bwd(const void* dy, long lddy, int dtype, const void* q, long ldq, const void* e, long lde, const float* mean, const float* rstd,
                                        const float* gamma, const float* dres_in, long ldr, float* dx, long ldo, void* dcast, long ldc, float* part, float* dgamma, float* dbeta,
                                        float* colsum, float beta, int M, int C, void* stream) {
  if ((dtype != CLIMB_DT_F32 && dtype != CLIMB_DT_BF16) || !ck_ok(q, ldq, e, lde, M, C) || lddy < C || ldo < C || (dres_in && ldr < C) || (dcast && ldc < C))
    return CLIMB_EINVAL;
  if (C > 1536 || M > (1 << 25)) return CLIMB_EUNSUPPORTED;
  if (M == 0) return CLIMB_OK;
  const bool few = a8ln_few(M, colsum != nullptr);
  if (!dy || !mean || !rstd || !gamma || !dx || (!few && !part)) return CLIMB_EINVAL;
  const int mode = row_mode(al(dy, lddy, 4) && al(dx, ldo, 4) && al(gamma, 0, 4) && (!dres_in || al(dres_in, ldr, 4)) && (!dcast || al(dcast, ldc, 4)), C, 4);
  hipStream_t st = (hipStream_t)stream;
#define LBL(MODE_, T_)                                                                                                                                                     \
  act8_ln_bwd_launch<T_, MODE_>(A8LnArgs<T_>{(const T_*)dy, lddy, (const signed char*)q, ldq, (const unsigned char*)e, lde, mean, rstd, gamma, dres_in, ldr, dx, ldo, (T_*)dcast, ldc}, \
                                part, dgamma, dbeta, beta, few, M, C, st)
  const int rc = dtype == CLIMB_DT_F32 ? BY_MODE(mode, LBL, float) : BY_MODE(mode, LBL, bf16_t);
#undef LBL
  return rc != CLIMB_OK || few ? rc : climb_colreduce3(part, 3L * C, climb_act8_layernorm_bwd_blocks(M), dgamma, dbeta, colsum, C, beta, stream);
}
