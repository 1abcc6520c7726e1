// int8 product with a scale for each token and each output channel:
//   C[m,n] = epi( (sum_k qa[m,k] qb[n,k]) sa[m] sb[n] + bias[n] ),   the sum in int32 (exact: K <= 2^17), everything after it in fp32, rounded once.
// v_mfma_i32_32x32x32_i8 (twice the 16-bit MFMA rate).  The weights are the MFMA's A operand and the tokens its B operand, so a lane of the accumulator
// owns ONE token and groups of 4 consecutive channels.
#include "rows8.h"
#include "gemm_bf16_nt.h"

typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(16))) int i32x16;

#define I8_BK 128          // bytes of K in a stage: one 128-byte line of every operand row

// LDS image of an operand tile: [rows][128 B], 16-byte chunk c of row r at position c ^ (r & 7): the fragment reads (16 bytes a lane, 32 rows x 2
// neighbouring chunks) then touch every bank group once.  global_load_lds writes LDS linearly, so the swizzle is applied to the SOURCE address.
template <int ROWS, int NT>
struct I8Src {
  static constexpr int CNT = ROWS * 8 / NT;
  unsigned off[CNT];          // per lane: byte offsets from the tile's first row
  __device__ __forceinline__ void init(int row0, int R, long ld) {
#pragma unroll
    for (int i = 0; i < CNT; ++i) {
      const int slot = i * NT + threadIdx.x, row = slot >> 3, c = (slot & 7) ^ (row & 7);
      off[i] = (unsigned)(min(row, R - 1 - row0) * (unsigned)ld) + c * 16;          // rows past the end repeat the last one: their results are not stored
    }
  }
  __device__ __forceinline__ void issue(const signed char* __restrict__ base, unsigned char* __restrict__ S) const {
    const int wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < CNT; ++i)
      __builtin_amdgcn_global_load_lds((gbl_void_t*)(base + off[i]), (lds_void_t*)(S + (i * NT + wave * 64) * 16), 16, 0, 0);
  }
};

template <typename TO>
__device__ __forceinline__ void i8_store4(TO* __restrict__ p, const float (&v)[4], int left, bool vec) {
  if (vec && left >= 4) st4(p, make_float4(v[0], v[1], v[2], v[3]));
  else
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) Act<TO>::st(p + i, v[i]);
}
__device__ __forceinline__ void i8_load4(const float* __restrict__ p, float (&v)[4], int left, bool vec) {
  if (vec && left >= 4) {
    const float4 r = ld4(p);
    v[0] = r.x; v[1] = r.y; v[2] = r.z; v[3] = r.w;
  } else
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < left ? p[i] : 0.f;
}

// WN x WM waves of (32 NI channels) x (32 MJ tokens); S stages in LDS.
template <typename TO, int EPI, int NI, int MJ, int WN, int WM, int S>
__global__ __launch_bounds__(64 * WN * WM) void gemm_i8_kernel(const signed char* __restrict__ A, long lda, const float* __restrict__ sa,
                                                               const signed char* __restrict__ B, long ldb, const float* __restrict__ sb, TO* __restrict__ C,
                                                               long ldc, int M, int N, int nk, const float* __restrict__ bias, const float* __restrict__ aux,
                                                               long ldaux, int vec) {
  constexpr int NT = 64 * WN * WM, BN = 32 * NI * WN, BM = 32 * MJ * WM, STAGE = (BN + BM) * I8_BK, LPT = I8Src<BN, NT>::CNT + I8Src<BM, NT>::CNT;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];          // S stages, then BM token scales
  float* sas = reinterpret_cast<float*>(smem + S * STAGE);
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, wn = wid % WN, wm = wid / WN, half = lane >> 5, l31 = lane & 31;
  int tm, tn;
  const int nbm = (M + BM - 1) / BM, nbn = (N + BN - 1) / BN;
  nt_tile<8>(nbm, nbn, tm, tn);
  const int m0 = tm * BM, n0 = tn * BN;
  I8Src<BN, NT> srcB;
  I8Src<BM, NT> srcA;
  srcB.init(n0, N, ldb);
  srcA.init(m0, M, lda);
  const signed char* Bp = B + (long)n0 * ldb;
  const signed char* Ap = A + (long)m0 * lda;
  for (int i = threadIdx.x; i < BM; i += NT) sas[i] = sa[min(m0 + i, M - 1)];
#pragma unroll
  for (int s = 0; s < S - 1; ++s)
    if (s < nk) {
      srcB.issue(Bp + s * I8_BK, smem + s * STAGE);
      srcA.issue(Ap + s * I8_BK, smem + s * STAGE + BN * I8_BK);
    }
  i32x16 acc[NI][MJ];
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < MJ; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;
  for (int kt = 0; kt < nk; ++kt) {
    if (S > 2 && kt + S - 2 < nk) wait_vmcnt<(S - 2) * LPT>();
    else wait_vmcnt<0>();
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();          // tile kt is in LDS for every wave, and every wave is done with the buffer the next loads go to
    __builtin_amdgcn_sched_barrier(0);
    if (kt + S - 1 < nk) {
      unsigned char* nb = smem + ((kt + S - 1) % S) * STAGE;
      srcB.issue(Bp + (long)(kt + S - 1) * I8_BK, nb);
      srcA.issue(Ap + (long)(kt + S - 1) * I8_BK, nb + BN * I8_BK);
    }
    const unsigned char* buf = smem + (kt % S) * STAGE + l31 * I8_BK;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      const unsigned co = (((ks * 2 + half) ^ (l31 & 7)) << 4);
      i32x4 fb[NI], fa[MJ];
#pragma unroll
      for (int i = 0; i < NI; ++i) fb[i] = *reinterpret_cast<const i32x4*>(buf + (wn * NI + i) * 32 * I8_BK + co);
#pragma unroll
      for (int j = 0; j < MJ; ++j) fa[j] = *reinterpret_cast<const i32x4*>(buf + (BN + (wm * MJ + j) * 32) * I8_BK + co);
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < MJ; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fb[i], fa[j], acc[i][j], 0, 0, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  __syncthreads();          // the epilogue turns its blocks through the stage buffers
  // Epilogue: a wave turns 32 tokens x 32 NI channels at a time through a private LDS region, so that bias, residual and C are read and written as whole
  // lines (a lane of the accumulator owns one token: direct stores would touch 32 rows with 8 - 16 bytes each).
  constexpr int CPR = NI * 8, PITCH = NI * 128, PERIOD = CPR % 64 == 0 ? CPR / 64 : (64 % CPR == 0 ? 1 : 3);
  static_assert(NI == 1 || NI == 2 || NI == 3 || NI == 4, "channel chunk of a lane: period 1 (8, 16, 32 chunks a row) or 3 (24)");
  unsigned char* stage = smem + wid * (32 * PITCH);
  const int nw = n0 + wn * NI * 32, mw = m0 + wm * MJ * 32;
  float sbv[PERIOD][4], bv[PERIOD][4];
#pragma unroll
  for (int p = 0; p < PERIOD; ++p) {
    const int n = nw + ((p * 64 + lane) % CPR) * 4;
    i8_load4(sb + n, sbv[p], N - n, vec);
    if (bias) i8_load4(bias + n, bv[p], N - n, vec);
    else
#pragma unroll
      for (int i = 0; i < 4; ++i) bv[p][i] = 0.f;
  }
#pragma unroll
  for (int j = 0; j < MJ; ++j) {
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<i32x4*>(stage + l31 * PITCH + ((i * 8 + ((2 * g + half) ^ (l31 & 7))) << 4)) =
            (i32x4){acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
    float rv[EPI == EPI_RESID ? NI * 4 : 1][4];
    if constexpr (EPI == EPI_RESID) {
#pragma unroll
      for (int p = 0; p < NI * 4; ++p) {
        const int q = p * 64 + lane, m = mw + j * 32 + q / CPR, n = nw + (q % CPR) * 4;
        i8_load4(aux + (long)m * ldaux + n, rv[p], m < M ? N - n : 0, vec);
      }
    }
#pragma unroll
    for (int p = 0; p < NI * 4; ++p) {
      const int q = p * 64 + lane, r = q / CPR, c = q % CPR, m = mw + j * 32 + r, n = nw + c * 4;
      const i32x4 a = *reinterpret_cast<const i32x4*>(stage + r * PITCH + (((c & ~7) | ((c ^ r) & 7)) << 4));
      if (m >= M || n >= N) continue;
      const float s = sas[m - m0];
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = fmaf((float)a[i], s * sbv[p % PERIOD][i], bv[p % PERIOD][i]);
        if (EPI == EPI_GELU) v[i] = gelu_phi<GeluDeg<TO>::v>(v[i]);
        if (EPI == EPI_RESID) v[i] += rv[EPI == EPI_RESID ? p : 0][i];
      }
      i8_store4(C + (long)m * ldc + n, v, N - n, vec);
    }
  }
}

template <typename TO, int EPI, int NI, int MJ, int WN, int WM, int S>
static int i8_launch(const signed char* A, long lda, const float* sa, const signed char* B, long ldb, const float* sb, TO* C, long ldc, int M, int N, int Kp,
                     const float* bias, const float* aux, long ldaux, int vec, hipStream_t st) {
  constexpr int BN = 32 * NI * WN, BM = 32 * MJ * WM, LDS = S * (BN + BM) * I8_BK + BM * 4;
  static_assert(LDS <= 160 * 1024 && WN * WM * NI * 4096 <= S * (BN + BM) * I8_BK, "LDS");
  const long tiles = (long)((M + BM - 1) / BM) * ((N + BN - 1) / BN);
  if (tiles >= (1L << 31)) return CLIMB_EUNSUPPORTED;
  auto k = gemm_i8_kernel<TO, EPI, NI, MJ, WN, WM, S>;
  if (LDS > 64 * 1024) {
    hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
    if (e != hipSuccess) return (int)e;
  }
  hipLaunchKernelGGL(k, dim3((unsigned)tiles), dim3(64 * WN * WM), LDS, st, A, lda, sa, B, ldb, sb, C, ldc, M, N, Kp / I8_BK, bias, aux, ldaux, vec);
  LAUNCH_CHECK();
  return CLIMB_OK;
}
template <typename TO, int EPI>
static int i8_pick(const signed char* A, long lda, const float* sa, const signed char* B, long ldb, const float* sb, TO* C, long ldc, int M, int N, int Kp,
                   const float* bias, const float* aux, long ldaux, int vec, hipStream_t st) {
  auto tiles = [&](int bm, int bn) { return (long)((M + bm - 1) / bm) * ((N + bn - 1) / bn); };
#define I8_GO(NI_, MJ_, WN_, WM_, S_) return i8_launch<TO, EPI, NI_, MJ_, WN_, WM_, S_>(A, lda, sa, B, ldb, sb, C, ldc, M, N, Kp, bias, aux, ldaux, vec, st)
  if (tiles(192, 192) >= 192) I8_GO(3, 3, 2, 2, 3);
  if (tiles(128, 128) >= 192) I8_GO(2, 2, 2, 2, 3);
  I8_GO(1, 1, 2, 2, 3);
#undef I8_GO
}
template <typename TO>
static int i8_epi(const signed char* A, long lda, const float* sa, const signed char* B, long ldb, const float* sb, TO* C, long ldc, int M, int N, int Kp, const float* bias,
                  int epi, const float* aux, long ldaux, int vec, hipStream_t st) {
  switch (epi) {
    case EPI_NONE: return i8_pick<TO, EPI_NONE>(A, lda, sa, B, ldb, sb, C, ldc, M, N, Kp, bias, aux, ldaux, vec, st);
    case EPI_GELU: return i8_pick<TO, EPI_GELU>(A, lda, sa, B, ldb, sb, C, ldc, M, N, Kp, bias, aux, ldaux, vec, st);
    case EPI_RESID: return i8_pick<TO, EPI_RESID>(A, lda, sa, B, ldb, sb, C, ldc, M, N, Kp, bias, aux, ldaux, vec, st);
  }
  return CLIMB_EINVAL;
}

extern "C" int climb_gemm_i8_nt(const void* A, long lda, const float* sa, const void* B, long ldb, const float* sb, void* C, long ldc, int c_dtype, int M, int N, int K,
                                const float* bias, int epi, const float* aux, long ldaux, void* stream) {
  const int Kp = (K + I8_BK - 1) / I8_BK * I8_BK;
  if (M < 0 || N <= 0 || K <= 0 || lda < Kp || ldb < Kp || lda % 16 || ldb % 16 || ldc < N || ((uintptr_t)A & 15) || ((uintptr_t)B & 15)) return CLIMB_EINVAL;
  if (epi != EPI_NONE && epi != EPI_GELU && epi != EPI_RESID) return CLIMB_EINVAL;
  if (epi == EPI_RESID && ldaux < N) return CLIMB_EINVAL;
  if (K > (1 << 17) || lda >= (1L << 22) || ldb >= (1L << 22)) return CLIMB_EUNSUPPORTED;          // int32 sums: 127^2 K < 2^31; 32-bit offsets inside a tile
  if (M == 0) return CLIMB_OK;
  if (!A || !sa || !B || !sb || !C || (epi == EPI_RESID && !aux)) return CLIMB_EINVAL;
  // whole 16-byte (16-bit C: 8-byte) pieces of 4 channels; anything else is read and written element by element
  const int vec = ldc % 4 == 0 && !((uintptr_t)C & 15) && !((uintptr_t)sb & 15) && !((uintptr_t)bias & 15) &&
                  (epi != EPI_RESID || (ldaux % 4 == 0 && !((uintptr_t)aux & 15)));
  hipStream_t st = (hipStream_t)stream;
  const signed char *a = (const signed char*)A, *b = (const signed char*)B;
  if (c_dtype == CLIMB_DT_F32) return i8_epi<float>(a, lda, sa, b, ldb, sb, (float*)C, ldc, M, N, Kp, bias, epi, aux, ldaux, vec, st);
  if (c_dtype == CLIMB_DT_BF16) return i8_epi<bf16_t>(a, lda, sa, b, ldb, sb, (bf16_t*)C, ldc, M, N, Kp, bias, epi, aux, ldaux, vec, st);
  return CLIMB_EINVAL;
}
