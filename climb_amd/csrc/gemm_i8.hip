// int8 product with a scale for each token and each output channel:
//   C[m,n] = epi( (sum_k qa[m,k] qb[n,k]) sa[m] sb[n] + bias[n] ),   the sum in int32 (exact: K <= 2^17), everything after it in fp32, rounded once.
// v_mfma_i32_32x32x32_i8 (twice the 16-bit MFMA rate).  Measured: 12288 x 768 -> 3072 with GELU to 16 bits 53 us (1.09 PFLOP/s; the matrix unit is busy 12 us of it at
// its peak clock, the epilogue's VALU ~20 us, 85 MB leave and enter HBM in ~15), 12288 x 3072 -> 768 + fp32 residual 41 us (1.41 PFLOP/s).  What bounds it is that these
// phases of a tile overlap only across the workgroups of a CU, at the 1.9 GHz the chip sustains under MFMA load.  The weights are the MFMA's A operand and the tokens its B operand, so a lane of the accumulator
// owns ONE token and groups of 4 consecutive channels.
#include <type_traits>
#include "rows8.h"
#include "gemm_bf16_nt.h"

typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(16))) int i32x16;

#define I8_BK 128          // the code rows are whole 128-byte pieces

// LDS image of an operand tile: [rows][128 bytes], 16-byte chunk c of row r at position c ^ i8_swz(r): the 16 rows that a fragment read (16 bytes a lane, 32 rows
// of one chunk) takes in a cycle lie in 16 different 16-byte slots of the 256-byte bank line.  global_load_lds writes LDS linearly, so the swizzle is applied to the
// SOURCE address.
__device__ __forceinline__ int i8_swz(int row) { return (row >> 1) & 7; }
template <int ROWS, int NT>
struct I8Src {
  static constexpr int CPR = I8_BK / 16, CNT = ROWS * CPR / NT;
  unsigned off[CNT];          // per lane: byte offsets from the tile's first row
  __device__ __forceinline__ void init(int row0, int R, long ld) {
#pragma unroll
    for (int i = 0; i < CNT; ++i) {
      const int slot = i * NT + threadIdx.x, row = slot / CPR, c = (slot % CPR) ^ i8_swz(row);
      off[i] = (unsigned)(min(row, R - 1 - row0) * (unsigned)ld) + c * 16;          // rows past the end repeat the last one: their results are not stored
    }
  }
  __device__ __forceinline__ void issue(const signed char* __restrict__ base, unsigned char* __restrict__ S) const {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
    for (int i = 0; i < CNT; ++i)
      __builtin_amdgcn_global_load_lds((gbl_void_t*)(base + off[i]), (lds_void_t*)(S + (i * NT + wave * 64) * 16), 16, 0, 0);
  }
};

template <typename TO>
__device__ __forceinline__ void i8_store4(TO* p, const float (&v)[4], int left, bool vec) {
  if (vec && left >= 4) st4(p, make_float4(v[0], v[1], v[2], v[3]));
  else
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) Act<TO>::st(p + i, v[i]);
}
__device__ __forceinline__ void i8_load4(const float* p, float (&v)[4], int left, bool vec) {
  if (vec && left >= 4) {
    const float4 r = ld4(p);
    v[0] = r.x; v[1] = r.y; v[2] = r.z; v[3] = r.w;
  } else
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < left ? p[i] : 0.f;
}

// WN x WM waves of (32 NI channels) x (32 MJ tokens); S stages in LDS.
template <typename TO, int EPI, int NI, int MJ, int WN, int WM, int S, int OCC>
__global__ __launch_bounds__(64 * WN * WM, OCC) void gemm_i8_kernel(const signed char* __restrict__ A, long lda, const float* __restrict__ sa,
                                                               const signed char* __restrict__ B, long ldb, const float* __restrict__ sb, TO* C,
                                                               long ldc, int M, int N, int nk, const float* __restrict__ bias, const float* aux,
                                                               long ldaux, int vec) {
  constexpr int BK = I8_BK, NT = 64 * WN * WM, BN = 32 * NI * WN, BM = 32 * MJ * WM, STAGE = (BN + BM) * BK, LPT = I8Src<BN, NT>::CNT + I8Src<BM, NT>::CNT;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];          // S stages, then the tile's token scales, channel scales and biases
  float *sas = reinterpret_cast<float*>(smem + S * STAGE), *sbs = sas + BM, *bs = sbs + BN;
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wn = wid % WN, wm = wid / WN, half = lane >> 5, l31 = lane & 31;
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
  // by DMA too, and first: they have landed when the first stage has, and no wait of the epilogue begins with them
  auto row_dma = [&](const float* __restrict__ src, int i0, int last, float* dst, int n) {
    for (int c = wid * 64; c < n; c += NT)
      __builtin_amdgcn_global_load_lds((gbl_void_t*)(src + min(i0 + c + lane, last)), (lds_void_t*)(dst + c), 4, 0, 0);
  };
  row_dma(sa, m0, M - 1, sas, BM);
  row_dma(sb, n0, N - 1, sbs, BN);
  if (bias) row_dma(bias, n0, N - 1, bs, BN);
#pragma unroll
  for (int s = 0; s < S; ++s)
    if (s < nk) {
      srcB.issue(Bp + s * BK, smem + s * STAGE);
      srcA.issue(Ap + s * BK, smem + s * STAGE + BN * BK);
    }
  i32x16 acc[NI][MJ];
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < MJ; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;
  // The fragments of a 32-byte step are read while the step before multiplies, behind its FIRST MFMA: while LDS DMA is on its way hipcc waits for every LDS
  // read before it uses one (lgkmcnt(0)), so reads issued ahead of that MFMA would be waited for with an idle matrix unit.  In the last step of a stage all of
  // its fragments are in registers, so that is where the workgroup meets: behind the barrier the stage's buffer takes the loads of the stage S ahead, and
  // the first fragments of the next one are read under this step's MFMAs.
  constexpr int KS = BK / 32;
  static_assert(KS % 2 == 0, "two fragment sets, the first of a stage always in set 0");
  i32x4 fb[2][NI], fa[2][MJ];
  const unsigned char* lbase = smem + l31 * BK;
  unsigned co[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) co[ks] = ((ks * 2 + half) ^ i8_swz(l31)) << 4;
  auto frags = [&](i32x4(&b)[NI], i32x4(&a)[MJ], const unsigned char* buf, unsigned c) {
#pragma unroll
    for (int i = 0; i < NI; ++i) b[i] = *reinterpret_cast<const i32x4*>(buf + (wn * NI + i) * 32 * BK + c);
#pragma unroll
    for (int j = 0; j < MJ; ++j) a[j] = *reinterpret_cast<const i32x4*>(buf + (BN + (wm * MJ + j) * 32) * BK + c);
  };
  auto arrive = [&](int more) {          // the oldest stage on its way has landed, `more` younger ones may still be out
    if (more >= S - 1) wait_vmcnt<(S - 1) * LPT>();
    else if (S > 2 && more == 1) wait_vmcnt<LPT>();
    else wait_vmcnt<0>();
    // ... and this wave's fragment reads of the stage before are back: behind the barrier the other waves' DMA overwrites that stage, while the first MFMA of a step
    // needs two of its fragments only
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
  };
  static_assert(S == 2 || S == 3, "arrive()");
  arrive(min(nk, S) - 1);
  bool far = false;          // a token of this wave whose scale asks for the general scaled_sum (the scales have landed with the first stage)
#pragma unroll
  for (int j = 0; j < MJ; ++j) far |= sas[wm * MJ * 32 + j * 32 + l31] > ROW_SCALE_PLAIN;
  const bool plain = vec && m0 + BM <= M && n0 + BN <= N && !__any(far);
  frags(fb[0], fa[0], lbase, co[0]);
  int cur = 0;          // stage buffer
  for (int kt = 0; kt < nk; ++kt) {
    const int nxt = cur + 1 == S ? 0 : cur + 1;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      acc[0][0] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fb[ks & 1][0], fa[ks & 1][0], acc[0][0], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);          // (one MFMA is under way; nothing is out of LDS now, see above)
      if (ks + 1 < KS) frags(fb[(ks + 1) & 1], fa[(ks + 1) & 1], lbase + cur * STAGE, co[ks + 1]);
      else if (kt + 1 < nk) {
        arrive(min(nk - kt - 2, S - 2));
        if (kt + S < nk) {
          srcB.issue(Bp + (long)(kt + S) * BK, smem + cur * STAGE);
          srcA.issue(Ap + (long)(kt + S) * BK, smem + cur * STAGE + BN * BK);
        }
        frags(fb[0], fa[0], lbase + nxt * STAGE, co[0]);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < MJ; ++j)
          if (i || j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fb[ks & 1][i], fa[ks & 1][j], acc[i][j], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
    cur = nxt;
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
    const int n = wn * NI * 32 + ((p * 64 + lane) % CPR) * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sbv[p][i] = sbs[n + i];
      bv[p][i] = bias ? bs[n + i] : 0.f;
    }
  }
  // `full`: the whole tile exists and is made of whole pieces, so nothing is tested on the way (tests cut the block into pieces that hipcc does not interleave)
  auto drain = [&](auto full_) {
    constexpr bool FULL = decltype(full_)::value;
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
          i8_load4(aux + (long)m * ldaux + n, rv[p], FULL ? 4 : (m < M ? N - n : 0), FULL || vec);
        }
      }
#pragma unroll
      for (int p = 0; p < NI * 4; ++p) {
        const int q = p * 64 + lane, r = q / CPR, c = q % CPR, m = mw + j * 32 + r, n = nw + c * 4;
        const i32x4 a = *reinterpret_cast<const i32x4*>(stage + r * PITCH + (((c & ~7) | ((c ^ r) & 7)) << 4));
        if (!FULL && (m >= M || n >= N)) continue;
        const float s = sas[m - m0];
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[i] = scaled_sum<FULL>(a[i], s, sbv[p % PERIOD][i], bv[p % PERIOD][i]);
          if (EPI == EPI_GELU) v[i] = gelu_phi<TO>(v[i]);
          if (EPI == EPI_RESID) v[i] += rv[EPI == EPI_RESID ? p : 0][i];
        }
        i8_store4(C + (long)m * ldc + n, v, FULL ? 4 : N - n, FULL || vec);
      }
    }
  };
  if (plain) drain(std::true_type{});
  else drain(std::false_type{});
}

template <typename TO, int EPI, int NI, int MJ, int WN, int WM, int S, int OCC>
static int i8_launch(const signed char* A, long lda, const float* sa, const signed char* B, long ldb, const float* sb, TO* C, long ldc, int M, int N, int Kp,
                     const float* bias, const float* aux, long ldaux, int vec, hipStream_t st) {
  constexpr int BK = I8_BK, BN = 32 * NI * WN, BM = 32 * MJ * WM, LDS = S * (BN + BM) * BK + (BM + 2 * BN) * 4;
  static_assert(BM % 64 == 0 && BN % 64 == 0 && LDS * OCC <= 160 * 1024 && WN * WM * NI * 4096 <= S * (BN + BM) * BK, "LDS");
  const long tiles = (long)((M + BM - 1) / BM) * ((N + BN - 1) / BN);
  if (tiles * (64 * WN * WM) >= (1L << 32)) return CLIMB_EUNSUPPORTED;          // (a launch holds less than 2^32 threads)
  auto k = gemm_i8_kernel<TO, EPI, NI, MJ, WN, WM, S, OCC>;
  if (LDS > 64 * 1024) {
    hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
    if (e != hipSuccess) return (int)e;
  }
  hipLaunchKernelGGL(k, dim3((unsigned)tiles), dim3(64 * WN * WM), LDS, st, A, lda, sa, B, ldb, sb, C, ldc, M, N, Kp / BK, bias, aux, ldaux, vec);
  LAUNCH_CHECK();
  return CLIMB_OK;
}
template <typename TO, int EPI>
static int i8_pick(const signed char* A, long lda, const float* sa, const signed char* B, long ldb, const float* sb, TO* C, long ldc, int M, int N, int Kp,
                   const float* bias, const float* aux, long ldaux, int vec, hipStream_t st) {
  auto tiles = [&](int bm, int bn) { return (long)((M + bm - 1) / bm) * ((N + bn - 1) / bn); };
#define I8_GO(NI_, MJ_, WN_, WM_, S_, OCC_) return i8_launch<TO, EPI, NI_, MJ_, WN_, WM_, S_, OCC_>(A, lda, sa, B, ldb, sb, C, ldc, M, N, Kp, bias, aux, ldaux, vec, st)
  // 192 x 192 tiles (twelve waves of 32 x 96, one workgroup a CU) where they fill one round of the chip or K is long: 12288 x 3072 -> 768 + residual 40 us (128 x 128:
  // 49), 12288 x 768 -> 768 + residual 20.5 (23).  128 x 128, two workgroups a CU, one's epilogue beside the other's products: 12288 x 768 -> 3072 45 us (192: 51), with
  // GELU 54 (63), -> 2304 36 (39).  64 x 64, three a CU, where the larger tiles leave CUs idle: 1024 x 768 -> 768 4.8 - 6.0 us (128: 9.1), 185 x 768 -> 3072 5.0 - 5.9 (9.2).
  const long t192 = tiles(192, 192);
  if (t192 >= 192 && (t192 <= 256 || Kp >= 1536)) I8_GO(3, 1, 2, 6, 3, 1);
  if (tiles(128, 128) >= 192) I8_GO(2, 2, 2, 2, 2, 2);
  I8_GO(1, 1, 2, 2, 3, 3);
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
  if (K > (1 << 30)) return CLIMB_EUNSUPPORTED;          // (before it is rounded up)
  const int Kp = (K + I8_BK - 1) / I8_BK * I8_BK;
  if (M < 0 || N <= 0 || K <= 0 || M > (1 << 30) || N > (1 << 30) || lda < Kp || ldb < Kp || lda % 16 || ldb % 16 || ldc < N || ((uintptr_t)A & 15) || ((uintptr_t)B & 15)) return CLIMB_EINVAL;
  if (epi != EPI_NONE && epi != EPI_GELU && epi != EPI_RESID) return CLIMB_EINVAL;
  if (epi == EPI_RESID && ldaux < N) return CLIMB_EINVAL;
  if (K > (1 << 17) || lda >= (1L << 22) || ldb >= (1L << 22)) return CLIMB_EUNSUPPORTED;          // int32 sums: 127^2 K < 2^31; 32-bit offsets inside a tile
  if (M == 0) return CLIMB_OK;
  if (!A || !sa || !B || !sb || !C || (epi == EPI_RESID && !aux)) return CLIMB_EINVAL;
  // whole 16-byte (16-bit C: 8-byte) pieces of 4 channels; anything else is read and written element by element
  const int vec = ldc % 4 == 0 && !((uintptr_t)C & 15) && (epi != EPI_RESID || (ldaux % 4 == 0 && !((uintptr_t)aux & 15)));
  hipStream_t st = (hipStream_t)stream;
  const signed char *a = (const signed char*)A, *b = (const signed char*)B;
  if (c_dtype == CLIMB_DT_F32) return i8_epi<float>(a, lda, sa, b, ldb, sb, (float*)C, ldc, M, N, Kp, bias, epi, aux, ldaux, vec, st);
  if (c_dtype == CLIMB_DT_BF16) return i8_epi<bf16_t>(a, lda, sa, b, ldb, sb, (bf16_t*)C, ldc, M, N, Kp, bias, epi, aux, ldaux, vec, st);
  return CLIMB_EINVAL;
}

// ------------------------------------------------------------------------------------------------ few tokens
// y = epi(rows8(x) W^T + bias) for M <= 8 tokens in ONE launch: a workgroup owns 16 channels, quantises the tokens itself (its weights are already on their
// way by then), its four waves share the reduction in 64-byte steps of v_mfma_i32_16x16x64_i8 and add their int32 sums through LDS.  Bound by latency: two
// dependent trips to memory and the launch.
// Against quantising in a launch of its own (768 channels, one / two launches): K = 768: 1 token 3.7 / 6.4 us, 4: 4.1 / 6.6, 8: 5.5 / 6.6, 16: 8.4 / 6.9; K = 3072:
// 7.3 / 12.7, 8.5 / 13.0, 13.3 / 13.1, 22.6 / 13.2 -- every workgroup quantises every token, so eight is where it stops paying.
#define FEW_M 8
#define FEW_STEPS 12          // 64-byte steps of a wave, held in registers: K <= 4 * 12 * 64
template <typename T, int MODE>
__global__ __launch_bounds__(256) void linear_i8_few_kernel(const T* __restrict__ x, long ldx, const signed char* __restrict__ W, long ldw, const float* __restrict__ sw,
                                                            void* y, long ldy, int y_dtype, int M, int N, int K, int Kp, const float* __restrict__ bias,
                                                            int epi, const float* aux, long ldaux) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];          // codes [16][Kp + 16] (8 rows written), sums [4][16][17], scales [16]
  const int pitch = Kp + 16, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l15 = lane & 15, n0 = blockIdx.x * 16;
  int* red = reinterpret_cast<int*>(smem + 16 * pitch);
  float* sc = reinterpret_cast<float*>(red + 4 * 16 * 17);
  const int steps = Kp / 64;
  i32x4 wf[FEW_STEPS];
  {
    const signed char* wp = W + (long)min(n0 + l15, N - 1) * ldw + (lane >> 4) * 16;
#pragma unroll
    for (int i = 0; i < FEW_STEPS; ++i)
      if (wave + 4 * i < steps) wf[i] = *reinterpret_cast<const i32x4*>(wp + (wave + 4 * i) * 64);
  }
  for (int r = wave; r < M; r += 4) {
    const T* xr = x + (long)r * ldx;
    unsigned mx = 0;
    float v[4];
#pragma unroll 3
    for (int c = lane * 4; c < K; c += 256) {
      row_ld<MODE, 4>(xr, c, K, v);
#pragma unroll
      for (int j = 0; j < 4; ++j) mx = max(mx, abs_bits(v[j]));
    }
    mx = lanes_umax<64>(mx);
    const float s = row_scale(mx), rs = 1.f / s;
    if (lane == 0) sc[r] = s;
    for (int c = lane * 4; c < Kp; c += 256) {          // (rowq4 asks the whole wave, so hipcc does not unroll this one; its loads hit L1)
      row_ld<MODE, 4>(xr, c, K, v);
      *reinterpret_cast<unsigned*>(smem + r * pitch + c) = rowq4(v, s, rs, mx >= 0x7f800000u);
    }
  }
  __syncthreads();
  i32x4 acc = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < FEW_STEPS; ++i)
    if (wave + 4 * i < steps) {          // (rows M .. 15 of the image are whatever LDS held: integers all the same, and their columns of the result are not read)
      const i32x4 tf = *reinterpret_cast<const i32x4*>(smem + l15 * pitch + (wave + 4 * i) * 64 + (lane >> 4) * 16);
      acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[i], tf, acc, 0, 0, 0);
    }
#pragma unroll
  for (int i = 0; i < 4; ++i) red[(wave * 16 + (lane >> 4) * 4 + i) * 17 + l15] = acc[i];
  __syncthreads();
  const int m = threadIdx.x >> 4, n = n0 + l15;          // (16 x 16 results, rows M .. 15 are not there)
  if (m >= M || n >= N) return;
  int sum = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) sum += red[(w * 16 + l15) * 17 + m];
  float v = scaled_sum(sum, sc[m], sw[n], bias ? bias[n] : 0.f);
  if (epi == EPI_GELU) v = y_dtype == CLIMB_DT_F32 ? gelu_phi<float>(v) : gelu_phi<bf16_t>(v);
  if (epi == EPI_RESID) v += aux[(long)m * ldaux + n];
  if (y_dtype == CLIMB_DT_F32) static_cast<float*>(y)[(long)m * ldy + n] = v;
  else static_cast<bf16_t*>(y)[(long)m * ldy + n] = f32_to_bf16(v);
}

static bool i8_few(int M, int K) { return M <= FEW_M && (K + I8_BK - 1) / I8_BK * I8_BK <= 4 * FEW_STEPS * 64; }

extern "C" int climb_rows8_quant(const void* x, long ldx, int dtype, void* q, long ldq, float* s, int M, int C, void* stream);
extern "C" long climb_linear_i8_workspace(int M, int K) {
  if (M < 0 || M > (1 << 30) || K <= 0 || K > (1 << 17)) return CLIMB_EINVAL;
  return i8_few(M, K) ? 0 : (long)M * ((K + I8_BK - 1) / I8_BK * I8_BK + 4);
}
extern "C" int climb_linear_i8(const void* x, long ldx, int dtype, const void* W, long ldw, const float* sw, void* y, long ldy, int y_dtype, int M, int N, int K,
                               const float* bias, int epi, const float* aux, long ldaux, void* workspace, long workspace_bytes, void* stream) {
  if (M < 0 || N <= 0 || K <= 0 || M > (1 << 30) || N > (1 << 27) || K > (1 << 17) || ldx < K || (dtype != CLIMB_DT_F32 && dtype != CLIMB_DT_BF16) || (y_dtype != CLIMB_DT_F32 && y_dtype != CLIMB_DT_BF16))
    return K > (1 << 17) ? CLIMB_EUNSUPPORTED : CLIMB_EINVAL;
  const int Kp = (K + I8_BK - 1) / I8_BK * I8_BK;
  if (ldw < Kp || ldw % 16 || ((uintptr_t)W & 15) || ldy < N || (epi != EPI_NONE && epi != EPI_GELU && epi != EPI_RESID) || (epi == EPI_RESID && ldaux < N)) return CLIMB_EINVAL;
  if (ldw >= (1L << 22)) return CLIMB_EUNSUPPORTED;
  if (M == 0) return CLIMB_OK;
  if (!x || !W || !sw || !y || (epi == EPI_RESID && !aux)) return CLIMB_EINVAL;
  if (i8_few(M, K)) {
    const int lds = 16 * (Kp + 16) + (4 * 16 * 17 + 16) * 4;
    const dim3 grid((N + 15) / 16), blk(256);
    hipStream_t st = (hipStream_t)stream;
#define FEW(T_, MODE_) \
  hipLaunchKernelGGL((linear_i8_few_kernel<T_, MODE_>), grid, blk, lds, st, (const T_*)x, ldx, (const signed char*)W, ldw, sw, y, ldy, y_dtype, M, N, K, Kp, bias, epi, aux, ldaux)
    if (dtype == CLIMB_DT_F32) { if (K < 4) FEW(float, 2); else FEW(float, 0); }
    else { if (K < 4) FEW(bf16_t, 2); else FEW(bf16_t, 0); }
#undef FEW
    LAUNCH_CHECK();
    return CLIMB_OK;
  }
  if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < climb_linear_i8_workspace(M, K)) return CLIMB_EINVAL;
  float* s = reinterpret_cast<float*>((char*)workspace + (long)M * Kp);
  const int rc = climb_rows8_quant(x, ldx, dtype, workspace, Kp, s, M, K, stream);
  return rc != CLIMB_OK ? rc : climb_gemm_i8_nt(workspace, Kp, s, W, ldw, sw, y, ldy, y_dtype, M, N, K, bias, epi, aux, ldaux, stream);
}
