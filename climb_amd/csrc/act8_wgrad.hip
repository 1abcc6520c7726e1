// Weight gradient of a linear layer whose input was kept as an 8-bit checkpoint (rows8.h):
//   C[n,k] = beta C[n,k] + sum_m dY[m,n] code[m,k] 2^e(m, k / 64),      dbias[n] = beta dbias[n] + sum_m dY[m,n]
// on the 16-bit MFMA.  code * 2^e is a number of the operand type, so the codes are expanded ONCE, on their way into LDS, and no product is rounded.
#include "rows8.h"
#include "gemm_bf16_nt.h"

#define WG_BR 64            // tokens in an LDS tile
#define WG_PITCH 256        // bytes of an LDS row: 128 columns
__device__ __forceinline__ int wg_swz(int row) { return (row & 3) << 2; }      // the 4 token rows of a transpose read lie in 4 different bank quarters

// 16 bytes from any address (the hardware reads unaligned words; hipcc makes one load of it), elements past `left` zero
__device__ __forceinline__ u32x4 wg_ld16(const bf16_t* __restrict__ p, int left) {
  u32x4 r = (u32x4){0u, 0u, 0u, 0u};
  if (left >= 8) __builtin_memcpy(&r, p, 16);
  else if (left > 0) {
    unsigned short h[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) h[i] = p[i];
    __builtin_memcpy(&r, h, 16);
  }
  return r;
}
// 8-token MFMA operand of output index col0 + (lane & 31), tokens mrow0 + (lane >> 5) * 8 + 0..7: two transpose reads
__device__ __forceinline__ bf16x8 wg_frag(const unsigned char* __restrict__ S, int mrow0, int col0, int lane) {
  const int g16 = lane >> 4, i = lane & 15, row = mrow0 + (g16 >> 1) * 8 + (i >> 2), col = col0 + (g16 & 1) * 16 + 4 * (i & 3);
  const unsigned char* p = S + row * WG_PITCH + (((col >> 3) ^ wg_swz(row)) << 4) + (col & 7) * 2;
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  union { s16x4 h[2]; bf16x8 b; } c;
  c.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p));
  c.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 4 * WG_PITCH));
  return c.b;
}

struct WgStage {
  u32x4 a[4], b[2];          // 8 gradients x 4 token rows, 16 codes x 2 token rows
  unsigned e[2];
};
__device__ __forceinline__ void wg_load(WgStage& s, const bf16_t* __restrict__ dY, long lddy, const signed char* __restrict__ q, long ldq,
                                        const unsigned char* __restrict__ e, long lde, int m0, int mend, int n0, int N, int k0, int K) {
  const int t = threadIdx.x;
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const int m = m0 + (t >> 4) + 16 * p, n = n0 + (t & 15) * 8;
    s.a[p] = wg_ld16(dY + (long)m * lddy + n, m < mend ? N - n : 0);
  }
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const int m = m0 + (t >> 3) + 32 * p, k = k0 + (t & 7) * 16;
    const bool ok = m < mend && k < K;          // (a piece that starts inside the row lies inside ldq; tokens past the end are zero codes of step 2^0)
    s.b[p] = ok ? *reinterpret_cast<const u32x4*>(q + (long)m * ldq + k) : (u32x4){0u, 0u, 0u, 0u};
    s.e[p] = ok ? e[(long)m * lde + (k >> 6)] : 127u;
  }
}
__device__ __forceinline__ void wg_store(const WgStage& s, unsigned char* __restrict__ As, unsigned char* __restrict__ Bs) {
  const int t = threadIdx.x;
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const int row = (t >> 4) + 16 * p;
    *reinterpret_cast<u32x4*>(As + row * WG_PITCH + (((t & 15) ^ wg_swz(row)) << 4)) = s.a[p];
  }
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const int row = (t >> 3) + 32 * p;
    const float step = act8_step(s.e[p]);
    unsigned h[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 v = act8_unpack4(s.b[p][i], step);
      h[2 * i] = pack_bf16x2(v.x, v.y);
      h[2 * i + 1] = pack_bf16x2(v.z, v.w);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
      *reinterpret_cast<u32x4*>(Bs + row * WG_PITCH + ((((t & 7) * 2 + i) ^ wg_swz(row)) << 4)) = (u32x4){h[4 * i], h[4 * i + 1], h[4 * i + 2], h[4 * i + 3]};
  }
}

// One workgroup: a 128 (n) x 128 (k) tile over the tokens [split * rows, + rows).  Four waves of 64 x 64.  PART: the sums go to `out` = [split][N * K]
// (and [split][N] for the bias behind them) for act8_wgrad_reduce_kernel, which adds them in the order of the splits; else straight into C.
template <bool PART>
__global__ __launch_bounds__(256) void act8_wgrad_kernel(const bf16_t* __restrict__ dY, long lddy, const signed char* __restrict__ q, long ldq,
                                                         const unsigned char* __restrict__ e, long lde, float* __restrict__ out, long ldc, float* __restrict__ dbias,
                                                         int M, int N, int K, int rows, int splits, float beta) {
  __shared__ __attribute__((aligned(16))) unsigned char smem[4 * WG_BR * WG_PITCH];          // two buffers of { dY, expanded codes }
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, wn = wid >> 1, wk = wid & 1, half = lane >> 5, l31 = lane & 31;
  const int nbn = (N + 127) / 128, nbk = (K + 127) / 128, tiles = nbn * nbk;
  int bid = blockIdx.x;
  {          // XCD-contiguous chunks: the workgroups of an XCD belong to the same token range, whose panels its L2 then holds once
    const int nwg = gridDim.x, c = nwg / 8, rr = nwg % 8, xcd = bid % 8, idx = bid / 8;
    bid = (xcd < rr ? xcd * (c + 1) : rr * (c + 1) + (xcd - rr) * c) + idx;
  }
  const int split = bid / tiles, tile = bid - split * tiles;
  const int ntile = nbn > nbk ? tile / nbk : tile % nbn, ktile = nbn > nbk ? tile % nbk : tile / nbn;      // the narrower operand is spanned first
  const int n0 = ntile * 128, k0 = ktile * 128, mbeg = split * rows, mend = min(M, mbeg + rows);
  f32x16 acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
  const bool do_bias = dbias != nullptr && ktile == 0;
  float bs[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) bs[i] = 0.f;
  WgStage st;
  const int nt = (mend - mbeg + WG_BR - 1) / WG_BR;
  if (nt > 0) wg_load(st, dY, lddy, q, ldq, e, lde, mbeg, mend, n0, N, k0, K);
  for (int t = 0; t < nt; ++t) {
    unsigned char* As = smem + (t & 1) * (2 * WG_BR * WG_PITCH);
    unsigned char* Bs = As + WG_BR * WG_PITCH;
    wg_store(st, As, Bs);
    if (do_bias) {
#pragma unroll
      for (int p = 0; p < 4; ++p)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          bs[2 * i] += h16lo_to_f32(st.a[p][i]);
          bs[2 * i + 1] += h16hi_to_f32(st.a[p][i]);
        }
    }
    if (t + 1 < nt) wg_load(st, dY, lddy, q, ldq, e, lde, mbeg + (t + 1) * WG_BR, mend, n0, N, k0, K);
    __syncthreads();          // (two buffers: the next store goes to the one that every wave has left by then)
#pragma unroll
    for (int ms = 0; ms < WG_BR / 16; ++ms) {
      bf16x8 fa[2], fb[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) fa[i] = wg_frag(As, ms * 16, wn * 64 + i * 32, lane);
#pragma unroll
      for (int j = 0; j < 2; ++j) fb[j] = wg_frag(Bs, ms * 16, wk * 64 + j * 32, lane);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = CLIMB_MFMA_H16(fa[i], fb[j], acc[i][j], 0, 0, 0);
    }
  }
  // a wave instruction writes 2 rows of 32 consecutive floats
  float* o = PART ? out + (long)split * N * K : out;
  const long ld = PART ? K : ldc;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int k = k0 + wk * 64 + j * 32 + l31;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int n = n0 + wn * 64 + i * 32 + (r & 3) + 8 * (r >> 2) + 4 * half;
        if (n < N && k < K) {
          float* p = o + (long)n * ld + k;
          *p = (!PART && beta != 0.f) ? fmaf(beta, *p, acc[i][j][r]) : acc[i][j][r];
        }
      }
    }
  if (do_bias) {          // 16 threads a column group of 8: through LDS, added in a fixed order
    __syncthreads();
    float* red = reinterpret_cast<float*>(smem);          // [16][128]
#pragma unroll
    for (int i = 0; i < 8; ++i) red[(threadIdx.x >> 4) * 128 + (threadIdx.x & 15) * 8 + i] = bs[i];
    __syncthreads();
    const int n = n0 + threadIdx.x;
    if (threadIdx.x < 128 && n < N) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) s += red[i * 128 + threadIdx.x];
      if (PART) out[(long)splits * N * K + (long)split * N + n] = s;
      else dbias[n] = beta != 0.f ? fmaf(beta, dbias[n], s) : s;
    }
  }
}
// C = beta C + the splits' sums, in the order of the splits
__global__ __launch_bounds__(256) void act8_wgrad_reduce_kernel(const float* __restrict__ part, float* __restrict__ C, long ldc, float* __restrict__ dbias, int N, int K,
                                                                int splits, float beta) {
  const long NK = (long)N * K;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < NK + (dbias ? N : 0); i += (long)gridDim.x * 256) {
    const bool w = i < NK;
    const float* p = w ? part + i : part + splits * NK + (i - NK);
    const long stride = w ? NK : N;
    float s = 0.f;
    for (int k = 0; k < splits; ++k) s += p[k * stride];
    const long n = w ? i / K : 0;
    float* o = w ? C + n * ldc + (i - n * K) : dbias + (i - NK);
    *o = beta != 0.f ? fmaf(beta, *o, s) : s;
  }
}

// token ranges the reduction is cut into: enough for two workgroups a CU, none shorter than 256 tokens (below that the second launch costs more)
static int wgrad_splits(int M, int N, int K) {
  const long tiles = (long)((N + 127) / 128) * ((K + 127) / 128);
  const long s = 512 / tiles, most = M / 256;
  const long r = s < most ? s : most;
  return r < 1 ? 1 : (int)r;
}
extern "C" long climb_act8_weight_grad_workspace(int M, int N, int K) {
  if (M < 0 || N <= 0 || K <= 0) return CLIMB_EINVAL;
  const int s = wgrad_splits(M, N, K);
  return s == 1 ? 0 : (long)s * ((long)N * K + N) * 4;
}
extern "C" int climb_act8_weight_grad(const void* dY, long lddy, const void* q, long ldq, const void* e, long lde, float* C, long ldc, float* dbias, int M, int N, int K,
                                      float beta, void* workspace, long workspace_bytes, void* stream) {
  if (M < 0 || M > (1 << 30) || N <= 0 || K <= 0 || lddy < N || ldc < K || ldq < K || ldq % 16 || ((uintptr_t)q & 15) || lde < (K + ACT8_GROUP - 1) / ACT8_GROUP || !C) return CLIMB_EINVAL;
  if (M > 0 && (!dY || !q || !e)) return CLIMB_EINVAL;
  if (((uintptr_t)dY & 1) || ((uintptr_t)C & 3) || ((uintptr_t)dbias & 3)) return CLIMB_EINVAL;
  const int splits = wgrad_splits(M, N, K);
  const long tiles = (long)((N + 127) / 128) * ((K + 127) / 128);
  if (tiles * splits >= (1L << 31)) return CLIMB_EUNSUPPORTED;
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)(tiles * splits)), blk(256);
  if (splits == 1) {
    hipLaunchKernelGGL((act8_wgrad_kernel<false>), grid, blk, 0, st, (const bf16_t*)dY, lddy, (const signed char*)q, ldq, (const unsigned char*)e, lde, C, ldc, dbias, M, N, K,
                       M > 0 ? M : 1, 1, beta);
    LAUNCH_CHECK();
    return CLIMB_OK;
  }
  if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < climb_act8_weight_grad_workspace(M, N, K)) return CLIMB_EINVAL;
  const int rows = ((M + splits - 1) / splits + WG_BR - 1) / WG_BR * WG_BR;
  hipLaunchKernelGGL((act8_wgrad_kernel<true>), grid, blk, 0, st, (const bf16_t*)dY, lddy, (const signed char*)q, ldq, (const unsigned char*)e, lde, (float*)workspace, K, dbias,
                     M, N, K, rows, splits, 0.f);
  LAUNCH_CHECK();
  const long work = (long)N * K + N;
  const unsigned rg = (unsigned)((work + 255) / 256 < 4096 ? (work + 255) / 256 : 4096);
  hipLaunchKernelGGL(act8_wgrad_reduce_kernel, dim3(rg), blk, 0, st, (const float*)workspace, C, ldc, dbias, N, K, splits, beta);
  LAUNCH_CHECK();
  return CLIMB_OK;
}
