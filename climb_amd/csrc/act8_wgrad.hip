// Weight gradient of a linear layer whose input was kept as an 8-bit checkpoint (rows8.h):
//   C[n,k] = beta C[n,k] + sum_m dY[m,n] code[m,k] 2^e(m, k / 64),      dbias[n] = beta dbias[n] + sum_m dY[m,n]
// on the 16-bit MFMA.  code * 2^e is a number of the operand type, so the codes are expanded ONCE, on their way into LDS, and no product is rounded.
#include <type_traits>
#include "rows8.h"
#include "gemm_bf16_nt.h"

#define WG_BR 64            // tokens in an LDS tile
#define WG_PITCH 256        // bytes of an LDS row: 128 columns
__device__ __forceinline__ int wg_swz(int row) { return (row & 3) << 2; }      // the 4 token rows of a transpose read lie in 4 different bank quarters

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

// 16 codes of a group with exponent byte e -> 16 numbers of the operand type, zeros for a token that is not there
__device__ __forceinline__ void wg_expand(u32x4 q, unsigned e, bool live, unsigned (&h)[8]) {
  const float step = live ? act8_step(e) : 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float4 v = act8_values4<bf16_t>(q[i], e, step);
    h[2 * i] = pack_bf16x2(v.x, v.y);
    h[2 * i + 1] = pack_bf16x2(v.z, v.w);
  }
}

// XCD-contiguous chunks of the launch: the workgroups of an XCD belong to the same token range, whose panels its L2 then holds once
__device__ __forceinline__ int wg_chunk() {
  const int id = blockIdx.x, nwg = gridDim.x, c = nwg / 8, rr = nwg % 8, xcd = id % 8;
  return (xcd < rr ? xcd * (c + 1) : rr * (c + 1) + (xcd - rr) * c) + id / 8;
}

struct WgStage {
  u32x4 a[4], b[2];          // 8 gradients x 4 token rows, 16 codes x 2 token rows
  unsigned e[2];
};
// The loads of a tile go out together, all of them unconditional (a load under a condition is waited for inside it): tokens past the end are read as the last
// one, pieces past the last column as the last piece; wg_store puts them right, or their results are not stored.  Any address: the hardware reads unaligned words.
// MODE 1: N % 8 == 0;  0: N >= 8, the piece that crosses the end is the row's last 8 columns, shifted down;  2: shorter rows, element by element.
template <int MODE>
__device__ __forceinline__ void wg_load(WgStage& s, const bf16_t* __restrict__ dY, long lddy, const signed char* __restrict__ q, long ldq,
                                        const unsigned char* __restrict__ e, long lde, int m0, int mend, int n0, int N, int k0, int K) {
  const int t = threadIdx.x;
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const int m = min(m0 + (t >> 4) + 16 * p, mend - 1), n = n0 + (t & 15) * 8;
    if constexpr (MODE == 2) {
      unsigned short h[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = dY[(long)m * lddy + min(n + i, N - 1)];
      __builtin_memcpy(&s.a[p], h, 16);
    } else {
      __builtin_memcpy(&s.a[p], dY + (long)m * lddy + min(n, N - 8), 16);
    }
  }
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const int m = min(m0 + (t >> 3) + 32 * p, mend - 1), k = min(k0 + (t & 7) * 16, (K - 1) & ~15);          // (a piece that starts inside the row lies inside ldq)
    s.b[p] = *reinterpret_cast<const u32x4*>(q + (long)m * ldq + k);
    s.e[p] = e[(long)m * lde + (k >> 6)];
  }
}
template <int MODE>
__device__ __forceinline__ void wg_store(WgStage& s, unsigned char* __restrict__ As, unsigned char* __restrict__ Bs, int left, int n0, int N) {
  const int t = threadIdx.x;
  if (MODE == 0 && n0 + 128 > N) {
    const int d = max(n0 + (t & 15) * 8 - (N - 8), 0);          // (8 and more: a piece past the end)
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      u32x4 v = s.a[p];
      if (d & 4) { v[0] = v[2]; v[1] = v[3]; }
      if (d & 2) { v[0] = v[1]; v[1] = v[2]; v[2] = v[3]; }
      if (d & 1) { v[0] = __builtin_amdgcn_alignbit(v[1], v[0], 16); v[1] = __builtin_amdgcn_alignbit(v[2], v[1], 16); v[2] = __builtin_amdgcn_alignbit(v[3], v[2], 16); v[3] >>= 16; }
      s.a[p] = v;
    }
  }
  if (left < WG_BR) {          // tokens past the end: gradients 0 (an infinity must not meet a zero code, and the bias sums run over all rows), codes of step 0
#pragma unroll
    for (int p = 0; p < 4; ++p)
      if ((t >> 4) + 16 * p >= left) s.a[p] = (u32x4){0u, 0u, 0u, 0u};
  }
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const int row = (t >> 4) + 16 * p;
    *reinterpret_cast<u32x4*>(As + row * WG_PITCH + (((t & 15) ^ wg_swz(row)) << 4)) = s.a[p];
  }
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const int row = (t >> 3) + 32 * p;
    unsigned h[8];
    wg_expand(s.b[p], s.e[p], row < left, h);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      *reinterpret_cast<u32x4*>(Bs + row * WG_PITCH + ((((t & 7) * 2 + i) ^ wg_swz(row)) << 4)) = (u32x4){h[4 * i], h[4 * i + 1], h[4 * i + 2], h[4 * i + 3]};
  }
}

// One workgroup: a 128 (n) x 128 (k) tile over the tokens [split * rows, + rows).  Four waves of 64 x 64.  PART: the sums go to `out` = [split][N * K]
// (and [split][N] for the bias behind them) for act8_wgrad_reduce_kernel, which adds them in the order of the splits; else straight into C.
// Bound by latency on few tokens (768 x 768 over 185: 7.5 us, 36 workgroups with three tiles each one after the other), by the expansion on many.
template <bool PART, int MODE>
__global__ __launch_bounds__(256) void act8_wgrad_kernel(const bf16_t* __restrict__ dY, long lddy, const signed char* __restrict__ q, long ldq,
                                                         const unsigned char* __restrict__ e, long lde, float* __restrict__ out, long ldc, float* __restrict__ dbias,
                                                         int M, int N, int K, int rows, int splits, float beta) {
  __shared__ __attribute__((aligned(16))) unsigned char smem[4 * WG_BR * WG_PITCH];          // two buffers of { dY, expanded codes }
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, wn = wid >> 1, wk = wid & 1, half = lane >> 5, l31 = lane & 31;
  const int nbn = (N + 127) / 128, nbk = (K + 127) / 128, tiles = nbn * nbk;
  const int bid = wg_chunk();
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
  if (nt > 0) wg_load<MODE>(st, dY, lddy, q, ldq, e, lde, mbeg, mend, n0, N, k0, K);
  for (int t = 0; t < nt; ++t) {
    unsigned char* As = smem + (t & 1) * (2 * WG_BR * WG_PITCH);
    unsigned char* Bs = As + WG_BR * WG_PITCH;
    wg_store<MODE>(st, As, Bs, mend - mbeg - t * WG_BR, n0, N);
    if (do_bias) {
#pragma unroll
      for (int p = 0; p < 4; ++p)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          bs[2 * i] += h16lo_to_f32(st.a[p][i]);
          bs[2 * i + 1] += h16hi_to_f32(st.a[p][i]);
        }
    }
    if (t + 1 < nt) wg_load<MODE>(st, dY, lddy, q, ldq, e, lde, mbeg + (t + 1) * WG_BR, mend, n0, N, k0, K);
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
  // a wave instruction writes 2 rows of 32 consecutive floats; old values are fetched 16 at a time, unconditionally (a place past the end: the last one)
  float* o = PART ? out + (long)split * N * K : out;
  const long ld = PART ? K : ldc;
  const bool acc_c = !PART && beta != 0.f;
  auto put = [&](auto full_) {
    constexpr bool FULL = decltype(full_)::value;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int k = k0 + wk * 64 + j * 32 + l31;
        float old[16];
        if (acc_c) {
#pragma unroll
          for (int r = 0; r < 16; ++r) old[r] = o[(long)min(n0 + wn * 64 + i * 32 + (r & 3) + 8 * (r >> 2) + 4 * half, N - 1) * ld + min(k, K - 1)];
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[i][j][r] = fmaf(beta, old[r], acc[i][j][r]);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int n = n0 + wn * 64 + i * 32 + (r & 3) + 8 * (r >> 2) + 4 * half;
          if (FULL || (n < N && k < K)) o[(long)n * ld + k] = acc[i][j][r];
        }
      }
  };
  if (n0 + 128 <= N && k0 + 128 <= K) put(std::true_type{});
  else put(std::false_type{});
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
// C = beta C + the splits' sums, in the order of the splits; the bias sums lie behind the splits' planes, `bplanes` of them.  V columns a thread.
template <int V>
__global__ __launch_bounds__(256) void act8_wgrad_reduce_kernel(const float* __restrict__ part, float* __restrict__ C, long ldc, float* __restrict__ dbias, int N, int K,
                                                                int splits, int bplanes, float beta) {
  const long NK = (long)N * K;
  for (long i = ((long)blockIdx.x * 256 + threadIdx.x) * V; i < NK; i += (long)gridDim.x * 256 * V) {
    float s[V];
#pragma unroll
    for (int j = 0; j < V; ++j) s[j] = 0.f;
    for (int k0 = 0; k0 < splits; k0 += 8) {          // eight planes' loads on their way at once; planes past the last are it again, not added
      float v[8][V];
#pragma unroll
      for (int k = 0; k < 8; ++k) __builtin_memcpy(v[k], part + (long)min(k0 + k, splits - 1) * NK + i, sizeof(v[k]));
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) s[j] += k0 + k < splits ? v[k][j] : 0.f;
    }
    const long n = i / K;          // (V divides K: one row)
    float* o = C + n * ldc + (i - n * K);
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = beta != 0.f ? fmaf(beta, o[j], s[j]) : s[j];
  }
  if (dbias)
    for (int n = blockIdx.x * 256 + threadIdx.x; n < N; n += gridDim.x * 256) {
      float s = 0.f;
      for (int k = 0; k < bplanes; ++k) s += part[(long)splits * NK + (long)k * N + n];
      dbias[n] = beta != 0.f ? fmaf(beta, dbias[n], s) : s;
    }
}

// ------------------------------------------------------------------------------------------------ large, aligned problems
// The same sum on 256 (n) x 256 (k) tiles, one workgroup of 8 waves a CU (4 x 2 waves of 64 x 128): a code is expanded once for 256 channels (the 128-tile
// kernel is bound by that VALU work).  Everything comes to LDS by DMA: a ring of 5 stages { gradients [32 tokens][256] , codes [32][256], exponents }, and two
// images of expanded codes.  The step that multiplies token tile t (two groups of 8 MFMAs)
//   - expands the codes of tile t + 1 in its first group (each lane expands the 16 codes it fetched itself, read from LDS a group earlier),
//   - meets the workgroup in the second group; behind the barrier the ring slot of tile t takes the DMA of tile t + 5, and the first fragments of tile t + 1
//     are read under the rest of the group.
// Measured, 3072 x 768 over 12288 tokens: 74 us (0.78 PFLOP/s) + 14 us of reduction in a trace, 85 together in a graph, against 109 for the 128-tile kernel with its own and 118 us for the vendor library's
// 16-bit product of the same shape.  Bounded by the loop: its LDS reads (taken out: - 16 us), its MFMAs (33 us at the clock the chip sustains), the expansion (- 8 us)
// and the final stores (- 7 us) overlap between the two waves of a SIMD only.
// As in gemm_i8.hip fragments are read behind the first MFMA of the group before, and no load goes to registers: hipcc would wait for all DMA with it.
#define WB_T 256
#define WB_BR 32
#define WB_PITCH 512
#define WB_IMG (WB_BR * WB_PITCH)                       // 16 KB
#define WB_CODES (WB_BR * WB_T)                         // 8 KB
#define WB_STAGE (WB_IMG + WB_CODES + 256)
#define WB_RING 5
#define WB_LDS (WB_RING * WB_STAGE + 2 * WB_IMG)
#define WB_LPT 4                                        // DMA instructions of a stage and lane: 2 gradients, 1 codes, 1 exponents
__device__ __forceinline__ bf16x8 wb_frag(const unsigned char* __restrict__ p) {
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  union { s16x4 h[2]; bf16x8 b; } c;
  c.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p));
  c.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 4 * WB_PITCH));
  return c.b;
}
__device__ __forceinline__ void wb_expand(u32x4 q, unsigned e4, bool live, unsigned char* __restrict__ Bs) {
  const int row = threadIdx.x >> 4, c16 = threadIdx.x & 15;
  unsigned h[8];
  wg_expand(q, (e4 >> ((c16 >> 2) * 8)) & 255u, live, h);
#pragma unroll
  for (int i = 0; i < 2; ++i)
    *reinterpret_cast<u32x4*>(Bs + row * WB_PITCH + (((c16 * 2 + i) ^ wg_swz(row)) << 4)) = (u32x4){h[4 * i], h[4 * i + 1], h[4 * i + 2], h[4 * i + 3]};
}
__global__ __launch_bounds__(512) void act8_wgrad_big_kernel(const bf16_t* __restrict__ dY, long lddy, const signed char* __restrict__ q, long ldq,
                                                             const unsigned char* __restrict__ e, long lde, float* __restrict__ out, int want_bias, int M, int N, int K,
                                                             int rows, int splits) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];          // the ring, then the two expanded images
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wn = wid >> 1, wk = wid & 1, half = lane >> 5, l31 = lane & 31;
  const int nbn = (N + WB_T - 1) / WB_T, nbk = (K + WB_T - 1) / WB_T, tiles = nbn * nbk;
  const int bid = wg_chunk();
  const int split = bid / tiles, tile = bid - split * tiles;
  const int ntile = nbn > nbk ? tile / nbk : tile % nbn, ktile = nbn > nbk ? tile % nbk : tile / nbn;
  const int n0 = ntile * WB_T, k0 = ktile * WB_T, mbeg = split * rows, mend = min(M, mbeg + rows);
  const int nt = (mend - mbeg + WB_BR - 1) / WB_BR;          // at least WB_RING (wgrad_plan)
  // DMA sources of a lane, relative to the first token of a stage; columns past the end repeat the last piece (their results are not stored), tokens past the
  // end the last one (their codes expand to zeros, their gradients are cleared)
  const int arow = threadIdx.x >> 5;          // rows arow and arow + 16 of the gradients
  const unsigned acol = (unsigned)min(n0 + (int)((threadIdx.x & 31) ^ wg_swz(arow)) * 8, N - 8) * 2, ldb = (unsigned)lddy * 2;
  const int qrow = threadIdx.x >> 4;
  const unsigned qcol = (unsigned)min(k0 + (int)(threadIdx.x & 15) * 16, (K - 1) & ~15);
  // running sources of the next stage to fetch, and its distance from the end
  const unsigned char* ap = reinterpret_cast<const unsigned char*>(dY + (long)mbeg * lddy);
  const signed char* qp = q + (long)mbeg * ldq;
  const unsigned char* ep = e + (long)mbeg * lde + (k0 >> 6);
  const long astep = (long)WB_BR * lddy * 2, qstep = (long)WB_BR * ldq, estep = (long)WB_BR * lde;
  int dleft = mend - mbeg;
  const unsigned av0 = (unsigned)arow * ldb + acol, av1 = (unsigned)(arow + 16) * ldb + acol, qv = (unsigned)qrow * (unsigned)ldq + qcol, ev = (unsigned)l31 * (unsigned)lde;
  auto dma = [&](unsigned char* S) {
    unsigned a0 = av0, a1 = av1, qo = qv, eo = ev;
    if (dleft < WB_BR) {
      const int last = dleft - 1;
      a0 = (unsigned)min(arow, last) * ldb + acol;
      a1 = (unsigned)min(arow + 16, last) * ldb + acol;
      qo = (unsigned)min(qrow, last) * (unsigned)ldq + qcol;
      eo = (unsigned)min(l31, last) * (unsigned)lde;
    }
    __builtin_amdgcn_global_load_lds((gbl_void_t*)(ap + a0), (lds_void_t*)(S + wid * 1024), 16, 0, 0);
    __builtin_amdgcn_global_load_lds((gbl_void_t*)(ap + a1), (lds_void_t*)(S + 8192 + wid * 1024), 16, 0, 0);
    __builtin_amdgcn_global_load_lds((gbl_void_t*)(qp + qo), (lds_void_t*)(S + WB_IMG + wid * 1024), 16, 0, 0);
    __builtin_amdgcn_global_load_lds((gbl_void_t*)(ep + eo), (lds_void_t*)(S + WB_IMG + WB_CODES), 4, 0, 0);          // (every wave fetches the 32 words of exponents: it
    ap += astep; qp += qstep; ep += estep; dleft -= WB_BR;                                                            // waits for its own loads only)
  };
  unsigned char* bimg = smem + WB_RING * WB_STAGE;
  // fragment addresses: A blocks 2 (n), B blocks 4 (k), rows ms * 16 + frow
  const int g16 = lane >> 4, i16 = lane & 15, frow = (g16 >> 1) * 8 + (i16 >> 2), fcol = (g16 & 1) * 16 + 4 * (i16 & 3);
  unsigned aoff[2], boff[4];
#pragma unroll
  for (int i = 0; i < 2; ++i) { const int c = wn * 64 + i * 32 + fcol; aoff[i] = frow * WB_PITCH + (((c >> 3) ^ wg_swz(frow)) << 4) + (c & 7) * 2; }
#pragma unroll
  for (int j = 0; j < 4; ++j) { const int c = wk * 128 + j * 32 + fcol; boff[j] = frow * WB_PITCH + (((c >> 3) ^ wg_swz(frow)) << 4) + (c & 7) * 2; }
  f32x16 acc[2][4];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
  float bsum[2] = {0.f, 0.f};
  bf16x8 fa[2][2], fb[2][4];
  auto frags = [&](bf16x8(&a)[2], bf16x8(&b)[4], const unsigned char* stage, const unsigned char* img, int ms) {
    const unsigned char *A = stage + ms * (16 * WB_PITCH), *B = img + ms * (16 * WB_PITCH);
#pragma unroll
    for (int i = 0; i < 2; ++i) a[i] = wb_frag(A + aoff[i]);
#pragma unroll
    for (int j = 0; j < 4; ++j) b[j] = wb_frag(B + boff[j]);
  };
  u32x4 raw;
  unsigned e4;
  auto raw_read = [&](const unsigned char* stage) {
    raw = *reinterpret_cast<const u32x4*>(stage + WB_IMG + threadIdx.x * 16);
    e4 = *reinterpret_cast<const unsigned*>(stage + WB_IMG + WB_CODES + qrow * 4);
  };
  // the gradients of tokens past the end become zero rows (an infinity must not meet a zero code, and the bias sums run over all rows): every lane clears what
  // it fetched itself, once that has landed and before the barrier behind which the stage is read
  const int valid = (mend - mbeg - 1) % WB_BR + 1;          // tokens of the last stage
  auto clear_tail = [&](unsigned char* stage) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (arow + 16 * i >= valid) *reinterpret_cast<u32x4*>(stage + i * 8192 + threadIdx.x * 16) = (u32x4){0u, 0u, 0u, 0u};
  };
  for (int t = 0; t < WB_RING; ++t) dma(smem + t * WB_STAGE);
  wait_vmcnt<(WB_RING - 2) * WB_LPT>();          // stages 0 and 1 have landed
  raw_read(smem);
  int qm = mend - mbeg - qrow;          // > 0: this lane's token of the tile it expands exists
  wb_expand(raw, e4, qm > 0, bimg);
  raw_read(smem + WB_STAGE);
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  frags(fa[0], fb[0], smem, bimg, 0);
  unsigned char *s0 = smem, *s1 = smem + WB_STAGE, *s2 = smem + 2 * WB_STAGE, *img = bimg, *img1 = bimg + WB_IMG;          // stages t, t + 1, t + 2; images t, t + 1
  int bias_in = want_bias && wk == 0 ? ktile : 1 << 30;          // tiles until this workgroup's next share of the bias sums
  // (the last steps expand and read what is left in LDS from earlier tiles: nothing of it is used)
  for (int t = 0; t < nt; ++t) {
    const bool bias_tile = bias_in == 0;
    bias_in = bias_tile ? nbk - 1 : bias_in - 1;
    qm -= WB_BR;
#pragma unroll
    for (int ms = 0; ms < 2; ++ms) {
      acc[0][0] = CLIMB_MFMA_H16(fa[ms][0], fb[ms][0], acc[0][0], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
      if (ms == 0) {
        frags(fa[1], fb[1], s0, img, 1);
        __builtin_amdgcn_sched_barrier(0);
        wb_expand(raw, e4, qm > 0, img1);
      } else {
        if (t + WB_RING - 1 < nt) wait_vmcnt<(WB_RING - 3) * WB_LPT>();          // stage t + 2 has landed, t + 3 and t + 4 may be out
        else wait_vmcnt<0>();
        if (t + 3 == nt && valid < WB_BR) clear_tail(s2);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        frags(fa[0], fb[0], s1, img1, 0);
        raw_read(s2);
        if (t + WB_RING < nt) dma(s0);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (i || j) acc[i][j] = CLIMB_MFMA_H16(fa[ms][i], fb[ms][j], acc[i][j], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
      if (bias_tile) {          // (a fragment holds 8 tokens of one channel; the tiles are dealt to the workgroups that share the channels)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          union { bf16x8 b; unsigned u[4]; } c;
          c.b = fa[ms][i];
#pragma unroll
          for (int w = 0; w < 4; ++w) bsum[i] += h16lo_to_f32(c.u[w]) + h16hi_to_f32(c.u[w]);
        }
      }
    }
    s0 = s1; s1 = s2;
    s2 = s2 == smem + (WB_RING - 1) * WB_STAGE ? smem : s2 + WB_STAGE;
    unsigned char* x = img; img = img1; img1 = x;
  }
  float* o = out + (long)split * N * K;
  auto put = [&](auto full_) {
    constexpr bool FULL = decltype(full_)::value;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = k0 + wk * 128 + j * 32 + l31;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int n = n0 + wn * 64 + i * 32 + (r & 3) + 8 * (r >> 2) + 4 * half;
          if (FULL || (n < N && k < K)) o[(long)n * K + k] = acc[i][j][r];
        }
      }
  };
  if (n0 + WB_T <= N && k0 + WB_T <= K) put(std::true_type{});
  else put(std::false_type{});
  if (want_bias && wk == 0) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float s = bsum[i] + __shfl_xor(bsum[i], 32, 64);
      const int n = n0 + wn * 64 + i * 32 + l31;
      if (half == 0 && n < N) out[(long)splits * N * K + ((long)split * nbk + ktile) * N + n] = s;
    }
  }
}

// The plan of a problem: which kernel, and into how many token ranges the reduction is cut.
//   small: 128 x 128 tiles, two workgroups a CU, ranges of 256 tokens or more on average (with less the second launch costs more), the last one shorter
//   big:   256 x 256 tiles, one workgroup a CU; needs whole 16-byte pieces of the gradients, whole words of exponents, tiles for at least 24 CUs, and tokens for
//          ranges of 768 or more on average.  At most ten ranges of 64-token tiles, 12 or more a range before rounding up, leave the last one 4 tiles or more: 193
//          tokens, which fill the ring.  Its partial sums are 256 KB a workgroup whatever the problem, twice what the small tiles write: with fewer tiles (more ranges) that
//          outweighs the faster loop.  Both kernels with the reduction, us, big / small, N x K over M tokens: 3072 x 768 over 12288 85 / 109, over 4096 47 / 44, over
//          2048 39 / 31; 2304 x 768 over 12288 70 / 79; 768 x 768 over 12288 58 / 38; 512 x 512 over 12288 60 / 31.
// Ranges of 128 tokens in place of 256 (small): 2304 x 768 over 400 20 us (12), 768 x 768 over 1024 20 (15), 260 x 384 over 700 12 (14).
struct WgPlan { bool big; int splits, rows; long ws; };
static_assert(WB_LDS <= 160 * 1024, "LDS");
static WgPlan wgrad_plan(int M, int N, int K, bool aligned) {
  WgPlan p;
  const long bt = (long)((N + WB_T - 1) / WB_T) * ((K + WB_T - 1) / WB_T), st = (long)((N + 127) / 128) * ((K + 127) / 128);
  const long mtiles = ((long)M + WG_BR - 1) / WG_BR, bs = bt <= 256 ? 256 / bt : 1;
  p.big = aligned && N % 8 == 0 && bt >= 24 && bt <= 256 && bs * bt >= 192 && mtiles >= 12 * bs;
  long s = 512 / st, most = M / 256;
  s = p.big ? bs : (s < most ? s : most);
  if (s < 1) s = 1;
  p.rows = M > 0 ? (int)((mtiles + s - 1) / s * WG_BR) : 1;
  p.splits = M > 0 ? (int)(((long)M + p.rows - 1) / p.rows) : 1;          // (no range is empty)
  const long bplanes = p.big ? (long)p.splits * ((K + WB_T - 1) / WB_T) : p.splits;
  p.ws = p.splits == 1 && !p.big ? 0 : ((long)p.splits * N * K + bplanes * N) * 4;
  return p;
}
extern "C" long climb_act8_weight_grad_workspace(int M, int N, int K) {
  if (M < 0 || M > (1 << 30) || N <= 0 || N > (1 << 30) || K <= 0 || K > (1 << 30)) return CLIMB_EINVAL;
  const long a = wgrad_plan(M, N, K, true).ws, b = wgrad_plan(M, N, K, false).ws;          // (alignments are not known here)
  return a > b ? a : b;
}
extern "C" int climb_act8_weight_grad(const void* dY, long lddy, const void* q, long ldq, const void* e, long lde, float* C, long ldc, float* dbias, int M, int N, int K,
                                      float beta, void* workspace, long workspace_bytes, void* stream) {
  if (M < 0 || M > (1 << 30) || N <= 0 || N > (1 << 30) || K <= 0 || K > (1 << 30) || lddy < N || ldc < K || ldq < K || ldq % 16 || ((uintptr_t)q & 15) || lde < (K + ACT8_GROUP - 1) / ACT8_GROUP || !C)
    return CLIMB_EINVAL;
  if (M > 0 && (!dY || !q || !e)) return CLIMB_EINVAL;
  if (((uintptr_t)dY & 1) || ((uintptr_t)C & 3) || ((uintptr_t)dbias & 3)) return CLIMB_EINVAL;
  const WgPlan p = wgrad_plan(M, N, K, lddy % 8 == 0 && !((uintptr_t)dY & 15) && lde % 4 == 0 && !((uintptr_t)e & 3) && lddy < (1L << 24) && ldq < (1L << 24) && lde < (1L << 24));
  const long tiles = (long)((N + 127) / 128) * ((K + 127) / 128);
  if (tiles * p.splits >= (1L << 24)) return CLIMB_EUNSUPPORTED;          // (a launch holds less than 2^32 threads)
  hipStream_t st = (hipStream_t)stream;
  const bf16_t* dy = (const bf16_t*)dY;
  const signed char* qc = (const signed char*)q;
  const unsigned char* ec = (const unsigned char*)e;
#define WGL(PART_, MODE_, G_, O_, LD_, ...) \
  hipLaunchKernelGGL((act8_wgrad_kernel<PART_, MODE_>), G_, dim3(256), 0, st, dy, lddy, qc, ldq, ec, lde, O_, LD_, dbias, M, N, K, __VA_ARGS__)
#define WGS(PART_, ...)                               \
  do {                                                \
    if (N % 8 == 0) WGL(PART_, 1, __VA_ARGS__);       \
    else if (N > 8) WGL(PART_, 0, __VA_ARGS__);       \
    else WGL(PART_, 2, __VA_ARGS__);                  \
  } while (0)
  if (p.ws == 0) {
    WGS(false, dim3((unsigned)tiles), C, ldc, M > 0 ? M : 1, 1, beta);
    LAUNCH_CHECK();
    return CLIMB_OK;
  }
  if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < p.ws) return CLIMB_EINVAL;
  float* ws = (float*)workspace;
  int bplanes = p.splits;
  if (p.big) {
    const int nbk = (K + WB_T - 1) / WB_T, lds = WB_LDS;
    if ((long)M - (long)(p.splits - 1) * p.rows <= (WB_RING - 1) * WB_BR) return CLIMB_EUNSUPPORTED;          // (the kernel fetches a whole ring ahead)
    bplanes *= nbk;
    hipError_t err = hipFuncSetAttribute(reinterpret_cast<const void*>(act8_wgrad_big_kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (err != hipSuccess) return (int)err;
    hipLaunchKernelGGL(act8_wgrad_big_kernel, dim3((N + WB_T - 1) / WB_T * nbk * p.splits), dim3(512), lds, st, dy, lddy, qc, ldq, ec, lde, ws, dbias != nullptr, M, N, K, p.rows,
                       p.splits);
  } else {
    WGS(true, dim3((unsigned)(tiles * p.splits)), ws, K, p.rows, p.splits, 0.f);
  }
#undef WGS
#undef WGL
  LAUNCH_CHECK();
  const bool v4 = K % 4 == 0 && ldc % 4 == 0;
  const long pieces = ((long)N * K / (v4 ? 4 : 1) + 255) / 256;
  const dim3 rg((unsigned)(pieces < 1 ? 1 : (pieces < 4096 ? pieces : 4096)));
  if (v4) hipLaunchKernelGGL((act8_wgrad_reduce_kernel<4>), rg, dim3(256), 0, st, ws, C, ldc, dbias, N, K, p.splits, bplanes, beta);
  else hipLaunchKernelGGL((act8_wgrad_reduce_kernel<1>), rg, dim3(256), 0, st, ws, C, ldc, dbias, N, K, p.splits, bplanes, beta);
  LAUNCH_CHECK();
  return CLIMB_OK;
}
