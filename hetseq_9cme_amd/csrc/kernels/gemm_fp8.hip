// Products of e4m3 operands with one power-of-two scale per row and block of 128 (hx_quant.h):
//
//   C[M][N] (+)= sum over k blocks b of 2^(ea[m][b] + eb[n][b]) sum_k A[m][k] B[n][k]   (+ bias[n])
//
// A [M][Kp] and B [N][Kp] are codes with rows padded to whole blocks (the padding is zero), so the
// three products of a linear layer -- y = Q(x) Q(W)^T, dx = Q(dy) Q(W^T)^T, dW = Q(dy^T) Q(x^T)^T --
// are this one shape on the copies that split8 writes.
//
// Two ways through the matrix cores:
//  * fast: v_mfma_scale_f32_32x32x64_f8f6f4 on the codes, the block scales as its E8M0 operands (no
//    vector instruction at all for the scaling).  The instruction keeps about 16 bits below the
//    largest product of a small group: relative error 1.5e-5 (normal data) to 3e-5 (spread over
//    decades) of the result, whatever the depth -- 1/100 of a bf16 rounding, so it carries every
//    product whose result is rounded to bf16.
//  * exact: the codes decoded to bf16 with their scale (v_cvt_scalef32_pk_bf16_fp8, exact) after the
//    LDS read, and v_mfma_f32_32x32x16_bf16, which sums exact products in fp32 (1e-7): the products
//    whose result is kept in fp32 (weight gradients, fp32 activations).  Half the matrix rate.
#include <algorithm>

#include "hx_gemm.h"
#include "hx_launch.h"
#include "hx_quant.h"

namespace {

using namespace hx::g;
using hx::bf2f;
using hx::q8::bf16x2;
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8v __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2v __attribute__((ext_vector_type(2)));

__device__ __forceinline__ void raw_barrier() { asm volatile("s_barrier" ::: "memory"); }

// 8 codes (two words of a fragment) -> bf16 values times s
__device__ __forceinline__ bf16x8v decode8(int w0, int w1, float s) {
  const bf16x2v a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, s, false);
  const bf16x2v b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, s, true);
  const bf16x2v c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, s, false);
  const bf16x2v d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, s, true);
  return bf16x8v{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// C[M][N] on a BM x BN tile per workgroup, (BM / WM)(BN / WN) waves of WM x WN.
// LDS: NS stages of KS codes of every row of the tile, filled by LDS-DMA, and two slots of scale
// words (one word = 4 blocks of a row).  A k block is two 64-deep halves: while the MFMAs of one run
// on fragments in registers, the fragments of the next are read.  A stage is opened (`open`) by a
// counted vmcnt and one raw barrier, which also frees the stage before it for the next DMA.
template <int BM, int BN, int WM, int WN, int KS, int NS, int WGS, bool EXACT, bool OB>
__global__ __launch_bounds__((BM / WM) * (BN / WN) * 64, (BM / WM) * (BN / WN) * WGS / 4) void gemm_fp8_k(HxGemm8 g) {
  constexpr int NWM = BM / WM, NWN = BN / WN, NW = NWM * NWN;
  constexpr int MB = WM / 32, NB = WN / 32;
  static_assert(KS == 64 || KS == 128, "stage depth");
  constexpr int RPP = 1024 / KS;                       // rows per 1-KiB DMA piece
  constexpr int KA = BM / RPP, KB = BN / RPP, J = (KA + KB) / NW;
  static_assert((KA + KB) % NW == 0 && BM % RPP == 0 && BN % RPP == 0, "whole DMA pieces per wave");
  static_assert(BM <= 256 && BN <= 256 && NW >= 2, "one DMA piece of scale words per operand");
  constexpr int STAGE = (BM + BN) * KS, SCALES = NS * STAGE;   // + 2 slots x (A, B, spare) x 1 KiB
  extern __shared__ __attribute__((aligned(16))) char lds[];

  const int TM = (g.M + BM - 1) / BM, TN = (g.N + BN - 1) / BN, total = TM * TN;
  const int per = (total * g.ks + 7) / 8;
  const int work0 = (blockIdx.x % 8) * per + blockIdx.x / 8;   // tiles dealt XCD by XCD
  if (work0 >= total * g.ks || (int)(blockIdx.x / 8) >= per) return;   // uniform per workgroup
  const int z = work0 / total, work = work0 - z * total;
  const int nt = work % TN, mt = work / TN;
  const int m0 = mt * BM, n0 = nt * BN;
  // k blocks of this slab: whole groups of four (one scale word)
  const int groups = (g.nkb + 3) / 4, gper = (groups + g.ks - 1) / g.ks;
  const int kb0 = min(z * gper * 4, g.nkb), kb1 = min(kb0 + gper * 4, g.nkb);

  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wv % NWM, wn = wv / NWM, h = lane >> 5, l32 = lane & 31;

  const int mrows = min(BM, g.M - m0), nrows = min(BN, g.N - n0);
  const u32x4 ra = rsrc_of(g.A + (int64_t)m0 * g.lda, (uint32_t)(mrows * g.lda));
  const u32x4 rb = rsrc_of(g.B + (int64_t)n0 * g.ldb, (uint32_t)(nrows * g.ldb));
  const int64_t sam = (g.M + 3) & ~3, sbn = (g.N + 3) & ~3;
  const u32x4 rsa = rsrc_of(g.sa + m0, (uint32_t)((groups * sam - m0) * 4));
  const u32x4 rsb = rsrc_of(g.sb + n0, (uint32_t)((groups * sbn - n0) * 4));
  const uint32_t lds0 = (uint32_t)(size_t)(lds_void*)lds;

  // lane L of a DMA piece fetches (row L / (KS / 16), 16-B chunk c) so that the lane-linear LDS
  // write lands chunk c of row r at position c ^ swz(r): fragment reads are free of bank conflicts
  uint32_t voff[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int q = wv + NW * j, r = (q < KA ? q : q - KA) * RPP + lane / (KS / 16);
    const int c = (lane % (KS / 16)) ^ (KS == 128 ? (r >> 1) & 7 : (r >> 2) & 3);
    voff[j] = (uint32_t)(r * (q < KA ? g.lda : g.ldb) + 16 * c);
  }
  constexpr int SPB = 128 / KS;   // stages per k block
  const int st1 = (kb1 - kb0) * SPB;
  auto dma = [&](int st) {
    // past the slab's end: an offset past every buffer (zeros, no memory traffic, still counted)
    const uint32_t ko = st < st1 ? (uint32_t)(kb0 * 128 + st * KS) : 0x80000000u;
    const uint32_t base = lds0 + (uint32_t)(st % NS) * STAGE;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int q = wv + NW * j;
      dma16(q < KA ? ra : rb, base + 1024u * q, voff[j] + ko);
    }
  };
  auto dma_scales = [&](int grp) {   // scale words of k blocks 4 grp .. + 3: wave 0 A's rows, wave 1 B's
    const uint32_t dst = lds0 + SCALES + (uint32_t)(grp & 1) * 3072 + (wv == 0 ? 0 : wv == 1 ? 1024 : 2048);
    const uint32_t off = wv < 2 && grp < groups ? (uint32_t)(grp * (wv == 0 ? sam : sbn) * 4) + 16 * lane : 0x80000000u;
    dma16(wv == 0 ? rsa : rsb, dst, off);
  };
  auto open = [&](int st) {   // stage st readable by every wave; the slot of stage st - 1 refilled
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    dma_wait<(NS - 2) * J>();
    raw_barrier();
    dma(st - 1 + NS);
  };

  f32x16 acc[MB][NB];
#pragma unroll
  for (int a = 0; a < MB; ++a)
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[a][b] = f32x16{0};

  struct Fr {
    i32x8 a[MB], b[NB];
  };
  auto frag = [&](const char* st, int row, int half) {
    const int r = row + l32;
    const char* p = st + r * KS;
    const int sw = KS == 128 ? (r >> 1) & 7 : (r >> 2) & 3;
    const i32x4 lo = *reinterpret_cast<const i32x4*>(p + 16 * ((4 * half + h) ^ sw));
    const i32x4 hi = *reinterpret_cast<const i32x4*>(p + 16 * ((4 * half + 2 + h) ^ sw));
    return i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  };
  auto read = [&](int st, int half, Fr& F) {
    const char* p = lds + (st % NS) * STAGE;
#pragma unroll
    for (int a = 0; a < MB; ++a) F.a[a] = frag(p, wm * WM + 32 * a, half);
#pragma unroll
    for (int b = 0; b < NB; ++b) F.b[b] = frag(p + BM * KS, wn * WN + 32 * b, half);
  };
  uint32_t wa[MB], wb[NB];   // scale words, the current block's byte lowest
  auto read_scales = [&](int grp) {
    const uint32_t* p = reinterpret_cast<const uint32_t*>(lds + SCALES + (grp & 1) * 3072);
#pragma unroll
    for (int a = 0; a < MB; ++a) wa[a] = p[wm * WM + 32 * a + l32];
#pragma unroll
    for (int b = 0; b < NB; ++b) wb[b] = p[256 + wn * WN + 32 * b + l32];
  };
  // rows of the result run along n (the first MFMA operand), so a lane holds 4 consecutive columns
  auto mma = [&](const Fr& F) {
    if constexpr (!EXACT) {
#pragma unroll
      for (int a = 0; a < MB; ++a)
#pragma unroll
        for (int b = 0; b < NB; ++b)
          acc[a][b] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(F.b[b], F.a[a], acc[a][b], 0, 0, 0, wb[b], 0, wa[a]);
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        bf16x8v fb[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) fb[b] = decode8(F.b[b][2 * q], F.b[b][2 * q + 1], hx::q8::scale_of(wb[b] & 0xffu));
#pragma unroll
        for (int a = 0; a < MB; ++a) {
          const bf16x8v fa = decode8(F.a[a][2 * q], F.a[a][2 * q + 1], hx::q8::scale_of(wa[a] & 0xffu));
#pragma unroll
          for (int b = 0; b < NB; ++b) acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fb[b], fa, acc[a][b], 0, 0, 0);
        }
      }
    }
  };

  if (kb0 < kb1) {
    dma_scales(kb0 / 4);
#pragma unroll
    for (int i = 0; i < NS; ++i) dma(i);
    dma_wait<(NS - 1) * J>();   // the scale words and stage 0 landed
    raw_barrier();
    Fr F0, F1;
    read(0, 0, F0);
    for (int kb = kb0; kb < kb1; ++kb) {
      if ((kb & 3) == 0) {
        read_scales(kb >> 2);
        dma_scales((kb >> 2) + 1);
      } else {
#pragma unroll
        for (int a = 0; a < MB; ++a) wa[a] >>= 8;
#pragma unroll
        for (int b = 0; b < NB; ++b) wb[b] >>= 8;
      }
      const int st = (kb - kb0) * SPB;
      if constexpr (SPB == 2) {
        open(st + 1);
        read(st + 1, 0, F1);
      } else {
        read(st, 1, F1);
      }
      mma(F0);
      open(st + SPB);   // (past the end: a stale slot is read, and not used)
      read(st + SPB, 0, F0);
      mma(F1);
    }
  }
  dma_wait<0>();
  __syncthreads();

  // ---- epilogue: 32 rows of the wave's tile at a time through its own piece of LDS, 16-B row stores
  using OutT = std::conditional_t<OB, uint16_t, float>;
  constexpr int ES = OB ? 2 : 4, RS = WN * ES + 16;
  static_assert(NW * 32 * RS <= NS * STAGE, "staging fits the stages");
  char* my = lds + wv * 32 * RS;
  OutT* C = (OutT*)g.C + (int64_t)z * g.c_zs;
  const int cn = n0 + wn * WN;
#pragma unroll
  for (int a = 0; a < MB; ++a) {
    const int rbase = m0 + wm * WM + 32 * a;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int lc = 32 * b + 8 * q + 4 * h, c = cn + lc;
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[i] = acc[a][b][4 * q + i];
          if (g.bias && c + i < g.N) v[i] += g.bias[c + i];
          if (g.beta && rbase + l32 < g.M && c + i < g.N) {
            const OutT o = C[(int64_t)(rbase + l32) * g.ldc + c + i];
            if constexpr (OB) v[i] += bf2f(o);
            else v[i] += o;
          }
        }
        if constexpr (OB) *reinterpret_cast<uint2*>(my + l32 * RS + lc * 2) = make_uint2(bf16x2(v[0], v[1]), bf16x2(v[2], v[3]));
        else *reinterpret_cast<float4*>(my + l32 * RS + lc * 4) = make_float4(v[0], v[1], v[2], v[3]);
      }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the wave's own writes; no other wave reads them
    constexpr int CH = WN * ES / 16, RPI = 64 / CH, EPC = 16 / ES;
#pragma unroll
    for (int i = 0; i < 32 / RPI; ++i) {
      const int lr = i * RPI + lane / CH, lc = (lane % CH) * EPC, r = rbase + lr, c = cn + lc;
      const uint4 v = *reinterpret_cast<const uint4*>(my + lr * RS + lc * ES);
      if (r < g.M && c < g.N) {
        OutT* p = C + (int64_t)r * g.ldc + c;
        if (g.vec) {
          *reinterpret_cast<uint4*>(p) = v;
        } else {
          const OutT* e = reinterpret_cast<const OutT*>(&v);
#pragma unroll
          for (int k = 0; k < EPC; ++k)
            if (c + k < g.N) p[k] = e[k];
        }
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // read before the next 32 rows overwrite
  }
}

// out[M][N] = sum of ks slabs (+ bias) (+ out), 4 elements per thread
template <bool OB>
__global__ __launch_bounds__(256) void fp8_slabs_k(const float* __restrict__ part, void* __restrict__ out_, int64_t ldc,
                                                 int M, int N, int ks, const float* __restrict__ bias, int beta, int vec) {
  using OutT = std::conditional_t<OB, uint16_t, float>;
  OutT* out = (OutT*)out_;
  const int64_t total = (int64_t)M * N;
  for (int64_t i = (blockIdx.x * 256LL + threadIdx.x) * 4; i < total; i += gridDim.x * 1024LL) {
    if (vec) {   // N % 4 == 0: one row, 16-B aligned
      float4 s = *reinterpret_cast<const float4*>(part + i);
      for (int z = 1; z < ks; ++z) {
        const float4 x = *reinterpret_cast<const float4*>(part + z * total + i);
        s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w;
      }
      const int64_t r = i / N;
      const int c = (int)(i - r * N);
      float v[4] = {s.x, s.y, s.z, s.w};
      OutT* p = out + r * ldc + c;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (bias) v[k] += bias[c + k];
        if (beta) v[k] += hx::io<OutT>::ld(p + k);
      }
      if constexpr (OB) *reinterpret_cast<uint2*>(p) = make_uint2(bf16x2(v[0], v[1]), bf16x2(v[2], v[3]));
      else *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
      for (int k = 0; k < 4 && i + k < total; ++k) {
        float s = part[i + k];
        for (int z = 1; z < ks; ++z) s += part[z * total + i + k];
        const int64_t r = (i + k) / N;
        const int c = (int)(i + k - r * N);
        OutT* p = out + r * ldc + c;
        if (bias) s += bias[c];
        if (beta) s += hx::io<OutT>::ld(p);
        hx::io<OutT>::st(p, s);
      }
    }
  }
}

template <int BM, int BN, int WM, int WN, int KS, int NS, int WGS, bool EXACT, bool OB>
int launch(const HxGemm8& g, hipStream_t s) {
  constexpr int NT = (BM / WM) * (BN / WN) * 64;
  constexpr int LDS = NS * (BM + BN) * KS + 6144;
  auto k = gemm_fp8_k<BM, BN, WM, WN, KS, NS, WGS, EXACT, OB>;
  static const hipError_t ok = hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
  if (ok != hipSuccess) return 1;
  const int64_t total = (int64_t)((g.M + BM - 1) / BM) * ((g.N + BN - 1) / BN) * g.ks;
  k<<<(unsigned)((total + 7) / 8 * 8), NT, LDS, s>>>(g);
  return hipGetLastError() == hipSuccess ? 0 : 1;
}
template <bool EXACT, bool OB>
int launch_cfg(const HxGemm8& g, int cfg, hipStream_t s) {
  switch (cfg) {
    case 0: return launch<256, 128, 128, 64, 64, 3, 2, EXACT, OB>(g, s);
    case 1: return launch<128, 128, 64, 64, 128, 2, 2, EXACT, OB>(g, s);
    case 2: return launch<64, 64, 32, 32, 128, 2, 4, EXACT, OB>(g, s);
  }
  return 1;
}
constexpr int kBM[3] = {256, 128, 64}, kBN[3] = {128, 128, 64};

}  // namespace

// the tile: the largest whose tiles give every CU one (a larger tile reads less LDS and L2 per product)
int hx_gemm_fp8_plan(int M, int N) {
  for (int c = 0; c < 2; ++c)
    if ((int64_t)((M + kBM[c] - 1) / kBM[c]) * ((N + kBN[c] - 1) / kBN[c]) >= hx_cu_slots()) return c;
  return 2;
}
// split-K slabs: as many as keep one workgroup per CU, of at least 4 scale groups (2048 deep)
int hx_gemm_fp8_ks(int M, int N, int nkb, int cfg) {
  const int64_t tiles = (int64_t)((M + kBM[cfg] - 1) / kBM[cfg]) * ((N + kBN[cfg] - 1) / kBN[cfg]);
  const int groups = (nkb + 3) / 4;
  const int ks = (int)std::min<int64_t>(hx_cu_slots() / std::max<int64_t>(tiles, 1), groups / 4);
  return std::max(ks, 1);
}

int hx_gemm_fp8(const HxGemm8& g, int cfg, int exact, int out_bf16, hipStream_t s) {
  if (out_bf16) return exact ? launch_cfg<true, true>(g, cfg, s) : launch_cfg<false, true>(g, cfg, s);
  return exact ? launch_cfg<true, false>(g, cfg, s) : launch_cfg<false, false>(g, cfg, s);
}

void hx_gemm_fp8_slabs(const float* part, void* out, int out_bf16, int64_t ldc, int M, int N, int ks, const float* bias,
                       int beta, int vec, hipStream_t s) {
  const unsigned grid = (unsigned)std::min<int64_t>(((int64_t)M * N + 1023) / 1024, 4096);
  if (out_bf16) fp8_slabs_k<true><<<grid, 256, 0, s>>>(part, out, ldc, M, N, ks, bias, beta, vec);
  else fp8_slabs_k<false><<<grid, 256, 0, s>>>(part, out, ldc, M, N, ks, bias, beta, vec);
}
