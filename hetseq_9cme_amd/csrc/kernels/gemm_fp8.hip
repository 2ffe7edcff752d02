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
//    vector instruction at all for the scaling).  The instruction sums 8 consecutive products at a time
//    and cuts each of them, towards zero, at 2^-13 of the largest 2^(ea + eb) among the 8 (ea, eb: the
//    codes' exponents); the sums of 8 are added in fp32.  That is 1.3e-5 (normal data) to 6e-5 (widths spread
//    over decades) of a result in the mean, whatever the depth -- 1/300 to 1/65 of half a bf16 step, so it
//    carries every product whose result is rounded to bf16 -- and, for codes that are not subnormal, at most
//    2^-10 of sum |a||b|.
//  * exact: the codes decoded to bf16 with their scale (v_cvt_scalef32_pk_bf16_fp8, exact) after the
//    LDS read, and v_mfma_f32_32x32x16_bf16, which sums exact products in fp32 (1e-7): the products
//    whose result is kept in fp32 (weight gradients, fp32 activations).  Half the matrix rate, and a
//    decoding instruction (half rate itself) for every 4 codes of a fragment.
//
// Measured alone, calls back to back (M x K x N, us, TFLOP/s): 16384 x 4096 x 1024 56, 2440; 16384 x 1024 x 4096 77,
// 1780 and 8192 x 1024 x 4096 41, 1690 (134 and 67 MB of results); 16384 x 2304 x 768 31, 1855; exact: 8192 x 1024
// x 4096 75, 920; with its slab sums 1024 x 16384 x 4096 119 .. 124, 1110 .. 1156 and 2304 x 16384 x 768 65 .. 67, 860 .. 900;
// 1312 x 768 x 768 5.8.  The library's e4m3 and bf16 products of 8192^3 run at 2600 and 1150.
#include <algorithm>
#include <atomic>

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

// a wave-uniform descriptor chosen from two, kept in scalar registers
__device__ __forceinline__ u32x4 pick(bool first, const u32x4& a, const u32x4& b) {
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = __builtin_amdgcn_readfirstlane(first ? a[i] : b[i]);
  return r;
}

__device__ __forceinline__ void raw_barrier() { asm volatile("s_barrier" ::: "memory"); }

// 8 codes (two words of a fragment) -> bf16 values times s
__device__ __forceinline__ bf16x8v decode8(int w0, int w1, float s) {
  const bf16x2v a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, s, false);
  const bf16x2v b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, s, true);
  const bf16x2v c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, s, false);
  const bf16x2v d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, s, true);
  return bf16x8v{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// C[M][N] in tiles of BM x BN, (BM / WM)(BN / WN) waves of WM x WN, one k block (128 codes of every row)
// per stage, two stages of LDS.  Persistent: a workgroup takes the tiles (and slabs) of its XCD's share
// in turn, and its streams of stages, scale words and biases run on from one tile into the next, so the
// first loads of a tile are under way while the one before it is stored.
//
// The 256 x 256 tile's 128 accumulators and fragments leave it short of registers: 8 (bf16 results), 6 (fp32 slabs) and
// 33 (exact) are spilled, outside the main loop, and read back in the epilogue.  Where result rows are not 16-B aligned (g.vec = 0)
// those reads lie between the stores and each waits for the stores before it, and a store's 16 B may cross lines: 8192 x
// 1024 x 4097 takes 72 us (exact 92) where x 4096 takes 41 (75), 16384 x 4096 x 1023 66 where x 1024 takes 56.
//
// A k block is two 64-deep halves: while the MFMAs of one run on fragments in registers, the fragments
// of the next are read.  A stage is opened (`open`) by a counted vmcnt and one raw barrier, which also
// frees the stage before it for the next DMA.
template <int BM, int BN, int WM, int WN, int WGS, bool EXACT, bool OB>
__global__ __launch_bounds__((BM / WM) * (BN / WN) * 64, (BM / WM) * (BN / WN) * WGS / 4) void gemm_fp8_k(HxGemm8 g) {
  constexpr int NWM = BM / WM, NWN = BN / WN, NW = NWM * NWN;
  constexpr int MB = WM / 32, NB = WN / 32;
  constexpr int KA = BM / 8, KB = BN / 8, J = (KA + KB) / NW;   // 1-KiB DMA pieces (8 rows) per stage; per wave
  static_assert((KA + KB) % NW == 0, "whole DMA pieces per wave");
  static_assert(BM <= 256 && BN <= 256 && NW >= 3, "one DMA piece of scale words per operand");
  // LDS: two stages, two slots of scale words (A 1 KiB, B 1 KiB; one word = 4 k blocks of a row), the
  // biases of three tiles, and where idle DMA pieces land.  Tile i's bias lies in slot i % 3.  It is fetched
  // in tile i - 1, of up to 4 k blocks before that tile's first barrier, when a slower wave may still be
  // reading the bias of tile i - 2 in its epilogue: two slots would give it tile i's.  The slot's tile before,
  // i - 3, was read by every wave before the barriers of tile i - 2.
  constexpr int STAGE = (BM + BN) * 128, SCALES = 2 * STAGE, BIAS = SCALES + 4096, SPARE = BIAS + 3 * 1024;
  constexpr int STORES = MB * NB * (OB ? 2 : 4);   // of a lane in the epilogue
  static_assert(STORES < 63, "counted by vmcnt");
  extern __shared__ __attribute__((aligned(16))) char lds[];

  const int TM = (g.M + BM - 1) / BM, TN = (g.N + BN - 1) / BN, tiles = TM * TN;
  // work items (slab, tile) dealt XCD by XCD: items [x per, x per + per) to the workgroups of XCD x
  const int per = (tiles * g.ks + 7) / 8, step = gridDim.x / 8;
  const int first = (blockIdx.x % 8) * per + blockIdx.x / 8;
  const int end = min((int)(blockIdx.x % 8) * per + per, tiles * g.ks);
  if (first >= end) return;   // uniform per workgroup
  // k blocks of a slab: whole groups of four
  const int groups = (g.nkb + 3) / 4, gper = (groups + g.ks - 1) / g.ks;
  struct Item {
    int m0, n0, z, kb0, n;
  };
  auto item = [&](int w) {
    Item t;
    t.z = w / tiles;
    const int r = w - t.z * tiles;
    t.m0 = r / TN * BM;
    t.n0 = (r - r / TN * TN) * BN;
    t.kb0 = t.z * gper * 4;
    t.n = min(gper * 4, g.nkb - t.kb0);   // >= 1: the plan makes no empty slab
    return t;
  };

  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wv % NWM, wn = wv / NWM, h = lane >> 5, l32 = lane & 31;
  const int64_t sam = (g.M + 3) & ~3, sbn = (g.N + 3) & ~3;
  const uint32_t lds0 = (uint32_t)(size_t)(lds_void*)lds;
  constexpr uint32_t NONE = 0x80000000u;   // an offset past every buffer: zeros, no memory traffic, still counted

  // Lane L of a DMA piece fetches 16-B chunk L % 8 ^ swz of row L / 8 so that the
  // lane-linear LDS write lands chunk c of row r at position c ^ (r / 2 % 8): fragment reads are free of
  // bank conflicts
  uint32_t voff[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int q = wv + NW * j, r = (q < KA ? q : q - KA) * 8 + lane / 8;
    voff[j] = (uint32_t)(r * (q < KA ? g.lda : g.ldb) + 16 * ((lane % 8) ^ ((r >> 1) & 7)));
  }
  // what a tile's DMA needs; `next` is the tile after the one in work (its loads start two stages early)
  struct Src {
    u32x4 a, b, x;   // A's and B's rows; wave 0: scale words of A's rows, wave 1: of B's, wave 2: the bias
    uint32_t ko, so;   // byte offsets of the first k block in a row, of the first scale words (NONE: no such tile)
  };
  auto source = [&](const Item& t, bool some) {
    Src s;
    s.a = rsrc_of(g.A + (int64_t)t.m0 * g.lda, (uint32_t)(min(BM, g.M - t.m0) * g.lda));
    s.b = rsrc_of(g.B + (int64_t)t.n0 * g.ldb, (uint32_t)(min(BN, g.N - t.n0) * g.ldb));
    const char* p = (const char*)(wv == 0 ? (const void*)(g.sa + t.m0) : wv == 1 ? (const void*)(g.sb + t.n0) : (const void*)(g.bias + t.n0));
    const uint32_t bytes = wv == 0 ? (uint32_t)((groups * sam - t.m0) * 4) : wv == 1 ? (uint32_t)((groups * sbn - t.n0) * 4)
                           : wv == 2 && g.bias ? (uint32_t)(g.N - t.n0) * 4 : 0u;
    s.x = rsrc_of(p, bytes);
    s.ko = some ? (uint32_t)t.kb0 * 128u : NONE;
    s.so = !some ? NONE : wv < 2 ? (uint32_t)((t.kb0 >> 2) * (wv == 0 ? sam : sbn) * 4) : 0u;
    return s;
  };
  auto dma_one = [&](const u32x4& a, const u32x4& b, uint32_t ko, int slot, int j) {
    const int q = wv + NW * j;
    dma16(pick(q < KA, a, b), lds0 + (uint32_t)slot * STAGE + 1024u * q, voff[j] + ko);
  };
  // the scale words of k blocks 4 grp .. + 3 of a tile, and with its first ones the bias
  auto dma_scales = [&](const u32x4& x, uint32_t so, int grp, int slot, int bslot) {
    const uint32_t dst = wv < 2 ? SCALES + slot * 2048 + wv * 1024 : wv == 2 && grp == 0 ? BIAS + bslot * 1024 : (uint32_t)SPARE;
    const uint32_t off = wv < 2 ? so + (uint32_t)(grp * (wv == 0 ? sam : sbn) * 4) : wv == 2 && grp == 0 ? so : NONE;
    dma16(pick(true, x, x), lds0 + dst, off + 16 * lane);
  };

  f32x16 acc[MB][NB];
  auto frag = [&](const char* st, int row, int half) {
    const int r = row + l32;
    const char* p = st + r * 128;
    const int sw = (r >> 1) & 7;
    const i32x4 lo = *reinterpret_cast<const i32x4*>(p + 16 * ((4 * half + h) ^ sw));
    const i32x4 hi = *reinterpret_cast<const i32x4*>(p + 16 * ((4 * half + 2 + h) ^ sw));
    return i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  };
  i32x8 fa[MB], fb[2][NB];   // A's fragments are read again as soon as their MFMAs are issued, B's by turns
  auto read_a = [&](int slot, int half, int a) { fa[a] = frag(lds + slot * STAGE, wm * WM + 32 * a, half); };
  auto read_b = [&](int slot, int half, i32x8 (&f)[NB]) {
#pragma unroll
    for (int b = 0; b < NB; ++b) f[b] = frag(lds + slot * STAGE + BM * 128, wn * WN + 32 * b, half);
  };
  uint32_t wa[MB], wb[NB];   // scale words, the current block's byte lowest
  auto read_scales = [&](int slot) {
    const uint32_t* p = reinterpret_cast<const uint32_t*>(lds + SCALES + slot * 2048);
#pragma unroll
    for (int a = 0; a < MB; ++a) wa[a] = p[wm * WM + 32 * a + l32];
#pragma unroll
    for (int b = 0; b < NB; ++b) wb[b] = p[256 + wn * WN + 32 * b + l32];
  };
  auto open = [&](uint32_t stores) {   // the next stage readable by every wave, the one before it free
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    // its DMA is the oldest in flight; in a tile's first block the tile before it may still be storing
    // (in one asm block: a branch that the compiler sees splits the MFMA sequence, which costs registers)
    asm volatile("s_cmp_lg_u32 %0, 0\n\ts_cbranch_scc1 .Lopen%=\n\ts_waitcnt vmcnt(0)\n.Lopen%=:\n\ts_waitcnt vmcnt(%1)"
                 ::"s"(__builtin_amdgcn_readfirstlane(stores)), "n"(STORES) : "memory", "scc");
    raw_barrier();
  };
  // The MFMAs of one half, and between them the reads of the next half's fragments (OPEN: of the next
  // stage, and the DMA pieces of the stage after it) -- one after the other as written: a wave that
  // issued its reads first would hold its MFMAs back until the LDS had served all waves' reads.  The
  // stage is opened under the first MFMAs.
  // Rows of the result run along n (the first MFMA operand): a lane holds 4 consecutive columns.
  auto half_step = [&](const i32x8 (&bc)[NB], i32x8 (&bn)[NB], int slot, auto open_it, uint32_t stores, const u32x4& sa_, const u32x4& sb_,
                       uint32_t ko) {
    constexpr bool OPEN = decltype(open_it)::value;
    const int ns = OPEN ? slot ^ 1 : slot, half = OPEN ? 0 : 1;
    bf16x8v db[4][NB];
    if constexpr (EXACT)
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int b = 0; b < NB; ++b) db[q][b] = decode8(bc[b][2 * q], bc[b][2 * q + 1], hx::q8::scale_of(wb[b] & 0xffu));
#pragma unroll
    for (int a = 0; a < MB; ++a) {
      if constexpr (!EXACT) {
#pragma unroll
        for (int b = 0; b < NB; ++b)
          acc[a][b] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(bc[b], fa[a], acc[a][b], 0, 0, 0, wb[b], 0, wa[a]);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const bf16x8v da = decode8(fa[a][2 * q], fa[a][2 * q + 1], hx::q8::scale_of(wa[a] & 0xffu));
#pragma unroll
          for (int b = 0; b < NB; ++b) acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(db[q][b], da, acc[a][b], 0, 0, 0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      if (a == 0) {
        if constexpr (OPEN) open(stores);
        read_b(ns, half, bn);
      }
      read_a(ns, half, a);
      if constexpr (OPEN)
#pragma unroll
        for (int j = 0; j < J; ++j)
          if (j * MB / J == a) dma_one(sa_, sb_, ko, slot, j);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  // ---- epilogue: a lane holds 4 consecutive columns of a row per quad of registers, the other half wave
  // the next 4; bf16 quads change places in pairs so that every store is 16 B per lane
  using OutT = std::conditional_t<OB, uint16_t, float>;
  constexpr int ST = OB ? 2 : 4;   // stores of a 32 x 32 block
  auto store = [&](const Item& t, int bslot_) {
    constexpr int ES = sizeof(OutT), PER = 16 / ES;
    OutT* C = (OutT*)g.C + (int64_t)t.z * g.c_zs + (int64_t)t.m0 * g.ldc + t.n0;
    const hx::Buf rc(C, g.vec ? (uint32_t)((min(BM, g.M - t.m0) * g.ldc - t.n0) * ES) : 0u);
    const int srow = wm * WM + (lane & 15), scol = wn * WN + PER * (((lane >> 4) & 1) * 2 + h);
    const uint32_t so = (uint32_t)((srow * g.ldc + scol) * ES);
    const float* bias = reinterpret_cast<const float*>(lds + BIAS + bslot_ * 1024);
#pragma unroll
    for (int a = 0; a < MB; ++a) {
      const int lr = wm * WM + 32 * a + l32;
      const bool in = t.m0 + lr < g.M;
      const OutT* row = C + (int64_t)lr * g.ldc - t.n0;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        float v[4][4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int lc = wn * WN + 32 * b + 8 * q + 4 * h, c = t.n0 + lc;
          float4 bb = make_float4(0.f, 0.f, 0.f, 0.f);
          if (g.bias) bb = *reinterpret_cast<const float4*>(bias + lc);
          v[q][0] = acc[a][b][4 * q] + bb.x;
          v[q][1] = acc[a][b][4 * q + 1] + bb.y;
          v[q][2] = acc[a][b][4 * q + 2] + bb.z;
          v[q][3] = acc[a][b][4 * q + 3] + bb.w;
          if (g.beta && in) {
            if (g.vec) {
              if (c < g.N) {
                if constexpr (OB) {
                  const uint2 w = *reinterpret_cast<const uint2*>(row + c);
                  v[q][0] += __uint_as_float(w.x << 16); v[q][1] += __uint_as_float(w.x & 0xffff0000u);
                  v[q][2] += __uint_as_float(w.y << 16); v[q][3] += __uint_as_float(w.y & 0xffff0000u);
                } else {
                  const float4 w = *reinterpret_cast<const float4*>(row + c);
                  v[q][0] += w.x; v[q][1] += w.y; v[q][2] += w.z; v[q][3] += w.w;
                }
              }
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (c + i < g.N) v[q][i] += hx::io<OutT>::ld(row + c + i);
            }
          }
        }
        // A store: 16 rows, 4 lanes of 16 B to a row.  (The products leave 32 rows of 32 B to a store; groups
        // of 16 lanes change places between the registers of two.  Whole 64-B pieces of a line: 8192 x 1024
        // x 4096 38.0 -> 36.4 us, 16384 x 1024 x 4096 71.0 -> 67.4.)
        uint32_t w[ST][4];   // store s: 16 B a lane
        if constexpr (OB) {
#pragma unroll
          for (int q = 0; q < 4; q += 2) {   // columns 8 q + 8 h .. + 8 after the exchange
            const auto x = __builtin_amdgcn_permlane32_swap(bf16x2(v[q][0], v[q][1]), bf16x2(v[q + 1][0], v[q + 1][1]), false, false);
            const auto y = __builtin_amdgcn_permlane32_swap(bf16x2(v[q][2], v[q][3]), bf16x2(v[q + 1][2], v[q + 1][3]), false, false);
            w[q / 2][0] = x[0]; w[q / 2][1] = y[0]; w[q / 2][2] = x[1]; w[q / 2][3] = y[1];
          }
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int i = 0; i < 4; ++i) w[q][i] = __float_as_uint(v[q][i]);
        }
#pragma unroll
        for (int s = 0; s < ST; s += 2)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const auto x = __builtin_amdgcn_permlane16_swap(w[s][i], w[s + 1][i], false, false);
            w[s][i] = x[0];
            w[s + 1][i] = x[1];
          }
#pragma unroll
        for (int s = 0; s < ST; ++s) {
          const int r = 32 * a + 16 * (s & 1), c = 32 * b + 2 * PER * (s & ~1);   // from srow, scol
          const bool ok = srow < g.M - t.m0 - r && scol < g.N - t.n0 - c;
          if (g.vec) {   // every lane of every store is issued (outside the result: dropped), so they can be counted
            __builtin_amdgcn_raw_buffer_store_b128(u32x4{w[s][0], w[s][1], w[s][2], w[s][3]}, rc.r, ok ? so : NONE,
                                                   (int)((r * g.ldc + c) * ES), 0);
          } else if (ok) {   // rows of any stride: 16 B at any element, and the last ones singly
            OutT* p = C + (srow + r) * g.ldc + scol + c;
            const int left = g.N - t.n0 - c - scol;
            if (left >= PER) {
              hx::q8::store16(p, u32x4{w[s][0], w[s][1], w[s][2], w[s][3]});
            } else {
#pragma unroll
              for (int i = 0; i < PER; ++i)
                if (i < left) {
                  if constexpr (OB) p[i] = (uint16_t)(w[s][i >> 1] >> (16 * (i & 1)));
                  else p[i] = __uint_as_float(w[s][i]);
                }
            }
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if (!g.vec) dma_wait<0>();   // stores that `open` does not count
  };

  Item t = item(first);
  Src src = source(t, true);
  bool more = first + step < end;
  Item u = item(more ? first + step : first);
  Src nxt = source(u, more);
  dma_scales(src.x, src.so, 0, 0, 0);
#pragma unroll
  for (int i = 0; i < 2; ++i) {   // (a tile of one block is its workgroup's only one: `launch`)
    const uint32_t ko = i < t.n ? src.ko + 128u * i : NONE;
#pragma unroll
    for (int j = 0; j < J; ++j) dma_one(src.a, src.b, ko, i, j);
  }
  dma_wait<J>();   // the first scale words and stage 0 landed
  raw_barrier();
  read_b(0, 0, fb[0]);
#pragma unroll
  for (int a = 0; a < MB; ++a) read_a(0, 0, a);
  int slot = 0, gslot = 0, tslot = 0;
  for (int w = first;;) {
#pragma unroll
    for (int a = 0; a < MB; ++a)
#pragma unroll
      for (int b = 0; b < NB; ++b) acc[a][b] = f32x16{0};
    for (int kb = 0; kb < t.n; ++kb) {
      if ((kb & 3) == 0) {
        read_scales(gslot);
        gslot ^= 1;
        const bool here = kb + 4 < t.n;
        dma_scales(pick(here, src.x, nxt.x), here ? src.so : nxt.so, here ? (kb >> 2) + 1 : 0, gslot, tslot == 2 ? 0 : tslot + 1);
      } else {
#pragma unroll
        for (int a = 0; a < MB; ++a) wa[a] >>= 8;
#pragma unroll
        for (int b = 0; b < NB; ++b) wb[b] >>= 8;
      }
      const int k2 = kb + 2 - t.n;   // the stage to fetch: of this tile, or block k2 (0, 1) of the next
      const bool here = k2 < 0;
      const uint32_t ko = here ? src.ko + 128u * (kb + 2) : more ? nxt.ko + 128u * k2 : NONE;
      half_step(fb[0], fb[1], slot, std::false_type{}, 0u, src.a, src.b, 0u);
      half_step(fb[1], fb[0], slot, std::true_type{}, (uint32_t)(kb == 0 && w != first), pick(here, src.a, nxt.a),
                pick(here, src.b, nxt.b), ko);
      slot ^= 1;
    }
    store(t, tslot);
    if (!more) break;
    w += step;
    tslot = tslot == 2 ? 0 : tslot + 1;
    t = u;
    src = nxt;
    more = w + step < end;
    u = item(more ? w + step : w);
    nxt = source(u, more);
  }
  dma_wait<0>();   // no DMA piece may land after the workgroup's LDS has been given away
}

// out[M][N] = sum of ks slabs (+ bias) (+ out), 4 elements per thread
template <bool OB>
__device__ __forceinline__ void sum_slabs(const HxSlabs& j, int64_t first, int64_t step) {
  using OutT = std::conditional_t<OB, uint16_t, float>;
  const float* part = j.part;
  OutT* out = (OutT*)j.out;
  const int64_t total = (int64_t)j.M * j.N;
  for (int64_t i = first * 4; i < total; i += step * 4) {
    if (j.vec) {   // N % 4 == 0: one row, 16-B aligned
      float4 s = *reinterpret_cast<const float4*>(part + i);
      for (int z = 1; z < j.ks; ++z) {
        const float4 x = *reinterpret_cast<const float4*>(part + z * total + i);
        s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w;
      }
      const int64_t r = i / j.N;
      const int c = (int)(i - r * j.N);
      float v[4] = {s.x, s.y, s.z, s.w};
      OutT* p = out + r * j.ldc + c;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (j.bias) v[k] += j.bias[c + k];
        if (j.beta) v[k] += hx::io<OutT>::ld(p + k);
      }
      if constexpr (OB) *reinterpret_cast<uint2*>(p) = make_uint2(bf16x2(v[0], v[1]), bf16x2(v[2], v[3]));
      else *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
      for (int k = 0; k < 4 && i + k < total; ++k) {
        float s = part[i + k];
        for (int z = 1; z < j.ks; ++z) s += part[z * total + i + k];
        const int64_t r = (i + k) / j.N;
        const int c = (int)(i + k - r * j.N);
        OutT* p = out + r * j.ldc + c;
        if (j.bias) s += j.bias[c];
        if (j.beta) s += hx::io<OutT>::ld(p);
        hx::io<OutT>::st(p, s);
      }
    }
  }
}

// What a layer's products leave to add up -- the slabs of up to two of them, and split8's column sums per
// row tile -- in one launch: the parts take workgroups [0, end[0]), [end[0], end[1]) and the rest.
// (Alone, the sums of a bias gradient take 4.9 us after 16384 x 2304.)
__global__ __launch_bounds__(256) void fp8_finish_k(HxFinish f) {
  __shared__ float red[8][32];
  const int bid = blockIdx.x;
  if (bid < f.end[1]) {
    const int i = bid >= f.end[0];
    const HxSlabs& j = f.slabs[i];
    const int64_t first = (int64_t)(bid - (i ? f.end[0] : 0)) * 256 + threadIdx.x, step = (int64_t)(f.end[i] - (i ? f.end[0] : 0)) * 256;
    if (j.bf16) sum_slabs<true>(j, first, step);
    else sum_slabs<false>(j, first, step);
    return;
  }
  const int c = (bid - f.end[1]) * 32 + (threadIdx.x & 31), w = threadIdx.x >> 5;
  float s = 0.f;
  if (c < f.cols) {
#pragma unroll 8
    for (int r = w; r < f.rows; r += 8) s += f.part[(int64_t)r * f.cols + c];
  }
  red[w][threadIdx.x & 31] = s;
  __syncthreads();
  if (w == 0 && c < f.cols) {
#pragma unroll
    for (int k = 1; k < 8; ++k) s += red[k][threadIdx.x];
    f.sum[c] = s;
  }
}

// ---------------------------------------------------------------- few rows
// y = Q(x) W^T (+ bias) of unquantised x, in one launch: 16 rows and 16 output features per workgroup, the k
// blocks dealt over its waves.  A wave reads its W codes straight into registers (32 B of a row per lane: a
// whole 128-B line per row), rounds its 32 x values per lane to e4m3 (the block's maximum is 4 lanes), runs
// both through exact bf16 MFMAs, and the waves' sums are added in LDS in wave order.  Bound by latency (one
// token through 768 x 2304: 1.8 MB of codes, 4.0 us; 41 rows through 1024 x 1024: 4.2) and, as rows are
// added, by the rounding, which every workgroup does for itself: groups of rows in one workgroup share the W
// codes but leave CUs idle (41 rows, 64 workgroups of 16 waves: 6.9 us).  Splitting the reduction inside
// the workgroup keeps up to 16 waves of loads in flight where a tile per wave would leave one.
template <typename T>
struct Row32;   // 32 consecutive values of a row, of which n are inside
template <>
struct Row32<float> {
  float v[32];
  __device__ void load(const float* p, int n) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float t[8];
      hx::q8::load_upto<float>(p + 8 * q, n - 8 * q, t);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[8 * q + i] = t[i];
    }
  }
  __device__ float at(int i) const { return v[i]; }
  __device__ uint32_t top() const {   // the largest magnitude's bits
    uint32_t a = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) a = max(a, __float_as_uint(v[i]) & 0x7fffffffu);
    return a;
  }
  __device__ uint32_t code(int j, float s) const { return hx::q8::e4m3x4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3], s); }
};
template <>
struct Row32<uint16_t> {
  uint32_t w[16];   // packed bf16 pairs
  __device__ void load(const uint16_t* p, int n) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int m = n - 8 * q;
      if (m >= 8) {
        const hx::q8::u32v4 t = hx::q8::load16(p + 8 * q);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[4 * q + i] = t[i];
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          w[4 * q + i] = (2 * i < m ? (uint32_t)p[8 * q + 2 * i] : 0u) | (2 * i + 1 < m ? (uint32_t)p[8 * q + 2 * i + 1] << 16 : 0u);
      }
    }
  }
  __device__ float at(int i) const { return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16); }
  __device__ uint32_t top() const {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    u16x2 m = __builtin_bit_cast(u16x2, w[0] & 0x7fff7fffu);
#pragma unroll
    for (int i = 1; i < 16; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu));
    return (uint32_t)max(m[0], m[1]) << 16;
  }
  __device__ uint32_t code(int j, float s) const { return hx::q8::e4m3x4(w[2 * j], w[2 * j + 1], s); }
};

template <typename T>
__global__ __launch_bounds__(1024) void fp8_rows_k(HxRows8 g) {
  __shared__ float red[16][256];   // a wave's sums
  const int nk = blockDim.x / 64;
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, h = lane >> 4;
  const int n0 = blockIdx.x * 16, n = n0 + l16, r0 = blockIdx.y * 16, r = r0 + l16;
  const int64_t sbn = (g.N + 3) & ~3;
  f32x4 acc = {0, 0, 0, 0};
  for (int kb = wv; kb < g.nkb; kb += nk) {
    const int k0 = kb * 128 + 32 * h;
    uint4 w0 = make_uint4(0, 0, 0, 0), w1 = w0;
    uint32_t sw = 0x7f7f7f7fu;
    if (n < g.N) {
      const uint4* p = reinterpret_cast<const uint4*>(g.B + (int64_t)n * g.ldb + k0);
      w0 = p[0];
      w1 = p[1];
      sw = g.sb[(kb >> 2) * sbn + n];
    }
    Row32<T> x;
    x.load((const T*)g.x + (int64_t)r * g.ldx + k0, r < g.M ? g.K - k0 : 0);
    const float ws = hx::q8::scale_of((sw >> (8 * (kb & 3))) & 0xffu);
    const uint32_t wc[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
    bf16x8v wd[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) wd[q] = decode8(wc[2 * q], wc[2 * q + 1], ws);
    uint32_t a = x.top();
    a = max(a, (uint32_t)__shfl_xor((int)a, 16, 64));
    a = max(a, (uint32_t)__shfl_xor((int)a, 32, 64));
    if (__builtin_expect(a >= 0x7f800000u, 0)) {   // something not finite (the row's 4 lanes agree): the maximum of the rest
      a = 0;
#pragma unroll
      for (int i = 0; i < 32; ++i) a = max(a, __float_as_uint(hx::q8::finite_abs(x.at(i))));
      a = max(a, (uint32_t)__shfl_xor((int)a, 16, 64));
      a = max(a, (uint32_t)__shfl_xor((int)a, 32, 64));
    }
    const float xs = hx::q8::exp2i(hx::q8::block_exp<hx::q8::E4M3>(__uint_as_float(a)));
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const bf16x8v xd = decode8((int)x.code(2 * q, xs), (int)x.code(2 * q + 1, xs), xs);
      acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wd[q], xd, acc, 0, 0, 0);
    }
  }
  *reinterpret_cast<f32x4*>(&red[wv][4 * lane]) = acc;
  __syncthreads();
  const int e = threadIdx.x;   // element e of the 16 x 16 block: lane e / 4, register e % 4
  if (e < 256) {
    float v = 0.f;
    for (int k = 0; k < nk; ++k) v += red[k][e];
    const int rr = r0 + ((e >> 2) & 15), c = n0 + 4 * (e >> 6) + (e & 3);
    if (rr < g.M && c < g.N) {
      if (g.bias) v += g.bias[c];
      hx::io<T>::st((T*)g.y + (int64_t)rr * g.N + c, v);
    }
  }
}

template <int BM, int BN, int WM, int WN, int WGS, bool EXACT, bool OB>
int launch(const HxGemm8& g, hipStream_t s) {
  constexpr int NT = (BM / WM) * (BN / WN) * 64;
  constexpr int LDS = 2 * (BM + BN) * 128 + 4096 + 3 * 1024 + 1024;   // stages, scale words, biases, spare
  auto k = gemm_fp8_k<BM, BN, WM, WN, WGS, EXACT, OB>;
  static std::atomic<uint64_t> allowed{0};   // devices on which the kernel may take this much LDS
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return 1;
  const uint64_t bit = 1ull << (dev & 63);
  if (!(allowed.load(std::memory_order_relaxed) & bit)) {
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, LDS) != hipSuccess) return 1;
    allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  const int64_t items = (int64_t)((g.M + BM - 1) / BM) * ((g.N + BN - 1) / BN) * g.ks;
  if (items > 0x7ffffff0) return 1;
  // one workgroup per item, at most what the CUs hold at a time -- but where an item is one k block, which
  // leaves no room for the next one's first two stages
  const int gper = ((g.nkb + 3) / 4 + g.ks - 1) / g.ks * 4, last = g.nkb - (g.ks - 1) * gper;
  if (last < 1) return 1;
  const int64_t all = (items + 7) / 8;
  const int64_t n = last < 2 ? all : std::min<int64_t>(all, std::max(hx_cu_slots() * WGS / 8, 1));
  k<<<(unsigned)(8 * n), NT, LDS, s>>>(g);
  return hipGetLastError() == hipSuccess ? 0 : 1;
}
template <bool EXACT, bool OB>
int launch_cfg(const HxGemm8& g, int cfg, hipStream_t s) {
  switch (cfg) {
    case 0: return launch<256, 256, 128, 64, 1, EXACT, OB>(g, s);
    case 1: return launch<256, 192, 64, 96, 1, EXACT, OB>(g, s);
    case 2: return launch<128, 128, 64, 64, 2, EXACT, OB>(g, s);
    case 3: return launch<64, 64, 32, 32, 4, EXACT, OB>(g, s);
  }
  return 1;
}
constexpr int kBM[4] = {256, 256, 128, 64}, kBN[4] = {256, 192, 128, 64};

// Time in us of a product whose busiest CU gets n tiles of nkb k blocks: f + f1 nkb + n (t + t1 nkb),
// fitted (non-negative least squares, 6 - 15 %) to 46 products of 128 .. 16384 tokens with the widths of
// BERT-base and BERT-large.  A k block of a 256 x 256 tile takes 1.1 us with every CU at work (3.9 PF;
// exact 2.2 us: 1.9 PF), which is the power limit: the instructions alone, on such data, run at 3.8 and
// 1.8 PF.  Each large tile pays 5 - 12 us of first loads and stores; 256 x 192 fits widths of 768 and
// 2304; the small tiles fill the chip with few rows.  The choice is on average 1 - 2 % from the best.
struct Cost {
  double f, f1, t, t1;
};
constexpr Cost kCost[2][4] = {{{0, 0, 6.3, 1.116}, {0, 0, 5.2, 1.0}, {0.67, 0, 1.78, 0.587}, {0.33, 0.153, 0.76, 0.197}},
                              {{0, 0, 12.6, 2.234}, {0, 0, 8.6, 1.826}, {1.05, 0, 2.55, 0.961}, {1.02, 0.152, 0.95, 0.31}}};

}  // namespace

// The tile and the number of split-K slabs with the least predicted time.  Slabs are whole scale groups
// (512 deep); their cost: a second launch (3 us) and fp32 slabs written and read at 8 bytes per ns.
void hx_gemm_fp8_plan(int M, int N, int nkb, int exact, int* cfg, int* ks) {
  const int slots = hx_cu_slots(), groups = (nkb + 3) / 4;
  double best = 1e30;
  *cfg = 3;
  *ks = 1;
  for (int c = 0; c < 4; ++c) {
    const int64_t tiles = (int64_t)((M + kBM[c] - 1) / kBM[c]) * ((N + kBN[c] - 1) / kBN[c]);
    for (int k = 1; k <= 16 && k <= groups; ++k) {
      const int per = (groups + k - 1) / k;
      if (k > 1 && (groups + per - 1) / per != k) continue;   // (an empty slab)
      const Cost& q = kCost[exact ? 1 : 0][c];
      const double n = (double)((tiles * k + slots - 1) / slots), kb = k == 1 ? nkb : 4.0 * per;
      double t = q.f + q.f1 * kb + n * (q.t + q.t1 * kb);
      if (k > 1) t += 3.0 + 8.0 * k * M * (double)N / 8e6;
      if (t < best) {
        best = t;
        *cfg = c;
        *ks = k;
      }
    }
  }
}

// Whether fp8_rows_k takes the product: its time grows with the 16 x 16 x 128 blocks of work, and with the depth
// (16 waves take it by turns); split8 and gemm_fp8_k, two launches, are 8 - 14 us at these sizes.  bf16, us here /
// there: 1 x 4096 x 1024 7.1 / 12.1, 100 x 768 x 768 4.6 / 9.0, 256 x 1024 x 1024 (8192 blocks) 8.0 / 10.1, 512 x 768 x 768 (9216) 9.8 /
// 9.4, 1 x 16384 x 1024 20 / 17; fp32: 256 x 768 x 768 (4608) 7.6 / 9.5, 128 x 768 x 2304 (6912) 11.0 / 9.8.
int hx_fp8_rows_fit(int64_t M, int64_t N, int64_t nkb, int bf16) {
  return nkb <= 64 && (M + 15) / 16 * ((N + 15) / 16) * nkb <= (bf16 ? 8192 : 5632);
}

int hx_fp8_rows(const HxRows8& g, int bf16, hipStream_t s) {
  if (g.M < 1 || g.M > 65535 * 16) return 1;   // (grid)
  const dim3 grid((unsigned)((g.N + 15) / 16), (unsigned)((g.M + 15) / 16));
  const unsigned nt = g.nkb > 8 ? 1024 : 512;   // waves that the k blocks keep busy
  if (bf16) fp8_rows_k<uint16_t><<<grid, nt, 0, s>>>(g);
  else fp8_rows_k<float><<<grid, nt, 0, s>>>(g);
  return 0;
}

int hx_gemm_fp8(const HxGemm8& g, int cfg, int exact, int out_bf16, hipStream_t s) {
  if (out_bf16) return exact ? 1 : launch_cfg<false, true>(g, cfg, s);   // (a bf16 result needs no exact sums)
  return exact ? launch_cfg<true, false>(g, cfg, s) : launch_cfg<false, false>(g, cfg, s);
}

void hx_fp8_finish(HxFinish f, hipStream_t s) {
  auto blocks = [](const HxSlabs& j) { return (int)std::min<int64_t>(((int64_t)j.M * j.N + 1023) / 1024, 4096); };
  f.end[0] = f.n > 0 ? blocks(f.slabs[0]) : 0;
  f.end[1] = f.end[0] + (f.n > 1 ? blocks(f.slabs[1]) : 0);
  const int grid = f.end[1] + (f.sum ? (f.cols + 31) / 32 : 0);
  if (grid > 0) fp8_finish_k<<<(unsigned)grid, 256, 0, s>>>(f);
}
