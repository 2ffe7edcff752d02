// 8-bit blocks (hx_quant.h): operands of the e4m3 products, and activations kept for the backward.
//
//  * split8      x [R, C] -> its e4m3 codes blocked along the columns (the operand of a product that
//                contracts over C) and / or its e4m3 codes blocked along the rows, transposed to
//                [C, R] (the operand of a product that contracts over R), and the column sums (a
//                bias gradient) -- one read of x.
//  * gelu8_fwd   out = gelu(y + b), and y kept as int8 blocks
//  * gelu8_bwd   dy = dout gelu'(y^ + b) with y^ decoded from the blocks, and the column sums of dy
//  * pack8 / unpack8   x <-> its int8 blocks
#include <type_traits>

#include "hx_launch.h"
#include "hx_quant.h"
#include "hx_reduce.h"

namespace {

using namespace hx;
using namespace hx::q8;
constexpr int NT = 256;

// ---------------------------------------------------------------- split8
// One 128 x 128 tile per workgroup of 512; thread t holds rows 4 (t / 16) .. + 4, columns 8 (t % 16) ..
// + 8: a wave reads 4 rows of 256 (bf16) or 512 B at a time, a row block's maximum is one DPP row of 16
// lanes, and the thread's 4 consecutive rows are 4 consecutive bytes of a transposed row.
// Bound by memory where there are many tiles (dy of 16384 x 2304 bf16: 152 MB read and written in 34 us,
// 4.4 TB/s; x of 16384 x 4096 with a 1024 x 4096 weight: 294 MB in 59 us, 5.0; a large copy runs at 5.1),
// by one tile's chain of loads, maxima and stores where there are few (1312 x 768: 6.5 us).  512 threads and
// 4 rows a thread: 256 threads of 8 rows took 44 us for the first of these and 12 for the last.
constexpr int SNT = 512, SR = 4;   // threads of a split8 workgroup, rows per thread
constexpr uint32_t kInf = 0x7f800000u;

// A thread's R x 8 values, their magnitudes as fp32 bits compared as integers (an infinity or NaN
// then shows as a maximum >= kInf, and the block's finite maximum is taken again), and their codes.
// One row's int8 codes come from one fma each: x 2^-e + 1.5 2^23 rounds to a whole number (nearest even),
// whose low byte is the code; a block with something not finite takes the careful path.
constexpr float kWhole = 12582912.f;   // 1.5 2^23
__device__ __forceinline__ uint32_t low_bytes(float a, float b, float c, float d) {
  const uint32_t ab = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x0c0c0400u);
  const uint32_t cd = __builtin_amdgcn_perm(__float_as_uint(d), __float_as_uint(c), 0x0c0c0400u);
  return __builtin_amdgcn_perm(cd, ab, 0x05040100u);
}

template <int R>
struct TileF32 {
  float v[R][8];
  __device__ void load(const void* x, int64_t at, int i, int n) { load_upto<float>((const float*)x + at, n, v[i]); }
  __device__ static uint32_t mag(float x) { return __float_as_uint(x) & 0x7fffffffu; }
  __device__ uint32_t row_max(int i) const {
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) m = max(m, mag(v[i][k]));
    return m;
  }
  __device__ void col_max(uint32_t (&m)[8]) const {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      m[k] = 0;
#pragma unroll
      for (int i = 0; i < R; ++i) m[k] = max(m[k], mag(v[i][k]));
    }
  }
  __device__ float at(int i, int k) const { return v[i][k]; }
  __device__ void set_row(int i, const float (&f)[8]) {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[i][k] = f[k];
  }
  __device__ uint2 row_codes(int i, float s) const {
    return make_uint2(e4m3x4(v[i][0], v[i][1], v[i][2], v[i][3], s), e4m3x4(v[i][4], v[i][5], v[i][6], v[i][7], s));
  }
  __device__ uint32_t col_codes(int k, float s) const { return e4m3x4(v[0][k], v[1][k], v[2][k], v[3][k], s); }
};

// the same on packed bf16 pairs (word j: columns 2 j, 2 j + 1)
template <int R>
struct TileBf16 {
  uint32_t w[R][4];
  __device__ void load(const void* x, int64_t at, int i, int n) {
    const uint16_t* p = (const uint16_t*)x + at;
    if (n >= 8) {
      const u32v4 a = load16(p);
      w[i][0] = a[0]; w[i][1] = a[1]; w[i][2] = a[2]; w[i][3] = a[3];
      return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      w[i][j] = (2 * j < n ? (uint32_t)p[2 * j] : 0u) | (2 * j + 1 < n ? (uint32_t)p[2 * j + 1] << 16 : 0u);
  }
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  __device__ static u16x2 mag2(uint32_t x) { return __builtin_bit_cast(u16x2, x & 0x7fff7fffu); }
  __device__ uint32_t row_max(int i) const {
    const u16x2 m = __builtin_elementwise_max(__builtin_elementwise_max(mag2(w[i][0]), mag2(w[i][1])),
                                              __builtin_elementwise_max(mag2(w[i][2]), mag2(w[i][3])));
    return (uint32_t)max(m[0], m[1]) << 16;
  }
  __device__ void col_max(uint32_t (&m)[8]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      u16x2 a = mag2(w[0][j]);
#pragma unroll
      for (int i = 1; i < R; ++i) a = __builtin_elementwise_max(a, mag2(w[i][j]));
      m[2 * j] = (uint32_t)a[0] << 16;
      m[2 * j + 1] = (uint32_t)a[1] << 16;
    }
  }
  __device__ void set_row(int i, const float (&f)[8]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) w[i][j] = bf16x2(f[2 * j], f[2 * j + 1]);
  }
  __device__ float at(int i, int k) const { return __uint_as_float(k & 1 ? w[i][k >> 1] & 0xffff0000u : w[i][k >> 1] << 16); }
  __device__ uint2 row_codes(int i, float s) const { return make_uint2(e4m3x4(w[i][0], w[i][1], s), e4m3x4(w[i][2], w[i][3], s)); }
  __device__ uint32_t col_codes(int k, float s) const {
    const uint32_t sel = k & 1 ? 0x07060302u : 0x05040100u;   // (row i, row i + 1) of column k as a pair
    return e4m3x4(__builtin_amdgcn_perm(w[1][k >> 1], w[0][k >> 1], sel), __builtin_amdgcn_perm(w[3][k >> 1], w[2][k >> 1], sel), s);
  }
};

template <typename T>
using Row8 = std::conditional_t<sizeof(T) == 4, TileF32<1>, TileBf16<1>>;
// a lane's 8 entries of a block (row i of 16 lanes) -> their int8 codes; e: the block's exponent
template <typename Row>
__device__ __forceinline__ uint2 int8_block(const Row& x, int i, int& e) {
  uint32_t m = max16u(x.row_max(i));
  if (__builtin_expect(m >= kInf, 0)) {   // (the 16 lanes agree)
    m = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) m = max(m, __float_as_uint(finite_abs(x.at(i, k))));
    e = block_exp<Int8>(__uint_as_float(max16u(m)));
    const float is = exp2i(-e);
    return make_uint2(int8x4(x.at(i, 0) * is, x.at(i, 1) * is, x.at(i, 2) * is, x.at(i, 3) * is),
                      int8x4(x.at(i, 4) * is, x.at(i, 5) * is, x.at(i, 6) * is, x.at(i, 7) * is));
  }
  e = block_exp<Int8>(__uint_as_float(m));
  const float is = exp2i(-e);
  float f[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) f[k] = fmaf(x.at(i, k), is, kWhole);
  return make_uint2(low_bytes(f[0], f[1], f[2], f[3]), low_bytes(f[4], f[5], f[6], f[7]));
}

struct Split8Lds {
  // transposed codes, 128 rows of 128 B; 16-B chunk ch of row c at ch ^ (c / 8 % 8): the writes of a
  // wave (16 columns, 8 apart, of one chunk) and the reads (8 chunks of a row) spread over the banks
  uint8_t tile[128 * 128];
  uint32_t redm[SNT / 64][128];
  float reds[SNT / 64][128];
};

// `Step`: what is done to a tile between its load and its codes (rows r0 .., columns c0 .. of a thread's);
// it may give the column sums of its own
struct NoStep {
  static constexpr bool sums = false;
  template <typename Tile>
  __device__ void operator()(Tile&, int, int, const HxSplit8&, float (&)[8]) const {}
};
template <typename Tile, typename Step = NoStep>
__device__ __forceinline__ void split8_tile(const HxSplit8& a, int bid, Split8Lds& lds, const Step& step = {}) {
  auto& tile = lds.tile;
  auto& redm = lds.redm;
  auto& reds = lds.reds;
  const int t = threadIdx.x, cg = t & 15, rg = t >> 4, w = t >> 6;
  const int nc = (a.C + 127) / 128;
  const int cb = bid % nc, rb = bid / nc;
  const int c0 = cb * 128 + 8 * cg, r0 = rb * 128 + SR * rg;
  const int64_t Rs = (a.R + 3) & ~3, Cs = (a.C + 3) & ~3;
  const int Cp = (a.C + 127) / 128 * 128, Rp = (a.R + 127) / 128 * 128;
  Tile x;
#pragma unroll
  for (int i = 0; i < SR; ++i) x.load(a.x, (int64_t)(r0 + i) * a.ld + c0, i, r0 + i < a.R ? a.C - c0 : 0);
  float own[8];
  step(x, r0, c0, a, own);
  if (a.q) {
#pragma unroll
    for (int i = 0; i < SR; ++i) {
      uint32_t m = max16u(x.row_max(i));
      if (__builtin_expect(m >= kInf, 0)) {   // (a row's 16 lanes agree)
        m = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) m = max(m, __float_as_uint(finite_abs(x.at(i, k))));
        m = max16u(m);
      }
      const int e = block_exp<E4M3>(__uint_as_float(m));
      if (r0 + i < a.R) {
        *reinterpret_cast<uint2*>(a.q + (int64_t)(r0 + i) * Cp + c0) = x.row_codes(i, exp2i(e));
        if (cg == 0) a.s[((cb >> 2) * Rs + r0 + i) * 4 + (cb & 3)] = (uint8_t)(e + 127);
      }
    }
  }
  if (!a.qt && !a.colpart) return;
  // column maxima and sums: the wave's four row groups by shuffles, the waves through LDS
  if (a.qt) {
    uint32_t m[8];
    x.col_max(m);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (__builtin_expect(m[k] >= kInf, 0)) {
        m[k] = 0;
#pragma unroll
        for (int i = 0; i < SR; ++i) m[k] = max(m[k], __float_as_uint(finite_abs(x.at(i, k))));
      }
      m[k] = max(m[k], (uint32_t)__shfl_xor((int)m[k], 16, 64));
      m[k] = max(m[k], (uint32_t)__shfl_xor((int)m[k], 32, 64));
    }
    if ((t & 63) < 16) {
      *reinterpret_cast<uint4*>(&redm[w][8 * cg]) = make_uint4(m[0], m[1], m[2], m[3]);
      *reinterpret_cast<uint4*>(&redm[w][8 * cg + 4]) = make_uint4(m[4], m[5], m[6], m[7]);
    }
  }
  if (a.colpart) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      float s = Step::sums ? own[k] : (x.at(0, k) + x.at(1, k)) + (x.at(2, k) + x.at(3, k));
      s += __shfl_xor(s, 16, 64);
      s += __shfl_xor(s, 32, 64);
      if ((t & 63) < 16) reds[w][8 * cg + k] = s;
    }
  }
  __syncthreads();
  if (a.colpart && t < 128 && cb * 128 + t < a.C) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < SNT / 64; ++k) s += reds[k][t];
    a.colpart[(int64_t)rb * a.C + cb * 128 + t] = s;
  }
  if (!a.qt) return;
  // one thread per column folds the waves' maxima into the column's exponent
  if (t < 128) {
    uint32_t m = redm[0][t];
#pragma unroll
    for (int k = 1; k < SNT / 64; ++k) m = max(m, redm[k][t]);
    const int e = block_exp<E4M3>(__uint_as_float(m));
    redm[0][t] = __float_as_uint(exp2i(e));
    if (cb * 128 + t < a.C) a.st[((rb >> 2) * Cs + cb * 128 + t) * 4 + (rb & 3)] = (uint8_t)(e + 127);
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const int c = 8 * cg + k;
    *reinterpret_cast<uint32_t*>(tile + c * 128 + 16 * ((rg >> 2) ^ (cg & 7)) + 4 * (rg & 3)) =
        x.col_codes(k, __uint_as_float(redm[0][c]));
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 128 * 8 / SNT; ++i) {   // 128 transposed rows of 8 x 16 B
    const int c = SNT / 8 * i + (t >> 3), ch = t & 7;
    if (cb * 128 + c < a.C)
      *reinterpret_cast<uint4*>(a.qt + (int64_t)(cb * 128 + c) * Rp + rb * 128 + 16 * ch) =
          *reinterpret_cast<const uint4*>(tile + c * 128 + 16 * (ch ^ ((c >> 3) & 7)));
  }
}

__device__ __forceinline__ int split8_tiles(const HxSplit8& a) { return ((a.C + 127) / 128) * ((a.R + 127) / 128); }

// the tiles of a, then those of b (TB = void: a alone)
template <typename TA, typename TB>
__global__ __launch_bounds__(SNT) void split8_k(HxSplit8 a, HxSplit8 b) {
  __shared__ __attribute__((aligned(16))) Split8Lds lds;
  if constexpr (std::is_same_v<TB, void>) {
    split8_tile<TA>(a, blockIdx.x, lds);
  } else {
    const int na = split8_tiles(a);   // uniform over the workgroup
    if ((int)blockIdx.x < na) split8_tile<TA>(a, blockIdx.x, lds);
    else split8_tile<TB>(b, blockIdx.x - na, lds);
  }
}

// every weight of an encoder at once (ops.fp8_weights): one launch per forward instead of one per layer
__global__ __launch_bounds__(SNT) void split8_many_k(HxSplit8Batch d) {
  __shared__ __attribute__((aligned(16))) Split8Lds lds;
  int i = 0;
  while (i + 1 < d.n && (int)blockIdx.x >= d.start[i + 1]) ++i;   // uniform over the workgroup
  const HxSplit8 a{0, d.W[i], d.C[i], d.R[i], d.C[i], d.q[i], d.s[i], d.qt[i], d.st[i], nullptr};
  split8_tile<TileF32<SR>>(a, blockIdx.x - d.start[i], lds);
}

// ---------------------------------------------------------------- bias + GELU with an int8 checkpoint
// gelu(u) = u Phi(u), Phi(u) = (1 + erf(z)) / 2 with z = u / 1.41421 (the model's truncated constant).
// erfc by Abramowitz & Stegun 7.1.26 (a degree-5 polynomial in 1 / (1 + p |z|) times exp(-z^2), error at
// most 1.5e-7), its constants taken with u: the exponential is the derivative's too.  Both directions move
// 5 bytes per bf16 element; 16384 x 4096 takes 69 us forward (4.9 TB/s; a large copy runs at 5.1) and 74
// us back (4.5: the derivative's arithmetic on what int8 decodes to takes what is left), 41 x 4096 3.2 and 5.2.
// Back, a workgroup takes 128 columns of kRowChunk rows: 512 columns at a time left 41 rows with 8
// workgroups (11 us); every row loaded before the first is used took 87 us (registers).
struct Gelu {
  float cdf, bell;   // Phi(u), exp(-z^2)
};
__device__ __forceinline__ Gelu gelu_parts(float u) {
  constexpr float ic = 1.0f / 1.41421f;
  const float t = __builtin_amdgcn_rcpf(fmaf(fabsf(u), 0.3275911f * ic, 1.0f));
  const float bell = __builtin_amdgcn_exp2f(u * u * (-1.4426950408889634f * ic * ic));
  float p = fmaf(0.5f * 1.061405429f, t, 0.5f * -1.453152027f);
  p = fmaf(p, t, 0.5f * 1.421413741f);
  p = fmaf(p, t, 0.5f * -0.284496736f);
  p = fmaf(p, t, 0.5f * 0.254829592f);
  const float half = p * t * bell;   // erfc(|z|) / 2
  return {u >= 0.f ? 1.0f - half : half, bell};
}

// codes [rows][nb][128], scale bytes [rows][nb]; 16 lanes per block, 8 elements per lane
template <typename T>
__global__ __launch_bounds__(NT) void gelu8_fwd_k(const T* __restrict__ y, const float* __restrict__ b,
                                                T* __restrict__ out, uint8_t* __restrict__ q, uint8_t* __restrict__ s,
                                                int64_t nblk, int nb, int N) {
  const int l16 = threadIdx.x & 15;
  for (int64_t i = (blockIdx.x * (int64_t)NT + threadIdx.x) >> 4; i < nblk; i += (int64_t)gridDim.x * (NT / 16)) {
    const int64_t r = i / nb;
    const int c0 = (int)(i - r * nb) * 128 + 8 * l16, n = N - c0;
    Row8<T> x;
    x.load(y, r * N + c0, 0, n);
    if (q) {   // (null: no backward)
      int e;
      *reinterpret_cast<uint2*>(q + i * 128 + 8 * l16) = int8_block(x, 0, e);
      if (l16 == 0) s[i] = (uint8_t)(e + 127);
    }
    float v[8], bb[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) bb[k] = 0.f;
    if (b) load_upto<float>(b + c0, n, bb);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float u = x.at(0, k) + bb[k];
      v[k] = u * gelu_parts(u).cdf;
    }
    store_upto<T>(out + r * N + c0, n, v);
  }
}

// a workgroup: one block column (128 columns), kRowChunk rows, 16 rows at a time
template <typename T>
__global__ __launch_bounds__(NT) void gelu8_bwd_k(const T* __restrict__ dout, const uint8_t* __restrict__ q,
                                                const uint8_t* __restrict__ s, const float* __restrict__ b,
                                                T* __restrict__ dy, float* __restrict__ partial, int64_t rows, int nb, int N) {
  __shared__ float red[16][128];
  const int l16 = threadIdx.x & 15, rg = threadIdx.x >> 4;
  const int cb = blockIdx.x % nb, chunk = blockIdx.x / nb, c0 = cb * 128 + 8 * l16, n = N - c0;
  const int64_t r1 = min((int64_t)(chunk + 1) * kRowChunk, rows);
  float bb[8], sum[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) bb[k] = sum[k] = 0.f;
  if (b) load_upto<float>(b + c0, n, bb);
  for (int64_t r = (int64_t)chunk * kRowChunk + rg; r < r1; r += 16) {
    const int64_t i = r * nb + cb;
    float d[8];
    load_upto<T>(dout + r * N + c0, n, d);
    const uint2 w = *reinterpret_cast<const uint2*>(q + i * 128 + 8 * l16);
    float yv[8];
    int8_vals(w, scale_of(s[i]), yv);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float u = yv[k] + bb[k];
      const Gelu g = gelu_parts(u);
      // d/du u Phi(u) = Phi + u exp(-z^2) / (1.41421 sqrt(pi))
      d[k] *= fmaf(u * (0.5641895835477563f / 1.41421f), g.bell, g.cdf);
      sum[k] += d[k];
    }
    store_upto<T>(dy + r * N + c0, n, d);
  }
  if (!partial) return;
#pragma unroll
  for (int k = 0; k < 8; ++k) red[rg][8 * l16 + k] = sum[k];
  __syncthreads();
  if (threadIdx.x < 128 && cb * 128 + threadIdx.x < N) {
    float a = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) a += red[k][threadIdx.x];
    partial[(int64_t)chunk * N + cb * 128 + threadIdx.x] = a;
  }
}

// ---------------------------------------------------------------- GELU on the way to a product's operand
// Between the two products of a feed-forward layer the GELU's result is read by the second one only, and
// its input's gradient by the first one's gradient products only: they go straight to e4m3 codes (both
// blockings, as split8) and the tensors themselves are never written.  Same arithmetic, and the same
// rounding to T in between, as gelu8 and split8 one after the other: equal bits.  5 bytes per bf16 element
// each way where those move 9; 16384 x 4096 takes 91 us forward and 109 back in the layer (76 and 94 at best; fp32 100 and
// 141; bytes alone 66).  Vector instructions issue in 96 % of the forward's cycles (counted) and in 75 % of the backward's, whose
// waves wait for their two loads for half of their time; 64 registers for a fourth workgroup per CU spill and cost more (91 / 122
// where it was 87 / 114).
struct GeluStep {   // y -> gelu(y + b), y's int8 blocks kept (q null: not kept)
  static constexpr bool sums = false;
  const float* b;
  uint8_t *q, *s;
  template <typename Tile>
  __device__ void operator()(Tile& x, int r0, int c0, const HxSplit8& a, float (&)[8]) const {
    const int nb = (a.C + 127) / 128, l16 = threadIdx.x & 15;
    float bb[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) bb[k] = 0.f;
    if (b) load_upto<float>(b + c0, a.C - c0, bb);
#pragma unroll
    for (int i = 0; i < SR; ++i) {
      const bool in = r0 + i < a.R;
      if (q) {
        int e;
        const uint2 codes = int8_block(x, i, e);
        const int64_t blk = (int64_t)(r0 + i) * nb + c0 / 128;
        if (in) {
          *reinterpret_cast<uint2*>(q + blk * 128 + 8 * l16) = codes;
          if (l16 == 0) s[blk] = (uint8_t)(e + 127);
        }
      }
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float u = x.at(i, k) + bb[k];
        v[k] = in ? u * gelu_parts(u).cdf : 0.f;   // (columns past the last: gelu(0) = 0)
      }
      x.set_row(i, v);
    }
  }
};
struct GeluBackStep {   // dout -> dout gelu'(y^ + b), and its column sums (of the values before their rounding to T)
  static constexpr bool sums = true;
  const float* b;
  const uint8_t *q, *s;
  template <typename Tile>
  __device__ void operator()(Tile& x, int r0, int c0, const HxSplit8& a, float (&sum)[8]) const {
    const int nb = (a.C + 127) / 128, l16 = threadIdx.x & 15;
    uint2 w[SR];
    float sc[SR];
#pragma unroll
    for (int i = 0; i < SR; ++i) {
      const int64_t blk = (int64_t)(r0 + i) * nb + c0 / 128;
      const bool in = r0 + i < a.R;
      w[i] = in ? *reinterpret_cast<const uint2*>(q + blk * 128 + 8 * l16) : make_uint2(0, 0);
      sc[i] = in ? scale_of(s[blk]) : 1.f;
    }
    float bb[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) bb[k] = sum[k] = 0.f;
    if (b) load_upto<float>(b + c0, a.C - c0, bb);
#pragma unroll
    for (int i = 0; i < SR; ++i) {
      float d[8], yv[8];
      int8_vals(w[i], sc[i], yv);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float u = yv[k] + bb[k];
        const Gelu g = gelu_parts(u);
        d[k] = x.at(i, k) * fmaf(u * (0.5641895835477563f / 1.41421f), g.bell, g.cdf);
        sum[k] += d[k];
      }
      x.set_row(i, d);
    }
  }
};
template <typename Tile, typename Step>
__global__ __launch_bounds__(SNT) void gelu8_split_k(HxSplit8 a, Step step) {
  __shared__ __attribute__((aligned(16))) Split8Lds lds;
  split8_tile<Tile>(a, blockIdx.x, lds, step);
}

// ---------------------------------------------------------------- pack8 / unpack8
// One pass, 16 lanes to a block; bound by memory: 16384 x 1024 fp32 (84 MB) 15 us in and 16 back (5.2 - 5.8 TB/s, part
// of it from the last level cache), 1312 x 768 bf16 2.8 us.
template <typename T>
__global__ __launch_bounds__(NT) void pack8_k(const T* __restrict__ x, uint8_t* __restrict__ q, uint8_t* __restrict__ s,
                                            int64_t nblk, int nb, int N) {
  const int l16 = threadIdx.x & 15;
  for (int64_t i = (blockIdx.x * (int64_t)NT + threadIdx.x) >> 4; i < nblk; i += (int64_t)gridDim.x * (NT / 16)) {
    const int64_t r = i / nb;
    const int c0 = (int)(i - r * nb) * 128 + 8 * l16;
    Row8<T> v;
    v.load(x, r * N + c0, 0, N - c0);
    int e;
    *reinterpret_cast<uint2*>(q + i * 128 + 8 * l16) = int8_block(v, 0, e);
    if (l16 == 0) s[i] = (uint8_t)(e + 127);
  }
}

template <typename T>
__global__ __launch_bounds__(NT) void unpack8_k(const uint8_t* __restrict__ q, const uint8_t* __restrict__ s,
                                              T* __restrict__ x, int64_t nblk, int nb, int N) {
  const int l16 = threadIdx.x & 15;
  for (int64_t i = (blockIdx.x * (int64_t)NT + threadIdx.x) >> 4; i < nblk; i += (int64_t)gridDim.x * (NT / 16)) {
    const int64_t r = i / nb;
    const int c0 = (int)(i - r * nb) * 128 + 8 * l16;
    const uint2 w = *reinterpret_cast<const uint2*>(q + i * 128 + 8 * l16);
    float v[8];
    int8_vals(w, scale_of(s[i]), v);
    store_upto<T>(x + r * N + c0, N - c0, v);
  }
}

inline unsigned stream_grid(int64_t nblk) {   // one pass up to 16 workgroups per CU, then grid-stride
  const int64_t g = (nblk + NT / 16 - 1) / (NT / 16);
  return (unsigned)(g < 4096 ? g : 4096);
}

}  // namespace

int hx_split8_row_tiles(int64_t R) { return (int)((R + 127) / 128); }

void hx_split8(const HxSplit8* jobs, int n, hipStream_t stream) {
  auto tiles = [](const HxSplit8& j) { return (unsigned)(((j.C + 127) / 128) * (int64_t)((j.R + 127) / 128)); };
  const HxSplit8 &a = jobs[0], &b = jobs[n > 1 ? 1 : 0];
  if (n == 1) {
    if (a.bf16) split8_k<TileBf16<SR>, void><<<tiles(a), SNT, 0, stream>>>(a, b);
    else split8_k<TileF32<SR>, void><<<tiles(a), SNT, 0, stream>>>(a, b);
    return;
  }
  const unsigned grid = tiles(a) + tiles(b);
  if (a.bf16 && b.bf16) split8_k<TileBf16<SR>, TileBf16<SR>><<<grid, SNT, 0, stream>>>(a, b);
  else if (a.bf16) split8_k<TileBf16<SR>, TileF32<SR>><<<grid, SNT, 0, stream>>>(a, b);
  else if (b.bf16) split8_k<TileF32<SR>, TileBf16<SR>><<<grid, SNT, 0, stream>>>(a, b);
  else split8_k<TileF32<SR>, TileF32<SR>><<<grid, SNT, 0, stream>>>(a, b);
}

void hx_gelu8_split_fwd(const HxSplit8& a, const float* b, uint8_t* q, uint8_t* s, hipStream_t stream) {
  const unsigned grid = (unsigned)(((a.C + 127) / 128) * (int64_t)((a.R + 127) / 128));
  const GeluStep step{b, q, s};
  if (a.bf16) gelu8_split_k<TileBf16<SR>><<<grid, SNT, 0, stream>>>(a, step);
  else gelu8_split_k<TileF32<SR>><<<grid, SNT, 0, stream>>>(a, step);
}

void hx_gelu8_split_bwd(const HxSplit8& a, const float* b, const uint8_t* q, const uint8_t* s, hipStream_t stream) {
  const unsigned grid = (unsigned)(((a.C + 127) / 128) * (int64_t)((a.R + 127) / 128));
  const GeluBackStep step{b, q, s};
  if (a.bf16) gelu8_split_k<TileBf16<SR>><<<grid, SNT, 0, stream>>>(a, step);
  else gelu8_split_k<TileF32<SR>><<<grid, SNT, 0, stream>>>(a, step);
}

void hx_split8_many(const HxSplit8Batch& d, hipStream_t stream) {
  split8_many_k<<<d.start[d.n], SNT, 0, stream>>>(d);
}

void hx_gelu8_fwd(int bf16, const void* y, const float* b, void* out, uint8_t* q, uint8_t* s, int64_t rows, int N,
                  hipStream_t stream) {
  const int nb = (N + 127) / 128;
  const int64_t nblk = rows * nb;
  if (bf16) gelu8_fwd_k<uint16_t><<<stream_grid(nblk), NT, 0, stream>>>((const uint16_t*)y, b, (uint16_t*)out, q, s, nblk, nb, N);
  else gelu8_fwd_k<float><<<stream_grid(nblk), NT, 0, stream>>>((const float*)y, b, (float*)out, q, s, nblk, nb, N);
}

int hx_gelu8_chunks(int64_t rows) { return (int)((rows + kRowChunk - 1) / kRowChunk); }

void hx_gelu8_bwd(int bf16, const void* dout, const uint8_t* q, const uint8_t* s, const float* b, void* dy,
                  float* partial, float* db, int64_t rows, int N, hipStream_t stream) {
  const int nb = (N + 127) / 128;
  const unsigned grid = (unsigned)(nb * (int64_t)hx_gelu8_chunks(rows));
  if (bf16) gelu8_bwd_k<uint16_t><<<grid, NT, 0, stream>>>((const uint16_t*)dout, q, s, b, (uint16_t*)dy, partial, rows, nb, N);
  else gelu8_bwd_k<float><<<grid, NT, 0, stream>>>((const float*)dout, q, s, b, (float*)dy, partial, rows, nb, N);
  if (partial != db) fold_rows(partial, hx_gelu8_chunks(rows), N, N, N, db, nullptr, nullptr, 0, stream);
}

void hx_pack8(int bf16, const void* x, uint8_t* q, uint8_t* s, int64_t rows, int N, hipStream_t stream) {
  const int nb = (N + 127) / 128;
  const int64_t nblk = rows * nb;
  if (bf16) pack8_k<uint16_t><<<stream_grid(nblk), NT, 0, stream>>>((const uint16_t*)x, q, s, nblk, nb, N);
  else pack8_k<float><<<stream_grid(nblk), NT, 0, stream>>>((const float*)x, q, s, nblk, nb, N);
}

void hx_unpack8(int bf16, const uint8_t* q, const uint8_t* s, void* x, int64_t rows, int N, hipStream_t stream) {
  const int nb = (N + 127) / 128;
  const int64_t nblk = rows * nb;
  if (bf16) unpack8_k<uint16_t><<<stream_grid(nblk), NT, 0, stream>>>(q, s, (uint16_t*)x, nblk, nb, N);
  else unpack8_k<float><<<stream_grid(nblk), NT, 0, stream>>>(q, s, (float*)x, nblk, nb, N);
}
