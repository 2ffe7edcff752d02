// 8-bit blocks (hx_quant.h): operands of the e4m3 products, and activations kept for the backward.
//
//  * split8      x [R, C] -> its e4m3 codes blocked along the columns (the operand of a product that
//                contracts over C) and / or its e4m3 codes blocked along the rows, transposed to
//                [C, R] (the operand of a product that contracts over R), and the column sums (a
//                bias gradient) -- one read of x.
//  * gelu8_fwd   out = gelu(y + b), and y kept as int8 blocks
//  * gelu8_bwd   dy = dout gelu'(y^ + b) with y^ decoded from the blocks, and the column sums of dy
//  * pack8 / unpack8   x <-> its int8 blocks
#include "hx_launch.h"
#include "hx_quant.h"
#include "hx_reduce.h"

namespace {

using namespace hx;
using namespace hx::q8;
constexpr int NT = 256;

// ---------------------------------------------------------------- split8
// One 128 x 128 tile per workgroup; thread t holds rows 8 (t / 16) .. + 8, columns 8 (t % 16) .. + 8,
// so a wave reads 4 rows of 256 (bf16) or 512 B at a time, a row block's maximum is 16 lanes, and
// the thread's 8 consecutive rows are 8 consecutive bytes of a transposed row.
struct Split8 {
  const void* x;
  int64_t ld;
  int R, C;
  uint8_t* q;        // [R, Cp] codes blocked along the columns (null: not wanted), Cp = 128 ceil(C / 128)
  uint8_t* s;        // their scale bytes: block b of row r at ((b / 4) Rs + r) 4 + b % 4, Rs = R rounded up to 4
  uint8_t* qt;       // [C, Rp] codes blocked along the rows (null: not wanted)
  uint8_t* st;
  float* colpart;    // [row tiles][C] column sums (null: not wanted)
  int vec;
};

template <typename T>
__global__ __launch_bounds__(NT) void split8_k(Split8 a) {
  __shared__ __attribute__((aligned(16))) uint8_t tile[128 * 144];   // transposed codes, rows of 128 + 16
  __shared__ float redm[4][128], reds[4][128];
  const int t = threadIdx.x, cg = t & 15, rg = t >> 4, w = t >> 6;
  const int nc = (a.C + 127) / 128;
  const int cb = blockIdx.x % nc, rb = blockIdx.x / nc;
  const int c0 = cb * 128 + 8 * cg, r0 = rb * 128 + 8 * rg;
  const int64_t Rs = (a.R + 3) & ~3, Cs = (a.C + 3) & ~3;
  const int Cp = (a.C + 127) / 128 * 128, Rp = (a.R + 127) / 128 * 128;
  float v[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    load_upto<T>((const T*)a.x + (int64_t)(r0 + i) * a.ld + c0, r0 + i < a.R ? a.C - c0 : 0, a.vec, v[i]);
  if (a.q) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float m = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) m = fmaxf(m, finite_abs(v[i][k]));
      const int e = block_exp<E4M3>(max16(m));
      const float is = exp2i(-e);
      if (r0 + i < a.R) {
        const uint2 o = make_uint2(e4m3x4(v[i][0] * is, v[i][1] * is, v[i][2] * is, v[i][3] * is),
                                   e4m3x4(v[i][4] * is, v[i][5] * is, v[i][6] * is, v[i][7] * is));
        *reinterpret_cast<uint2*>(a.q + (int64_t)(r0 + i) * Cp + c0) = o;
        if (cg == 0) a.s[((cb >> 2) * Rs + r0 + i) * 4 + (cb & 3)] = (uint8_t)(e + 127);
      }
    }
  }
  if (!a.qt && !a.colpart) return;
  // column maxima and sums: the wave's four row groups by shuffles, the four waves through LDS
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    float m = 0.f, s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      m = fmaxf(m, finite_abs(v[i][k]));
      s += v[i][k];
    }
    m = fmaxf(m, __shfl_xor(m, 16, 64));
    m = fmaxf(m, __shfl_xor(m, 32, 64));
    s += __shfl_xor(s, 16, 64);
    s += __shfl_xor(s, 32, 64);
    if ((t & 63) < 16) {
      redm[w][8 * cg + k] = m;
      reds[w][8 * cg + k] = s;
    }
  }
  __syncthreads();
  if (a.colpart && t < 128 && cb * 128 + t < a.C)
    a.colpart[(int64_t)rb * a.C + cb * 128 + t] = (reds[0][t] + reds[1][t]) + (reds[2][t] + reds[3][t]);
  if (!a.qt) return;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const int c = 8 * cg + k;
    const int e = block_exp<E4M3>(fmaxf(fmaxf(redm[0][c], redm[1][c]), fmaxf(redm[2][c], redm[3][c])));
    const float is = exp2i(-e);
    *reinterpret_cast<uint2*>(tile + c * 144 + 8 * rg) =
        make_uint2(e4m3x4(v[0][k] * is, v[1][k] * is, v[2][k] * is, v[3][k] * is),
                   e4m3x4(v[4][k] * is, v[5][k] * is, v[6][k] * is, v[7][k] * is));
    if (rg == 0 && cb * 128 + c < a.C) a.st[((rb >> 2) * Cs + cb * 128 + c) * 4 + (rb & 3)] = (uint8_t)(e + 127);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {   // 128 transposed rows of 8 x 16 B
    const int c = 32 * i + (t >> 3), ch = t & 7;
    if (cb * 128 + c < a.C)
      *reinterpret_cast<uint4*>(a.qt + (int64_t)(cb * 128 + c) * Rp + rb * 128 + 16 * ch) =
          *reinterpret_cast<const uint4*>(tile + c * 144 + 16 * ch);
  }
}

// ---------------------------------------------------------------- bias + GELU with an int8 checkpoint
// gelu(u) = u Phi(u), Phi(u) = (1 + erf(z)) / 2 with z = u / 1.41421 (the model's truncated constant).
// erfc by Abramowitz & Stegun 7.1.26 (a degree-5 polynomial in 1 / (1 + p z) times exp(-z^2), error
// at most 1.5e-7): its exponential is the derivative's too.
struct Gelu {
  float cdf, bell;   // Phi(u), exp(-z^2)
};
__device__ __forceinline__ Gelu gelu_parts(float u) {
  const float z = u * (1.0f / 1.41421f);
  const float az = fabsf(z);
  const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f, az, 1.0f));
  const float bell = __expf(-z * z);
  float p = fmaf(1.061405429f, t, -1.453152027f);
  p = fmaf(p, t, 1.421413741f);
  p = fmaf(p, t, -0.284496736f);
  p = fmaf(p, t, 0.254829592f);
  const float half = 0.5f * p * t * bell;   // erfc(|z|) / 2
  return {z >= 0.f ? 1.0f - half : half, bell};
}

// codes [rows][nb][128], scale bytes [rows][nb]; 16 lanes per block, 8 elements per lane
template <typename T>
__global__ __launch_bounds__(NT) void gelu8_fwd_k(const T* __restrict__ y, const float* __restrict__ b,
                                                T* __restrict__ out, uint8_t* __restrict__ q, uint8_t* __restrict__ s,
                                                int64_t nblk, int nb, int N, int vec) {
  const int l16 = threadIdx.x & 15;
  for (int64_t i = (blockIdx.x * (int64_t)NT + threadIdx.x) >> 4; i < nblk; i += (int64_t)gridDim.x * (NT / 16)) {
    const int64_t r = i / nb;
    const int c0 = (int)(i - r * nb) * 128 + 8 * l16, n = N - c0;
    float v[8], bb[8];
    load_upto<T>(y + r * N + c0, n, vec, v);
    float m = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) m = fmaxf(m, finite_abs(v[k]));
    const int e = block_exp<Int8>(max16(m));
    const float is = exp2i(-e);
    *reinterpret_cast<uint2*>(q + i * 128 + 8 * l16) =
        make_uint2(int8x4(v[0] * is, v[1] * is, v[2] * is, v[3] * is), int8x4(v[4] * is, v[5] * is, v[6] * is, v[7] * is));
    if (l16 == 0) s[i] = (uint8_t)(e + 127);
#pragma unroll
    for (int k = 0; k < 8; ++k) bb[k] = 0.f;
    if (b) load_upto<float>(b + c0, n, vec, bb);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float u = v[k] + bb[k];
      v[k] = u * gelu_parts(u).cdf;
    }
    store_upto<T>(out + r * N + c0, n, vec, v);
  }
}

// a workgroup: one block column (128 columns), kRowChunk rows, 16 rows at a time
template <typename T>
__global__ __launch_bounds__(NT) void gelu8_bwd_k(const T* __restrict__ dout, const uint8_t* __restrict__ q,
                                                const uint8_t* __restrict__ s, const float* __restrict__ b,
                                                T* __restrict__ dy, float* __restrict__ partial, int64_t rows, int nb,
                                                int N, int vec) {
  __shared__ float red[16][128];
  const int l16 = threadIdx.x & 15, rg = threadIdx.x >> 4;
  const int cb = blockIdx.x % nb, chunk = blockIdx.x / nb, c0 = cb * 128 + 8 * l16, n = N - c0;
  const int64_t r1 = min((int64_t)(chunk + 1) * kRowChunk, rows);
  float bb[8], sum[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) bb[k] = sum[k] = 0.f;
  if (b) load_upto<float>(b + c0, n, vec, bb);
  for (int64_t r = (int64_t)chunk * kRowChunk + rg; r < r1; r += 16) {
    const int64_t i = r * nb + cb;
    float d[8];
    load_upto<T>(dout + r * N + c0, n, vec, d);
    const uint2 w = *reinterpret_cast<const uint2*>(q + i * 128 + 8 * l16);
    const float sc = scale_of(s[i]);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float u = int8_val(k < 4 ? w.x : w.y, k & 3, sc) + bb[k];
      const Gelu g = gelu_parts(u);
      // d/du u Phi(u) = Phi + u exp(-z^2) / (1.41421 sqrt(pi))
      d[k] *= fmaf(u * (0.5641895835477563f / 1.41421f), g.bell, g.cdf);
      sum[k] += d[k];
    }
    store_upto<T>(dy + r * N + c0, n, vec, d);
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

// ---------------------------------------------------------------- pack8 / unpack8
template <typename T>
__global__ __launch_bounds__(NT) void pack8_k(const T* __restrict__ x, uint8_t* __restrict__ q, uint8_t* __restrict__ s,
                                            int64_t nblk, int nb, int N, int vec) {
  const int l16 = threadIdx.x & 15;
  for (int64_t i = (blockIdx.x * (int64_t)NT + threadIdx.x) >> 4; i < nblk; i += (int64_t)gridDim.x * (NT / 16)) {
    const int64_t r = i / nb;
    const int c0 = (int)(i - r * nb) * 128 + 8 * l16;
    float v[8];
    load_upto<T>(x + r * N + c0, N - c0, vec, v);
    float m = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) m = fmaxf(m, finite_abs(v[k]));
    const int e = block_exp<Int8>(max16(m));
    const float is = exp2i(-e);
    *reinterpret_cast<uint2*>(q + i * 128 + 8 * l16) =
        make_uint2(int8x4(v[0] * is, v[1] * is, v[2] * is, v[3] * is), int8x4(v[4] * is, v[5] * is, v[6] * is, v[7] * is));
    if (l16 == 0) s[i] = (uint8_t)(e + 127);
  }
}

template <typename T>
__global__ __launch_bounds__(NT) void unpack8_k(const uint8_t* __restrict__ q, const uint8_t* __restrict__ s,
                                              T* __restrict__ x, int64_t nblk, int nb, int N, int vec) {
  const int l16 = threadIdx.x & 15;
  for (int64_t i = (blockIdx.x * (int64_t)NT + threadIdx.x) >> 4; i < nblk; i += (int64_t)gridDim.x * (NT / 16)) {
    const int64_t r = i / nb;
    const int c0 = (int)(i - r * nb) * 128 + 8 * l16;
    const uint2 w = *reinterpret_cast<const uint2*>(q + i * 128 + 8 * l16);
    const float sc = scale_of(s[i]);
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = int8_val(k < 4 ? w.x : w.y, k & 3, sc);
    store_upto<T>(x + r * N + c0, N - c0, vec, v);
  }
}

inline unsigned stream_grid(int64_t nblk) {   // one pass up to 16 workgroups per CU, then grid-stride
  const int64_t g = (nblk + NT / 16 - 1) / (NT / 16);
  return (unsigned)(g < 4096 ? g : 4096);
}

}  // namespace

int hx_split8_row_tiles(int64_t R) { return (int)((R + 127) / 128); }

void hx_split8(int bf16, const void* x, int64_t ld, int R, int C, uint8_t* q, uint8_t* s, uint8_t* qt, uint8_t* st,
               float* colpart, float* colsum, int vec, hipStream_t stream) {
  Split8 a{x, ld, R, C, q, s, qt, st, colpart, vec};
  const unsigned grid = (unsigned)(((C + 127) / 128) * (int64_t)((R + 127) / 128));
  if (bf16) split8_k<uint16_t><<<grid, NT, 0, stream>>>(a);
  else split8_k<float><<<grid, NT, 0, stream>>>(a);
  if (colpart) fold_rows(colpart, hx_split8_row_tiles(R), C, C, C, colsum, nullptr, nullptr, 0, stream);
}

void hx_gelu8_fwd(int bf16, const void* y, const float* b, void* out, uint8_t* q, uint8_t* s, int64_t rows, int N,
                  int vec, hipStream_t stream) {
  const int nb = (N + 127) / 128;
  const int64_t nblk = rows * nb;
  if (bf16) gelu8_fwd_k<uint16_t><<<stream_grid(nblk), NT, 0, stream>>>((const uint16_t*)y, b, (uint16_t*)out, q, s, nblk, nb, N, vec);
  else gelu8_fwd_k<float><<<stream_grid(nblk), NT, 0, stream>>>((const float*)y, b, (float*)out, q, s, nblk, nb, N, vec);
}

int hx_gelu8_chunks(int64_t rows) { return (int)((rows + kRowChunk - 1) / kRowChunk); }

void hx_gelu8_bwd(int bf16, const void* dout, const uint8_t* q, const uint8_t* s, const float* b, void* dy,
                  float* partial, float* db, int64_t rows, int N, int vec, hipStream_t stream) {
  const int nb = (N + 127) / 128;
  const unsigned grid = (unsigned)(nb * (int64_t)hx_gelu8_chunks(rows));
  if (bf16) gelu8_bwd_k<uint16_t><<<grid, NT, 0, stream>>>((const uint16_t*)dout, q, s, b, (uint16_t*)dy, partial, rows, nb, N, vec);
  else gelu8_bwd_k<float><<<grid, NT, 0, stream>>>((const float*)dout, q, s, b, (float*)dy, partial, rows, nb, N, vec);
  if (partial) fold_rows(partial, hx_gelu8_chunks(rows), N, N, N, db, nullptr, nullptr, 0, stream);
}

void hx_pack8(int bf16, const void* x, uint8_t* q, uint8_t* s, int64_t rows, int N, int vec, hipStream_t stream) {
  const int nb = (N + 127) / 128;
  const int64_t nblk = rows * nb;
  if (bf16) pack8_k<uint16_t><<<stream_grid(nblk), NT, 0, stream>>>((const uint16_t*)x, q, s, nblk, nb, N, vec);
  else pack8_k<float><<<stream_grid(nblk), NT, 0, stream>>>((const float*)x, q, s, nblk, nb, N, vec);
}

void hx_unpack8(int bf16, const uint8_t* q, const uint8_t* s, void* x, int64_t rows, int N, int vec, hipStream_t stream) {
  const int nb = (N + 127) / 128;
  const int64_t nblk = rows * nb;
  if (bf16) unpack8_k<uint16_t><<<stream_grid(nblk), NT, 0, stream>>>(q, s, (uint16_t*)x, nblk, nb, N, vec);
  else unpack8_k<float><<<stream_grid(nblk), NT, 0, stream>>>(q, s, (float*)x, nblk, nb, N, vec);
}
