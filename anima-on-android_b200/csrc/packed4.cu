// packed4.cu -- packing 16-bit rows to 4 bits, unpacking them, and matrix-vector products
// with packed weights (format: packed4.cuh).
//
//   quantize4_kernel    x [rows, K] 16-bit -> codes [rows, K/2], scales [rows, K/32]
//   dequantize4_kernel  back to fp32 / fp16 / bf16 values
//   matvec4_kernel      y[e] = f(x[e]) W[e]^T + add, a few rows x against E packed matrices
#include <algorithm>

#include "packed4.cuh"

namespace anima {

// ---------------------------------------------------------------- packing
// One thread reads 8 consecutive values (16 bytes) and writes one code word; the four lanes of
// a group agree on the value of largest magnitude x* by shuffles.  s = -x* / 8 in fp16 (exact
// unless it is subnormal), n = floor(x / s + 1/2) clamped to [-8, 7].
//
// The quotient is computed as x * (1 / s) with a bias of 2^-17 instead of being divided.  That
// gives the same n: x and s are 16-bit values, so x / s is either exactly at a border between two
// codes or at least 2^-13 away from it (|x - s (k + 1/2)| is a multiple of 2^(e_s - 12), e_s the
// exponent of s), while the product and the sum are off by less than 2^-19.  Adding 2^23 rounds
// the sum to a whole number, which is then the low bits of 0x4b000000 + n + 8.
struct Quant4Params {
  const void* x;
  uint32_t* codes;
  __half* scales;
  long long n1, n2;           // inner row counts: row = (a * n1 + b) * n2 + c
  long long s0, s1, s2;       // element strides of a, b, c
  long long units;            // rows * K / 8
  int upr;                    // units per row, K / 8
  int contiguous;             // rows are K elements apart: unit u starts at 8 u
};

template <bool kBf16>
__device__ __forceinline__ void widen8(const uint4& u, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (kBf16) {
      f[2 * k] = __uint_as_float(w[k] << 16);
      f[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
    } else {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
      f[2 * k] = v.x;
      f[2 * k + 1] = v.y;
    }
  }
}

template <bool kBf16>
__device__ __forceinline__ const uint4* unit_ptr(const Quant4Params& p, long long u) {
  const uint16_t* x = static_cast<const uint16_t*>(p.x);
  if (p.contiguous) return reinterpret_cast<const uint4*>(x + 8 * u);
  const long long row = u / p.upr;
  const long long c = row % p.n2, ab = row / p.n2;
  return reinterpret_cast<const uint4*>(x + (ab / p.n1) * p.s0 + (ab % p.n1) * p.s1 + c * p.s2 +
                                        8 * (u - row * p.upr));
}

template <bool kBf16>
__global__ void __launch_bounds__(256) quantize4_kernel(const Quant4Params p) {
  const int lane = threadIdx.x & 31;
  // units is a multiple of 16, so the lanes of a group leave the loop together
  for (long long u = (long long)blockIdx.x * blockDim.x + threadIdx.x; u < p.units;
       u += (long long)gridDim.x * blockDim.x) {
    const uint32_t mask = __activemask();
    float x[8];
    widen8<kBf16>(__ldg(unit_ptr<kBf16>(p, u)), x);
    float hi = x[0], lo = x[0];
    bool fine = true;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      hi = fmaxf(hi, x[e]);
      lo = fminf(lo, x[e]);
      fine = fine && fabsf(x[e]) <= 65504.f;  // false for NaN
    }
    if (!fine) hi = INFINITY;
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      hi = fmaxf(hi, __shfl_xor_sync(mask, hi, o));
      lo = fminf(lo, __shfl_xor_sync(mask, lo, o));
    }
    const bool bad = hi == INFINITY;
    const __half s = bad ? __ushort_as_half(0x7fff) : __float2half_rn((hi >= -lo ? hi : lo) * -0.125f);
    const float sf = __half2float(s);
    const float r = bad || sf == 0.f ? 0.f : 1.0f / sf;
    constexpr float kBias = 8.0f + 7.62939453125e-06f;  // + 2^-17
    uint32_t w = 0;
#pragma unroll
    for (int k = 7; k >= 0; --k) {
      const int e = 2 * (k & 3) + (k >> 2);  // the value at nibble k
      const float t = fminf(fmaxf(fmaf(bad ? 0.f : x[e], r, kBias), 0.f), 15.25f);
      // round(t) with t a bias past each half: floor(x / s + 1/2) + 8
      w = w * 16u + (__float_as_uint(t + 8388608.f) - 0x4b000000u);
    }
    const long long word = (u & ~15ll) + 4 * (u & 3) + ((u >> 2) & 3);
    p.codes[word] = w;
    if ((lane & 3) == 0) p.scales[u >> 2] = s;
  }
}

// ---------------------------------------------------------------- unpacking
// One thread reads 4 code words (16 bytes: values 32 g + 8 i .. + 7 of the four groups) and the
// block's 4 scales and writes four runs of 8 values.  n * s is exact in fp32 and rounded once.
template <int kDt>
__device__ __forceinline__ void store8(void* y, long long at, uint32_t w, float s) {
  uint32_t n[4];
  p4::numbers_f16(w, n);
  float f[8];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&n[k]));
    f[2 * k] = v.x * s;
    f[2 * k + 1] = v.y * s;
  }
  if (kDt == ANIMA_DTYPE_F32) {
    float4* o = reinterpret_cast<float4*>(static_cast<float*>(y) + at);
    o[0] = make_float4(f[0], f[1], f[2], f[3]);
    o[1] = make_float4(f[4], f[5], f[6], f[7]);
  } else {
    uint32_t o[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      o[k] = kDt == ANIMA_DTYPE_BF16 ? pack_bf16x2(f[2 * k], f[2 * k + 1])
                                     : pack_f16x2(f[2 * k], f[2 * k + 1]);
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(y) + at) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

template <int kDt>
__global__ void __launch_bounds__(256)
    dequantize4_kernel(const uint4* __restrict__ codes, const uint2* __restrict__ scales, void* y,
                       long long quads) {
  for (long long u = (long long)blockIdx.x * blockDim.x + threadIdx.x; u < quads;
       u += (long long)gridDim.x * blockDim.x) {
    const uint4 c = __ldg(codes + u);
    const float4 s = p4::scales4(__ldg(scales + (u >> 2)));
    const long long at = (u >> 2) * p4::kBlock + 8 * (u & 3);
    store8<kDt>(y, at, c.x, s.x);
    store8<kDt>(y, at + 32, c.y, s.y);
    store8<kDt>(y, at + 64, c.z, s.z);
    store8<kDt>(y, at + 96, c.w, s.w);
  }
}

// ---------------------------------------------------------------- matrix-vector products
// y[e, m, n] = sum_k f(x[e, m, k]) W[e, n, k] + add[e, m, n], f the identity or SiLU.
//
// Sixteen rows of W are the A operand of m16n8k16 and the rows x its eight columns, so up to
// eight columns cost what one does.  The products are of whole numbers n (packed4.cuh) and 16-bit
// x, exact; a group's partial sum is taken from a zeroed accumulator and multiplied by the group's
// scale in fp32.  fp32 rows (and SiLU's results) become three bf16 columns each, x = x0 + x1 + x2
// with x1 and x2 the rounded remainders: 24 bits together, so nothing of x is lost, and the three
// column sums are added at the end.
//
// A CTA of 8 warps takes tiles of 16 rows of W; `split` warps share a tile, taking its 128-value
// blocks in turn, and their sums meet in shared memory in a fixed order.  The columns are
// staged in shared memory once per matrix, rows 64 bytes past a multiple of 256 so that the
// quads of two columns fill the 128 bytes of a wavefront.
struct Mv4Params {
  const void* x;
  const uint8_t* codes;
  const __half* scales;
  const float* add;
  void* out;
  long long xe, xm, ae, am, oe, om;
  long long items;       // E * tile groups
  int N, K, M, groups;   // groups: tile groups of one matrix
  int split, tiles;      // warps per tile, tiles per group (8 / split)
  int silu, x_dtype, out_dtype;
};

constexpr int kMvThreads = 256;

__device__ __forceinline__ float load_x(const Mv4Params& p, long long at) {
  if (p.x_dtype == ANIMA_DTYPE_F32) return __ldg(static_cast<const float*>(p.x) + at);
  const uint16_t u = __ldg(static_cast<const uint16_t*>(p.x) + at);
  return p.x_dtype == ANIMA_DTYPE_BF16 ? __uint_as_float((uint32_t)u << 16)
                                       : __half2float(__ushort_as_half(u));
}

// kParts: columns per row of x (3: bf16 parts of an fp32 value, 1: the 16-bit value itself);
// kNB: blocks of eight columns.
template <bool kBf16, int kParts, int kNB>
__global__ void __launch_bounds__(kMvThreads) matvec4_kernel(const Mv4Params p) {
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int j = lane >> 2, i = lane & 3;
  const int cols = p.M * kParts;
  const int stride = p.K + 32;  // elements between staged columns
  uint16_t* const xs = reinterpret_cast<uint16_t*>(smem);
  float* const red = reinterpret_cast<float*>(smem + (size_t)cols * stride * 2);
  const int s = warp % p.split, t = warp / p.split;
  const int blocks = p.K / p4::kBlock;
  const long long lo = p.items * blockIdx.x / gridDim.x, hi = p.items * (blockIdx.x + 1) / gridDim.x;
  long long staged = -1;
  for (long long it = lo; it < hi; ++it) {
    const long long e = it / p.groups;
    const int tile = (int)(it - e * p.groups) * p.tiles + t;
    if (e != staged) {
      __syncthreads();  // the previous matrix's columns are no longer read
      for (int c = threadIdx.x; c < p.M * p.K; c += kMvThreads) {
        const int m = c / p.K, k = c - m * p.K;
        float v = load_x(p, e * p.xe + m * p.xm + k);
        if (p.silu) v = v / (1.0f + expf(-v));
        if (kParts == 1) {
          xs[m * stride + k] = kBf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v))
                                     : __half_as_ushort(__float2half_rn(v));
        } else {
#pragma unroll
          for (int q = 0; q < kParts; ++q) {
            const __nv_bfloat16 b = __float2bfloat16_rn(v);
            xs[(m * kParts + q) * stride + k] = __bfloat16_as_ushort(b);
            const float f = __bfloat162float(b);
            v = isinf(f) ? 0.f : v - f;
          }
        }
      }
      staged = e;
      __syncthreads();
    }
    float acc[kNB][4];
#pragma unroll
    for (int b = 0; b < kNB; ++b)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[b][c] = 0.f;
    const int n0 = tile * 16;
    // rows past the matrix read its last row; their sums are not stored
    const long long r0 = e * p.N + min(n0 + j, p.N - 1), r1 = e * p.N + min(n0 + j + 8, p.N - 1);
    const uint4* c0 = reinterpret_cast<const uint4*>(p.codes + r0 * (p.K / 2)) + i;
    const uint4* c1 = reinterpret_cast<const uint4*>(p.codes + r1 * (p.K / 2)) + i;
    const uint2* s0 = reinterpret_cast<const uint2*>(p.scales + r0 * (p.K / p4::kGroup));
    const uint2* s1 = reinterpret_cast<const uint2*>(p.scales + r1 * (p.K / p4::kGroup));
#pragma unroll 2
    for (int blk = s; blk < blocks; blk += p.split) {
      const uint4 u0 = __ldg(c0 + 4 * blk), u1 = __ldg(c1 + 4 * blk);
      const float4 f0 = p4::scales4(__ldg(s0 + blk)), f1 = p4::scales4(__ldg(s1 + blk));
      const uint32_t w0[4] = {u0.x, u0.y, u0.z, u0.w}, w1[4] = {u1.x, u1.y, u1.z, u1.w};
      const float g0[4] = {f0.x, f0.y, f0.z, f0.w}, g1[4] = {f1.x, f1.y, f1.z, f1.w};
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        uint32_t a[4], b[4];
        p4::numbers<kBf16>(w0[g], a);
        p4::numbers<kBf16>(w1[g], b);
#pragma unroll
        for (int nb = 0; nb < kNB; ++nb) {
          uint4 xv = make_uint4(0u, 0u, 0u, 0u);
          if (nb * 8 + j < cols)
            xv = *reinterpret_cast<const uint4*>(xs + (nb * 8 + j) * stride + blk * p4::kBlock +
                                                 32 * g + 8 * i);
          float d[4] = {0.f, 0.f, 0.f, 0.f};
          p4::mma16816<kBf16>(d, a[0], b[0], a[1], b[1], xv.x, xv.y);
          p4::mma16816<kBf16>(d, a[2], b[2], a[3], b[3], xv.z, xv.w);
          acc[nb][0] = fmaf(g0[g], d[0], acc[nb][0]);
          acc[nb][1] = fmaf(g0[g], d[1], acc[nb][1]);
          acc[nb][2] = fmaf(g1[g], d[2], acc[nb][2]);
          acc[nb][3] = fmaf(g1[g], d[3], acc[nb][3]);
        }
      }
    }
    // red[warp][row][column]
    constexpr int kCols = 8 * kNB;
    float* const mine = red + warp * 16 * kCols;
#pragma unroll
    for (int nb = 0; nb < kNB; ++nb) {
      *reinterpret_cast<float2*>(mine + j * kCols + nb * 8 + 2 * i) = make_float2(acc[nb][0], acc[nb][1]);
      *reinterpret_cast<float2*>(mine + (j + 8) * kCols + nb * 8 + 2 * i) =
          make_float2(acc[nb][2], acc[nb][3]);
    }
    __syncthreads();
    for (int o = threadIdx.x; o < p.tiles * 16 * p.M; o += kMvThreads) {
      const int row = o & 15, m = (o >> 4) % p.M, tt = (o >> 4) / p.M;
      const int n = ((int)(it - e * p.groups) * p.tiles + tt) * 16 + row;
      if (n >= p.N) continue;
      float y = 0.f;
      for (int q = 0; q < p.split; ++q)
#pragma unroll
        for (int c = 0; c < kParts; ++c)
          y += red[((tt * p.split + q) * 16 + row) * kCols + m * kParts + c];
      if (p.add) y += __ldg(p.add + e * p.ae + m * p.am + n);
      const long long at = e * p.oe + m * p.om + n;
      if (p.out_dtype == ANIMA_DTYPE_F32)
        static_cast<float*>(p.out)[at] = y;
      else
        static_cast<uint16_t*>(p.out)[at] = p.out_dtype == ANIMA_DTYPE_BF16
                                                ? __bfloat16_as_ushort(__float2bfloat16_rn(y))
                                                : __half_as_ushort(__float2half_rn(y));
    }
    __syncthreads();  // the sums are read before the next tile's are written
  }
}

// ---------------------------------------------------------------- launchers
static int stream_grid(long long work, int per_block, int sm_count, int waves) {
  const long long g = (work + per_block - 1) / per_block, cap = (long long)sm_count * waves;
  return (int)(g < 1 ? 1 : g > cap ? cap : g);
}

int quantize4_launch(const void* x, int dtype, long long n0, long long n1, long long n2,
                     long long s0, long long s1, long long s2, int K, void* codes, void* scales,
                     int sm_count, cudaStream_t st) {
  Quant4Params p;
  p.x = x;
  p.codes = static_cast<uint32_t*>(codes);
  p.scales = static_cast<__half*>(scales);
  p.n1 = n1;
  p.n2 = n2;
  p.s0 = s0;
  p.s1 = s1;
  p.s2 = s2;
  p.upr = K / 8;
  p.units = n0 * n1 * n2 * p.upr;
  p.contiguous = (n2 == 1 || s2 == K) && (n1 == 1 || s1 == n2 * K) && (n0 == 1 || s0 == n1 * n2 * K);
  const int grid = stream_grid(p.units, 256, sm_count, 8);
  if (dtype == ANIMA_DTYPE_BF16)
    quantize4_kernel<true><<<grid, 256, 0, st>>>(p);
  else
    quantize4_kernel<false><<<grid, 256, 0, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? ANIMA_OK : ANIMA_ERR_CUDA;
}

int dequantize4_launch(const void* codes, const void* scales, void* y, int dtype, long long rows,
                       int K, int sm_count, cudaStream_t st) {
  const long long quads = rows * (K / 32);
  const int grid = stream_grid(quads, 256, sm_count, 8);
  const uint4* c = static_cast<const uint4*>(codes);
  const uint2* s = static_cast<const uint2*>(scales);
  if (dtype == ANIMA_DTYPE_F32)
    dequantize4_kernel<ANIMA_DTYPE_F32><<<grid, 256, 0, st>>>(c, s, y, quads);
  else if (dtype == ANIMA_DTYPE_BF16)
    dequantize4_kernel<ANIMA_DTYPE_BF16><<<grid, 256, 0, st>>>(c, s, y, quads);
  else
    dequantize4_kernel<ANIMA_DTYPE_F16><<<grid, 256, 0, st>>>(c, s, y, quads);
  return cudaGetLastError() == cudaSuccess ? ANIMA_OK : ANIMA_ERR_CUDA;
}

template <bool kBf16, int kParts, int kNB>
static int mv4_t(const Mv4Params& p, int sm_count, cudaStream_t st) {
  auto kern = matvec4_kernel<kBf16, kParts, kNB>;
  const size_t smem = (size_t)p.M * kParts * (p.K + 32) * 2 + 8 * 16 * 8 * kNB * sizeof(float);
  if (smem > 227 * 1024) return ANIMA_ERR_SHAPE;
  if (smem > 48 * 1024 && cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (int)smem) != cudaSuccess) {
    cudaGetLastError();
    return ANIMA_ERR_CUDA;
  }
  int per_sm = (int)(227 * 1024 / (smem + 1024));
  if (per_sm > 4) per_sm = 4;
  const int grid = (int)std::min<long long>(p.items, (long long)sm_count * per_sm);
  kern<<<grid, kMvThreads, smem, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? ANIMA_OK : ANIMA_ERR_CUDA;
}

// Rows of x of one launch: eight fp32 rows are 24 columns, sixteen 16-bit rows 16; fewer where
// their columns would not fit shared memory.
static int mv4_rows(int K, int parts) {
  const int most = parts == 3 ? 8 : 16;
  const int fit = (int)((227 * 1024 - 8 * 16 * 24 * 4) / ((size_t)parts * (K + 32) * 2));
  return most < fit ? most : fit;
}

int matvec4_launch(const AnimaMatvec4Args* a, int sm_count, cudaStream_t st) {
  const int parts = a->x_dtype == ANIMA_DTYPE_F32 || a->silu ? 3 : 1;
  const int rows = mv4_rows(a->K, parts);
  if (rows < 1) return ANIMA_ERR_SHAPE;
  Mv4Params p;
  p.codes = static_cast<const uint8_t*>(a->codes);
  p.scales = static_cast<const __half*>(a->scales);
  p.xe = a->x_stride[0];
  p.xm = a->x_stride[1];
  p.ae = a->add_stride[0];
  p.am = a->add_stride[1];
  p.oe = a->out_stride[0];
  p.om = a->out_stride[1];
  p.N = a->N;
  p.K = a->K;
  p.silu = a->silu;
  p.x_dtype = a->x_dtype;
  p.out_dtype = a->out_dtype;
  // Warps that share a tile: as many as leave each two blocks of its rows.
  p.split = 1;
  while (p.split < 8 && p.K / p4::kBlock >= 4 * p.split) p.split *= 2;
  p.tiles = 8 / p.split;
  const int ntiles = (p.N + 15) / 16;
  p.groups = (ntiles + p.tiles - 1) / p.tiles;
  p.items = (long long)a->E * p.groups;
  const int xs = a->x_dtype == ANIMA_DTYPE_F32 ? 4 : 2, os = a->out_dtype == ANIMA_DTYPE_F32 ? 4 : 2;
  for (int m0 = 0; m0 < a->M; m0 += rows) {
    p.M = std::min(rows, a->M - m0);
    p.x = static_cast<const char*>(a->x) + m0 * p.xm * xs;
    p.out = static_cast<char*>(a->out) + m0 * p.om * os;
    p.add = a->add ? static_cast<const float*>(a->add) + m0 * p.am : nullptr;
    const int nb = (p.M * parts + 7) / 8;
    int rc;
    if (parts == 3)
      rc = nb == 1 ? mv4_t<true, 3, 1>(p, sm_count, st)
                   : nb == 2 ? mv4_t<true, 3, 2>(p, sm_count, st) : mv4_t<true, 3, 3>(p, sm_count, st);
    else if (a->x_dtype == ANIMA_DTYPE_BF16)
      rc = nb == 1 ? mv4_t<true, 1, 1>(p, sm_count, st) : mv4_t<true, 1, 2>(p, sm_count, st);
    else
      rc = nb == 1 ? mv4_t<false, 1, 1>(p, sm_count, st) : mv4_t<false, 1, 2>(p, sm_count, st);
    if (rc != ANIMA_OK) return rc;
  }
  return ANIMA_OK;
}

}  // namespace anima
