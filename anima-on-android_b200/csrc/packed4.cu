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
// a group agree on its largest values of either sign, (max x, max -x) as a pair, by shuffles.
// s = -x* / 8 in fp16 (exact unless it is subnormal), n = floor(x / s + 1/2) clamped to [-8, 7].
//
// The quotient is not divided: x and s are 16-bit values, so x / s is either exactly at a border
// between two codes or at least 2^-13 away from it (|x - s (k + 1/2)| is a multiple of 2^(e_s - 12),
// e_s the exponent of s), while products with an approximate 1 / s are off by less than 2^-19.  So
// with t = saturate(x / (16 s) + 17/32 + 2^-18), the sum t (16 - 2^-14) + 2^23 - 1/2 rounds to
// 2^23 + n + 8: at a border the bias leaves between 2^-18 and 2^-14 above it, and t = 1 gives 15.
// (With a clamp on both sides, tests of every value and a true reciprocal this took 106 us for 132 M
// values, bound by instructions; the floor is 52.)
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
__device__ __forceinline__ float2 widen2(uint32_t w) {
  if (kBf16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
// Pairwise maximum; NaN wins.
template <bool kBf16>
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  uint32_t r;
  if (kBf16)
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ const uint4* unit_ptr(const Quant4Params& p, long long u) {
  const uint16_t* x = static_cast<const uint16_t*>(p.x);
  if (p.contiguous) return reinterpret_cast<const uint4*>(x + 8 * u);
  const long long row = u / p.upr;
  const long long c = row % p.n2, ab = row / p.n2;
  return reinterpret_cast<const uint4*>(x + (ab / p.n1) * p.s0 + (ab % p.n1) * p.s1 + c * p.s2 +
                                        8 * (u - row * p.upr));
}

template <bool kBf16>
__device__ __forceinline__ void quantize_unit(const Quant4Params& p, long long u, const uint4& v, uint32_t mask) {
  constexpr uint32_t kSign = 0x80008000u;
  const uint32_t w4[4] = {v.x, v.y, v.z, v.w};
  const uint32_t hi2 = max2<kBf16>(max2<kBf16>(v.x, v.y), max2<kBf16>(v.z, v.w));
  const uint32_t lo2 = max2<kBf16>(max2<kBf16>(v.x ^ kSign, v.y ^ kSign), max2<kBf16>(v.z ^ kSign, v.w ^ kSign));
  // (max x, max -x) of the eight values, then of the group
  uint32_t m = max2<kBf16>(__byte_perm(hi2, lo2, 0x5410), __byte_perm(hi2, lo2, 0x7632));
  m = max2<kBf16>(m, __shfl_xor_sync(mask, m, 1));
  m = max2<kBf16>(m, __shfl_xor_sync(mask, m, 2));
  const float2 top = widen2<kBf16>(m);
  const bool fine = fmaxf(top.x, top.y) <= 65504.f && top.x == top.x && top.y == top.y;
  const __half s = fine ? __float2half_rn((top.x >= top.y ? top.x : -top.y) * -0.125f) : __ushort_as_half(0x7fff);
  const float sf = __half2float(s);
  const float r = sf == 0.f ? 0.f : 0.0625f * rcp_approx(sf);
  constexpr float kBias = 0.53125f + 3.814697265625e-06f;  // 17/32 + 2^-18
  constexpr float kMul = 16.0f - 6.103515625e-05f;         // 16 - 2^-14
  float x[8];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 f = widen2<kBf16>(w4[k]);
    x[2 * k] = f.x;
    x[2 * k + 1] = f.y;
  }
  uint32_t w = 0;
  if (__any_sync(mask, fabsf(sf) < 6.103515625e-05f)) {  // a subnormal s may be rounded below |x*| / 8
#pragma unroll
    for (int k = 7; k >= 0; --k) {
      const float t = fmaxf(__saturatef(fmaf(x[2 * (k & 3) + (k >> 2)], r, kBias)), 0.03125f);
      w = w * 16u + __float_as_uint(fmaf(t, kMul, 8388607.5f));
    }
  } else {
#pragma unroll
    for (int k = 7; k >= 0; --k) {
      const float t = __saturatef(fmaf(x[2 * (k & 3) + (k >> 2)], r, kBias));  // the value at nibble k
      w = w * 16u + __float_as_uint(fmaf(t, kMul, 8388607.5f));
    }
  }
  w -= 0xfb000000u;  // what the exponent bits 0x4b000000 of the eight sums added up to
  p.codes[(u & ~15ll) + 4 * (u & 3) + ((u >> 2) & 3)] = fine ? w : 0x88888888u;
  if ((u & 3) == 0) p.scales[u >> 2] = s;
}

template <bool kBf16>
__global__ void __launch_bounds__(256) quantize4_kernel(const Quant4Params p) {
  // units is a multiple of 16, so the lanes of a group leave the loop together
  const long long step = (long long)gridDim.x * blockDim.x;
  for (long long u = (long long)blockIdx.x * blockDim.x + threadIdx.x; u < p.units; u += 2 * step) {
    const uint32_t mask = __activemask();
    const bool two = u + step < p.units;
    const uint4 v0 = __ldg(unit_ptr(p, u));
    uint4 v1 = make_uint4(0u, 0u, 0u, 0u);
    if (two) v1 = __ldg(unit_ptr(p, u + step));
    quantize_unit<kBf16>(p, u, v0, mask);
    if (two) quantize_unit<kBf16>(p, u + step, v1, __activemask());
  }
}

// ---------------------------------------------------------------- unpacking
// One lane per run of 8 values, in value order, so a warp's stores are one contiguous run (with
// a lane per 16 bytes of codes, each store touched eight 64-byte pieces: 110 us against 57 for
// 132 M values to bf16).  Value run v of a block (v = 4 g + i) is word 4 i + g of its codes.  n * s
// is exact in fp32 and rounded once.
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
    dequantize4_kernel(const uint32_t* __restrict__ codes, const __half* __restrict__ scales, void* y,
                       long long words) {
  constexpr int kU = 4;  // runs per lane and round, loaded before any is converted
  const long long step = (long long)gridDim.x * blockDim.x;
  for (long long u0 = (long long)blockIdx.x * blockDim.x + threadIdx.x; u0 < words; u0 += kU * step) {
    uint32_t w[kU];
    __half s[kU];
#pragma unroll
    for (int k = 0; k < kU; ++k) {
      const long long u = u0 + k * step;
      if (u < words) {
        w[k] = __ldg(codes + ((u & ~15ll) + 4 * (u & 3) + ((u >> 2) & 3)));
        s[k] = __ldg(scales + (u >> 2));
      }
    }
#pragma unroll
    for (int k = 0; k < kU; ++k) {
      const long long u = u0 + k * step;
      if (u < words) store8<kDt>(y, 8 * u, w[k], __half2float(s[k]));
    }
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
// A CTA of 8 warps works on one matrix, on a run of tiles of 16 rows of W; `split` warps share a
// tile, taking its 128-value blocks in turn, and their sums meet in shared memory in a fixed
// order.  A warp streams its blocks (1 KB of codes, 128 bytes of scales) through a private ring
// of cp.async stages that runs on across tiles; each lane fetches the codes that it will read
// itself.  The columns are staged in shared memory once, rows 64 bytes past a multiple of 256 so
// that the quads of two columns fill the 128 bytes of a wavefront.
struct Mv4Params {
  const void* x;
  const uint8_t* codes;
  const __half* scales;
  const float* add;
  void* out;
  long long xe, xm, ae, am, oe, om;
  int N, K, M;
  int parts;             // CTAs per matrix
  int groups;            // tile groups of one matrix (8 / split tiles each)
  int split;             // warps per tile
  int silu, x_dtype, out_dtype;
};

constexpr int kMvThreads = 256;
constexpr int kMvStage = 16 * 64 + 16 * 8;  // bytes of a block of 16 rows

__device__ __forceinline__ float load_x(const Mv4Params& p, long long at) {
  if (p.x_dtype == ANIMA_DTYPE_F32) return __ldg(static_cast<const float*>(p.x) + at);
  const uint16_t u = __ldg(static_cast<const uint16_t*>(p.x) + at);
  return p.x_dtype == ANIMA_DTYPE_BF16 ? __uint_as_float((uint32_t)u << 16)
                                       : __half2float(__ushort_as_half(u));
}

// kParts: columns per row of x (3: bf16 parts of an fp32 value, which take columns 4 m .. 4 m + 2,
// so that a row's sum needs one exchange between neighbour lanes; 1: the 16-bit value itself);
// kNB: blocks of eight columns; kStages: ring stages (4; 3 for rows so long that their columns
// need the room).  Columns without a row repeat another one's data: columns do not mix.
template <bool kBf16, int kParts, int kNB, int kStages>
__global__ void __launch_bounds__(kMvThreads, 3) matvec4_kernel(const Mv4Params p) {
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int kOuts = kParts == 3 ? 1 : 4;  // results of a lane per block of columns
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int j = lane >> 2, i = lane & 3;
  const int stride = p.K + 32;  // elements between staged columns
  const uint32_t ring = smem_u32(smem) + warp * kStages * kMvStage;
  float* const red = reinterpret_cast<float*>(smem + 8 * kStages * kMvStage);
  uint16_t* const xs = reinterpret_cast<uint16_t*>(red + 8 * 32 * kNB * kOuts);
  const int s = warp % p.split, t = warp / p.split, tiles = 8 / p.split;
  const int blocks = p.K / p4::kBlock;
  const int e = blockIdx.x / p.parts, part = blockIdx.x - e * p.parts;
  const int g_lo = (int)((long long)p.groups * part / p.parts);
  const int g_hi = (int)((long long)p.groups * (part + 1) / p.parts);

  // The block sequence of this warp: (group, block) with block = s, s + split, ...  A lane
  // fetches its 16 bytes of rows j and j + 8, lanes i = 0, 1 their scales.  Rows past the
  // matrix repeat its last one; their results are not stored.
  const uint8_t* const codes = p.codes + (long long)e * p.N * (p.K / 2) + i * 16;
  const uint8_t* const scales = reinterpret_cast<const uint8_t*>(p.scales) + (long long)e * p.N * (p.K / 16);
  const uint8_t *c0 = codes, *c1 = codes, *sp = scales;
  int ld_g = g_lo, ld_blk = s;
  uint32_t ld_at = ring;
  const int tile_rows = 16 * tiles;  // from a warp's tile to its next
  const long long c_next = (long long)tile_rows * (p.K / 2) - (long long)((blocks - s - 1) / p.split + 1) * p.split * 64;
  const long long s_next = (long long)tile_rows * (p.K / 16) - (long long)((blocks - s - 1) / p.split + 1) * p.split * 8;
  int ld_n = (g_lo * tiles + t) * 16;  // first row of the tile being fetched
  auto tile_start = [&]() {
    const int n = ld_n + j;
    const int n0 = min(n, p.N - 1), n1 = min(n + 8, p.N - 1);
    c0 = codes + (long long)n0 * (p.K / 2) + s * 64;
    c1 = codes + (long long)n1 * (p.K / 2) + s * 64;
    sp = scales + (long long)(i == 0 ? n0 : n1) * (p.K / 16) + s * 8;
  };
  auto fetch = [&]() {
    if (ld_g < g_hi) {
      p4::cp16(ld_at + lane * 16, c0);
      p4::cp16(ld_at + 512 + lane * 16, c1);
      if (i < 2) p4::cp8(ld_at + 1024 + (i * 8 + j) * 8, sp);
      c0 += p.split * 64;
      c1 += p.split * 64;
      sp += p.split * 8;
      ld_blk += p.split;
      if (ld_blk >= blocks) {
        ld_blk = s;
        ++ld_g;
        ld_n += tile_rows;
        if (ld_n + 16 <= p.N) {
          c0 += c_next;
          c1 += c_next;
          sp += s_next;
        } else {
          tile_start();
        }
      }
    }
    p4::cp_commit();
    ld_at = ld_at == ring + (kStages - 1) * kMvStage ? ring : ld_at + kMvStage;
  };
  tile_start();
#pragma unroll
  for (int k = 0; k < kStages - 1; ++k) fetch();

  for (int m = 0; m < p.M; ++m) {
    const long long from = (long long)e * p.xe + (long long)m * p.xm;
    uint16_t* const to = xs + m * kParts * stride;
#pragma unroll 4
    for (int k = 2 * threadIdx.x; k < p.K; k += 2 * kMvThreads) {
      float v0 = load_x(p, from + k), v1 = load_x(p, from + k + 1);
      if (p.silu) {
        v0 = __fdividef(v0, 1.0f + expf(-v0));
        v1 = __fdividef(v1, 1.0f + expf(-v1));
      }
      if (kParts == 1) {
        *reinterpret_cast<uint32_t*>(to + k) = kBf16 ? pack_bf16x2(v0, v1) : pack_f16x2(v0, v1);
      } else {
#pragma unroll
        for (int q = 0; q < kParts; ++q) {
          const uint32_t b = pack_bf16x2(v0, v1);
          *reinterpret_cast<uint32_t*>(to + q * stride + k) = b;
          const float f0 = __uint_as_float(b << 16), f1 = __uint_as_float(b & 0xffff0000u);
          v0 = isinf(f0) ? 0.f : v0 - f0;
          v1 = isinf(f1) ? 0.f : v1 - f1;
        }
      }
    }
  }
  uint32_t xa[kNB];  // this lane's column of x, at its eight values of a group
#pragma unroll
  for (int nb = 0; nb < kNB; ++nb) {
    const int col = kParts == 3 ? min(nb * 2 + (j >> 2), p.M - 1) * 3 + min(j & 3, 2) : min(nb * 8 + j, p.M - 1);
    xa[nb] = smem_u32(xs + col * stride + 8 * i);
  }
  __syncthreads();

  // Result r of this lane for column block nb is row `row + out_row(r)`, row m = out_m(nb, r) of x.
  auto out_row = [&](int r) { return kParts == 3 ? 0 : 8 * (r >> 1); };
  auto out_m = [&](int nb, int r) { return kParts == 3 ? nb * 2 + (i >> 1) : nb * 8 + 2 * i + (r & 1); };
  int row = (g_lo * tiles + t) * 16 + j + (kParts == 3 ? 8 * (i & 1) : 0);
  long long out_at[kNB], add_at[kNB];
#pragma unroll
  for (int nb = 0; nb < kNB; ++nb) {
    out_at[nb] = (long long)e * p.oe + (long long)out_m(nb, 0) * p.om + row;
    add_at[nb] = (long long)e * p.ae + (long long)out_m(nb, 0) * p.am + row;
  }

  uint32_t at = ring;
  for (int grp = g_lo; grp < g_hi; ++grp) {
    float y[kNB][kOuts];
#pragma unroll
    for (int nb = 0; nb < kNB; ++nb)
#pragma unroll
      for (int r = 0; r < kOuts; ++r) {
        y[nb][r] = 0.f;
        if (p.add && s == 0 && row + out_row(r) < p.N && out_m(nb, r) < p.M)
          y[nb][r] = __ldg(p.add + add_at[nb] + (r & 1) * p.am + out_row(r));
      }
    float acc[kNB][4];
#pragma unroll
    for (int b = 0; b < kNB; ++b)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[b][c] = 0.f;
    for (int blk = s; blk < blocks; blk += p.split) {
      p4::cp_wait<kStages - 2>();
      __syncwarp();
      fetch();  // into the slot read in the last round
      const uint4 u0 = p4::lds16(at + lane * 16), u1 = p4::lds16(at + 512 + lane * 16);
      const float4 f0 = p4::scales4(p4::lds8(at + 1024 + j * 8));
      const float4 f1 = p4::scales4(p4::lds8(at + 1024 + (8 + j) * 8));
      at = at == ring + (kStages - 1) * kMvStage ? ring : at + kMvStage;
      const uint32_t w0[4] = {u0.x, u0.y, u0.z, u0.w}, w1[4] = {u1.x, u1.y, u1.z, u1.w};
      const float g0[4] = {f0.x, f0.y, f0.z, f0.w}, g1[4] = {f1.x, f1.y, f1.z, f1.w};
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        uint32_t a[4], b[4];
        p4::numbers<kBf16>(w0[g], a);
        p4::numbers<kBf16>(w1[g], b);
#pragma unroll
        for (int nb = 0; nb < kNB; ++nb) {
          const uint4 xv = p4::lds16(xa[nb] + blk * (2 * p4::kBlock) + 64 * g);
          float d[4];
          p4::mma16816_zero<kBf16>(d, a[0], b[0], a[1], b[1], xv.x, xv.y);
          p4::mma16816<kBf16>(d, a[2], b[2], a[3], b[3], xv.z, xv.w);
          acc[nb][0] = fmaf(g0[g], d[0], acc[nb][0]);
          acc[nb][1] = fmaf(g0[g], d[1], acc[nb][1]);
          acc[nb][2] = fmaf(g1[g], d[2], acc[nb][2]);
          acc[nb][3] = fmaf(g1[g], d[3], acc[nb][3]);
        }
      }
    }
#pragma unroll
    for (int nb = 0; nb < kNB; ++nb) {
      if (kParts == 3) {
        float v0 = acc[nb][0] + ((i & 1) ? 0.f : acc[nb][1]);
        float v1 = acc[nb][2] + ((i & 1) ? 0.f : acc[nb][3]);
        v0 += __shfl_xor_sync(0xffffffffu, v0, 1);
        v1 += __shfl_xor_sync(0xffffffffu, v1, 1);
        y[nb][0] += (i & 1) ? v1 : v0;
      } else {
#pragma unroll
        for (int r = 0; r < kOuts; ++r) y[nb][r] += acc[nb][r];
      }
    }
    if (p.split > 1) {  // the warps of a tile are neighbours: the first adds the others' results
#pragma unroll
      for (int nb = 0; nb < kNB; ++nb)
#pragma unroll
        for (int r = 0; r < kOuts; ++r) red[((warp * kNB + nb) * kOuts + r) * 32 + lane] = y[nb][r];
      __syncthreads();
      if (s == 0)
        for (int q = 1; q < p.split; ++q)
#pragma unroll
          for (int nb = 0; nb < kNB; ++nb)
#pragma unroll
            for (int r = 0; r < kOuts; ++r) y[nb][r] += red[(((warp + q) * kNB + nb) * kOuts + r) * 32 + lane];
    }
    if (s == 0) {
#pragma unroll
      for (int nb = 0; nb < kNB; ++nb)
#pragma unroll
        for (int r = 0; r < kOuts; ++r) {
          if (row + out_row(r) >= p.N || out_m(nb, r) >= p.M) continue;
          const float v = y[nb][r];
          const long long o = out_at[nb] + (r & 1) * p.om + out_row(r);
          if (p.out_dtype == ANIMA_DTYPE_F32)
            static_cast<float*>(p.out)[o] = v;
          else
            static_cast<uint16_t*>(p.out)[o] = p.out_dtype == ANIMA_DTYPE_BF16
                                                   ? __bfloat16_as_ushort(__float2bfloat16_rn(v))
                                                   : __half_as_ushort(__float2half_rn(v));
        }
    }
    if (p.split > 1) __syncthreads();  // the sums are read before the next tile's are written
    row += tile_rows;
#pragma unroll
    for (int nb = 0; nb < kNB; ++nb) {
      out_at[nb] += tile_rows;
      add_at[nb] += tile_rows;
    }
  }
  p4::cp_wait<0>();
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
  const int grid = stream_grid(p.units, 512, sm_count, 8);
  if (dtype == ANIMA_DTYPE_BF16)
    quantize4_kernel<true><<<grid, 256, 0, st>>>(p);
  else
    quantize4_kernel<false><<<grid, 256, 0, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? ANIMA_OK : ANIMA_ERR_CUDA;
}

int dequantize4_launch(const void* codes, const void* scales, void* y, int dtype, long long rows,
                       int K, int sm_count, cudaStream_t st) {
  const long long words = rows * (K / 8);
  const int grid = stream_grid(words, 1024, sm_count, 8);
  const uint32_t* c = static_cast<const uint32_t*>(codes);
  const __half* s = static_cast<const __half*>(scales);
  if (dtype == ANIMA_DTYPE_F32)
    dequantize4_kernel<ANIMA_DTYPE_F32><<<grid, 256, 0, st>>>(c, s, y, words);
  else if (dtype == ANIMA_DTYPE_BF16)
    dequantize4_kernel<ANIMA_DTYPE_BF16><<<grid, 256, 0, st>>>(c, s, y, words);
  else
    dequantize4_kernel<ANIMA_DTYPE_F16><<<grid, 256, 0, st>>>(c, s, y, words);
  return cudaGetLastError() == cudaSuccess ? ANIMA_OK : ANIMA_ERR_CUDA;
}

constexpr size_t kMaxSmem = 227 * 1024;
constexpr size_t mv4_fixed_smem(int nb, int outs, int stages) {
  return 8 * stages * kMvStage + 8 * 32 * nb * outs * sizeof(float);
}

template <bool kBf16, int kParts, int kNB, int kStages>
static int mv4_t(Mv4Params p, int E, int sm_count, cudaStream_t st) {
  auto kern = matvec4_kernel<kBf16, kParts, kNB, kStages>;
  const size_t smem = mv4_fixed_smem(kNB, kParts == 3 ? 1 : 4, kStages) + (size_t)p.M * kParts * (p.K + 32) * 2;
  if (smem > kMaxSmem) return ANIMA_ERR_SHAPE;
  static SmemAttr attr;
  if (!attr.raise((const void*)kern, smem)) return ANIMA_ERR_CUDA;
  // Warps that share a tile, and CTAs per matrix: the split whose busiest warp has the least to do,
  // in blocks, a tile's ends counted as one.
  const int ntiles = (p.N + 15) / 16, blocks = p.K / p4::kBlock;
  const int per_sm = std::max(1, std::min(3, (int)(kMaxSmem / (smem + 1024))));
  const long long slots = (long long)per_sm * sm_count;
  long long best = 0;
  for (int split = 1; split <= 8 && split <= blocks; split *= 2) {
    const long long groups = ((long long)ntiles * split + 7) / 8;
    const long long parts = std::min(groups, std::max(1LL, slots / E));
    const long long waves = (E * parts + slots - 1) / slots;
    const long long cost = waves * ((groups + parts - 1) / parts) * ((blocks + split - 1) / split + 1);
    if (split == 1 || cost < best) {
      best = cost;
      p.split = split;
      p.groups = (int)groups;
      p.parts = (int)parts;
    }
  }
  if ((long long)E * p.parts > 0x7fffffffLL) return ANIMA_ERR_SHAPE;
  kern<<<E * p.parts, kMvThreads, smem, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? ANIMA_OK : ANIMA_ERR_CUDA;
}

// Rows of x of one launch: eight fp32 rows or sixteen 16-bit ones; fewer where their columns
// would not fit shared memory, and a shorter ring where not even one would.
static int mv4_rows(int K, int parts, int* stages) {
  const size_t row = (size_t)parts * (K + 32) * 2;
  *stages = 4;
  const int fit = (int)((kMaxSmem - mv4_fixed_smem(2, 4, 4)) / row);
  if (fit >= 1) return std::min(parts == 3 ? 8 : 16, fit);
  *stages = 3;
  return kMaxSmem - mv4_fixed_smem(1, 4, 3) >= row ? 1 : 0;
}

int matvec4_launch(const AnimaMatvec4Args* a, int sm_count, cudaStream_t st) {
  const int parts = a->x_dtype == ANIMA_DTYPE_F32 || a->silu ? 3 : 1;
  int stages;
  const int rows = mv4_rows(a->K, parts, &stages);
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
  const int xs = a->x_dtype == ANIMA_DTYPE_F32 ? 4 : 2, os = a->out_dtype == ANIMA_DTYPE_F32 ? 4 : 2;
  for (int m0 = 0; m0 < a->M; m0 += rows) {
    p.M = std::min(rows, a->M - m0);
    p.x = static_cast<const char*>(a->x) + m0 * p.xm * xs;
    p.out = static_cast<char*>(a->out) + m0 * p.om * os;
    p.add = a->add ? static_cast<const float*>(a->add) + m0 * p.am : nullptr;
    const int nb = parts == 3 ? (p.M + 1) / 2 : (p.M + 7) / 8;
    const bool bf = parts == 3 || a->x_dtype == ANIMA_DTYPE_BF16;
    int rc;
    if (stages == 3)
      rc = parts == 3 ? mv4_t<true, 3, 1, 3>(p, a->E, sm_count, st)
           : bf       ? mv4_t<true, 1, 1, 3>(p, a->E, sm_count, st)
                      : mv4_t<false, 1, 1, 3>(p, a->E, sm_count, st);
    else if (parts == 3)
      rc = nb == 1   ? mv4_t<true, 3, 1, 4>(p, a->E, sm_count, st)
           : nb == 2 ? mv4_t<true, 3, 2, 4>(p, a->E, sm_count, st)
                     : mv4_t<true, 3, 4, 4>(p, a->E, sm_count, st);
    else if (bf)
      rc = nb == 1 ? mv4_t<true, 1, 1, 4>(p, a->E, sm_count, st) : mv4_t<true, 1, 2, 4>(p, a->E, sm_count, st);
    else
      rc = nb == 1 ? mv4_t<false, 1, 1, 4>(p, a->E, sm_count, st) : mv4_t<false, 1, 2, 4>(p, a->E, sm_count, st);
    if (rc != ANIMA_OK) return rc;
  }
  return ANIMA_OK;
}

}  // namespace anima
