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
// Replayed from a graph, 132 M bf16 values take 59 us (5.7 TB/s; 52 at the copy rate), bound by the integer pipe.  With tests
// of every value, clamps on both sides and a true reciprocal they took 106 (at 71 otherwise).
struct Quant4Params {
  const void* x;
  uint32_t* codes;
  __half* scales;
  long long n1, n2;           // inner row counts: row = (a * n1 + b) * n2 + c
  long long s0, s1, s2;       // element strides of a, b, c
  long long units;            // rows * K / 8
  int upr;                    // units per row, K / 8
};

template <bool kBf16>
__device__ __forceinline__ float2 widen2(uint32_t w) {
  if (kBf16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
// Pairwise maximum and minimum; NaN wins.
template <bool kBf16>
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  uint32_t r;
  if (kBf16)
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <bool kBf16>
__device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) {
  uint32_t r;
  if (kBf16)
    asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else
    asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

template <bool kContiguous>
__device__ __forceinline__ const uint4* unit_ptr(const Quant4Params& p, long long u) {
  const uint16_t* x = static_cast<const uint16_t*>(p.x);
  if (kContiguous) return reinterpret_cast<const uint4*>(x + 8 * u);
  const long long row = u / p.upr;
  const long long c = row % p.n2, ab = row / p.n2;
  return reinterpret_cast<const uint4*>(x + (ab / p.n1) * p.s0 + (ab % p.n1) * p.s1 + c * p.s2 +
                                        8 * (u - row * p.upr));
}

template <bool kBf16>
__device__ __forceinline__ void quantize_unit(const Quant4Params& p, long long u, const uint4& v, bool store) {
  constexpr uint32_t kSign = 0x80008000u, mask = 0xffffffffu;
  const uint32_t w4[4] = {v.x, v.y, v.z, v.w};
  const uint32_t hi2 = max2<kBf16>(max2<kBf16>(v.x, v.y), max2<kBf16>(v.z, v.w));
  const uint32_t lo2 = min2<kBf16>(min2<kBf16>(v.x, v.y), min2<kBf16>(v.z, v.w)) ^ kSign;
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
  if (store) {
    p.codes[(u & ~15ll) + 4 * (u & 3) + ((u >> 2) & 3)] = fine ? w : 0x88888888u;
    if ((u & 3) == 0) p.scales[u >> 2] = s;
  }
}

template <bool kBf16, bool kContiguous>
__global__ void __launch_bounds__(256) quantize4_kernel(const Quant4Params p) {
  // A warp's lanes stay together to its last unit: those past the end (the upper half of a warp at most, units
  // being a multiple of 16) exchange zeros and store nothing.  (Masks per group of four lanes: 84 us against 57.)
  constexpr int kStep = 256;  // a block takes runs of 512 units (rounds spread over the grid: 65 us against 61)
  const int lane = threadIdx.x & 31;
  const long long first = (long long)blockIdx.x * (2 * kStep) + (threadIdx.x - lane);
  for (long long w = first; w < p.units; w += (long long)gridDim.x * (2 * kStep)) {
    const long long u = w + lane;
    if (w + kStep + 32 <= p.units) {
      const uint4 v0 = __ldg(unit_ptr<kContiguous>(p, u)), v1 = __ldg(unit_ptr<kContiguous>(p, u + kStep));
      quantize_unit<kBf16>(p, u, v0, true);
      quantize_unit<kBf16>(p, u + kStep, v1, true);
      continue;
    }
    const bool one = u < p.units, two = u + kStep < p.units;
    uint4 v0 = make_uint4(0u, 0u, 0u, 0u), v1 = v0;
    if (one) v0 = __ldg(unit_ptr<kContiguous>(p, u));
    if (two) v1 = __ldg(unit_ptr<kContiguous>(p, u + kStep));
    quantize_unit<kBf16>(p, u, v0, one);
    if (w + kStep < p.units) quantize_unit<kBf16>(p, u + kStep, v1, two);
  }
}

// ---------------------------------------------------------------- unpacking
// One lane per run of 8 values, in value order, so a warp's stores are one contiguous run (with
// a lane per 16 bytes of codes, each store touched eight 64-byte pieces: 110 us against 65 for
// 132 M values to bf16; now 56, 6.0 TB/s).  Value run v of a block (v = 4 g + i) is word 4 i + g of its codes.  n * s
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

// Runs per lane and round, loaded before any is converted (132 M values: bf16 in 56 us with four, 58 with
// two, 80 with one; fp32 in 139 with four, 128 with two).
__host__ __device__ constexpr int deq_runs(int dtype) { return dtype == ANIMA_DTYPE_F32 ? 2 : 4; }

template <int kDt>
__global__ void __launch_bounds__(256)
    dequantize4_kernel(const uint32_t* __restrict__ codes, const __half* __restrict__ scales, void* y,
                       long long words) {
  constexpr int kU = deq_runs(kDt);
  constexpr int step = 256;
  const long long first = (long long)blockIdx.x * (kU * step) + threadIdx.x;
  for (long long u0 = first; u0 < words; u0 += (long long)gridDim.x * (kU * step)) {
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
// Sixteen rows of W are the A operand of an MMA and the rows x its columns, so eight columns
// cost what one does, and every product is of whole numbers and exact (packed4.cuh); a group's sum
// is multiplied by the group's scale in fp32.
//
// 16-bit rows (kF16, kBf16) are a column each of m16n8k16, codes unpacked to n in their type.
//
// fp32 rows and SiLU's results (kParts) are three bf16 columns each: a value cut after 8 and after 16 bits is
// the exact sum of three bf16, whatever stands beside it.  Per group of 32, x is first scaled by the power of
// two that takes the largest to 2^100 (2^126 at most), so that sums of parts stay in fp32's range and the
// lowest parts in bf16's.  (As whole numbers of 2^-30 of a group's largest value, in four base-256 digits for the
// whole-number MMA, 84 x 6144 x 256 took a fifth less, and values far below the group's largest lost their bits.)
//
// Replayed from a graph, 84 matrices of 6144 x 256 with two fp32 rows take 23.4 us (3.3 TB/s of codes, scales and results; 12 at
// the copy rate), bound by instruction issue, the unpacking to bf16 first, and some 3 us of start, when x
// is staged.  One 6144 x 2048 matrix and row takes 5.7 us, one 21504 x 2048 with SiLU and two rows 12.6.
//
// A CTA of 8 warps works on one matrix, on a run of tiles of 16 rows of W; `split` warps share a
// tile, taking its 128-value blocks in turn, and their sums meet in shared memory in a fixed
// order.  A warp streams its blocks (1 KB of codes, 128 bytes of scales) through a private ring
// of cp.async stages that runs on across tiles; each lane fetches the codes that it will read
// itself.  The columns are staged in shared memory once, with a row stride that spreads the columns
// that a wavefront reads over all banks.
struct Mv4Params {
  const void* x;
  const uint8_t* codes;
  const __half* scales;
  const float* add;
  void* out;
  long long xe, xm, ae, am, oe, om;
  int N, K, M;
  int parts;             // CTAs per matrix
  int g_each, g_more;    // tile groups (8 / split tiles) of a CTA; the first g_more have one more
  int log_split;         // log2 of the warps per tile
  int silu, x_dtype, out_dtype;
  int x_aligned;         // every row of x starts on 16 bytes
};

constexpr int kMvThreads = 256;
constexpr int kMvStage = 16 * 64 + 16 * 8;  // bytes of a block of 16 rows

__device__ __forceinline__ float load_x(const Mv4Params& p, long long at) {
  if (p.x_dtype == ANIMA_DTYPE_F32) return __ldg(static_cast<const float*>(p.x) + at);
  const uint16_t u = __ldg(static_cast<const uint16_t*>(p.x) + at);
  return p.x_dtype == ANIMA_DTYPE_BF16 ? __uint_as_float((uint32_t)u << 16)
                                       : __half2float(__ushort_as_half(u));
}

enum { kF16 = 0, kBf16 = 1, kParts = 2 };

// Bytes between staged columns, and of all staged data.
__host__ __device__ constexpr int mv4_stride(int K) {
  return 2 * K + 64;
}
template <int kMode>
__host__ __device__ constexpr size_t mv4_staged(int M, int K, int nb) {
  return kMode == kParts ? (size_t)3 * M * mv4_stride(K) + (size_t)(K / 32) * nb * 8 : (size_t)M * mv4_stride(K);
}

// Eight values of x, SiLU applied if asked for.
__device__ __forceinline__ void load_x8(const Mv4Params& p, long long at, float (&v)[8]) {
  if (p.x_dtype == ANIMA_DTYPE_F32 && p.x_aligned) {
    const float4* x = reinterpret_cast<const float4*>(static_cast<const float*>(p.x) + at);
    const float4 a = __ldg(x), b = __ldg(x + 1);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = load_x(p, at + k);
  }
  if (p.silu)
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = v[k] / (1.0f + expf(-v[k]));  // a true quotient: __fdividef is 0 from 2^126 on
}

// Stages the rows of x in three parts.  A lane takes 8 values; the four lanes of a group share its scale.
// cols: part q of row m at column 3 m + q; xscale[g][m]: what the group's sums are multiplied by, 2^-a.
__device__ __forceinline__ void stage_parts(const Mv4Params& p, int e, int nb, uint8_t* cols, float* xscale) {
  const int stride = mv4_stride(p.K), runs = p.K / 8;
  const uint32_t group = 0xfu << (threadIdx.x & 28);  // K / 8 is a multiple of 16: its lanes stay together
  for (int c = threadIdx.x; c < p.M * runs; c += kMvThreads) {
    const int m = c / runs, r = c - m * runs;
    float v[8];
    load_x8(p, (long long)e * p.xe + (long long)m * p.xm + 8 * r, v);
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(v[k]) & 0x7fffffffu);
    top = max(top, __shfl_xor_sync(group, top, 1));
    top = max(top, __shfl_xor_sync(group, top, 2));
    const bool finite = top < 0x7f800000u;
    const int E = max((int)(top >> 23), 1) - 126;  // largest magnitude below 2^E
    const int a = finite ? min(100 - E, 126) : 0;
    const float f = __int_as_float((a + 127) << 23);
    uint32_t part[3][8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float y = v[k] * f;
      part[0][k] = __float_as_uint(y) & 0xffff0000u;
      const float y1 = y - __uint_as_float(part[0][k]);
      part[1][k] = __float_as_uint(y1) & 0xffff0000u;
      part[2][k] = __float_as_uint(y1 - __uint_as_float(part[1][k]));
      if (!finite) {  // infinities and NaN decide the sums alone
        part[0][k] = isnan(v[k]) ? 0x7fff0000u : isinf(v[k]) ? __float_as_uint(v[k]) : 0u;
        part[1][k] = part[2][k] = 0u;
      }
    }
#pragma unroll
    for (int q = 0; q < 3; ++q)
      *reinterpret_cast<uint4*>(cols + (size_t)(3 * m + q) * stride + 16 * r) =
          make_uint4(__byte_perm(part[q][0], part[q][1], 0x7632), __byte_perm(part[q][2], part[q][3], 0x7632),
                     __byte_perm(part[q][4], part[q][5], 0x7632), __byte_perm(part[q][6], part[q][7], 0x7632));
    if ((r & 3) == 0) xscale[(r >> 2) * 2 * nb + m] = __int_as_float((127 - a) << 23);
  }
}

// kNB: blocks of eight columns (two fp32 rows or eight 16-bit ones); kStages: ring stages (4; 2 for rows
// so long that their columns need the room).  Columns without a row repeat another one's data:
// columns do not mix.
template <int kMode, int kNB, int kStages>
__global__ void __launch_bounds__(kMvThreads, 3) matvec4_kernel(const Mv4Params p) {
  extern __shared__ __align__(128) uint8_t smem[];
  grid_dependency_wait();  // launched while the kernel before it drains
  constexpr bool kWide = kMode == kParts;
  constexpr int kOuts = kWide ? 1 : 4;  // results of a lane per block of columns
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int j = lane >> 2, i = lane & 3;
  const int stride = mv4_stride(p.K);
  const uint32_t ring = smem_u32(smem) + warp * kStages * kMvStage;
  float* const red = reinterpret_cast<float*>(smem + 8 * kStages * kMvStage);
  uint8_t* const cols = reinterpret_cast<uint8_t*>(red + 8 * 32 * kNB * kOuts);
  float* const xscale = reinterpret_cast<float*>(cols + (size_t)3 * p.M * stride);  // kParts
  const int split = 1 << p.log_split;
  const int s = warp & (split - 1), t = warp >> p.log_split, tiles = 8 >> p.log_split;
  const int blocks = p.K / p4::kBlock;
  const int e = blockIdx.x / p.parts, part = blockIdx.x - e * p.parts;
  const int g_lo = part * p.g_each + min(part, p.g_more), g_hi = g_lo + p.g_each + (part < p.g_more ? 1 : 0);

  // The block sequence of this warp: (group, block) with block = s, s + split, ...  A lane
  // fetches its 16 bytes of rows j and j + 8, lanes i = 0, 1 their scales.  Rows past the
  // matrix repeat its last one; their results are not stored.
  const uint8_t* const codes = p.codes + (long long)e * p.N * (p.K / 2) + i * 16;
  const uint8_t* const scales = reinterpret_cast<const uint8_t*>(p.scales) + (long long)e * p.N * (p.K / 16);
  const uint8_t *c0 = codes, *c1 = codes, *sp = scales;
  int ld_g = g_lo, ld_blk = s;
  uint32_t ld_at = ring;
  const int tile_rows = 16 * tiles;  // from a warp's tile to its next
  const int rounds = ((blocks - s - 1) >> p.log_split) + 1;
  const long long c_next = (long long)tile_rows * (p.K / 2) - (long long)rounds * split * 64;
  const long long s_next = (long long)tile_rows * (p.K / 16) - (long long)rounds * split * 8;
  int ld_n = (g_lo * tiles + t) * 16;  // first row of the tile being fetched
  auto tile_start = [&]() {
    const int n0 = min(ld_n + j, p.N - 1), n1 = min(ld_n + j + 8, p.N - 1);
    c0 = codes + (long long)n0 * (p.K / 2) + s * 64;
    c1 = codes + (long long)n1 * (p.K / 2) + s * 64;
    sp = scales + (long long)(i == 0 ? n0 : n1) * (p.K / 16) + s * 8;
  };
  auto fetch = [&]() {
    if (ld_g < g_hi) {
      p4::cp16(ld_at + lane * 16, c0);
      p4::cp16(ld_at + 512 + lane * 16, c1);
      if (i < 2) p4::cp8(ld_at + 1024 + (i * 8 + j) * 8, sp);
      c0 += split * 64;
      c1 += split * 64;
      sp += split * 8;
      ld_blk += split;
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

  if constexpr (kWide) {
    stage_parts(p, e, kNB, cols, xscale);
  } else {  // 16-bit rows as they are
    const uint16_t* const x = static_cast<const uint16_t*>(p.x) + (long long)e * p.xe;
    if (p.x_aligned) {
      const int runs = p.K / 8;
      for (int c = threadIdx.x; c < p.M * runs; c += kMvThreads) {
        const int m = c / runs, r = c - m * runs;
        p4::cp16(smem_u32(cols) + m * stride + 16 * r, x + (long long)m * p.xm + 8 * r);
      }
      p4::cp_commit();
      p4::cp_wait<0>();
    } else {
      for (int m = 0; m < p.M; ++m) {
        uint16_t* const to = reinterpret_cast<uint16_t*>(cols + (size_t)m * stride);
#pragma unroll 4
        for (int k = threadIdx.x; k < p.K; k += kMvThreads) to[k] = __ldg(x + (long long)m * p.xm + k);
      }
    }
  }
  uint32_t xa[kNB];  // this lane's column of x, at its eight values of a group
#pragma unroll
  for (int nb = 0; nb < kNB; ++nb) {
    const int col = kWide ? 3 * min(nb * 2 + (j >> 2), p.M - 1) + min(j & 3, 2) : min(nb * 8 + j, p.M - 1);
    xa[nb] = smem_u32(cols) + col * stride + 16 * i;
  }
  const uint32_t fa = smem_u32(xscale) + 4 * (i >> 1);
  __syncthreads();

  // Result r of this lane for column block nb is row `row + out_row(r)`, row m = out_m(nb, r) of x.
  auto out_row = [&](int r) { return kWide ? 0 : 8 * (r >> 1); };
  auto out_m = [&](int nb, int r) { return kWide ? nb * 2 + (i >> 1) : nb * 8 + 2 * i + (r & 1); };
  int row = (g_lo * tiles + t) * 16 + j + (kWide ? 8 * (i & 1) : 0);
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
          y[nb][r] = p.add[add_at[nb] + (r & 1) * p.am + out_row(r)];  // may be out: a plain load
      }
    float acc[kNB][4];
#pragma unroll
    for (int b = 0; b < kNB; ++b)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[b][c] = 0.f;
    uint64_t acc2[kNB][2];  // kParts: the same as pairs
#pragma unroll
    for (int b = 0; b < kNB; ++b) acc2[b][0] = acc2[b][1] = 0ull;
    for (int blk = s; blk < blocks; blk += split) {
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
        p4::numbers<kMode != kF16>(w0[g], a);
        p4::numbers<kMode != kF16>(w1[g], b);
#pragma unroll
        for (int nb = 0; nb < kNB; ++nb) {
          const uint4 xv = p4::lds16(xa[nb] + blk * (2 * p4::kBlock) + 64 * g);
          float d[4];
          p4::mma16816_zero<kMode != kF16>(d, a[0], b[0], a[1], b[1], xv.x, xv.y);
          p4::mma16816<kMode != kF16>(d, a[2], b[2], a[3], b[3], xv.z, xv.w);
          if constexpr (kWide) {  // the scale of W first: that of x may be near fp32's ends
            const float sx = p4::lds4(fa + ((blk * 4 + g) * kNB + nb) * 8);
            const uint64_t s0 = f2pack(g0[g], g0[g]), s1 = f2pack(g1[g], g1[g]), sx2 = f2pack(sx, sx);
            acc2[nb][0] = fma2(fma2(f2pack(d[0], d[1]), s0, 0ull), sx2, acc2[nb][0]);
            acc2[nb][1] = fma2(fma2(f2pack(d[2], d[3]), s1, 0ull), sx2, acc2[nb][1]);
          } else {
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[nb][c] = fmaf(c < 2 ? g0[g] : g1[g], d[c], acc[nb][c]);
          }
        }
      }
    }
#pragma unroll
    for (int nb = 0; nb < kNB; ++nb) {
      if constexpr (kWide) {  // parts 0 and 1 of rows j and j + 8, or part 2 (twice), and the other lane's
        f2unpack(acc2[nb][0], acc[nb][0], acc[nb][1]);
        f2unpack(acc2[nb][1], acc[nb][2], acc[nb][3]);
        float v0 = (i & 1) ? acc[nb][0] : acc[nb][0] + acc[nb][1];
        float v1 = (i & 1) ? acc[nb][2] : acc[nb][2] + acc[nb][3];
        v0 += __shfl_xor_sync(0xffffffffu, v0, 1);
        v1 += __shfl_xor_sync(0xffffffffu, v1, 1);
        y[nb][0] += (i & 1) ? v1 : v0;
      } else {
#pragma unroll
        for (int r = 0; r < kOuts; ++r) y[nb][r] += acc[nb][r];
      }
    }
    if (split > 1) {  // the warps of a tile are neighbours: the first adds the others' results
#pragma unroll
      for (int nb = 0; nb < kNB; ++nb)
#pragma unroll
        for (int r = 0; r < kOuts; ++r) red[((warp * kNB + nb) * kOuts + r) * 32 + lane] = y[nb][r];
      __syncthreads();
      if (s == 0)
        for (int q = 1; q < split; ++q)
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
    if (split > 1) __syncthreads();  // the sums are read before the next tile's are written
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
// Blocks of a streaming kernel that takes one round each.  132 M values (bf16) unpack in 56 us so, 59 with
// 32 blocks an SM and 65 with 8; packing is capped at 64 blocks an SM (by an earlier form: 61 us, 68 without, 71 with 8).
static int stream_grid(long long work, int per_block) {
  return (int)std::min<long long>((work + per_block - 1) / per_block, 1 << 30);
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
  // rows K elements apart: unit u starts at 8 u
  const bool contiguous = (n2 == 1 || s2 == K) && (n1 == 1 || s1 == n2 * K) && (n0 == 1 || s0 == n1 * n2 * K);
  const int grid = std::min(64 * sm_count, stream_grid(p.units, 512));
  if (dtype == ANIMA_DTYPE_BF16)
    (contiguous ? quantize4_kernel<true, true> : quantize4_kernel<true, false>)<<<grid, 256, 0, st>>>(p);
  else
    (contiguous ? quantize4_kernel<false, true> : quantize4_kernel<false, false>)<<<grid, 256, 0, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? ANIMA_OK : ANIMA_ERR_CUDA;
}

int dequantize4_launch(const void* codes, const void* scales, void* y, int dtype, long long rows,
                       int K, cudaStream_t st) {
  const long long words = rows * (K / 8);
  const int grid = stream_grid(words, 256 * deq_runs(dtype));
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

constexpr size_t mv4_fixed_smem(int nb, int outs, int stages) {
  return 8 * stages * kMvStage + 8 * 32 * nb * outs * sizeof(float);
}

template <int kMode, int kNB, int kStages>
static int mv4_t(Mv4Params p, int E, int sm_count, cudaStream_t st) {
  auto kern = matvec4_kernel<kMode, kNB, kStages>;
  const size_t smem = mv4_fixed_smem(kNB, kMode == kParts ? 1 : 4, kStages) + mv4_staged<kMode>(p.M, p.K, kNB);
  if (smem > kMaxSmem) return ANIMA_ERR_SHAPE;
  static SmemAttr attr;
  if (!attr.raise((const void*)kern, smem)) return ANIMA_ERR_CUDA;
  // Warps that share a tile, and CTAs per matrix: the split whose busiest warp has the least to do,
  // in blocks, a tile's ends counted as one.
  const int ntiles = (p.N + 15) / 16, blocks = p.K / p4::kBlock;
  const int per_sm = std::max(1, std::min(3, (int)(kMaxSmem / (smem + 1024))));
  const long long slots = (long long)per_sm * sm_count;
  long long best = 0;
  for (int lg = 0; lg <= 3 && (1 << lg) <= blocks; ++lg) {
    const int split = 1 << lg;
    const long long groups = ((long long)ntiles * split + 7) / 8;
    const long long parts = std::min(groups, std::max(1LL, slots / E));
    const long long waves = (E * parts + slots - 1) / slots;
    const long long cost = waves * ((groups + parts - 1) / parts) * ((blocks + split - 1) / split + 1);
    if (lg == 0 || cost < best) {
      best = cost;
      p.log_split = lg;
      p.parts = (int)parts;
      p.g_each = (int)(groups / parts);
      p.g_more = (int)(groups % parts);
    }
  }
  if ((long long)E * p.parts > 0x7fffffffLL) return ANIMA_ERR_SHAPE;
  return launch_dependent(kern, E * p.parts, kMvThreads, smem, st, p);
}

// Rows of x of one launch: eight fp32 rows or sixteen 16-bit ones; fewer where their columns
// would not fit shared memory, and a shorter ring where not even one would.
static int mv4_rows(int K, bool wide, int* stages) {
  *stages = 4;
  for (int m = wide ? 8 : 16; m > 0; --m) {
    const size_t staged = wide ? mv4_staged<kParts>(m, K, m <= 2 ? 1 : m <= 4 ? 2 : 4) : mv4_staged<kF16>(m, K, 1);
    if (staged + mv4_fixed_smem(wide ? 4 : 2, wide ? 1 : 4, 4) <= kMaxSmem) return m;
  }
  *stages = 2;
  const size_t staged = wide ? mv4_staged<kParts>(1, K, 1) : mv4_staged<kF16>(1, K, 1);
  return staged + mv4_fixed_smem(1, wide ? 1 : 4, 2) <= kMaxSmem ? 1 : 0;
}

int matvec4_launch(const AnimaMatvec4Args* a, int sm_count, cudaStream_t st) {
  const bool wide = a->x_dtype == ANIMA_DTYPE_F32 || a->silu;
  int stages;
  const int rows = mv4_rows(a->K, wide, &stages);
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
  p.x_aligned = ((reinterpret_cast<uintptr_t>(a->x) | (uintptr_t)(xs * p.xe) | (uintptr_t)(xs * p.xm)) & 15u) == 0;
  for (int m0 = 0; m0 < a->M; m0 += rows) {
    p.M = std::min(rows, a->M - m0);
    p.x = static_cast<const char*>(a->x) + m0 * p.xm * xs;
    p.out = static_cast<char*>(a->out) + m0 * p.om * os;
    p.add = a->add ? static_cast<const float*>(a->add) + m0 * p.am : nullptr;
    const bool bf = a->x_dtype == ANIMA_DTYPE_BF16, one = p.M <= 8;
    int rc;
    if (stages == 2)
      rc = wide ? mv4_t<kParts, 1, 2>(p, a->E, sm_count, st)
           : bf   ? mv4_t<kBf16, 1, 2>(p, a->E, sm_count, st)
                  : mv4_t<kF16, 1, 2>(p, a->E, sm_count, st);
    else if (wide)
      rc = p.M <= 2   ? mv4_t<kParts, 1, 4>(p, a->E, sm_count, st)
           : p.M <= 4 ? mv4_t<kParts, 2, 4>(p, a->E, sm_count, st)
                      : mv4_t<kParts, 4, 4>(p, a->E, sm_count, st);
    else if (bf)
      rc = one ? mv4_t<kBf16, 1, 4>(p, a->E, sm_count, st) : mv4_t<kBf16, 2, 4>(p, a->E, sm_count, st);
    else
      rc = one ? mv4_t<kF16, 1, 4>(p, a->E, sm_count, st) : mv4_t<kF16, 2, 4>(p, a->E, sm_count, st);
    if (rc != ANIMA_OK) return rc;
  }
  return ANIMA_OK;
}

}  // namespace anima
