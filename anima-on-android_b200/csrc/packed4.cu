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
// 132 M bf16 values take 61 us (5.6 TB/s; 52 at the copy rate), bound by the integer pipe.  With tests
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
__device__ __forceinline__ void quantize_unit(const Quant4Params& p, long long u, const uint4& v, uint32_t mask) {
  constexpr uint32_t kSign = 0x80008000u;
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
  p.codes[(u & ~15ll) + 4 * (u & 3) + ((u >> 2) & 3)] = fine ? w : 0x88888888u;
  if ((u & 3) == 0) p.scales[u >> 2] = s;
}

template <bool kBf16, bool kContiguous>
__global__ void __launch_bounds__(256) quantize4_kernel(const Quant4Params p) {
  // units is a multiple of 16, so the lanes of a group leave the loop together
  constexpr int kStep = 256;  // a block takes runs of 512 units (rounds spread over the grid: 65 us against 61)
  const long long first = (long long)blockIdx.x * (2 * kStep) + threadIdx.x;
  for (long long u = first; u < p.units; u += (long long)gridDim.x * (2 * kStep)) {
    const uint32_t mask = __activemask();
    const bool two = u + kStep < p.units;
    const uint4 v0 = __ldg(unit_ptr<kContiguous>(p, u));
    uint4 v1 = make_uint4(0u, 0u, 0u, 0u);
    if (two) v1 = __ldg(unit_ptr<kContiguous>(p, u + kStep));
    quantize_unit<kBf16>(p, u, v0, mask);
    if (two) quantize_unit<kBf16>(p, u + kStep, v1, __activemask());
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
// fp32 rows and SiLU's results (kDigits) are four columns each of the whole-number MMA m16n8k32.  Per
// group of 32, x is scaled by the power of two that takes the largest below 2^30, rounded to a whole
// number and written in four signed base-256 digits, so nothing above 2^-31 of the group's largest
// magnitude is lost, more than an fp32 sum keeps.  A word's codes are its bytes' halves, c = n + 8, three
// instructions for eight where bf16 takes eleven; the 8 goes into the accumulator's start value, -8
// sum(digits), together with the 1.5 * 2^23 that makes the whole sum an fp32's low bits.
//
// 84 matrices of 6144 x 256 with two fp32 rows take 19.6 us (4.0 TB/s of codes, scales and results; 12 at
// the copy rate): 194 instructions a block of 16 x 128 weights at 0.65 a cycle and scheduler, of which
// the tile's ends are a fifth with two blocks a row, and about 3 us of start, when x is staged.
// As three bf16 columns a row, codes unpacked to bf16, they took 24.  One 6144 x 2048 matrix and row
// takes 5.1 us, one 21504 x 2048 with SiLU and two rows 10.8.
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

enum { kF16 = 0, kBf16 = 1, kDigits = 2 };

// Bytes between staged columns, and of all staged data.
template <int kMode>
__host__ __device__ constexpr int mv4_stride(int K) {
  return kMode == kDigits ? K + 32 : 2 * K + 64;
}
template <int kMode>
__host__ __device__ constexpr size_t mv4_staged(int M, int K, int nb) {
  return kMode == kDigits ? (size_t)4 * M * mv4_stride<kMode>(K) + (size_t)(K / 32) * nb * 72
                          : (size_t)M * mv4_stride<kMode>(K);
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
    for (int k = 0; k < 8; ++k) v[k] = __fdividef(v[k], 1.0f + expf(-v[k]));
}

// Stages the rows of x as digits.  A lane takes 8 values; the four lanes of a group share its
// exponent.  cols: digit q of value e at [4 m + q][32 g + 8 i + place of e], in the order in which the
// code words' halves come (values 0 4 1 5, then 2 6 3 7).  start[g][pair of columns]: the start values of
// a lane's four accumulators; xscale[g][m]: the group's scale 2^(E - 6), E with largest magnitude
// below 2^E.
__device__ __forceinline__ void stage_digits(const Mv4Params& p, int e, int nb, uint8_t* cols, uint4* start,
                                             float* xscale) {
  const int stride = mv4_stride<kDigits>(p.K), runs = p.K / 8;
  for (int c = threadIdx.x; c < p.M * runs; c += kMvThreads) {
    const uint32_t mask = __activemask();  // K / 8 is a multiple of 16: a group's lanes stay together
    const int m = c / runs, r = c - m * runs;
    float v[8];
    load_x8(p, (long long)e * p.xe + (long long)m * p.xm + 8 * r, v);
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(v[k]) & 0x7fffffffu);
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) top = max(top, __shfl_xor_sync(mask, top, o));
    const int E = max((int)(top >> 23), 1) - 126;
    uint32_t t[8];
    float scale;
    if (top < 0x7f800000u) {
      const int s0 = (30 - E) / 2, s1 = 30 - E - s0;  // in two steps: neither leaves fp32
      const float f0 = __int_as_float((s0 + 127) << 23), f1 = __int_as_float((s1 + 127) << 23);
#pragma unroll
      for (int k = 0; k < 8; ++k)  // the signed digits as bytes: add 128 to the lower three, then flip
        t[k] = ((uint32_t)__float2int_rn(v[k] * f0 * f1) + 0x00808080u) ^ 0x00808080u;
      scale = E - 6 >= -126 ? __int_as_float((E - 6 + 127) << 23) : __int_as_float(1 << (E - 6 + 149));
    } else {
      // one infinity makes its products infinite or NaN and hides the rest; anything else is NaN
      int odd = 0;  // infinities of the group, two for a NaN
#pragma unroll
      for (int k = 0; k < 8; ++k) odd += isnan(v[k]) ? 2 : isinf(v[k]) ? 1 : 0;
      const uint32_t group = 0xfu << (threadIdx.x & 28);  // its four lanes come here together
      odd += __shfl_xor_sync(group, odd, 1);
      odd += __shfl_xor_sync(group, odd, 2);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        t[k] = isinf(v[k]) ? (v[k] > 0.f ? 0x01010101u : 0xffffffffu) : 0u;
      scale = odd == 1 ? INFINITY : NAN;
    }
    uint32_t sum[4];
    const int g = r >> 2, i = r & 3;
#pragma unroll
    for (int q = 0; q < 4; ++q) {  // digit q is byte 3 - q
      const uint32_t sel = (uint32_t)(3 - q) | (uint32_t)(7 - q) << 4;
      const uint32_t lo = __byte_perm(__byte_perm(t[0], t[4], sel), __byte_perm(t[1], t[5], sel), 0x5410);
      const uint32_t hi = __byte_perm(__byte_perm(t[2], t[6], sel), __byte_perm(t[3], t[7], sel), 0x5410);
      *reinterpret_cast<uint2*>(cols + (size_t)(4 * m + q) * stride + 32 * g + 8 * i) = make_uint2(lo, hi);
      int s = __dp4a((int)lo, 0x01010101, __dp4a((int)hi, 0x01010101, 0));
      s += __shfl_xor_sync(mask, s, 1);
      s += __shfl_xor_sync(mask, s, 2);
      sum[q] = 0x4b400000u - 8u * (uint32_t)s;
    }
    if (i < 2)  // pair 2 m: digits 0 and 1; pair 2 m + 1: digits 2 and 3
      start[g * 4 * nb + 2 * m + i] = i ? make_uint4(sum[2], sum[3], sum[2], sum[3]) : make_uint4(sum[0], sum[1], sum[0], sum[1]);
    if (i == 2) xscale[g * 2 * nb + m] = scale;
  }
}

// kNB: blocks of eight columns (two fp32 rows or eight 16-bit ones); kStages: ring stages (4; 2 for rows
// so long that their columns need the room).  Columns without a row repeat another one's data:
// columns do not mix.
template <int kMode, int kNB, int kStages>
__global__ void __launch_bounds__(kMvThreads, 3) matvec4_kernel(const Mv4Params p) {
  extern __shared__ __align__(128) uint8_t smem[];
  grid_dependency_wait();  // launched while the kernel before it drains
  constexpr bool kDig = kMode == kDigits;
  constexpr int kOuts = kDig ? 1 : 4;  // results of a lane per block of columns
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int j = lane >> 2, i = lane & 3;
  const int stride = mv4_stride<kMode>(p.K);
  const uint32_t ring = smem_u32(smem) + warp * kStages * kMvStage;
  float* const red = reinterpret_cast<float*>(smem + 8 * kStages * kMvStage);
  uint8_t* const cols = reinterpret_cast<uint8_t*>(red + 8 * 32 * kNB * kOuts);
  uint4* const start = reinterpret_cast<uint4*>(cols + (size_t)4 * p.M * stride);  // kDigits
  float* const xscale = reinterpret_cast<float*>(start + (p.K / 32) * 4 * kNB);
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

  if constexpr (kDig) {
    stage_digits(p, e, kNB, cols, start, xscale);
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
    const int col = kDig ? 4 * min(nb * 2 + (j >> 2), p.M - 1) + (j & 3) : min(nb * 8 + j, p.M - 1);
    xa[nb] = smem_u32(cols) + col * stride + (kDig ? 8 : 16) * i;
  }
  const uint32_t sa = smem_u32(start) + 16 * i, fa = smem_u32(xscale) + 4 * (i >> 1);
  __syncthreads();

  // Result r of this lane for column block nb is row `row + out_row(r)`, row m = out_m(nb, r) of x.
  auto out_row = [&](int r) { return kDig ? 0 : 8 * (r >> 1); };
  auto out_m = [&](int nb, int r) { return kDig ? nb * 2 + (i >> 1) : nb * 8 + 2 * i + (r & 1); };
  int row = (g_lo * tiles + t) * 16 + j + (kDig ? 8 * (i & 1) : 0);
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
    uint64_t acc2[kNB][2];  // kDigits: the same as pairs
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
        if constexpr (kDig) {
          constexpr uint32_t kHalf = 0x0f0f0f0fu;
          const uint32_t a0 = w0[g] & kHalf, a2 = (w0[g] >> 4) & kHalf;
          const uint32_t a1 = w1[g] & kHalf, a3 = (w1[g] >> 4) & kHalf;
#pragma unroll
          for (int nb = 0; nb < kNB; ++nb) {
            const uint2 xv = p4::lds8(xa[nb] + blk * p4::kBlock + 32 * g);
            const uint4 c4 = p4::lds16(sa + ((blk * 4 + g) * kNB + nb) * 64);
            const float sx = p4::lds4(fa + ((blk * 4 + g) * kNB + nb) * 8);
            int d[4];
            p4::mma16832(d, a0, a1, a2, a3, xv.x, xv.y, c4);
            const float s0 = g0[g] * sx, s1 = g1[g] * sx;
            const uint64_t off = f2pack(-12582912.f, -12582912.f);
            const uint64_t v0 = add2(f2pack(__int_as_float(d[0]), __int_as_float(d[1])), off);
            const uint64_t v1 = add2(f2pack(__int_as_float(d[2]), __int_as_float(d[3])), off);
            acc2[nb][0] = fma2(f2pack(s0, s0), v0, acc2[nb][0]);
            acc2[nb][1] = fma2(f2pack(s1, s1), v1, acc2[nb][1]);
          }
        } else {
          uint32_t a[4], b[4];
          p4::numbers<kMode == kBf16>(w0[g], a);
          p4::numbers<kMode == kBf16>(w1[g], b);
#pragma unroll
          for (int nb = 0; nb < kNB; ++nb) {
            const uint4 xv = p4::lds16(xa[nb] + blk * (2 * p4::kBlock) + 64 * g);
            float d[4];
            p4::mma16816_zero<kMode == kBf16>(d, a[0], b[0], a[1], b[1], xv.x, xv.y);
            p4::mma16816<kMode == kBf16>(d, a[2], b[2], a[3], b[3], xv.z, xv.w);
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[nb][c] = fmaf(c < 2 ? g0[g] : g1[g], d[c], acc[nb][c]);
          }
        }
      }
    }
#pragma unroll
    for (int nb = 0; nb < kNB; ++nb) {
      if constexpr (kDig) {  // digits 2 (i % 2) and the next of rows j and j + 8, then the other lane's
        const float f = (i & 1) ? 1.52587890625e-05f : 1.0f;  // 2^-16
        f2unpack(acc2[nb][0], acc[nb][0], acc[nb][1]);
        f2unpack(acc2[nb][1], acc[nb][2], acc[nb][3]);
        float v0 = fmaf(acc[nb][1], 0.00390625f, acc[nb][0]) * f;
        float v1 = fmaf(acc[nb][3], 0.00390625f, acc[nb][2]) * f;
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
// 32 blocks an SM and 65 with 8; packing is capped at 64 blocks an SM: 61 us, 68 without, 71 with 8.
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

constexpr size_t kMaxSmem = 227 * 1024;
constexpr size_t mv4_fixed_smem(int nb, int outs, int stages) {
  return 8 * stages * kMvStage + 8 * 32 * nb * outs * sizeof(float);
}

template <int kMode, int kNB, int kStages>
static int mv4_t(Mv4Params p, int E, int sm_count, cudaStream_t st) {
  auto kern = matvec4_kernel<kMode, kNB, kStages>;
  const size_t smem = mv4_fixed_smem(kNB, kMode == kDigits ? 1 : 4, kStages) + mv4_staged<kMode>(p.M, p.K, kNB);
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
static int mv4_rows(int K, bool digits, int* stages) {
  *stages = 4;
  for (int m = digits ? 8 : 16; m > 0; --m) {
    const size_t staged = digits ? mv4_staged<kDigits>(m, K, m <= 2 ? 1 : m <= 4 ? 2 : 4) : mv4_staged<kF16>(m, K, 1);
    if (staged + mv4_fixed_smem(digits ? 4 : 2, digits ? 1 : 4, 4) <= kMaxSmem) return m;
  }
  *stages = 2;
  const size_t staged = digits ? mv4_staged<kDigits>(1, K, 1) : mv4_staged<kF16>(1, K, 1);
  return staged + mv4_fixed_smem(1, digits ? 1 : 4, 2) <= kMaxSmem ? 1 : 0;
}

int matvec4_launch(const AnimaMatvec4Args* a, int sm_count, cudaStream_t st) {
  const bool digits = a->x_dtype == ANIMA_DTYPE_F32 || a->silu;
  int stages;
  const int rows = mv4_rows(a->K, digits, &stages);
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
      rc = digits ? mv4_t<kDigits, 1, 2>(p, a->E, sm_count, st)
           : bf   ? mv4_t<kBf16, 1, 2>(p, a->E, sm_count, st)
                  : mv4_t<kF16, 1, 2>(p, a->E, sm_count, st);
    else if (digits)
      rc = p.M <= 2   ? mv4_t<kDigits, 1, 4>(p, a->E, sm_count, st)
           : p.M <= 4 ? mv4_t<kDigits, 2, 4>(p, a->E, sm_count, st)
                      : mv4_t<kDigits, 4, 4>(p, a->E, sm_count, st);
    else if (bf)
      rc = one ? mv4_t<kBf16, 1, 4>(p, a->E, sm_count, st) : mv4_t<kBf16, 2, 4>(p, a->E, sm_count, st);
    else
      rc = one ? mv4_t<kF16, 1, 4>(p, a->E, sm_count, st) : mv4_t<kF16, 2, 4>(p, a->E, sm_count, st);
    if (rc != ANIMA_OK) return rc;
  }
  return ANIMA_OK;
}

}  // namespace anima
