// attn_kv4.cu -- attention over K and V held packed in 4 bits (format: packed4.cuh):
// out = softmax(q K^T * scale) V per (batch, head), D = 128, key-padding lengths per sample.
//
// Two ways, chosen by rows_path below:
//   little work: kv4_rows_kernel reads the packed cache directly, eight query rows at a time;
//   more:        attn_kv4_tile.cu, on the tensor cores, unpacks K and V in the kernel.
// Neither writes the cache out in 16 bits: scratch holds partial results only, of slices at most 64
// times 130 floats a query row, and of long chains 128 KB a CTA.
//
// kv4_rows_kernel.  One cluster per (batch, head, block of query rows); its CTAs and their
// warps take 32-key blocks in turn, each warp with its own running maximum, sum and output, so
// there is no synchronisation inside the loop.  A warp streams its blocks through a private ring
// of cp.async stages.  Per block:
//   S^T = K Q^T   m16n8k16 with 16 keys as rows and 8 query rows as columns.  The products of
//                 codes and 16-bit q are exact; a group's sum comes from a zeroed
//                 accumulator and is multiplied by the key's scale of that group in fp32.
//   P             exp2 of the scaled scores against a running maximum that only moves when a
//                 score exceeds it by more than 8 (a factor 256), as in the core kernel.
//   O^T += V^T P^T  16 dims as rows, 16 keys as k.  All rows of a tile lie in one group of V, so
//                 the key's scale of that group goes into P in fp32, and the product P s is
//                 split into two bf16 parts, hi + lo (16 bits of it): V's codes stay exact
//                 and small scales do not underflow, as they would in fp16.  movmatrix turns the
//                 accumulator's layout of P^T into the operand's.
// At the end the warps' outputs meet in shared memory, then the cluster's CTAs read one
// another's over distributed shared memory, each writing its share of the output.  Where heads are
// few and the cache long, several clusters share a unit's keys and write fp32 partials, which
// kv4_merge_kernel joins.  No atomics; the order of all sums is fixed.
//
// One row against 65536 keys, 32 heads: 60 us replayed from a graph, 5.0 TB/s of the cache (46 us at the copy
// rate), 67 a call whose inputs change; 65536 blocks of 32 keys take 544 instructions each, nearly half of them on the
// integer pipe, which takes one every other cycle.  One SM's two CTAs are no faster with more warps.  One
// row against 512 keys takes 5.3 us, seven rows against 1237 9.6 (calls from Python 10.7 and 11.3).
#include <algorithm>
#include <atomic>

#include "attn_kv4.cuh"
#include "packed4.cuh"

namespace anima {

namespace kv4 {

constexpr int kD = 128;
constexpr int kKeys = 32;                  // keys per block
constexpr int kCodeBytes = kKeys * 64;     // codes of one block of K or V
constexpr int kScaleBytes = kKeys * 8;
constexpr int kStageBytes = 2 * kCodeBytes + 2 * kScaleBytes;
constexpr float kRescale = 8.0f;           // log2 units

struct Params {
  const uint16_t* q;
  const uint8_t* kc;
  const uint8_t* ks;
  const uint8_t* vc;
  const uint8_t* vs;
  const int* valid;
  void* out;
  float* part;         // partials, or nullptr: write the output
  long long ob, oh, os;
  int H, S_q, S_kv;
  int nqb;             // units (blocks of query rows) per (batch, head)
  int units;
  int nsplit;          // clusters that share a unit's keys
  int out_f32;         // out is fp32, else of q's type
  float scale_log2;
};

using p4::cp16;
using p4::cp16_if;
using p4::cp8;
using p4::cp8_if;
using p4::cp_commit;
using p4::cp_wait;
using p4::lds16;
using p4::lds8;
template <bool kBf16>
__device__ __forceinline__ float2 widen(uint32_t w) {
  if (kBf16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
// Transposes an 8 x 8 matrix of 16-bit values held two to a lane (row lane / 4).
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float ld_cluster(uint32_t a) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}

template <int kW>
constexpr size_t smem_bytes(int stages, int rows) {
  const size_t ring = (size_t)kW * stages * kStageBytes;
  const size_t merge = (size_t)(kW + 1) * kv4_part_floats(rows) * sizeof(float);
  return ring > merge ? ring : merge;
}

// kBf16: type of q and out (else fp16); kOne: the form for a single row, else up to eight; kW:
// warps; kNS: stages.
//
// A single row has the eight columns to itself.  For S^T its q is scaled by a power of two below 2^30, and
// the whole part and 2^31 times the rest are written in four signed base-256 digits each, the columns, so
// that an fp16 value is exact and a bf16 one down to 2^-54 of the row's largest.  The MMA
// is the one of whole numbers (m16n8k32) on c = n + 8: three instructions unpack eight codes where
// fp16 takes nine and bf16 eleven, and the sums are exact (1 x 65536, 32 heads: 66 -> 60 us).  For O^T
// the columns of P are the row's four group-scaled forms, high parts in columns 0 .. 3 and low parts in
// 4 .. 7: one operand, made once, serves all eight dim tiles, and of a tile of group g
// columns g and 4 + g count.
template <bool kBf16, bool kOne, int kW, int kNS>
__global__ void __launch_bounds__(32 * kW) kv4_rows_kernel(const Params p) {
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int kRows = kOne ? 1 : 8;
  constexpr int kStep = kOne ? 2 : 1;  // of the four accumulators, those that differ
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int j = lane >> 2, i = lane & 3;
  uint32_t ncta;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(ncta));
  const int rank = (int)cluster_rank();
  grid_dependency_wait();  // launched while the kernel before it drains
  const int cluster = blockIdx.x / ncta;
  const int slice = cluster / p.units, unit = cluster - slice * p.units;
  const int bh = unit / p.nqb, row0 = (unit - bh * p.nqb) * kRows;
  const int b = bh / p.H;
  const int len = p.valid ? min(max(__ldg(p.valid + b), 0), p.S_kv) : p.S_kv;
  const int nblk = (len + kKeys - 1) / kKeys;
  const int step = (int)ncta * kW * p.nsplit;

  // Query rows as B fragments: word order and pairs match packed4's (group g, lane i).
  uint4 qf[4];
  const int qrow = kOne ? 0 : row0 + j;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    qf[g] = make_uint4(0u, 0u, 0u, 0u);
    if (qrow < p.S_q)
      qf[g] = __ldg(reinterpret_cast<const uint4*>(p.q + ((long long)bh * p.S_q + qrow) * kD + 32 * g + 8 * i));
  }
  float sl2 = p.scale_log2;
  uint2 qd[4];       // kOne: digit j of this lane's eight values of group g, in the codes' order
  uint64_t base[4];  // and what its two columns' sums start from, 1.5 * 2^23 + 8 sum(digits)
  if constexpr (kOne) {
    uint32_t top = 0;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const uint32_t w[4] = {qf[g].x, qf[g].y, qf[g].z, qf[g].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 v = widen<kBf16>(w[k]);
        top = max(top, max(__float_as_uint(v.x) & 0x7fffffffu, __float_as_uint(v.y) & 0x7fffffffu));
      }
    }
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int E = max((int)(top >> 23), 1) - 126;  // |q| < 2^E
    const int e0 = (30 - E) / 2, e1 = 30 - E - e0;  // in two steps: neither factor leaves fp32
    const float f0 = __int_as_float((e0 + 127) << 23), f1 = __int_as_float((e1 + 127) << 23);
    const int s0 = (E - 6) / 2, s1 = E - 6 - s0;
    sl2 = top >= 0x7f800000u
              ? NAN
              : fminf(sl2 * __int_as_float((s0 + 127) << 23) * __int_as_float((s1 + 127) << 23), 3.402823466e38f);
    auto whole = [&](float v) {  // this column's whole number of a value, its signed digits as bytes
      const float y = v * f0 * f1;
      const int n = __float2int_rn(y);
      const int part = j < 4 ? n : __float2int_rn((y - (float)n) * 2147483648.f);
      return ((uint32_t)part + 0x00808080u) ^ 0x00808080u;
    };
    const uint32_t sel = (uint32_t)(3 - (j & 3)) | (uint32_t)(7 - (j & 3)) << 4;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const uint32_t w[4] = {qf[g].x, qf[g].y, qf[g].z, qf[g].w};
      uint32_t t[8];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 v = widen<kBf16>(w[k]);
        t[2 * k] = whole(v.x);
        t[2 * k + 1] = whole(v.y);
      }
      qd[g].x = __byte_perm(__byte_perm(t[0], t[4], sel), __byte_perm(t[1], t[5], sel), 0x5410);
      qd[g].y = __byte_perm(__byte_perm(t[2], t[6], sel), __byte_perm(t[3], t[7], sel), 0x5410);
      int x = __dp4a((int)qd[g].x, 0x01010101, __dp4a((int)qd[g].y, 0x01010101, 0));
      x += __shfl_xor_sync(0xffffffffu, x, 1);
      x += __shfl_xor_sync(0xffffffffu, x, 2);
      const float x0 = (float)(12582912 + 8 * __shfl_sync(0xffffffffu, x, 8 * i));
      const float x1 = (float)(12582912 + 8 * __shfl_sync(0xffffffffu, x, 8 * i + 4));
      base[g] = f2pack(-x0, -x1);
    }
  }

  const uint32_t ring = smem_u32(smem) + warp * kNS * kStageBytes;
  const long long row_base = (long long)bh * p.S_kv;
  // 16-byte code chunk c of key k sits at chunk c ^ ((k >> 1) & 3): the four even (or odd)
  // keys that a V fragment reads at once then lie in different banks.
  // This lane's chunks of a block lie 8 keys apart: offsets of the first, and of its scales.
  const uint32_t put0 = (lane >> 2) * 64 + (((lane & 3) ^ ((lane >> 3) & 3)) << 4);
  const uint8_t* const kc = p.kc + row_base * 64 + lane * 16;
  const uint8_t* const vc = p.vc + row_base * 64 + lane * 16;
  const uint8_t* const ks = p.ks + row_base * 8 + lane * 8;
  const uint8_t* const vs = p.vs + row_base * 8 + lane * 8;
  auto load = [&](int t, int slot) {
    const uint32_t st = ring + slot * kStageBytes;
    const long long at = (long long)t * kCodeBytes, sat = (long long)t * kScaleBytes;
    if ((t + 1) * kKeys <= len) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        cp16(st + put0 + c * 512, kc + at + c * 512);
        cp16(st + kCodeBytes + put0 + c * 512, vc + at + c * 512);
      }
      cp8(st + 2 * kCodeBytes + lane * 8, ks + sat);
      cp8(st + 2 * kCodeBytes + kScaleBytes + lane * 8, vs + sat);
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const bool take = t * kKeys + 8 * c + (lane >> 2) < len;
        cp16_if(st + put0 + c * 512, take ? kc + at + c * 512 : p.kc, take);
        cp16_if(st + kCodeBytes + put0 + c * 512, take ? vc + at + c * 512 : p.vc, take);
      }
      const bool take = t * kKeys + lane < len;
      cp8_if(st + 2 * kCodeBytes + lane * 8, take ? ks + sat : p.ks, take);
      cp8_if(st + 2 * kCodeBytes + kScaleBytes + lane * 8, take ? vs + sat : p.vs, take);
    }
  };

  float o[8][4];  // O^T: tile 2 g + h of dims, rows j and j + 8; columns 2 i, 2 i + 1
#pragma unroll
  for (int t = 0; t < 8; ++t)
#pragma unroll
    for (int c = 0; c < 4; ++c) o[t][c] = 0.f;
  // of query rows 2 i, 2 i + 1; l: this lane's keys only
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

  const int first = (slice * (int)ncta + rank) * kW + warp;
  int ahead = first;
#pragma unroll
  for (int s = 0; s < kNS - 1; ++s) {
    if (ahead < nblk) load(ahead, s);
    cp_commit();
    ahead += step;
  }
  int slot = 0;
  for (int t = first; t < nblk; t += step) {
    cp_wait<kNS - 2>();
    __syncwarp();
    {
      const int put = slot == 0 ? kNS - 1 : slot - 1;  // the slot read in the last round
      if (ahead < nblk) load(ahead, put);
      cp_commit();
      ahead += step;
    }
    const uint32_t st = ring + slot * kStageBytes;
    slot = slot + 1 == kNS ? 0 : slot + 1;

    float sc[2][4];  // scores of keys 16 u + j (0, 1) and 16 u + j + 8 (2, 3)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int k0 = 16 * u + j;
      const uint32_t swz = (uint32_t)(i ^ ((k0 >> 1) & 3)) << 4;  // the same for key k0 + 8
      const uint4 c0 = lds16(st + k0 * 64 + swz), c1 = lds16(st + (k0 + 8) * 64 + swz);
      const float4 f0 = p4::scales4(lds8(st + 2 * kCodeBytes + k0 * 8));
      const float4 f1 = p4::scales4(lds8(st + 2 * kCodeBytes + (k0 + 8) * 8));
      const uint32_t w0[4] = {c0.x, c0.y, c0.z, c0.w}, w1[4] = {c1.x, c1.y, c1.z, c1.w};
      const float g0[4] = {f0.x, f0.y, f0.z, f0.w}, g1[4] = {f1.x, f1.y, f1.z, f1.w};
#pragma unroll
      for (int c = 0; c < 4; ++c) sc[u][c] = 0.f;
      if constexpr (kOne) {
        constexpr uint32_t kHalf = 0x0f0f0f0fu, kStart = 0x4b400000u;
        uint64_t s0 = 0ull, s1 = 0ull;  // of keys k0 and k0 + 8: columns 2 i, 2 i + 1
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          int d[4];
          p4::mma16832(d, w0[g] & kHalf, w1[g] & kHalf, (w0[g] >> 4) & kHalf, (w1[g] >> 4) & kHalf, qd[g].x,
                       qd[g].y, make_uint4(kStart, kStart, kStart, kStart));
          s0 = fma2(f2pack(g0[g], g0[g]), add2(f2pack(__int_as_float(d[0]), __int_as_float(d[1])), base[g]), s0);
          s1 = fma2(f2pack(g1[g], g1[g]), add2(f2pack(__int_as_float(d[2]), __int_as_float(d[3])), base[g]), s1);
        }
        // the digits 2 i and the next together, then the other lanes'
        const float f = __int_as_float((127 - 16 * (i & 1) - 31 * (i >> 1)) << 23);
        float a, b;
        f2unpack(s0, a, b);
        a = fmaf(b, 0.00390625f, a) * f;
        a += __shfl_xor_sync(0xffffffffu, a, 2);
        sc[u][0] = a + __shfl_xor_sync(0xffffffffu, a, 1);
        f2unpack(s1, a, b);
        a = fmaf(b, 0.00390625f, a) * f;
        a += __shfl_xor_sync(0xffffffffu, a, 2);
        sc[u][2] = a + __shfl_xor_sync(0xffffffffu, a, 1);
      } else {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          uint32_t x[4], y[4];
          p4::numbers<kBf16>(w0[g], x);
          p4::numbers<kBf16>(w1[g], y);
          float d[4];
          p4::mma16816_zero<kBf16>(d, x[0], y[0], x[1], y[1], qf[g].x, qf[g].y);
          p4::mma16816<kBf16>(d, x[2], y[2], x[3], y[3], qf[g].z, qf[g].w);
#pragma unroll
          for (int c = 0; c < 4; ++c) sc[u][c] = fmaf(c < 2 ? g0[g] : g1[g], d[c], sc[u][c]);
        }
      }
    }
    // scores in log2 units; keys at or past len are masked
    const int left = len - t * kKeys;
    bool over = false;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int c = 0; c < 4; c += kStep) {
        const float v = sc[u][c] * sl2;
        sc[u][c] = 16 * u + j + 8 * (c >> 1) < left ? v : -INFINITY;
        over = over || sc[u][c] > m[c & 1] + kRescale;
      }
    if (__any_sync(0xffffffffu, over)) {
#pragma unroll
      for (int r = 0; r < (kOne ? 1 : 2); ++r) {
        float x = fmaxf(fmaxf(sc[0][r], sc[0][r + 2]), fmaxf(sc[1][r], sc[1][r + 2]));
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
        const float mn = fmaxf(m[r], x);
        const float alpha = m[r] == -INFINITY ? 0.f : ex2_approx(m[r] - mn);
        m[r] = mn;
        l[r] *= alpha;
#pragma unroll
        for (int q = 0; q < 8; ++q)
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (kOne || (c & 1) == r) o[q][c] *= alpha;
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      // the four V rows of this lane: keys 2 i, 2 i + 1 and those plus 8
      uint4 vw[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int k = 16 * u + 2 * i + (c & 1) + 8 * (c >> 1);
        vw[c] = lds16(st + kCodeBytes + k * 64 + (((j >> 1) ^ ((k >> 1) & 3)) << 4));
      }
      const int k0 = 16 * u + j;
      const uint2 s0 = lds8(st + 2 * kCodeBytes + kScaleBytes + k0 * 8);
      const uint2 s1 = lds8(st + 2 * kCodeBytes + kScaleBytes + (k0 + 8) * 8);
      const uint32_t w[4][4] = {{vw[0].x, vw[1].x, vw[2].x, vw[3].x}, {vw[0].y, vw[1].y, vw[2].y, vw[3].y},
                                {vw[0].z, vw[1].z, vw[2].z, vw[3].z}, {vw[0].w, vw[1].w, vw[2].w, vw[3].w}};
#pragma unroll
      for (int c = 0; c < 4; c += kStep) {
        const float mu = m[c & 1];
        const float e = ex2_approx(sc[u][c] - (mu == -INFINITY ? 0.f : mu));
        sc[u][c] = e;
        l[c & 1] += e;
      }
      const uint32_t half = (j & 1) ? 0x7632u : 0x5410u;
      float g0[4], g1[4];
      uint32_t one0 = 0, one1 = 0;  // the single row's operand
      if constexpr (kOne) {
        // columns 2 i, 2 i + 1: groups 2 (i % 2) and the next, high parts for i < 2
        const uint32_t h0 = (i & 1) ? s0.y : s0.x, h1 = (i & 1) ? s1.y : s1.x;
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&h0));
        const float2 c = __half22float2(*reinterpret_cast<const __half2*>(&h1));
        const float p0 = sc[u][0] * a.x, p1 = sc[u][0] * a.y;
        const float p2 = sc[u][2] * c.x, p3 = sc[u][2] * c.y;
        one0 = pack_bf16x2(p0, p1);
        one1 = pack_bf16x2(p2, p3);
        const uint32_t l0 = pack_bf16x2(p0 - __uint_as_float(one0 << 16), p1 - __uint_as_float(one0 & 0xffff0000u));
        const uint32_t l1 = pack_bf16x2(p2 - __uint_as_float(one1 << 16), p3 - __uint_as_float(one1 & 0xffff0000u));
        one0 = transpose8(i < 2 ? one0 : l0);
        one1 = transpose8(i < 2 ? one1 : l1);
      } else {
        const float4 f0 = p4::scales4(s0), f1 = p4::scales4(s1);
        g0[0] = f0.x, g0[1] = f0.y, g0[2] = f0.z, g0[3] = f0.w;
        g1[0] = f1.x, g1[1] = f1.y, g1[2] = f1.z, g1[3] = f1.w;
      }
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        // a lane's dims in group g: 32 g + 8 (j / 2) + j % 2 + {0, 2, 4, 6}, one half word
        uint32_t x[4], y[4];
        p4::numbers_bf16(__byte_perm(w[g][0], w[g][1], half), x);
        p4::numbers_bf16(__byte_perm(w[g][2], w[g][3], half), y);
        if constexpr (kOne) {
          p4::mma16816<true>(o[2 * g], x[0], x[1], y[0], y[1], one0, one1);
          p4::mma16816<true>(o[2 * g + 1], x[2], x[3], y[2], y[3], one0, one1);
        } else {
          const float p0 = sc[u][0] * g0[g], p1 = sc[u][1] * g0[g];
          const float p2 = sc[u][2] * g1[g], p3 = sc[u][3] * g1[g];
          const uint32_t h0 = pack_bf16x2(p0, p1), h1 = pack_bf16x2(p2, p3);
          const uint32_t l0 = pack_bf16x2(p0 - __uint_as_float(h0 << 16), p1 - __uint_as_float(h0 & 0xffff0000u));
          const uint32_t l1 = pack_bf16x2(p2 - __uint_as_float(h1 << 16), p3 - __uint_as_float(h1 & 0xffff0000u));
          const uint32_t b0 = transpose8(h0), b1 = transpose8(h1), e0 = transpose8(l0), e1 = transpose8(l1);
          p4::mma16816<true>(o[2 * g], x[0], x[1], y[0], y[1], b0, b1);
          p4::mma16816<true>(o[2 * g + 1], x[2], x[3], y[2], y[3], b0, b1);
          p4::mma16816<true>(o[2 * g], x[0], x[1], y[0], y[1], e0, e1);
          p4::mma16816<true>(o[2 * g + 1], x[2], x[3], y[2], y[3], e0, e1);
        }
      }
    }
  }
  cp_wait<0>();
  __syncthreads();  // the rings become the merge area

  // Per-warp results to shared memory: O [row][dim], m, l.
  constexpr int kPart = (int)kv4_part_floats(kRows);
  float* const parts = reinterpret_cast<float*>(smem);
  {
    float* const mine = parts + warp * kPart;
#pragma unroll
    for (int r = 0; r < (kOne ? 1 : 2); ++r) {
      float x = l[r];
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
      const int row = kOne ? 0 : 2 * i + r;
      if (j == 0 && (!kOne || i == 0)) {
        mine[kRows * kD + row] = m[r];
        mine[kRows * kD + kRows + row] = x;
      }
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        // tile q = 2 g + h: row j is nibble 2 h of the half word, row j + 8 nibble 2 h + 1
        const int g = q >> 1, d0 = 32 * g + 8 * (j >> 1) + (j & 1) + 4 * (q & 1);
        if constexpr (kOne) {  // column g is in lanes i = g / 2, column 4 + g two lanes on
          const float lo = o[q][g & 1] + __shfl_xor_sync(0xffffffffu, o[q][g & 1], 2);
          const float hi = o[q][(g & 1) + 2] + __shfl_xor_sync(0xffffffffu, o[q][(g & 1) + 2], 2);
          if (i == (g >> 1)) {
            mine[d0] = lo;
            mine[d0 + 2] = hi;
          }
        } else {
          mine[row * kD + d0] = o[q][r];
          mine[row * kD + d0 + 2] = o[q][r + 2];
        }
      }
    }
  }
  __syncthreads();
  float* const own = parts + kW * kPart;
  for (int e = threadIdx.x; e < kRows * kD; e += 32 * kW) {
    const int row = e / kD;
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < kW; ++w) mx = fmaxf(mx, parts[w * kPart + kRows * kD + row]);
    float acc = 0.f, sum = 0.f;
#pragma unroll
    for (int w = 0; w < kW; ++w) {
      const float mw = parts[w * kPart + kRows * kD + row];
      const float f = mw == -INFINITY ? 0.f : ex2_approx(mw - mx);
      acc = fmaf(f, parts[w * kPart + e], acc);
      sum = fmaf(f, parts[w * kPart + kRows * kD + kRows + row], sum);
    }
    own[e] = acc;
    if (e % kD == 0) {
      own[kRows * kD + row] = mx;
      own[kRows * kD + kRows + row] = sum;
    }
  }
  cluster_sync();
  const uint32_t own_a = smem_u32(own);
  const int per = (kRows * kD + (int)ncta - 1) / (int)ncta;
  const int end = min(kRows * kD, (rank + 1) * per);
  for (int e = rank * per + threadIdx.x; e < end; e += 32 * kW) {
    const int row = e / kD;
    float mx = -INFINITY;
    for (uint32_t c = 0; c < ncta; ++c)
      mx = fmaxf(mx, ld_cluster(mapa_shared(own_a + (kRows * kD + row) * 4, c)));
    float acc = 0.f, sum = 0.f;
    for (uint32_t c = 0; c < ncta; ++c) {
      const uint32_t base = mapa_shared(own_a, c);
      const float mc = ld_cluster(base + (kRows * kD + row) * 4);
      const float f = mc == -INFINITY ? 0.f : ex2_approx(mc - mx);
      acc = fmaf(f, ld_cluster(base + e * 4), acc);
      sum = fmaf(f, ld_cluster(base + (kRows * kD + kRows + row) * 4), sum);
    }
    if (p.part) {
      float* const part = p.part + ((long long)slice * p.units + unit) * kPart;
      part[e] = acc;
      if (e % kD == 0) {
        part[kRows * kD + row] = mx;
        part[kRows * kD + kRows + row] = sum;
      }
    } else if (row0 + row < p.S_q) {
      const float v = sum == 0.f ? 0.f : acc / sum;  // no valid key: zeros
      const long long at = b * p.ob + (bh % p.H) * p.oh + (long long)(row0 + row) * p.os + e % kD;
      if (p.out_f32)
        static_cast<float*>(p.out)[at] = v;
      else
        static_cast<uint16_t*>(p.out)[at] = kBf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v))
                                                  : __half_as_ushort(__float2half_rn(v));
    }
  }
  cluster_sync();  // no CTA leaves while another reads its shared memory
}

}  // namespace kv4

// Whether the packed cache is read directly.  Up to 16 rows always; beyond, the rows' passes over the
// cache (and, below 256 keys, their starts) cost more than the tile kernel's start (some 8 us) once
// heads x rows x keys exceed 2^20, twice that from 4096 keys and four times that from 32768, where the
// tile kernel has slices to join.  Measured, us, from graphs, this way against the tile kernel, heads x rows x keys:
// 4 x 1024 x 130 12.2 / 12.1, 32 x 128 x 130 12.2 / 9.2, 4 x 512 x 512 12.2 / 16.7, 32 x 64 x 512 12.2 / 13.6,
// 4 x 1024 x 512 18.8 / 17.7, 32 x 64 x 2048 28.0 / 21.0, 1 x 512 x 4096 16.2 / 23.6, 16 x 32 x 4096
// 16.2 / 21.1, 4 x 256 x 4096 26.2 / 24.0, 4 x 32 x 16384 18.6 / 27.7, 4 x 64 x 16384 26.1 / 28.3, 1 x 64 x
// 65536 28.9 / 41.7, 1 x 128 x 65536 45.3 / 41.7.
static bool rows_path(long long bh, long long S_q, long long S_kv) {
  const long long most = 1LL << (20 + (S_kv >= 4096) + (S_kv >= 32768));
  return S_q <= 16 || bh * S_q * std::max(S_kv, 256LL) <= most;
}
constexpr int kRowsStages = 3;
template <bool kBf16, bool kOne, int kW>
static int rows_t(const kv4::Params& p, int ncta, cudaStream_t st) {
  auto kern = kv4::kv4_rows_kernel<kBf16, kOne, kW, kRowsStages>;
  constexpr size_t smem = kv4::smem_bytes<kW>(kRowsStages, kOne ? 1 : 8);
  static SmemAttr attr;
  if (!attr.raise((const void*)kern, smem)) return ANIMA_ERR_CUDA;
  return launch_clusters(kern, p.units * p.nsplit * ncta, ncta, 32 * kW, smem, st, p);
}

// Clusters of `ncta` CTAs of eight warps that the device holds at once; one cluster lies in one group of SMs,
// and what is left over of a group stays empty, so this is less than two CTAs an SM (32 of eight on 148 SMs).  Asked for once.
template <bool kOne>
static int clusters_held(int ncta, int sm_count) {
  constexpr int kMaxDev = 64;
  static std::atomic<int> held[kMaxDev][9];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDev) return std::max(1, 2 * sm_count / ncta);
  int n = held[dev][ncta].load(std::memory_order_acquire);
  if (n > 0) return n;
  auto kern = kv4::kv4_rows_kernel<true, kOne, 8, kRowsStages>;
  constexpr size_t smem = kv4::smem_bytes<8>(kRowsStages, kOne ? 1 : 8);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ncta);
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = (unsigned)ncta;
  at.val.clusterDim.y = 1;
  at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMaxSmem) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n < 1) {
    cudaGetLastError();
    n = std::max(1, 2 * sm_count / ncta);
  }
  held[dev][ncta].store(n, std::memory_order_release);
  return n;
}

// How a call on rows_path is cut.
struct RowsPlan {
  int rows, nqb;   // query rows per unit, units per (batch, head)
  long long units;
  int warps, ncta, nsplit;
  size_t bytes;
};
static RowsPlan rows_plan(long long bh, int S_q, int S_kv, int sm_count) {
  RowsPlan r;
  r.rows = S_q > 1 ? 8 : 1;
  r.nqb = (S_q + r.rows - 1) / r.rows;
  r.units = bh * r.nqb;
  r.nsplit = 1;
  const int nblk = (S_kv + kv4::kKeys - 1) / kv4::kKeys;
  r.warps = nblk >= 128 ? 8 : 4;
  if (r.warps == 4) {
    // CTAs per cluster: as many as two to an SM have room for, while each of their warps has a block
    const long long room = std::max(1LL, 2LL * sm_count / r.units);
    r.ncta = (int)std::min<long long>(std::min<long long>((nblk + 3) / 4, room), 8);
  } else {
    // CTAs per cluster and clusters per unit (slices of its keys, four blocks a warp at least): the
    // shortest chain of blocks, in rounds of the clusters that the device holds, where a round's ends cost
    // 1.5 blocks of some 2 us and joining s slices 1.5 + s / 8.  In us from graphs, one cluster of eight against slices of one CTA, one
    // row, heads x keys: 20 x 65536 60.7 / 43.7, 32 x 65536 60.0 / 58.5, 32 x 16384 20.8 / 23.8, 37 x 16384
    // 31.1 / 25.3; two clusters of eight against those: 16 x 65536 37.4 / 38.0.
    r.ncta = 1;
    const int units = (int)std::min<long long>(r.units, 1 << 20);  // beyond, the cut is the same
    double best = 0;
    for (int c = 8; c >= 1; --c) {
      const int held = r.rows == 1 ? clusters_held<true>(c, sm_count) : clusters_held<false>(c, sm_count);
      const int per = 8 * c;  // warps of a cluster
      const int most = std::max(1, std::min(nblk / (4 * per), 64));
      for (int k = 1; k <= 5; ++k) {
        const int s = k < 5 ? k : held / units;  // the last: as many as fit in one round
        if (s > most || (k == 5 && s < 5)) continue;
        const double chain = (double)((nblk + per * s - 1) / (per * s));
        const double cost = (double)((units * s + held - 1) / held) * (chain + 1.5) + (s > 1 ? 1.5 + s * 0.125 : 0.0);
        if (best == 0 || cost < best) {
          best = cost;
          r.ncta = c;
          r.nsplit = s;
        }
      }
    }
  }
  r.bytes = r.nsplit > 1 ? (size_t)r.nsplit * r.units * kv4_part_floats(r.rows) * sizeof(float) : 0;
  return r;
}

size_t attn_kv4_workspace_bytes(int B, int H, int S_q, int S_kv, int sm_count) {
  const long long bh = (long long)B * H;
  if (rows_path(bh, S_q, S_kv)) return rows_plan(bh, S_q, S_kv, sm_count).bytes;
  return kv4_tile_plan((int)bh, S_q, S_kv, sm_count).bytes;
}

int attn_kv4_launch(const AnimaAttnKv4Args* a, int* status, int sm_count, cudaStream_t st) {
  const long long bh = (long long)a->B * a->H;
  const bool bf = a->dtype == ANIMA_DTYPE_BF16;
  const int* valid = (a->flags & ANIMA_FLAG_MASK) ? a->kv_valid_len : nullptr;
  auto room = [&](size_t need) { return need == 0 || (a->workspace && a->workspace_bytes >= need); };
  if (rows_path(bh, a->S_q, a->S_kv)) {
    const RowsPlan r = rows_plan(bh, a->S_q, a->S_kv, sm_count);
    if (!room(r.bytes)) return ANIMA_ERR_NOMEM;
    if (r.units * r.nsplit * r.ncta > 0x7fffffffLL) return ANIMA_ERR_SHAPE;
    kv4::Params p;
    p.q = static_cast<const uint16_t*>(a->q);
    p.kc = static_cast<const uint8_t*>(a->k_codes);
    p.ks = static_cast<const uint8_t*>(a->k_scales);
    p.vc = static_cast<const uint8_t*>(a->v_codes);
    p.vs = static_cast<const uint8_t*>(a->v_scales);
    p.valid = valid;
    p.out = a->out;
    p.part = r.nsplit > 1 ? static_cast<float*>(a->workspace) : nullptr;
    p.ob = a->out_stride[0];
    p.oh = a->out_stride[1];
    p.os = a->out_stride[2];
    p.H = a->H;
    p.S_q = a->S_q;
    p.S_kv = a->S_kv;
    p.nqb = r.nqb;
    p.units = (int)r.units;
    p.nsplit = r.nsplit;
    p.out_f32 = (a->flags & ANIMA_FLAG_OUT_F32) != 0;
    p.scale_log2 = std::min(a->scale * 1.4426950408889634f, 3.402823466e38f);
    int rc;
    if (r.warps == 8)
      rc = r.rows == 1 ? (bf ? rows_t<true, true, 8>(p, r.ncta, st) : rows_t<false, true, 8>(p, r.ncta, st))
                       : (bf ? rows_t<true, false, 8>(p, r.ncta, st) : rows_t<false, false, 8>(p, r.ncta, st));
    else
      rc = r.rows == 1 ? (bf ? rows_t<true, true, 4>(p, r.ncta, st) : rows_t<false, true, 4>(p, r.ncta, st))
                       : (bf ? rows_t<true, false, 4>(p, r.ncta, st) : rows_t<false, false, 4>(p, r.ncta, st));
    if (rc != ANIMA_OK || r.nsplit == 1) return rc;
    return kv4_merge_launch(a, p.part, r.nqb, r.rows, p.units, r.nsplit, sm_count, st);
  }
  const Kv4TilePlan t = kv4_tile_plan((int)bh, a->S_q, a->S_kv, sm_count);
  return room(t.bytes) ? kv4_tile_launch(a, t, status, sm_count, st) : ANIMA_ERR_NOMEM;
}

}  // namespace anima
