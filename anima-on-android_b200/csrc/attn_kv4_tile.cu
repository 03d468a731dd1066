// attn_kv4_tile.cu -- attention over packed K and V (packed4.cuh) for many query rows, on the
// tensor cores: tcgen05 MMAs with TMEM accumulators, K and V unpacked into shared memory by the
// CTA itself.  out = softmax(q K^T * scale) V per (batch, head), D = 128.
//
// Work unit = kNT 128-row query tiles of one (batch, head); its keys may be cut into slices, and
// (unit, slice) is a segment, streamed in 64-key tiles (one of more than kRun tiles in several runs, whose sums a CTA
// joins in scratch of its own).  The grid is persistent: a CTA takes
// segments c, c + G, ..., and moves from one to the next without draining (the next Q tile, K and V
// are under way while the last P V and the output of the segment before run).  A unit cut into
// slices writes fp32 partials (O, running max, running sum), which kv4_merge_kernel joins in slice
// order, so results repeat bit for bit.
//
// No operand loses bits that the result could show.  A value n s of K or V has up to 15 bits and is held as
// the exact sum of two 16-bit parts, P as two as well:
//   S = Q K_hi^T + Q K_lo^T                     fp16, q as it is, K exact
//   O += P_hi V_hi + P_lo V_hi + P_hi V_lo      bf16, V exact, P to 2^-17; the part left out is below 2^-17
// P is bf16 for its range: a weight is as right far below the row's largest as next to it, whatever the
// length of the cache (fp16 has nothing below 2^-25).  As one fp16 product each, with K, V and P rounded
// to 11 bits, the result was off by 3.1e-4 before its own rounding, and calls took two thirds of the time.
// bf16 query rows are first scaled by the power of two that brings their largest magnitude to
// [2^14, 2^15), which the row's softmax scale takes back, so a bf16 value keeps its eight bits down
// to 2^-31 of the row's largest.
//
// Warp roles (16 warps):
//   warps 0-3    softmax of query tile 0: thread = query row = TMEM lane.  Per key tile reads its S
//                row, updates max / sum, writes P's parts over S; at the end stores O.  A bf16 Q
//                tile is converted in place by its warpgroup before its first MMA.
//   warps 4-7    softmax of query tile 1 (kNT = 2), or unpack (kNT = 1, where a key tile feeds
//                half the MMA work).
//   warps 8-11   unpack: packed tiles into the parts' tiles in the 128-byte-swizzled layout of the MMA
//                operands.
//   warps 12, 14 MMA issuers of a query tile each (kNT = 2), or of Q K^T and P V; 12 owns the TMEM.
//   warp 13      TMA producer of the Q tiles.
//   warp 15      packed tiles from global memory by cp.async.
// An issuing warp runs converged and one elected lane issues: descriptors stay in uniform registers.  With
// one divergent thread issuing for both query tiles an MMA took 100 cycles beside busy softmax warps,
// against 48 (Q K^T, N = 64, shared memory) and 64 (P V) of the tensor core.
// Tensor memory: two S buffers of 64 columns per query tile, with P's parts over S, and O_0, O_1 of 128
// columns.  Q K^T runs a step ahead of P V, so the softmax of one step runs beside the MMAs of its neighbours.
//
// What bounds it: a step of two query tiles and 64 keys takes 3,010 cycles (traced) of 3,072 that its MMAs
// need, and the unpacking fills as much; the clock falls under that load (1.4 GHz).  256 rows against 8192
// keys, 32 heads: 82 us replayed from a graph; 64 rows 55 us, 2,500 cycles a step of 1,536 of MMAs, the rest unpacking and
// hand-offs.
#include <algorithm>

#include "attn_kv4.cuh"
#include "attn_shared.cuh"
#include "packed4.cuh"

namespace anima {
namespace kv4t {

using namespace attn;  // kD, kBM, drain_wait, stage/store_block, pack2

constexpr int kKeys = 64;                   // keys per tile
// Tiles of one chain of sums in tensor memory.  The tensor core cuts a sum off to fp32 after each of its 12 products a
// tile instead of rounding it, so what a chain loses grows with its length: 2e-5 of sum p |v| at 128 tiles, 1.4e-4 at
// 1024, 1.6e-3 at 4096.  Longer ones go on as runs, joined in rounded fp32 sums.
constexpr int kRun = 128;
constexpr int kPanel = 128 * 128;           // [128 rows][64 x 16-bit]
constexpr int kTile = 2 * kPanel;            // a Q tile
constexpr int kKvPanel = kKeys * 128;
constexpr int kPart = 2 * kKvPanel;          // the upper or lower parts of a K or V tile
constexpr int kMmaWarp12 = 12, kQWarp13 = 13, kRawWarp15 = 15;
constexpr int kThreads16 = 512;
// 512 threads launch with 128 registers each: 256 x 168 + 128 x 112 + 128 x 64 = 512 x 128.
constexpr uint32_t kRegsSoft = 168, kRegsUnpack = 112, kRegsMma = 64;
static_assert(2 * kRegsSoft + kRegsUnpack + kRegsMma == 4 * 128, "register split");

struct Params {
  const uint8_t* kc;
  const uint8_t* ks;
  const uint8_t* vc;
  const uint8_t* vs;
  const int* valid;
  void* out;
  float* part;         // partials, or nullptr: write the output
  float* fold;         // a CTA's O of the runs so far, [rows][128]
  long long ob, oh, os;
  int* status;
  int H, S_q, S_kv;
  int nqb;             // units per (batch, head)
  int units;
  int nsplit;
  int runs;            // runs of a segment
  int out_f32;         // out is fp32, else of q's type
  float scale_log2;
};

template <int kNT>
struct Smem {
  static constexpr int kUnpackWarps = kNT == 2 ? 4 : 8;
  static constexpr int kGroups = kKeys / 8 / kUnpackWarps;  // of eight keys, per tile and warp
  static constexpr int kRaw = kNT == 2 ? 3 : 8;             // stages of packed tiles
  uint8_t q[kNT][kTile];
  uint8_t kv[2][2][2][kPart];  // unpacked tiles of K, of V: two slots, upper and lower parts
  uint8_t raw[kRaw][kKeys * 72];  // codes, then scales
  float4 stage[kNT * 4][128];  // per softmax warp: one 32 x 32 16-bit block on its way to global
  uint64_t q_raw[2];           // Q tile as loaded
  uint64_t q_conv[2];          // bf16: converted
  uint64_t q_empty[2];
  uint64_t raw_full[kRaw];
  uint64_t raw_empty[kRaw];
  uint64_t kv_full[2][2];   // [K, V][slot]
  uint64_t kv_empty[2][2];
  uint64_t s_full[2][2];    // [query tile][buffer]
  uint64_t p_full[2][2];
  uint64_t o_full[2];
  uint64_t o_empty[2];
  uint64_t pv_done[2];
  uint64_t s_empty[2];      // [buffer], one query tile
  uint64_t mma_done[2];
  uint32_t tmem_base;
  int abort;
};
template <int kNT>
constexpr size_t smem_bytes() {
  return sizeof(Smem<kNT>) + 1024;
}
static_assert(smem_bytes<1>() <= 227 * 1024 && smem_bytes<2>() <= 227 * 1024, "shared memory budget");

// A run of a segment: key tiles [k0, k0 + n) of a unit.  Runs are numbered through, those of a segment in a row, and
// a CTA takes all of a segment.
struct Seg {
  int unit, slice, bh, b, q0, len, k0, n;
  bool last;  // of its segment
};
template <bool kLong>
__device__ __forceinline__ int after(const Params& p, int run) {
  if (!kLong) return run + (int)gridDim.x;
  ++run;
  return run % p.runs ? run : run + ((int)gridDim.x - 1) * p.runs;
}
template <bool kLong>
__device__ __forceinline__ Seg segment(const Params& p, int run, int rows) {
  Seg s;
  const int seg = kLong ? run / p.runs : run;
  run -= kLong ? seg * p.runs : seg;
  s.last = !kLong || run + 1 == p.runs;
  s.slice = seg / p.units;
  s.unit = seg - s.slice * p.units;
  s.bh = s.unit / p.nqb;
  s.q0 = (s.unit - s.bh * p.nqb) * rows;
  s.b = s.bh / p.H;
  s.len = p.valid ? min(max(__ldg(p.valid + s.b), 0), p.S_kv) : p.S_kv;
  const int tiles = (s.len + kKeys - 1) / kKeys;
  s.k0 = (int)((long long)tiles * s.slice / p.nsplit);
  s.n = (int)((long long)tiles * (s.slice + 1) / p.nsplit) - s.k0;
  if (kLong) {
    s.n = min(max(s.n - run * kRun, 0), kRun);
    s.k0 += run * kRun;
  }
  return s;
}

// One lane of a converged warp, the same one each time.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r != 0;
}

// Arrives on `bar` once all of this thread's asynchronous copies so far have landed.
__device__ __forceinline__ void cp_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// The m-th of the 2 n tiles of a segment in the order in which they are used: K_0 K_1 V_0 K_2 V_1 ...
// K_(n-1) V_(n-2) V_(n-1).
struct Item {
  int v, tile;  // V or K, key tile
};
__device__ __forceinline__ Item item_of(int m, int n) {
  if (m == 0 || m == 2 * n - 1) return {m > 0, m >> 1};
  return {~m & 1, (m & 1) ? (m + 1) >> 1 : (m >> 1) - 1};
}

// n s of four pairs as the sum of two fp16 (n: numbers in, upper parts out).  n s is a multiple of 2^-24
// of at most 15 bits, so what its rounding to 11 leaves is a value of fp16 too.
__device__ __forceinline__ void split_f16(uint32_t (&n)[4], uint32_t (&lo)[4], __half2 s) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const __half2 v = *reinterpret_cast<const __half2*>(&n[k]);
    const __half2 h = __hmul2(v, s);
    const __half2 l = __hfma2(v, s, __hneg2(h));
    n[k] = *reinterpret_cast<const uint32_t*>(&h);
    lo[k] = *reinterpret_cast<const uint32_t*>(&l);
  }
}
// The same in bf16, s in two parts (lower half, upper half of `s2`): 8 bits above, and what is left of n s
// below, at most 2^-8 of it and so at most 6 bits.
__device__ __forceinline__ void split_bf16(uint32_t (&n)[4], uint32_t (&lo)[4], uint32_t s2) {
  const __nv_bfloat162 s = *reinterpret_cast<const __nv_bfloat162*>(&s2);
  const __nv_bfloat162 s0 = __low2bfloat162(s), s1 = __high2bfloat162(s);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const __nv_bfloat162 v = *reinterpret_cast<const __nv_bfloat162*>(&n[k]);
    const __nv_bfloat162 h = __hmul2(v, s0);
    const __nv_bfloat162 l = __hfma2(v, s1, __hfma2(v, s0, __hneg2(h)));
    n[k] = *reinterpret_cast<const uint32_t*>(&h);
    lo[k] = *reinterpret_cast<const uint32_t*>(&l);
  }
}

// A thread's bf16 query row of a Q tile to fp16 in place, scaled; returns the factor that undoes it.
__device__ __forceinline__ float convert_row(uint8_t* tile, int row) {
  auto at = [&](int c) {
    return reinterpret_cast<uint4*>(tile + (c >> 3) * kPanel + row * 128 + (((c & 7) ^ (row & 7)) << 4));
  };
  uint4 v[16];
#pragma unroll
  for (int c = 0; c < 16; ++c) v[c] = *at(c);
  uint32_t top = 0;  // largest magnitude's bits
#pragma unroll
  for (int c = 0; c < 16; ++c) {
    const uint32_t w[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
#pragma unroll
    for (int k = 0; k < 4; ++k) top = max(top, max(w[k] & 0x7fffu, (w[k] >> 16) & 0x7fffu));
  }
  // With exponent e of the largest, scale by 2^(14 - e), in two steps so that neither factor leaves
  // fp32; zero, subnormal and non-finite rows are left as they are.
  const int ex = (int)(top >> 7);
  const int shift = ex == 0 || ex == 255 ? 0 : 14 - (ex - 127);
  const int s0 = shift / 2, s1 = shift - s0;
  const float f0 = __int_as_float((s0 + 127) << 23), f1 = __int_as_float((s1 + 127) << 23);
#pragma unroll
  for (int c = 0; c < 16; ++c) {
    uint32_t w[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
#pragma unroll
    for (int k = 0; k < 4; ++k)
      w[k] = pack_f16x2(__uint_as_float(w[k] << 16) * f0 * f1, __uint_as_float(w[k] & 0xffff0000u) * f0 * f1);
    *at(c) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return __int_as_float((127 - s0) << 23) * __int_as_float((127 - s1) << 23);
}

// kLong: segments of more than one run.
template <bool kBf16, int kNT, bool kLong>
__global__ void __launch_bounds__(kThreads16, 1)
    kv4_tile_kernel(const __grid_constant__ CUtensorMap tmap_q, const Params p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t pad = (1024u - (smem_u32(smem_raw) & 1023u)) & 1023u;
  Smem<kNT>& sm = *reinterpret_cast<Smem<kNT>*>(smem_raw + pad);
  constexpr int kUnpackWarps = Smem<kNT>::kUnpackWarps, kGroups = Smem<kNT>::kGroups, kRaw = Smem<kNT>::kRaw;
  constexpr int kRows = kNT * kBM;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort = &sm.abort;
  if (threadIdx.x == 0) {
    for (int k = 0; k < kRaw; ++k) {
      mbar_init(&sm.raw_full[k], 32);
      mbar_init(&sm.raw_empty[k], kUnpackWarps);
    }
    for (int i = 0; i < 2; ++i) {
      for (int k = 0; k < 2; ++k) {
        mbar_init(&sm.kv_full[i][k], kUnpackWarps);
        mbar_init(&sm.kv_empty[i][k], kNT);
        mbar_init(&sm.s_full[i][k], 1);
        mbar_init(&sm.p_full[i][k], kBM);
      }
      mbar_init(&sm.pv_done[i], 1);
      mbar_init(&sm.mma_done[i], 1);
      mbar_init(&sm.s_empty[i], 1);
      mbar_init(&sm.q_raw[i], 1);
      mbar_init(&sm.q_conv[i], kBM);
      mbar_init(&sm.q_empty[i], 1);
      mbar_init(&sm.o_full[i], 1);
      mbar_init(&sm.o_empty[i], kBM);
    }
    sm.abort = 0;
    fence_barrier_init();
  }
  if (warp == kMmaWarp12) {
    tmem_alloc(&sm.tmem_base, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;
  const int segs = p.units * p.nsplit * (kLong ? p.runs : 1);
  const int first = (int)blockIdx.x * (kLong ? p.runs : 1);
  // Launched as a programmatic dependent of the kernel before it on the stream: the set-up above
  // overlaps that kernel's end, and no global memory is touched before it has completed.
  grid_dependency_wait();
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    return mbar_wait(bar, parity, abort, p.status, ANIMA_ERR_TIMEOUT);
  };
  // Every role walks the same segments; `a` counts those with keys, `gg` their key-tile steps.

  if (warp >= kMmaWarp12) {
    regs_dec<kRegsMma>();
    if (warp == kQWarp13 && lane == 0) {
      // ---------------------------------------------------------- Q producer
      tma_prefetch_desc(&tmap_q);
      int a = 0;
      bool ok = true;
      for (int seg = first; seg < segs && ok; seg = after<kLong>(p, seg)) {
        const Seg s = segment<kLong>(p, seg, kRows);
        if (s.n <= 0) continue;
        for (int i = 0; i < kNT && ok; ++i) {
          if (a > 0 && !(ok = wait(&sm.q_empty[i], (uint32_t)(a - 1) & 1u))) break;
          mbar_arrive_expect_tx(&sm.q_raw[i], kTile);
          for (int pn = 0; pn < 2; ++pn)
            tma_load_3d(sm.q[i] + pn * kPanel, &tmap_q, &sm.q_raw[i], pn * 64, s.q0 + i * kBM, s.bh);
        }
        if (ok) ++a;
      }
      // every copy this thread started lands before the CTA may exit
      if (ok && a > 0)
        for (int i = 0; i < kNT; ++i) drain_wait(&sm.q_raw[i], (uint32_t)(a - 1) & 1u);
      if (!ok)  // an aborted round may have loaded tile 0 only
        for (int i = 0; i < kNT; ++i) {
          if (a > 0) drain_wait(&sm.q_raw[i], (uint32_t)(a - 1) & 1u);
          if (i == 0) drain_wait(&sm.q_raw[0], (uint32_t)a & 1u);
        }
    } else if (warp == kRawWarp15) {
      // ---------------------------------------------------------- packed tiles
      // 16-byte chunk c of key r's codes goes to row r ^ ((r >> 2) & 1), so that the two keys that a
      // quarter-warp of the unpacking reads lie in different banks.
      bool ok = true;
      int raw = 0, use = 0;
      for (int seg = first; seg < segs && ok; seg = after<kLong>(p, seg)) {
        const Seg s = segment<kLong>(p, seg, kRows);
        const long long row0 = (long long)s.bh * p.S_kv + (long long)s.k0 * kKeys;
        for (int m = 0; m < 2 * s.n; ++m) {
          const Item it = item_of(m, s.n);
          const bool got = wait(&sm.raw_empty[raw], ((uint32_t)use & 1u) ^ 1u);
          if (!(ok = __all_sync(0xffffffffu, got))) break;
          const int left = s.len - (s.k0 + it.tile) * kKeys;  // valid keys from this tile's first on
          const uint8_t* const codes = (it.v ? p.vc : p.kc) + (row0 + (long long)it.tile * kKeys) * 64 + lane * 16;
          const uint8_t* const scales = (it.v ? p.vs : p.ks) + (row0 + (long long)it.tile * kKeys) * 8 + lane * 8;
          const int r = lane >> 2;
          const uint32_t dst = smem_u32(sm.raw[raw]) + (r ^ (r >> 2)) * 64 + (lane & 3) * 16;
          const uint32_t sdst = smem_u32(sm.raw[raw]) + kKeys * 64 + lane * 8;
          if (left >= kKeys) {
#pragma unroll
            for (int c = 0; c < 8; ++c) p4::cp16(dst + c * 512, codes + c * 512);
#pragma unroll
            for (int c = 0; c < 2; ++c) p4::cp8(sdst + c * 256, scales + c * 256);
          } else {  // keys past the length read as zeros
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              const bool take = 8 * c + r < left;
              p4::cp16_if(dst + c * 512, take ? codes + c * 512 : p.kc, take);
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const bool take = 32 * c + lane < left;
              p4::cp8_if(sdst + c * 256, take ? scales + c * 256 : p.ks, take);
            }
          }
          cp_arrive(&sm.raw_full[raw]);
          if (++raw == kRaw) raw = 0, ++use;
        }
      }
      p4::cp_wait<0>();
    } else if (warp == kMmaWarp12 || warp == kMmaWarp12 + 2) {
      // ---------------------------------------------------------- MMA issuers: of a query tile each, or of Q K^T and P V
      // The warp runs converged and one elected lane issues, so that descriptors stay in uniform registers.
      const int who = __shfl_sync(0xffffffffu, (warp - kMmaWarp12) >> 1, 0);
      const int i = kNT == 1 ? 0 : who;
      const bool qk = kNT == 2 || who == 0, pv = kNT == 2 || who == 1;
      const bool leader = elect_one();
      constexpr uint32_t idesc_qk = make_idesc_f16(0u, kBM, kKeys, 0);  // fp16 Q and K
      constexpr uint32_t idesc_pv = make_idesc_f16(1u, kBM, kD, 1);     // bf16 P and V
      const uint64_t dk0 = sdesc_sw128(smem_u32(sm.kv[0]), 16, 1024);
      const uint64_t dv0 = sdesc_sw128(smem_u32(sm.kv[1]), kKvPanel, 1024);
      const uint64_t dq0 = sdesc_sw128(smem_u32(sm.q[0]), 16, 1024);
      auto s_at = [&](int t) { return tmem + (2 * i + (t & 1)) * kKeys; };
      // S_i of step t = Q_i (K_hi + K_lo)^T
      auto issue_qk = [&](int t) {
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          const uint64_t kb = desc_plus(dk0, (uint32_t)(2 * (t & 1) + part) * kPart);
          uint64_t bd[8], aq[8];
#pragma unroll
          for (int kk = 0; kk < 8; ++kk) {
            bd[kk] = desc_plus(kb, (kk >> 2) * kKvPanel + (kk & 3) * 32);
            aq[kk] = desc_plus(dq0, (uint32_t)i * kTile + (kk >> 2) * kPanel + (kk & 3) * 32);
          }
          if (leader) umma_ss_x8(s_at(t), aq, bd, idesc_qk, part);
        }
      };
      // O_i (+)= P_hi V_hi + P_lo V_hi + P_hi V_lo of step t
      auto issue_pv = [&](int t, bool acc) {
        const uint64_t vb = desc_plus(dv0, (uint32_t)(2 * (t & 1)) * kPart);
        const uint32_t tP = s_at(t), tO = tmem + 256 + i * kD;
        uint64_t bd[8];
        uint32_t a[8];
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          bd[kk] = desc_plus(vb, (kk & 3) * 2048);
          a[kk] = tP + kk * 8;
        }
        if (leader) umma_ts_x8(tO, a, bd, idesc_pv, acc ? 1u : 0u);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          if (leader) umma_ts(tO, a[kk], desc_plus(bd[kk], kPart), idesc_pv, 1u);
      };
      auto commit = [&](uint64_t* bar) {
        if (leader) umma_commit(bar);
      };
      bool ok = true;
      auto get = [&](uint64_t* bar, int phase) {
        const bool got = ok && wait(bar, (uint32_t)phase & 1u);
        ok = __all_sync(0xffffffffu, got);
        tc_fence_after();
      };
      int a = 0, gg = 0;
      for (int seg = first; seg < segs && ok; seg = after<kLong>(p, seg)) {
        const int n = segment<kLong>(p, seg, kRows).n;
        if (n <= 0) continue;
        // QK^T runs a step ahead of P V.  S of step t is in buffer t % 2, which P V of step t - 2 has to have left:
        // with two query tiles it is the same thread's and earlier in the pipe.
        if (qk) get(kBf16 ? &sm.q_conv[i] : &sm.q_raw[i], a);
        for (int g = -1; g < n; ++g) {
          const int t = gg + g, u = t + 1;
          if (qk && g + 1 < n) {
            if (kNT == 1 && u > 1) get(&sm.s_empty[u & 1], (u >> 1) - 1);
            get(&sm.kv_full[0][u & 1], u >> 1);
            if (!ok) break;
            issue_qk(u);
            commit(&sm.s_full[i][u & 1]);
            if (g + 2 == n) commit(&sm.q_empty[i]);
            commit(&sm.kv_empty[0][u & 1]);
          }
          if (!pv || g < 0) continue;
          get(&sm.kv_full[1][t & 1], t >> 1);
          get(&sm.p_full[i][t & 1], t >> 1);
          if (g == 0 && a > 0) get(&sm.o_empty[i], a - 1);
          if (!ok) break;
          issue_pv(t, g > 0);
          commit(&sm.pv_done[i]);
          if (kNT == 1) commit(&sm.s_empty[t & 1]);
          if (g + 1 == n) commit(&sm.o_full[i]);
          commit(&sm.kv_empty[1][t & 1]);
        }
        gg += n;
        ++a;
      }
      commit(&sm.mma_done[who]);
      drain_wait(&sm.mma_done[who], 0);
    }
    __syncwarp();
  } else if (warp >= 4 * kNT) {
    if (warp >= 8) regs_dec<kRegsUnpack>();
    // ------------------------------------------------------------ unpack
    // Eight rows at a time: lane 4 j + i has 16-byte chunk i (values 32 g + 8 i .. + 7 of the four
    // groups) of row 8 c + r(j), r exchanging bits 0 and 2 of j's order so that the two rows of
    // a quarter-warp's store lie in different halves of the swizzled 128 bytes.
    const int w = warp - 4 * kNT;
    const int i = lane & 3, jr = (((lane >> 2) & 1) << 2) | (lane >> 3);
    constexpr uint32_t kRawStage = kKeys * 72;
    const int r0 = w * kGroups * 8 + jr;  // this lane's first row of a tile; the others lie 8 apart
    const uint32_t raw0 = smem_u32(sm.raw[0]) + (r0 ^ ((r0 >> 2) & 1)) * 64 + i * 16;  // its codes in a stage,
    const uint32_t raws0 = smem_u32(sm.raw[0]) + kKeys * 64 + r0 * 8;                  // and the row's scales
    // where this lane's eight values of group g go: 16-byte chunk 4 (g % 2) + i of panel g / 2
    uint32_t put[2];
#pragma unroll
    for (int g = 0; g < 2; ++g) put[g] = r0 * 128 + (((4 * g + i) ^ (jr & 7)) << 4);
    bool ok = true;
    int raw = 0, use = 0, gg = 0;
    for (int seg = first, n; seg < segs && ok; seg = after<kLong>(p, seg), gg += n) {
    n = segment<kLong>(p, seg, kRows).n;
#pragma unroll 1
    for (int m = 0; m < 2 * n; ++m) {
      const Item it = item_of(m, n);
      const int t = gg + it.tile, slot = t & 1;
      const bool here = wait(&sm.raw_full[raw], (uint32_t)use & 1u);
      if (!(ok = __all_sync(0xffffffffu, here))) break;
      uint4 u[kGroups];
      uint2 s2[kGroups];
#pragma unroll
      for (int c = 0; c < kGroups; ++c) {
        u[c] = p4::lds16(raw0 + raw * kRawStage + c * 512);
        s2[c] = p4::lds8(raws0 + raw * kRawStage + c * 64);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.raw_empty[raw]);
      if (++raw == kRaw) raw = 0, ++use;
      const bool got = wait(&sm.kv_empty[it.v][slot], ((uint32_t)(t >> 1) & 1u) ^ 1u);
      if (!(ok = __all_sync(0xffffffffu, got))) break;
      const uint32_t dst = smem_u32(sm.kv[it.v][slot]);
#pragma unroll
      for (int c = 0; c < kGroups; ++c) {
        const uint32_t wd[4] = {u[c].x, u[c].y, u[c].z, u[c].w};
        const __half2 sa = *reinterpret_cast<const __half2*>(&s2[c].x);
        const __half2 sb = *reinterpret_cast<const __half2*>(&s2[c].y);
        auto put_parts = [&](int g, const uint32_t (&hi)[4], const uint32_t (&lo)[4]) {
          const uint32_t at = dst + (g >> 1) * kKvPanel + put[g & 1] + c * 1024;
          st_shared_v4(at, hi[0], hi[1], hi[2], hi[3]);
          st_shared_v4(at + kPart, lo[0], lo[1], lo[2], lo[3]);
        };
        uint32_t hi[4], lo[4];
        if (it.v == 0) {
          const __half2 sg[4] = {__low2half2(sa), __high2half2(sa), __low2half2(sb), __high2half2(sb)};
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            p4::numbers_f16(wd[g], hi);
            split_f16(hi, lo, sg[g]);
            put_parts(g, hi, lo);
          }
        } else {
          const float2 fa = __half22float2(sa), fb = __half22float2(sb);
          const float f[4] = {fa.x, fa.y, fb.x, fb.y};
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const float top = __bfloat162float(__float2bfloat16_rn(f[g]));
            p4::numbers_bf16(wd[g], hi);
            split_bf16(hi, lo, pack_bf16x2(top, f[g] - top));
            put_parts(g, hi, lo);
          }
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.kv_full[it.v][slot]);
    }
    }
  } else {
    regs_inc<kRegsSoft>();
    // ------------------------------------------------------------ softmax / epilogue
    const int i = warp >> 2;
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t lane_field = (uint32_t)(quarter * 32) << 16;
    const uint32_t tO = tmem + lane_field + 256 + i * 128;
    int a = 0, gg = 0;
    bool ok = true;
    // The scale of this thread's row of segment round `round`, never 0 or infinite; bf16: once its Q tile
    // is loaded, converts the row.
    auto in_range = [](float x) { return fminf(fmaxf(x, 1.4e-45f), 3.402823466e38f); };
    auto take_q = [&](int round) {
      if (!kBf16) return in_range(p.scale_log2);
      const bool got = wait(&sm.q_raw[i], (uint32_t)round & 1u);
      if (!(ok = __all_sync(0xffffffffu, got))) return 0.f;
      const float back = convert_row(sm.q[i], row);
      fence_proxy_async_smem();
      mbar_arrive(&sm.q_conv[i]);
      return in_range(p.scale_log2 * back);
    };
    auto more = [&](int seg) {  // whether a segment with keys follows
      for (seg = after<kLong>(p, seg); seg < segs; seg = after<kLong>(p, seg))
        if (segment<kLong>(p, seg, kRows).n > 0) return true;
      return false;
    };
    float sl2 = 0.f;
    bool have_q = false;
    // Of the segment's runs before this one, with O in p.fold: whether there are any, maximum, sum, and the scale of m.
    bool folded = false;
    float m_sum = 0.f, l_sum = 0.f, sl2_sum = 0.f;
    for (int seg = first; seg < segs && ok; seg = after<kLong>(p, seg)) {
    const Seg s = segment<kLong>(p, seg, kRows);
    const int n = s.n, grow = s.q0 + i * kBM + row;
    if (n > 0 && !have_q) {
      sl2 = take_q(a);
      if (!ok) break;
    }
    float m = -INFINITY, l = 0.f;  // m in units of S
    for (int g = 0; g < n; ++g) {
      const int t = gg + g;
      const int buf = t & 1;  // S and its barriers
      const uint32_t tS = tmem + lane_field + (2 * i + buf) * kKeys;
      const bool got = wait(&sm.s_full[i][buf], (uint32_t)(t >> 1) & 1u);
      if (!(ok = __all_sync(0xffffffffu, got))) break;
      tc_fence_after();
      uint32_t r[2][32];
      const int lim = s.len - (s.k0 + g) * kKeys;
      const bool full = lim >= kKeys;
      auto load_s = [&]() {
#pragma unroll
        for (int c = 0; c < 2; ++c) tmem_ld32(tS + c * 32, r[c]);
        tmem_ld_wait();
        if (!full) {
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (c * 32 + e >= lim) r[c][e] = __float_as_uint(-INFINITY);
        }
      };
#define SV(e) __uint_as_float(r[(e) >> 5][(e) & 31])
      auto row_max = [&]() {
        float acc[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) acc[k] = fmaxf(SV(2 * k), SV(2 * k + 1));
#pragma unroll
        for (int e = 16; e < kKeys; e += 16)
#pragma unroll
          for (int k = 0; k < 8; ++k) acc[k] = max3f(acc[k], SV(e + 2 * k), SV(e + 2 * k + 1));
        return max3f(max3f(acc[0], acc[1], acc[2]), max3f(acc[3], acc[4], acc[5]), fmaxf(acc[6], acc[7]));
      };
      uint64_t sum2[4];
      // 2^((S - mu) scale): the difference first, so that at the maximum itself it is exactly 0 however large
      // scores are (S scale - m with a rounded m is off by 16 once they pass 2^28).
      auto exp_pass = [&](float mu) {
        const float nb = (mu == -INFINITY) ? 0.f : -mu;
        const uint64_t scale2 = f2pack(sl2, sl2), base2 = f2pack(nb, nb);
#pragma unroll
        for (int k = 0; k < 4; ++k) sum2[k] = 0ull;
#pragma unroll
        for (int pr = 0; pr < kKeys / 2; ++pr) {
          float x0, x1;
          f2unpack(fma2(add2(f2pack(SV(2 * pr), SV(2 * pr + 1)), base2), scale2, 0ull), x0, x1);
          x0 = ex2_approx(x0);
          x1 = ex2_approx(x1);
          sum2[pr & 3] = add2(sum2[pr & 3], f2pack(x0, x1));
          r[pr >> 4][2 * (pr & 15)] = __float_as_uint(x0);
          r[pr >> 4][2 * (pr & 15) + 1] = __float_as_uint(x1);
        }
      };
      auto row_sum = [&]() {
        float sa, sb;
        f2unpack(add2(add2(sum2[0], sum2[1]), add2(sum2[2], sum2[3])), sa, sb);
        return sa + sb;
      };
      // As in the core kernel: P with the running max straight away; the row sum tells
      // whether it has to be redone with a larger one.
      load_s();
      float m_use = m, alpha = 1.f, sum;
      if (g == 0) {
        m_use = row_max();
        alpha = 0.f;
        exp_pass(m_use);
        sum = row_sum();
      } else {
        exp_pass(m);
        sum = row_sum();
        const bool check = !(sum <= 256.f) || (m == -INFINITY && sum > 0.f);
        if (__any_sync(0xffffffffu, check)) {
          load_s();
          const float m_tile = row_max();
          if (m == -INFINITY) {
            m_use = m_tile;
            alpha = 0.f;
          } else if ((m_tile - m) * sl2 > kRescaleThreshold) {
            m_use = m_tile;
            alpha = ex2_approx((m - m_tile) * sl2);
          }
          exp_pass(m_use);
          sum = row_sum();
        }
      }
      {  // P in two bf16 parts over S: upper in the first 32 columns, lower in the other 32
        uint32_t hi[32], lo[32];
#pragma unroll
        for (int k = 0; k < 32; ++k) {
          const float x0 = SV(2 * k), x1 = SV(2 * k + 1);
          hi[k] = pack_bf16x2(x0, x1);
          lo[k] = pack_bf16x2(x0 - __uint_as_float(hi[k] << 16), x1 - __uint_as_float(hi[k] & 0xffff0000u));
        }
        tmem_st32(tS, hi);
        tmem_st32(tS + 32, lo);
      }
#undef SV
      l = l * alpha + sum;
      if (__any_sync(0xffffffffu, g > 0 && alpha != 1.f)) {
        // the P V before this step may still run
        const bool idle = wait(&sm.pv_done[i], (uint32_t)(t - 1) & 1u);
        if (!(ok = __all_sync(0xffffffffu, idle))) break;
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t o[32];
          tmem_ld32(tO + c * 32, o);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
          tmem_st32(tO + c * 32, o);
        }
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&sm.p_full[i][buf]);
      m = m_use;
    }
    if (!ok) break;
    float sl2_of_m = sl2;  // the next segment's may be fetched before m is written
    if (n > 0) {
      // The next segment's Q tile, if any, has been loading since this one's last QK^T.
      have_q = kBf16 && more(seg);
      if (have_q) sl2 = take_q(a + 1);
      const bool got = ok && wait(&sm.o_full[i], (uint32_t)a & 1u);
      if (!(ok = __all_sync(0xffffffffu, got))) break;
      tc_fence_after();
    }
    {
      float f_old = 1.f, f_new = 1.f;  // factors of the O's
      if (kLong && folded) {
        if (n > 0) {
          const float M = fmaxf(m_sum, m);
          f_old = m_sum == -INFINITY ? 0.f : ex2_approx((m_sum - M) * sl2_of_m);
          f_new = m == -INFINITY ? 0.f : ex2_approx((m - M) * sl2_of_m);
          m = M;
          l = fmaf(l_sum, f_old, l * f_new);
        } else {
          m = m_sum;
          l = l_sum;
          sl2_of_m = sl2_sum;
        }
      }
      const bool some = n > 0 || (kLong && folded);
      float* const fold = p.fold + ((long long)blockIdx.x * kRows + i * kBM + row) * kD;  // kLong
      float4* const stage = sm.stage[warp];
      const int r0 = grow - lane;  // the warp's first row
      const int nvalid = p.S_q - r0;
      const bool direct = p.part == nullptr;
      const float inv = !direct ? 1.f : l == 0.f ? 0.f : 1.f / l;  // no key: zeros
      const long long urow = i * kBM + quarter * 32;
      float* const part = direct ? nullptr : p.part + ((long long)s.slice * p.units + s.unit) * kv4_part_floats(kRows);
      const long long out_at = (long long)s.b * p.ob + (long long)(s.bh % p.H) * p.oh + (long long)r0 * p.os;
#pragma unroll 1
      for (int c = 0; c < 4 && (s.last ? direct || some : n > 0); ++c) {
        float v[32];
        if (n > 0) {
          uint32_t o[32];
          tmem_ld32(tO + c * 32, o);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = __uint_as_float(o[e]);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = 0.f;
        }
        if (kLong && folded) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float4 x = *reinterpret_cast<const float4*>(fold + c * 32 + 4 * e);
            v[4 * e] = fmaf(x.x, f_old, v[4 * e] * f_new);
            v[4 * e + 1] = fmaf(x.y, f_old, v[4 * e + 1] * f_new);
            v[4 * e + 2] = fmaf(x.z, f_old, v[4 * e + 2] * f_new);
            v[4 * e + 3] = fmaf(x.w, f_old, v[4 * e + 3] * f_new);
          }
        }
        if (kLong && !s.last) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            *reinterpret_cast<float4*>(fold + c * 32 + 4 * e) = make_float4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
        } else if (direct && !p.out_f32) {
          store_block<kBf16 ? ANIMA_DTYPE_BF16 : ANIMA_DTYPE_F16>(static_cast<char*>(p.out) + out_at * 2, p.os * 2,
                                                                   nvalid, v, c, inv, stage, lane);
        } else if (!direct || lane < nvalid) {  // fp32: a partial, or the output
          float* const to = direct ? static_cast<float*>(p.out) + out_at + lane * p.os : part + (urow + lane) * kD;
#pragma unroll
          for (int e = 0; e < 8; ++e)
            *reinterpret_cast<float4*>(to + c * 32 + 4 * e) =
                make_float4(v[4 * e] * inv, v[4 * e + 1] * inv, v[4 * e + 2] * inv, v[4 * e + 3] * inv);
        }
      }
      if (s.last && !direct) {
        part[kRows * kD + urow + lane] = m == -INFINITY ? m : m * sl2_of_m;
        part[kRows * kD + kRows + urow + lane] = l;
      }
      if (kLong) {
        folded = !s.last && some;
        m_sum = m;
        l_sum = l;
        sl2_sum = sl2_of_m;
      }
    }
    if (n > 0) {
      tc_fence_before();
      mbar_arrive(&sm.o_empty[i]);
      gg += n;
      ++a;
    }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp12) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// Joins the slices of every query row: out = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s, in
// slice order.  One warp per row, four columns per lane; up to 64 slices.  part: [slice][unit][kv4_part_floats(rows)].
template <int kOut>
__global__ void __launch_bounds__(256)
    kv4_merge_kernel(const float* part, void* out, long long ob, long long oh, long long os, int H, int S_q,
                     int nqb, int rows, int units, int nsplit, long long total) {
  const int lane = threadIdx.x & 31;
  grid_dependency_wait();  // launched while the slices' kernel drains
  const long long stride = (long long)units * kv4_part_floats(rows);
  for (long long t = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5; t < total;
       t += ((long long)gridDim.x * blockDim.x) >> 5) {
    const int bh = (int)(t / S_q), s = (int)(t - (long long)bh * S_q);
    const int unit = bh * nqb + s / rows, r = s % rows;
    const float* const base = part + (long long)unit * kv4_part_floats(rows);
    const float* const mp = base + (long long)rows * kD + r;
    // lane k holds m and l of slices k and k + 32; a slice without keys has l = 0, and its O may not be
    // written
    float m[2], f[2], den = 0.f, M = -INFINITY;
    uint32_t some[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = lane + 32 * h;
      m[h] = k < nsplit ? mp[k * stride] : -INFINITY;
      f[h] = k < nsplit ? mp[k * stride + rows] : 0.f;
      M = fmaxf(M, m[h]);
    }
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      // only NaN scores leave the maximum at its start: their NaN sums come through
      const float l = f[h];
      some[h] = __ballot_sync(0xffffffffu, l != 0.f);
      f[h] = m[h] == -INFINITY ? 0.f : ex2_approx(m[h] - M);
      den = fmaf(f[h], l, den);
    }
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) den += __shfl_xor_sync(0xffffffffu, den, d);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    const float* const op = base + (long long)r * kD + lane * 4;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll 8
      for (int k = 32 * h; k < min(nsplit, 32 * h + 32); ++k) {
        const bool take = some[h] >> (k & 31) & 1u;
        const float fk = __shfl_sync(0xffffffffu, f[h], k & 31);  // finite where O is taken as 0
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        if (take) o = *reinterpret_cast<const float4*>(op + k * stride);
        acc.x = fmaf(fk, o.x, acc.x);
        acc.y = fmaf(fk, o.y, acc.y);
        acc.z = fmaf(fk, o.z, acc.z);
        acc.w = fmaf(fk, o.w, acc.w);
      }
    }
    const float inv = den == 0.f ? 0.f : 1.f / den;
    const long long at = (long long)(bh / H) * ob + (long long)(bh % H) * oh + (long long)s * os + lane * 4;
    if (kOut == ANIMA_DTYPE_F32) {
      *reinterpret_cast<float4*>(static_cast<float*>(out) + at) =
          make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
      continue;
    }
    uint32_t w0, w1;
    if (kOut == ANIMA_DTYPE_BF16) {
      w0 = pack_bf16x2(acc.x * inv, acc.y * inv);
      w1 = pack_bf16x2(acc.z * inv, acc.w * inv);
    } else {
      w0 = pack_f16x2(acc.x * inv, acc.y * inv);
      w1 = pack_f16x2(acc.z * inv, acc.w * inv);
    }
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + at) = make_uint2(w0, w1);
  }
}

}  // namespace kv4t

// How a call of many rows is cut: query tiles per unit, units, slices of the keys.
Kv4TilePlan kv4_tile_plan(int bh, int S_q, int S_kv, int sm_count) {
  Kv4TilePlan t;
  t.nt = S_q <= attn::kBM ? 1 : 2;
  t.nqb = (S_q + t.nt * attn::kBM - 1) / (t.nt * attn::kBM);
  t.units = (long long)bh * t.nqb;
  const long long tiles = (S_kv + kv4t::kKeys - 1) / kv4t::kKeys;
  // Slices: at most as many as the SMs hold in one round; the number with the least of the longest
  // chain of key tiles, some 1.65 us each, plus, if more than one, the merge: 2.7 tiles, and per slice 0.11
  // and 0.012 for every 256 rows.  In us from graphs, by slices: 32 units, 8 tiles: 22.2 whole, 23.1 in 2, 21.0 in 4; 16
  // units, 32 tiles: 63 whole, 30 in 4, 23.5 in 8; 8 units, 64 tiles: 30.0 in 8, 24.8 in 16; one unit,
  // 256 tiles: 69 in 8, 45 in 16, 34.6 in 32, 33.3 in 64.
  const long long most = std::min({sm_count / std::max(1LL, t.units), tiles, 64LL});
  t.nsplit = 1;
  double best = (double)tiles;
  for (int k = 2; k <= most; ++k) {
    const double cost = (double)((tiles + k - 1) / k) + 2.7 + k * (0.11 + 0.006 * (double)(t.units * t.nt));
    if (cost < best) {
      best = cost;
      t.nsplit = k;
    }
  }
  t.runs = (int)(((tiles + t.nsplit - 1) / t.nsplit + kv4t::kRun - 1) / kv4t::kRun);
  t.grid = (int)std::min<long long>(t.units * t.nsplit, sm_count);
  t.part_bytes = t.nsplit > 1 ? (size_t)(t.nsplit * t.units * kv4_part_floats(t.nt * attn::kBM)) * 4 : 0;
  t.bytes = t.part_bytes + (t.runs > 1 ? (size_t)t.grid * (t.nt * attn::kBM) * attn::kD * 4 : 0);
  return t;
}

template <bool kBf16, int kNT, bool kLong>
static int tile_t(const CUtensorMap& mq, const kv4t::Params& p, int grid, cudaStream_t st) {
  auto kern = kv4t::kv4_tile_kernel<kBf16, kNT, kLong>;
  constexpr size_t smem = kv4t::smem_bytes<kNT>();
  static SmemAttr attr;
  if (!attr.raise((const void*)kern, smem)) return ANIMA_ERR_CUDA;
  return launch_dependent(kern, grid, kv4t::kThreads16, smem, st, mq, p);
}

int kv4_merge_launch(const AnimaAttnKv4Args* a, const float* part, int nqb, int rows, int units, int nsplit,
                     int sm_count, cudaStream_t st) {
  const long long total = (long long)a->B * a->H * a->S_q;
  auto merge = (a->flags & ANIMA_FLAG_OUT_F32)   ? kv4t::kv4_merge_kernel<ANIMA_DTYPE_F32>
               : a->dtype == ANIMA_DTYPE_BF16 ? kv4t::kv4_merge_kernel<ANIMA_DTYPE_BF16>
                                              : kv4t::kv4_merge_kernel<ANIMA_DTYPE_F16>;
  const int grid = (int)std::min<long long>((total + 7) / 8, (long long)sm_count * 8);
  return launch_dependent(merge, grid, 256, 0, st, part, a->out, (long long)a->out_stride[0],
                          (long long)a->out_stride[1], (long long)a->out_stride[2], a->H, a->S_q, nqb, rows,
                          units, nsplit, total);
}

int kv4_tile_launch(const AnimaAttnKv4Args* a, const Kv4TilePlan& t, int* status, int sm_count, cudaStream_t st) {
  const bool bf = a->dtype == ANIMA_DTYPE_BF16;
  if (t.units * t.nsplit * t.runs > 1 << 30) return ANIMA_ERR_SHAPE;  // with one round of the grid below 2^31
  kv4t::Params p;
  p.kc = static_cast<const uint8_t*>(a->k_codes);
  p.ks = static_cast<const uint8_t*>(a->k_scales);
  p.vc = static_cast<const uint8_t*>(a->v_codes);
  p.vs = static_cast<const uint8_t*>(a->v_scales);
  p.valid = (a->flags & ANIMA_FLAG_MASK) ? a->kv_valid_len : nullptr;
  p.out = a->out;
  p.part = t.nsplit > 1 ? static_cast<float*>(a->workspace) : nullptr;
  p.fold = reinterpret_cast<float*>(static_cast<char*>(a->workspace) + t.part_bytes);
  p.ob = a->out_stride[0];
  p.oh = a->out_stride[1];
  p.os = a->out_stride[2];
  p.status = status;
  p.H = a->H;
  p.S_q = a->S_q;
  p.S_kv = a->S_kv;
  p.nqb = t.nqb;
  p.units = (int)t.units;
  p.nsplit = t.nsplit;
  p.runs = t.runs;
  p.out_f32 = (a->flags & ANIMA_FLAG_OUT_F32) != 0;
  p.scale_log2 = std::min(a->scale * 1.4426950408889634f, 3.402823466e38f);
  CUtensorMap mq;
  int rc = attn_head_map(&mq, a->q, a->dtype, a->B * a->H, a->S_q);
  if (rc != ANIMA_OK) return rc;
  auto go = [&](auto nt, auto is_long) {
    constexpr int kNT = decltype(nt)::value;
    constexpr bool kLong = decltype(is_long)::value;
    return bf ? tile_t<true, kNT, kLong>(mq, p, t.grid, st) : tile_t<false, kNT, kLong>(mq, p, t.grid, st);
  };
  auto of = [&](auto nt) { return t.runs > 1 ? go(nt, std::true_type()) : go(nt, std::false_type()); };
  rc = t.nt == 1 ? of(std::integral_constant<int, 1>()) : of(std::integral_constant<int, 2>());
  if (rc != ANIMA_OK || t.nsplit == 1) return rc;
  return kv4_merge_launch(a, p.part, t.nqb, t.nt * attn::kBM, p.units, t.nsplit, sm_count, st);
}

}  // namespace anima
