// attn_kv4.cuh -- host interface between the two kernels of the attention over packed K/V.
#pragma once
#include <stddef.h>

#include "common.cuh"

namespace anima {

// Tensor map of a [bh][rows][128] 16-bit operand, boxes of 128 rows x 64 elements, 128-byte
// swizzle (attn_fwd.cu).
int attn_head_map(CUtensorMap* map, const void* base, int op_dtype, int bh, int rows);

// Floats of a partial result of a unit: O [rows][128], m [rows], l [rows], and padding that keeps the
// next partial 16-byte aligned.
__host__ __device__ constexpr long long kv4_part_floats(int rows) { return ((long long)rows * 130 + 3) & ~3ll; }

// A call of many query rows (attn_kv4_tile.cu).
struct Kv4TilePlan {
  int nt;           // 128-row query tiles per unit
  int nqb;          // units per (batch, head)
  long long units;
  int nsplit;       // slices of a unit's keys
  int runs;         // runs of a slice's keys, one after another
  int grid;         // CTAs
  size_t part_bytes;  // workspace for the slices' partials,
  size_t bytes;       // and with a CTA's sums over runs behind them
};
Kv4TilePlan kv4_tile_plan(int bh, int S_q, int S_kv, int sm_count);
// Joins partials [slice][unit][kv4_part_floats(rows)] into a->out.
int kv4_merge_launch(const AnimaAttnKv4Args* a, const float* part, int nqb, int rows, int units, int nsplit,
                     int sm_count, cudaStream_t st);
int kv4_tile_launch(const AnimaAttnKv4Args* a, const Kv4TilePlan& t, int* status, int sm_count, cudaStream_t st);

}  // namespace anima
