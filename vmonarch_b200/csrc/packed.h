// Parameter blocks of the packed-sequence attention kernels (packed_fwd.cu, packed_bwd.cu).
#pragma once
#include <cuda.h>
#include <stdint.h>

#include "fea_params.h"

namespace vmb {

// One unit of a packed call's work, built on the host from the sequence lengths
// (vmb_packed_unit of include/vmonarch_b200.h, same layout).
//  forward and dQ : query rows [q_row, q_row + q_valid) (at most 256 / 128) of a sequence whose keys
//                   are rows [k_row, k_row + k_valid); local query r sees the keys below
//                   clamp(vis0 + r * causal, 0, k_valid); the unit walks key tiles [begin, end)
//                   (128 keys each). stat_row: the unit's first row in the padded statistics.
//  dK / dV        : key rows [k_row, k_row + k_valid) (at most 128) of a sequence whose queries are
//                   rows [q_row, q_row + q_valid); local key r is seen by the queries from
//                   vis0 + r on (all of them when not causal); the unit walks steps [begin, end) of
//                   its (query head of the group, 64-query tile) pairs, the tiles of a head counted
//                   from max(vis0, 0) / 64. stat_row: the sequence's first padded statistics row.
//                   The sequence's queries below `lone` see one key at most.
//  part           : -1, or the slot that a split unit's partial result goes to
struct PackedUnit {
  int32_t q_row, q_valid, k_row, k_valid, vis0, begin, end, part, stat_row, pieces, lone, pad;
};

struct PackedParams {
  const PackedUnit* units;
  const int32_t* joins;    // (first unit, pieces) of cut units
  int n_units, n_joins;
  int heads, kv_heads, group, head_chunk;  // head_chunk: (query or kv) heads whose units run together
  int dim, causal;
  int64_t q_total, k_total, stat_rows;     // stat_rows: rows of the padded statistics planes
  float sm_scale;
  const void *q, *k, *v, *dout;
  void *o, *o_low, *dq, *dk, *dv;  // o_low: the 16-bit rest that rounding o left out (may be NULL, forward)
  float* lse;              // [heads][q_total], natural logarithm
  float* stats;            // backward: planes nl, nc, row scales, each [heads][stat_rows]
  float* tile_scale;       // backward: least row scale of 128 rows, [heads][stat_rows / 128]
  float* centre;           // backward: mean of a sequence's first keys, [kv_heads][stat_rows / 128][128]
  float *part, *part_ml;   // split units: partial tiles and their (max, sum)
  View qv, kv, vv, ov, olv, dov, dqv, dkv, dvv;  // rows = tokens, s1 = head stride
  long long wait_limit;    // pipeline wait limit in cycles (0: the default ~2 s)
  int hold_loads;          // test of the timeout path: the producers issue no load
};

// Unit and head of a block: chunks of `chunk` heads outermost (their keys and values stay in L2),
// inside them the units in the host's order (most work first), heads innermost.
struct UnitHead {
  int unit, head;
};
#ifdef __CUDACC__
__host__ __device__ __forceinline__ UnitHead unit_of_block(int64_t block, int n_units, int heads, int chunk) {
  const int64_t per = (int64_t)n_units * chunk;
  const int c = (int)(block / per);
  const int rem = (int)(block - c * per);
  const int left = heads - c * chunk;
  const int g = left < chunk ? left : chunk;
  return UnitHead{rem / g, c * chunk + rem % g};
}

// 32 bytes to a 32-byte aligned global address (one sector, one store)
__device__ __forceinline__ void st_global_v8(void* ptr, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(ptr), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
// 32 columns of a row, as 16 packed words; whole sectors where rows are 32-byte aligned. dim: a multiple of 8.
__device__ __forceinline__ void store_row32(uint16_t* row, int col, int dim, bool sectors, const uint32_t* x) {
  if (sectors && col + 32 <= dim) {
    st_global_v8(row + col, x);
    st_global_v8(row + col + 16, x + 8);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (col + 8 * k < dim) *reinterpret_cast<uint4*>(row + col + 8 * k) = make_uint4(x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3]);
  }
}
// Whether the rows of a 16-bit tensor start at whole 32-byte sectors.
__device__ __forceinline__ bool whole_sectors(const void* t, const View& v) {
  return ((v.rs | v.s1) & 15) == 0 && (reinterpret_cast<uintptr_t>(t) & 31) == 0;
}
#endif

}  // namespace vmb
