// Products of rows grouped by expert (grouped.cu, grouped_tc.cu).
#pragma once

#include "common.cuh"

namespace bm {

// For every slot of a selection [T, k]: its place among the routed assignments (token_indices, offsets as bm_route_build makes them), or -1.
struct SlotArgs {
  const int32_t *topk_idx, *map, *token_indices, *offsets;
  int32_t* pos;                // [T * k]; null: nothing to do
  int slots, k, E, num_routed;
  int sparse;                  // most slots name experts that are not held here
  int distinct;                // slots of a token that name one expert share a row
  const int32_t* window;       // [2] tokens from, to: the others' slots are left alone; null: all
};

// y[i][n] = sum_k x[row(i)][k] * w[e][n][k] for offsets[e] <= i < offsets[e + 1], row(i) = index[i] (i itself when null).
// glu: w holds 2 N rows per expert, gate rows before up rows, and y[i][n] = silu(row n) * row (N + n).
// offsets null: one group of all `rows` rows.
struct GroupedArgs {
  const void* x;               // [x_rows, K]
  const void* w;               // [E, N or 2 N, K], of x's type
  const int32_t* offsets;      // [E + 1], device
  const int32_t* index;        // [rows], device; entries outside [0, x_rows) stand for rows of zeros
  void* y;                     // [rows, N]
  int x_rows, rows, K, N, E;
  int dtype, y_dtype;          // of x and w: BM_F16 or BM_BF16; of y: the same or BM_F32
  int glu;
  float* wide;                 // glu with fp16 y: [rows, N], gets the values that fp16 does not hold (their y is infinite); or null
  const float* x_wide;         // such values of x (fp16, in order, fp32 y); or null
  int expected;                // rows that the groups are expected to have, 0 = `rows`
  void* gathered;              // with an index: room for [rows, K], 16-byte aligned, or null
  SlotArgs slots;              // worked out beside the products
  int may_be_empty;            // offsets ascend, and offsets[E] = 0 is to be expected
  LaunchAfter after;
};

__device__ __forceinline__ int slot_expert(const SlotArgs& a, int i) {
  const int id = a.topk_idx[i];
  if (id < 0 || id >= a.num_routed) return -1;
  const int e = a.map ? a.map[id] : id;
  return e >= 0 && e < a.E ? e : -1;
}
// Slot i's place: the routing build keeps an expert's list in ascending (token, slot) order, so the token is found by bisection; an expert
// may be named twice.
__device__ __forceinline__ int slot_place(const SlotArgs& a, int i) {
  const int e = slot_expert(a, i), t = i / a.k;
  if (e < 0) return -1;
  int lo = a.offsets[e], hi = a.offsets[e + 1];
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a.token_indices[mid] < t) lo = mid + 1;
    else hi = mid;
  }
  if (!a.distinct)
    for (int j = t * a.k; j < i; ++j) lo += slot_expert(a, j) == e;
  return lo;
}

__device__ __forceinline__ int2 slot_range(const SlotArgs& a) {
  return a.window ? make_int2(__ldcg(a.window) * a.k, __ldcg(a.window + 1) * a.k) : make_int2(0, a.slots);
}

// The rows of group e, whatever the caller's table holds: inside [0, rows), ends not before they start.
__device__ __forceinline__ int2 group_rows(const int32_t* offsets, int e, int rows) {
  if (!offsets) return make_int2(0, rows);
  const int a = min(max(__ldg(offsets + e), 0), rows);
  return make_int2(a, min(max(__ldg(offsets + e + 1), a), rows));
}

__device__ __forceinline__ float silu_mul(float g, float u) { return __fdividef(g, 1.f + __expf(-g)) * u; }

// Whether rounding v to fp16 leaves a number (65520 is half way from the largest one to the next power of two).
__device__ __forceinline__ bool fits_fp16(float v) { return fabsf(v) < 65520.f; }

// Where the kernels of the dense products report a wait that gave up, and how long one waits (0: as if one had given up at the start).
struct DenseGuard {
  int* status;
  uint64_t limit_ns;
};
int dense_guard(DenseGuard* g);      // of the current device

// BM_ERR_UNSUPPORTED, with nothing launched, when a shape or pointer does not suit tiled copies (grouped_tc.cu).
int launch_grouped_tc(const GroupedArgs& a, cudaStream_t st);
// Whether rows picked by an index are brought into expert order before the products.
bool grouped_gathers(int expected, int E, int K);
// The tensor-core kernel, else the one that takes every shape.
int launch_grouped(const GroupedArgs& a, cudaStream_t st);

}  // namespace bm
