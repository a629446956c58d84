// Dense products beside the packed experts, grouped by expert: entry points, the kernel that takes every shape, and the weighted
// sum over a token's experts.
//   y[i] = x[row(i)] . W[e(i)]^T                                                             (bm_grouped_linear)
//   y[t] = residual[t] + sum_s w[t, s] * Wd[e] . (silu(Wg[e] . x[t]) * (Wu[e] . x[t]))       (bm_dense_experts_forward)
// The second is what a block runs for its un-quantised ("super") experts, which the reference runs one module at a time on the rows
// that torch.nonzero finds (bitsmoe/models/base_block.py:291-313): routing build, gate and up products with silu * mul, down products,
// weighted sum, on one stream and without a host round trip.
#include <algorithm>

#include "grouped.cuh"

namespace bm {

constexpr int GG_ROWS = 16, GG_COLS = 64, GG_K = 32, GG_THREADS = 256;

template <int D>
__device__ __forceinline__ float load16(const void* p, int64_t i) {
  return D == BM_F16 ? __half2float(static_cast<const __half*>(p)[i]) : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

// Rows a group from which a pass over the rows of x costs less than fetching them four at a time for every item.  128 groups, K 2048, N 1536, us
// by a pass first / by gather copies / with the rows in order: 8 rows 148 / 128 / 124, 32 rows 155 / 135 / 130, 48 rows 155 / 146 / 134, 64 rows 166 / 198 /
// 142, 128 rows 180 / 290 / 155, 512 rows 400 / 900 / 340: four rows of 128 bytes take the copy engine 57 cycles.
constexpr int GATHER_ROWS = 56;

// Any shape and alignment: a CTA takes 16 rows of a group and 64 output columns, element loads, fp32 FMA.
template <int D, bool GLU>
__global__ void __launch_bounds__(GG_THREADS) grouped_any_kernel(const GroupedArgs a) {
  __shared__ float xs[GG_K][GG_ROWS + 1], ws[GLU ? 2 : 1][GG_K][GG_COLS + 1];
  __shared__ int found[3];
  __shared__ int src[GG_ROWS];
  const int lane = threadIdx.x & 31, n0 = blockIdx.x * GG_COLS;
  grid_launch_dependents();
  grid_wait();
  for (int64_t tile = blockIdx.y;; tile += gridDim.y) {
    // the group of row tile `tile`: 32 groups at a time
    if (threadIdx.x < 32) {
      int64_t before = 0;
      if (lane == 0) found[0] = -1;
      for (int e0 = 0; e0 < a.E; e0 += 32) {
        const int e = e0 + lane;
        const int2 r = e < a.E ? group_rows(a.offsets, e, a.rows) : make_int2(0, 0);
        const int n = (r.y - r.x + GG_ROWS - 1) / GG_ROWS;
        int incl = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += v;
        }
        const int64_t first = before + incl - n;
        if (tile >= first && tile < first + n) {
          found[0] = e;
          found[1] = r.x + static_cast<int>(tile - first) * GG_ROWS;
          found[2] = r.y;
        }
        before += __shfl_sync(0xffffffffu, incl, 31);
        if (before > tile) break;
      }
    }
    __syncthreads();
    const int e = found[0], row0 = found[1], rows = min(GG_ROWS, found[2] - row0);
    if (e < 0) return;
    if (threadIdx.x < GG_ROWS) {
      int r = -1;
      if (threadIdx.x < rows) r = a.index ? __ldg(a.index + row0 + threadIdx.x) : row0 + threadIdx.x;
      src[threadIdx.x] = r >= 0 && r < a.x_rows ? r : -1;
    }
    __syncthreads();
    const int col = threadIdx.x & 63, rg = threadIdx.x >> 6;      // four rows of one column
    const int64_t w0 = static_cast<int64_t>(e) * (GLU ? 2 : 1) * a.N;
    float acc[GLU ? 2 : 1][4] = {};
    for (int k0 = 0; k0 < a.K; k0 += GG_K) {
      for (int i = threadIdx.x; i < GG_ROWS * GG_K; i += GG_THREADS) {
        const int r = i / GG_K, k = i % GG_K;
        xs[k][r] = src[r] >= 0 && k0 + k < a.K ? load16<D>(a.x, static_cast<int64_t>(src[r]) * a.K + k0 + k) : 0.f;
      }
#pragma unroll
      for (int h = 0; h < (GLU ? 2 : 1); ++h)
        for (int i = threadIdx.x; i < GG_COLS * GG_K; i += GG_THREADS) {
          const int c = i / GG_K, k = i % GG_K;
          ws[h][k][c] = n0 + c < a.N && k0 + k < a.K ? load16<D>(a.w, (w0 + static_cast<int64_t>(h) * a.N + n0 + c) * a.K + k0 + k) : 0.f;
        }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < GG_K; ++k)
#pragma unroll
        for (int h = 0; h < (GLU ? 2 : 1); ++h) {
          const float w = ws[h][k][col];
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[h][j] = fmaf(xs[k][4 * rg + j], w, acc[h][j]);
        }
      __syncthreads();
    }
    if (n0 + col < a.N)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (4 * rg + j < rows) {
          const int64_t o = static_cast<int64_t>(row0 + 4 * rg + j) * a.N + n0 + col;
          const float v = GLU ? silu_mul(acc[0][j], acc[GLU ? 1 : 0][j]) : acc[0][j];
          store_act(a.y, a.y_dtype, o, v);
          if (GLU && D == BM_F16 && a.wide && !fits_fp16(v)) a.wide[o] = v;
        }
    __syncthreads();
  }
}

// Rows picked by an index, in the order of the groups: out[i] = x[index[i]] for the rows that groups own.  A warp takes four rows at a time.
constexpr int GR_THREADS = 256, GR_ROWS = 4;
__global__ void __launch_bounds__(GR_THREADS) gather_rows_kernel(const uint4* __restrict__ x, const int32_t* __restrict__ index, const int32_t* __restrict__ offsets,
                                                                 int E, int x_rows, int rows, int pieces, uint4* __restrict__ out) {
  grid_launch_dependents();
  grid_wait();
  const int lane = threadIdx.x & 31, warps = gridDim.x * (GR_THREADS / 32), end = min(max(__ldg(offsets + E), 0), rows);
  for (int64_t i0 = static_cast<int64_t>(blockIdx.x * (GR_THREADS / 32) + (threadIdx.x >> 5)) * GR_ROWS; i0 < end; i0 += static_cast<int64_t>(warps) * GR_ROWS) {
    const uint4* src[GR_ROWS];
#pragma unroll
    for (int r = 0; r < GR_ROWS; ++r) {
      const int id = __ldg(index + min(i0 + r, static_cast<int64_t>(end - 1)));
      src[r] = id >= 0 && id < x_rows ? x + static_cast<int64_t>(id) * pieces : nullptr;
    }
#pragma unroll 2
    for (int c = lane; c < pieces; c += 32) {
      uint4 v[GR_ROWS];
#pragma unroll
      for (int r = 0; r < GR_ROWS; ++r) v[r] = src[r] ? __ldg(src[r] + c) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (int r = 0; r < GR_ROWS; ++r)
        if (i0 + r < end) out[(i0 + r) * pieces + c] = v[r];
    }
  }
}

__global__ void __launch_bounds__(256) slot_places_kernel(const SlotArgs a) {
  grid_launch_dependents();
  grid_wait();
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < a.slots) a.pos[i] = slot_place(a, i);
}

bool grouped_gathers(int expected, int E, int K) { return K % 8 == 0 && expected / E >= GATHER_ROWS; }

int launch_grouped(const GroupedArgs& args, cudaStream_t st) {
  GroupedArgs a = args;
  if (a.rows == 0 || a.E == 0) return BM_OK;
  if (a.index && a.gathered && a.x_rows > 0 && aligned16(a.x, a.w, a.gathered) && grouped_gathers(a.expected ? a.expected : a.rows, a.E, a.K)) {
    const int per = GR_THREADS / 32 * GR_ROWS, blocks = std::min((a.rows + per - 1) / per, 148 * 8);
    BM_CUDA(launch_after(a.after, 1, gather_rows_kernel, dim3(blocks), GR_THREADS, 0, st, static_cast<const uint4*>(a.x), a.index, a.offsets, a.E, a.x_rows,
                         a.rows, a.K / 8, static_cast<uint4*>(a.gathered)));
    BM_LAUNCH_CHECK("gather_rows_kernel");
    a.x = a.gathered; a.x_rows = a.rows; a.index = nullptr; a.after = AFTER_READS;
  }
  const int rc = launch_grouped_tc(a, st);
  if (rc != BM_ERR_UNSUPPORTED) return rc;
  if (a.slots.pos) {
    BM_CUDA(launch_after(a.after, 1, slot_places_kernel, dim3((a.slots.slots + 255) / 256), 256, 0, st, a.slots));
    BM_LAUNCH_CHECK("slot_places_kernel");
    a.after = AFTER_READS;
  }
  const int64_t tiles = a.rows / GG_ROWS + static_cast<int64_t>(a.E < a.rows ? a.E : a.rows) + 1;
  const dim3 grid((a.N + GG_COLS - 1) / GG_COLS, static_cast<unsigned>(tiles < 65535 ? tiles : 65535));
  auto* kernel = a.dtype == BM_F16 ? (a.glu ? grouped_any_kernel<BM_F16, true> : grouped_any_kernel<BM_F16, false>)
                                   : (a.glu ? grouped_any_kernel<BM_BF16, true> : grouped_any_kernel<BM_BF16, false>);
  BM_CUDA(launch_after(a.after, 1, kernel, grid, GG_THREADS, 0, st, a));
  BM_LAUNCH_CHECK("grouped_any_kernel");
  return BM_OK;
}

// y[t] = residual[t] + sum over the slots s of w[t, s] * d[place of (t, s)], in the order of the slots.  A thread owns four columns of a
// token and has the rows of eight slots in flight; bound by reading d (fp32: rounded to 16 bits between the products a second time, the
// result of a bf16 layer would be 1.7 times as far from the exact one as a single rounding; as it is 1.4).
constexpr int EC_THREADS = 128, EC_MAX_K = 32;
struct CombineArgs {
  const float* d;              // [T * k, H] in expert order
  const int32_t* pos;          // [T, k]
  const float* topk_w;
  const void* residual;
  void* y;
  int k, H, vec;               // vec: H % 4 == 0, y and the residual on 8-byte boundaries
  // fp16: what the down product was made of
  SlotArgs slots;
  const void *z, *w_down;      // [rows, I], [E, H, I]
  const float* wide;           // [rows, I], valid where z is not finite
  int I;
};
// A column of a row of d from z's values before their rounding.  The product between the two matrices of an expert may pass fp16's range
// where the sum over it does not: z is infinite there, and with it the row of d.
__device__ __forceinline__ float wide_down(const CombineArgs& a, int slot, int64_t at, int h) {
  const __half *z = static_cast<const __half*>(a.z) + at * a.I, *w = static_cast<const __half*>(a.w_down) + (static_cast<int64_t>(slot_expert(a.slots, slot)) * a.H + h) * a.I;
  float v = 0.f;
#pragma unroll 4
  for (int i = 0; i < a.I; ++i) {
    float f = __half2float(z[i]);
    if (!(fabsf(f) <= 65504.f)) f = a.wide[at * a.I + i];
    v = fmaf(__half2float(w[i]), f, v);
  }
  return v;
}
template <int D>
__device__ __forceinline__ float4 load4(const void* p, int64_t i) {
  const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
  if (D == BM_F16) {
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&v.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
    return make_float4(a.x, a.y, b.x, b.y);
  }
  return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u));
}
template <int D>
__global__ void __launch_bounds__(EC_THREADS) experts_combine_kernel(const CombineArgs a) {
  const int t = blockIdx.x, h = (blockIdx.y * EC_THREADS + threadIdx.x) * 4;
  grid_launch_dependents();
  grid_wait();
  if (h >= a.H) return;
  const int64_t o = static_cast<int64_t>(t) * a.H + h;
  const int n = min(4, a.H - h);
  float v[4] = {};
  if (a.residual) {
    if (a.vec) *reinterpret_cast<float4*>(v) = load4<D>(a.residual, o);
    else
      for (int j = 0; j < n; ++j) v[j] = load16<D>(a.residual, o + j);
  }
  for (int s0 = 0; s0 < a.k; s0 += 8) {
    float4 d[8];
    float w[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int at = s0 + u < a.k ? __ldg(a.pos + static_cast<int64_t>(t) * a.k + s0 + u) : -1;
      w[u] = at >= 0 ? __ldg(a.topk_w + static_cast<int64_t>(t) * a.k + s0 + u) : 0.f;
      d[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (at >= 0) {
        const float* src = a.d + static_cast<int64_t>(at) * a.H + h;
        if (a.vec) d[u] = __ldcs(reinterpret_cast<const float4*>(src));
        else {
          d[u].x = src[0];
          if (n > 1) d[u].y = src[1];
          if (n > 2) d[u].z = src[2];
          if (n > 3) d[u].w = src[3];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      v[0] = fmaf(w[u], d[u].x, v[0]);
      v[1] = fmaf(w[u], d[u].y, v[1]);
      v[2] = fmaf(w[u], d[u].z, v[2]);
      v[3] = fmaf(w[u], d[u].w, v[3]);
    }
  }
  if (D == BM_F16 && !(fabsf((v[0] + v[1]) + (v[2] + v[3])) < __int_as_float(0x7f800000)))
    // once more, slot by slot, with the rows of d that are not finite worked out anew
#pragma unroll 1
    for (int j = 0; j < n; ++j) {
      float sum = a.residual ? load16<D>(a.residual, o + j) : 0.f;
#pragma unroll 1
      for (int s = 0; s < a.k; ++s) {
        const int slot = t * a.k + s, at = a.pos[slot];
        if (at < 0) continue;
        float d = a.d[static_cast<int64_t>(at) * a.H + h + j];
        if (!(fabsf(d) < __int_as_float(0x7f800000))) d = wide_down(a, slot, at, h + j);
        sum = fmaf(a.topk_w[slot], d, sum);
      }
      v[0] = j == 0 ? sum : v[0]; v[1] = j == 1 ? sum : v[1]; v[2] = j == 2 ? sum : v[2]; v[3] = j == 3 ? sum : v[3];
    }
  uint16_t out[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) out[j] = D == BM_F16 ? __half_as_ushort(__float2half_rn(v[j])) : __bfloat16_as_ushort(__float2bfloat16_rn(v[j]));
  if (a.vec) *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.y) + o) = make_uint2(out[0] | out[1] << 16, out[2] | out[3] << 16);
  else
    for (int j = 0; j < n; ++j) static_cast<uint16_t*>(a.y)[o + j] = out[j];
}

struct DenseExpertsWs {
  size_t tok, rw, pos, off, route, xs, z, wide, d, total;
  DenseExpertsWs(int64_t T, int64_t k, int64_t E, int64_t H, int64_t I) {
    const size_t A = static_cast<size_t>(T * k);
    size_t at = 0;
    auto take = [&](size_t bytes) {
      const size_t here = at;
      at += align_up(bytes, 256);
      return here;
    };
    tok = take(A * 4);
    rw = take(A * 4);
    pos = take(A * 4);
    off = take(static_cast<size_t>(E + 1) * 4);
    route = take(bm_route_build_workspace_bytes(static_cast<int32_t>(T), static_cast<int32_t>(k), static_cast<int32_t>(E)));
    z = take(A * I * 2);
    wide = take(A * I * 4);
    d = xs = take(A * H * 4);      // rows of x in expert order are read before the down products are written
    total = at;
  }
};

}  // namespace bm

using namespace bm;

extern "C" size_t bm_grouped_linear_workspace_bytes(int32_t K, int32_t E, int32_t rows) {
  if (K <= 0 || E <= 0 || rows <= 0 || !grouped_gathers(rows, E, K)) return 0;
  return static_cast<size_t>(rows) * K * 2;
}

extern "C" int bm_grouped_linear(const void* x, int dtype, const void* w, int32_t x_rows, int32_t K, int32_t N, int32_t E,
                                 const int32_t* expert_offsets, const int32_t* token_indices, int32_t rows, void* y, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  bm::NvtxRange nvtx_range("bm_grouped_linear");
  BM_REQUIRE(x_rows >= 0 && rows >= 0 && K > 0 && N > 0 && E >= 0, BM_ERR_INVALID_ARG, "grouped_linear: bad sizes");
  BM_REQUIRE(dtype == BM_F16 || dtype == BM_BF16, BM_ERR_INVALID_ARG, "grouped_linear: x and the weights must be fp16 or bf16");
  if (rows == 0 || E == 0) return BM_OK;
  BM_REQUIRE((x || x_rows == 0) && w && expert_offsets && y, BM_ERR_INVALID_ARG, "grouped_linear: null pointer");
  BM_REQUIRE(token_indices || rows <= x_rows, BM_ERR_INVALID_ARG, "grouped_linear: %d rows without indices, x has %d", rows, x_rows);
  const size_t need = token_indices ? bm_grouped_linear_workspace_bytes(K, E, rows) : 0;
  BM_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 255u) == 0), BM_ERR_WORKSPACE,
             "grouped_linear: workspace must be 256-byte aligned and hold %zu bytes (%zu given)", need, workspace_bytes);
  GroupedArgs a{};
  a.gathered = need ? workspace : nullptr;
  a.x = x; a.w = w; a.offsets = expert_offsets; a.index = token_indices; a.y = y;
  a.x_rows = x_rows; a.rows = rows; a.K = K; a.N = N; a.E = E; a.dtype = a.y_dtype = dtype;
  a.after = AFTER_READS;
  return launch_grouped(a, static_cast<cudaStream_t>(stream));
}

extern "C" size_t bm_dense_experts_workspace_bytes(int32_t T, int32_t k, int32_t num_local, int32_t hidden, int32_t intermediate) {
  if (T <= 0 || k <= 0 || num_local <= 0 || hidden <= 0 || intermediate <= 0) return 0;
  return DenseExpertsWs(T, k, num_local, hidden, intermediate).total;
}

extern "C" int bm_dense_experts_forward(const void* x, int dtype, const int32_t* topk_idx, const float* topk_w, const int32_t* global_to_local,
                                        int32_t num_routed, int32_t T, int32_t k, int32_t num_local, const void* w_gate_up, const void* w_down,
                                        int32_t hidden, int32_t intermediate, const void* residual, void* y, void* workspace,
                                        size_t workspace_bytes, void* stream) {
  bm::NvtxRange nvtx_range("bm_dense_experts_forward");
  BM_REQUIRE(T >= 0 && k > 0 && num_local > 0 && num_routed > 0 && hidden > 0 && intermediate > 0, BM_ERR_INVALID_ARG, "dense_experts: bad sizes");
  BM_REQUIRE(dtype == BM_F16 || dtype == BM_BF16, BM_ERR_INVALID_ARG, "dense_experts: x and the weights must be fp16 or bf16");
  BM_REQUIRE(k <= EC_MAX_K, BM_ERR_UNSUPPORTED, "dense_experts: top_k=%d exceeds %d", k, EC_MAX_K);
  BM_REQUIRE(static_cast<int64_t>(T) * k < (1ll << 30), BM_ERR_UNSUPPORTED, "dense_experts: too many assignments");
  if (T == 0) return BM_OK;
  BM_REQUIRE(x && topk_idx && topk_w && w_gate_up && w_down && y, BM_ERR_INVALID_ARG, "dense_experts: null pointer");
  const DenseExpertsWs at(T, k, num_local, hidden, intermediate);
  BM_REQUIRE(workspace && workspace_bytes >= at.total && (reinterpret_cast<uintptr_t>(workspace) & 255u) == 0, BM_ERR_WORKSPACE,
             "dense_experts: workspace must be 256-byte aligned and hold %zu bytes (%zu given)", at.total, workspace_bytes);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  int32_t *tok = reinterpret_cast<int32_t*>(ws + at.tok), *off = reinterpret_cast<int32_t*>(ws + at.off);
  const int A = T * k;
  int rc = bm_route_build(topk_idx, topk_w, global_to_local, num_routed, T, k, num_local, 128, tok, off, reinterpret_cast<float*>(ws + at.rw), nullptr,
                          nullptr, ws + at.route, at.z - at.route, stream);
  if (rc) return rc;
  GroupedArgs g{};
  g.x = x; g.w = w_gate_up; g.offsets = off; g.index = tok; g.y = ws + at.z;
  g.x_rows = T; g.rows = A; g.K = hidden; g.N = intermediate; g.E = num_local; g.dtype = g.y_dtype = dtype; g.glu = 1;
  g.expected = static_cast<int>(static_cast<int64_t>(A) * num_local / std::max(num_routed, num_local));
  g.gathered = ws + at.xs;
  g.wide = dtype == BM_F16 ? reinterpret_cast<float*>(ws + at.wide) : nullptr;
  g.after = AFTER_READS;
  if ((rc = launch_grouped(g, st))) return rc;
  g.x = g.y; g.w = w_down; g.index = nullptr; g.y = ws + at.d; g.y_dtype = BM_F32;
  g.x_rows = A; g.K = intermediate; g.N = hidden; g.glu = 0;
  int32_t* pos = reinterpret_cast<int32_t*>(ws + at.pos);
  g.slots = SlotArgs{topk_idx, global_to_local, tok, off, pos, A, k, num_local, num_routed, g.expected < A / 4};
  if ((rc = launch_grouped(g, st))) return rc;
  CombineArgs c{};
  c.d = reinterpret_cast<const float*>(ws + at.d);
  c.pos = pos; c.topk_w = topk_w; c.residual = residual; c.y = y; c.k = k; c.H = hidden;
  c.slots = g.slots; c.z = ws + at.z; c.wide = reinterpret_cast<const float*>(ws + at.wide); c.w_down = w_down; c.I = intermediate;
  c.vec = hidden % 4 == 0 && ((reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(residual)) & 7u) == 0;
  BM_CUDA(launch_after(AFTER_READS, 1, dtype == BM_F16 ? experts_combine_kernel<BM_F16> : experts_combine_kernel<BM_BF16>,
                       dim3(T, (hidden + 4 * EC_THREADS - 1) / (4 * EC_THREADS)), EC_THREADS, 0, st, c));
  BM_LAUNCH_CHECK("experts_combine_kernel");
  return BM_OK;
}
