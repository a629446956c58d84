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
        float v = 0.f;
        if (src[r] >= 0 && k0 + k < a.K) {
          const int64_t o = static_cast<int64_t>(src[r]) * a.K + k0 + k;
          v = load16<D>(a.x, o);
          if (!GLU && D == BM_F16 && a.x_wide && !(fabsf(v) <= 65504.f)) v = a.x_wide[o];
        }
        xs[k][r] = v;
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
  const int lane = threadIdx.x & 31, warps = gridDim.x * (GR_THREADS / 32);
  int end = 0;                 // behind the last row that a group owns: offsets[E], unless the table does not ascend
  for (int e = lane; e < E; e += 32) end = max(end, group_rows(offsets, e, rows).y);
  end = __reduce_max_sync(0xffffffffu, end);
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
  const int2 r = slot_range(a);
  if (i >= r.x && i < r.y) a.pos[i] = slot_place(a, i);
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
  int T, k, H, vec;            // vec: H % 4 == 0, y and the residual on 8-byte boundaries
  const int32_t* window;       // [2] tokens from, to; null: all
};
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
  const int h = (blockIdx.y * EC_THREADS + threadIdx.x) * 4;
  grid_launch_dependents();
  grid_wait();
  if (h >= a.H) return;
  const int2 tokens = a.window ? make_int2(__ldcg(a.window), __ldcg(a.window + 1)) : make_int2(0, a.T);
  for (int t = tokens.x + blockIdx.x; t < tokens.y; t += gridDim.x) {
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
    uint16_t out[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] = D == BM_F16 ? __half_as_ushort(__float2half_rn(v[j])) : __bfloat16_as_ushort(__float2bfloat16_rn(v[j]));
    if (a.vec) *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.y) + o) = make_uint2(out[0] | out[1] << 16, out[2] | out[3] << 16);
    else
      for (int j = 0; j < n; ++j) static_cast<uint16_t*>(a.y)[o + j] = out[j];
  }
}

// Rows of scratch.  A short batch has one for every assignment, since all may name experts held here.  Where few are held most would stay empty: of 32768
// tokens of ten experts, three of 512 held (2048 hidden, 512), 3.7 GB for the 20 MB that are used.  Beyond 256 MB a token therefore has
// min(k, experts held) rows (slots that name the same expert share one), and beyond 1 GB, or four times the weights where that is more, the batch goes
// through in windows of tokens: a window takes all that is left when its rows fit, which the device finds out, and else as many tokens as fit
// for certain.  There are as many windows as that may need, the others find nothing to do, at 20 to 25 us each.  4096 / 16384 / 32768
// tokens of that layer took 61 / 141 / 242 us and 0.4 / 1.5 / 3.0 GB with a row for every assignment, and take 68 / 155 / 296 and 0.15 / 0.6 / 1.15
// (bf16, the output among them).
struct DenseRows {
  int64_t rows;
  int per, step;               // of a token at most; tokens that fit for certain
  DenseRows(int64_t T, int64_t k, int64_t E, int64_t H, int64_t I) {
    const double row = 4.0 * H + 6.0 * I, room = std::max(double(1ll << 30), 24.0 * E * H * I);
    per = static_cast<int>(T * k * row <= double(256ll << 20) ? k : std::min(k, E));
    const int64_t fit = static_cast<int64_t>(std::min(room / row, 1e9));
    rows = std::min(T * per, std::max<int64_t>(fit, per));
    step = static_cast<int>(rows / per);
  }
};

// Slots that name an expert of an earlier slot of their token are taken out of the selection: a warp per token.
__global__ void __launch_bounds__(256) experts_distinct_kernel(const SlotArgs a, int T, int32_t* idx) {
  grid_launch_dependents();
  grid_wait();
  const int t = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (t >= T) return;
  const int e = lane < a.k ? slot_expert(a, t * a.k + lane) : -1;
  const unsigned same = __match_any_sync(0xffffffffu, e);
  if (lane < a.k) idx[static_cast<int64_t>(t) * a.k + lane] = e >= 0 && __ffs(same) - 1 == lane ? a.topk_idx[t * a.k + lane] : -1;
}

struct WindowArgs {
  const int32_t *tok, *off;    // all rows: token of each, offsets [E + 1]
  int32_t *wtok, *woff;        // the window's
  int32_t* bounds;             // [2] its tokens from, to; of the window before on entry
  int T, E, rows, step, first; // rows there are; tokens that fit for certain
};
// One CTA: a thread per expert finds the window's part of its list (tokens ascend in it), warps copy it.
constexpr int EW_THREADS = 1024;
__global__ void __launch_bounds__(EW_THREADS) experts_window_kernel(const WindowArgs a) {
  __shared__ int from[EW_THREADS], sums[EW_THREADS / 32], start[EW_THREADS + 1];
  grid_launch_dependents();
  grid_wait();
  const int e = threadIdx.x, lane = e & 31, warp = e >> 5, t0 = a.first ? 0 : __ldcg(a.bounds + 1);
  const int begin = e < a.E ? a.off[e] : 0, end = e < a.E ? a.off[e + 1] : 0;
  auto first_of = [&](int t) {
    int lo = begin, hi = end;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (a.tok[mid] < t) lo = mid + 1;
      else hi = mid;
    }
    return lo;
  };
  auto inclusive = [&](int v) {      // over the block
    __syncthreads();
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int n = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += n;
    }
    if (lane == 31) sums[warp] = v;
    __syncthreads();
    for (int w = 0; w < warp; ++w) v += sums[w];
    return v;
  };
  const int lo = first_of(t0);
  from[e] = lo;
  start[e + 1] = inclusive(end - lo);
  __syncthreads();
  const int t1 = start[EW_THREADS] <= a.rows ? a.T : min(a.T, t0 + a.step);
  const int n = first_of(t1) - lo, upto = inclusive(n);
  start[e + 1] = upto;
  if (e == 0) {
    start[0] = 0;
    a.woff[0] = 0;
    a.bounds[0] = t0;
    a.bounds[1] = t1;
  }
  if (e < a.E) a.woff[e + 1] = upto;
  __syncthreads();
  const int share = max(1, EW_THREADS / 32 / a.E);       // warps that share an expert's list
  for (int x = warp / share; x < a.E; x += EW_THREADS / 32 / share)
#pragma unroll 4
    for (int i = start[x] + 32 * (warp % share) + lane; i < start[x + 1]; i += 32 * share) a.wtok[i] = a.tok[from[x] + i - start[x]];
}

struct DenseExpertsWs {
  DenseRows scratch;
  size_t tok, rw, pos, off, route, wtok, woff, bounds, xs, z, wide, d, total;
  DenseExpertsWs(int64_t T, int64_t k, int64_t E, int64_t H, int64_t I) : scratch(T, k, E, H, I) {
    const size_t A = static_cast<size_t>(T * k), R = static_cast<size_t>(scratch.rows);
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
    wtok = take(scratch.step < T ? R * 4 : 0);
    woff = take(static_cast<size_t>(E + 1) * 4);
    bounds = take(8);
    z = take(R * I * 2);
    wide = take(R * I * 4);
    d = xs = take(R * H * 4);      // rows of x in expert order are read before the down products are written
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
  int32_t *tok = reinterpret_cast<int32_t*>(ws + at.tok), *off = reinterpret_cast<int32_t*>(ws + at.off), *pos = reinterpret_cast<int32_t*>(ws + at.pos);
  int32_t *wtok = reinterpret_cast<int32_t*>(ws + at.wtok), *woff = reinterpret_cast<int32_t*>(ws + at.woff), *bounds = reinterpret_cast<int32_t*>(ws + at.bounds);
  const int A = T * k, rows = static_cast<int>(at.scratch.rows), step = at.scratch.step;
  const bool windows = step < T, distinct = at.scratch.per < k;
  SlotArgs slots{topk_idx, global_to_local, windows ? wtok : tok, windows ? woff : off, pos, A, k, num_local, num_routed, 0, distinct, windows ? bounds : nullptr};
  if (distinct) {
    BM_CUDA(launch_after(AFTER_READS, 1, experts_distinct_kernel, dim3((T + 7) / 8), 256, 0, st, slots, T, pos));       // until the places go there
    BM_LAUNCH_CHECK("experts_distinct_kernel");
  }
  int rc = bm_route_build(distinct ? pos : topk_idx, topk_w, global_to_local, num_routed, T, k, num_local, 128, tok, off, reinterpret_cast<float*>(ws + at.rw), nullptr,
                          nullptr, ws + at.route, at.wtok - at.route, stream);
  if (rc) return rc;
  for (int64_t t = 0; t < T; t += windows ? step : T) {
    if (windows) {
      const WindowArgs w{tok, off, wtok, woff, bounds, T, num_local, rows, step, t == 0};
      BM_CUDA(launch_after(AFTER_READS, 1, experts_window_kernel, dim3(1), EW_THREADS, 0, st, w));
      BM_LAUNCH_CHECK("experts_window_kernel");
    }
    GroupedArgs g{};
    g.x = x; g.w = w_gate_up; g.offsets = windows ? woff : off; g.index = windows ? wtok : tok; g.y = ws + at.z;
    g.x_rows = T; g.rows = rows; g.K = hidden; g.N = intermediate; g.E = num_local; g.dtype = g.y_dtype = dtype; g.glu = 1;
    g.expected = static_cast<int>(std::min<int64_t>(rows, std::max<int64_t>(1, static_cast<int64_t>(A) * num_local / std::max(num_routed, num_local))));
    g.gathered = ws + at.xs;
    g.wide = dtype == BM_F16 ? reinterpret_cast<float*>(ws + at.wide) : nullptr;
    g.after = AFTER_READS;
    g.may_be_empty = t > 0;
    if ((rc = launch_grouped(g, st))) return rc;
    slots.sparse = g.expected < A / 4;
    g.slots = slots;
    g.x_wide = g.wide;
    g.wide = nullptr;
    g.x = g.y; g.w = w_down; g.index = nullptr; g.y = ws + at.d; g.y_dtype = BM_F32;
    g.x_rows = rows; g.K = intermediate; g.N = hidden; g.glu = 0;
    if ((rc = launch_grouped(g, st))) return rc;
    CombineArgs c{};
    c.d = reinterpret_cast<const float*>(ws + at.d);
    c.pos = pos; c.topk_w = topk_w; c.residual = residual; c.y = y; c.T = T; c.k = k; c.H = hidden;
    c.window = slots.window;
    c.vec = hidden % 4 == 0 && ((reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(residual)) & 7u) == 0;
    const int columns = (hidden + 4 * EC_THREADS - 1) / (4 * EC_THREADS);
    BM_CUDA(launch_after(AFTER_READS, 1, dtype == BM_F16 ? experts_combine_kernel<BM_F16> : experts_combine_kernel<BM_BF16>,
                         dim3(windows ? std::min(T, std::max(1, 1332 / columns)) : T, columns), EC_THREADS, 0, st, c));
    BM_LAUNCH_CHECK("experts_combine_kernel");
  }
  return BM_OK;
}
