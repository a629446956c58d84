// Products of rows grouped by expert on tcgen05, for groups of any size: y[i] = x[row(i)] . W[e(i)]^T, or silu(gate) * up of it.
//
// The weights are the M operand and the rows the N operand: N goes in steps of 16, so that a group of 130 rows costs 144 columns
// where tiles of 128 rows would cost 256, and a group of one row costs 16.  A pair of CTAs (cluster of two, cta_group::2) takes an item =
// (expert, up to 256 of its rows, 256 weight rows): each CTA loads 128 weight rows and half of the item's rows, and the tensor cores
// read both halves, so that an SM fetches 32 KB per 64 columns of K for 128 x 256 sums (a lone CTA would need 48, which is more than an SM gets
// from L2 while its tensor core multiplies them).
//   warps 0, 3  producers: weight rows as tiled copies; rows of x as tiled copies or by tile::gather4 (four an instruction); all onto
//               the even CTA's barrier.  A copy costs its thread 50 cycles or more, a stage of nine on one warp more than its products
//   warp 1      MMA issue, in the even CTA for both: four tcgen05.mma (M = 256, N = the item's rows, K = 16) per stage
//   warps 4-11  epilogue: tensor memory -> registers (fragments of 16 weight rows x 8 rows) -> y.  stmatrix turns them round in
//               shared memory, so that a thread stores 16 bytes of a row of y.  With a gated pair the accumulator's lanes alternate between
//               16 gate rows and the 16 up rows that belong to them, so that a thread holds both sums of an output.
// The accumulator alternates between two halves of tensor memory.  Items are handed out round robin; which expert an item belongs
// to every CTA works out from the offsets, so that the host never reads them.  Waits are bounded; one that gives up raises the
// status word, and the pair leaves once its copies and products are done.
//
// Measured (bf16, K 2048, N 1536): 128 groups in order of 1 row 121 us (HBM floor 123), 128 rows 151, 512 rows 315 (1.3 PFLOP/s); one group of 65536 rows 290
// (1.42 PFLOP/s, what the library product reaches under the power limit).  Few rows are bound by HBM, many by the tensor pipe at its
// sustained clock, one to eight groups of one row (11 to 13 us) by start, first data and end of the launch.
#include <cuda.h>

#include <cstring>

#include "grouped.cuh"
#include "tc05.cuh"

namespace bm {

bool encode_map16(CUtensorMap* map, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box);

constexpr int GC_THREADS = 384, GC_EPI0 = 4, GC_EPI_WARPS = 8, GC_K = 64, GC_ROWS = 256, GC_MAX_STAGES = 16, GC_MAX_E = 1024;
constexpr int GC_TURN_PITCH = 80, GC_TURN_BYTES = 32 * GC_TURN_PITCH;      // 32 rows of 64 (gated pair: 32) bytes: eight rows hit eight bank groups
constexpr int GC_A_BYTES = 128 * GC_K * 2, GC_BOX = 32;
// The ring: slices of 128 weight rows and half of the rows of the longest item that the offsets make, a stage holds one, two or four.
constexpr int GC_RING = 6 * 2 * GC_A_BYTES;
// Where the items would leave most pairs idle they are cut along the weight rows: a CTA takes 32 `quarters` of them instead of 128, the rest of
// its rows of the accumulator is not looked at.
constexpr int gc_smem_bytes(int E) { return GC_RING + GC_EPI_WARPS * GC_TURN_BYTES + 1024 + (3 * E + 1) * 4; }

struct GcParams {
  CUtensorMap x, x8;           // 32 rows in order (one row of a gather), 8
  CUtensorMap w, w32;          // 128 weight rows, or 32 (of a gated pair 16 and 16)
  const int32_t* offsets;
  const int32_t* index;
  void* y;
  float* wide;
  const float* x_wide;
  const __half *xp, *wp;       // x and w, for the sums that x_wide makes necessary
  DenseGuard guard;
  int x_rows, rows, K, N, E, slices, vec, whole;     // vec: y takes 16-byte stores; whole: w describes a gated pair in blocks of 16 rows
  SlotArgs slots;
  int may_be_empty;
};

// Copies into this CTA's shared memory, signalled on `bar` (shared::cluster address, of either CTA of the pair): four rows, tiles.
__device__ __forceinline__ void tma_gather4_pair(void* dst, const CUtensorMap* map, int x, int4 r, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(
          tc::smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(r.x), "r"(r.y), "r"(r.z), "r"(r.w), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];" ::"r"(
                   tc::smem_u32(dst)),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void tma_load_3d_pair(void* dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
                   tc::smem_u32(dst)),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void tma_load_4d_pair(void* dst, const CUtensorMap* map, int x, int y, int z, int w, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
                   tc::smem_u32(dst)),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void tma_load_5d_pair(void* dst, const CUtensorMap* map, int x, int y, int z, int w, int v, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(
                   tc::smem_u32(dst)),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(v), "r"(bar)
               : "memory");
}
// K-major operand tile of 128-byte rows, 8-row groups 1024 bytes apart, 128-byte swizzle
__device__ __forceinline__ uint64_t gc_desc(uint32_t saddr) {
  return static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4) | (1ull << 16) | (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// Group e has ceil(rows / 256) pieces of (nearly) equal size, each with `blocks` items along the weight rows.
struct GcTable {
  const int *first, *start, *count;     // [E + 1] pieces before the group; its first row; its rows
  int blocks;
};
// Rows of the pieces of a group of n rows, a multiple of 16 (a lesser last one apart).
__device__ __forceinline__ int gc_piece(int n) {
  const int pieces = (n + GC_ROWS - 1) / GC_ROWS;
  return pieces ? ((n + pieces - 1) / pieces + 15) & ~15 : 0;
}
struct GcItem {
  int e, row0, rows, block;
  __device__ int n() const { return (rows + 15) & ~15; }
  // A product waits for the sum that the one before wrote: 112 cycles however few rows there are, where 256 rows take 128.  Few rows
  // get two or four sums that take the products in turn and are added up at the end.
  __device__ int parts() const { return rows <= 64 ? 4 : rows <= 128 ? 2 : 1; }
};
__device__ __forceinline__ GcItem gc_item(const GcTable& tab, int item, int& e) {
  const int piece = item / tab.blocks;
  while (piece >= tab.first[e + 1]) ++e;
  const int i = piece - tab.first[e], n = tab.count[e], size = gc_piece(n);
  GcItem it;
  it.e = e;
  it.block = item - piece * tab.blocks;
  it.row0 = tab.start[e] + i * size;
  it.rows = min(size, n - i * size);       // at least one: size < 256 only where 16 (pieces - 1) < n / pieces
  return it;
}

// Places of the slots by warp `w` of those that take part: one a CTA, or where few of the slots are held here, and the products therefore short, the
// epilogue warps before their first item too.
__device__ __forceinline__ void gc_places(const SlotArgs& a, int w, int lane) {
  const int warps = a.sparse ? 1 + GC_EPI_WARPS : 1;
  if (a.pos && w < warps) {
    const int2 r = slot_range(a);
    for (int i = r.x + (blockIdx.x * warps + w) * 32 + lane; i < r.y; i += gridDim.x * warps * 32) a.pos[i] = slot_place(a, i);
  }
}

template <bool BF16>
__device__ __forceinline__ uint32_t gc_pack(float a, float b) {
  if (BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// Four 8 x 8 fragments, turned round: lane 8 m + j names the 16 bytes that column j of fragment m goes to.
__device__ __forceinline__ void stmatrix_x4_trans(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// x is the product between the two matrices of an expert, which may pass fp16's range where the sums over it do not: x is infinite there, and with
// it the whole row of y.  Such rows of this CTA's items are summed up here again, from x's values before their rounding, four columns a
// warp; where those are infinite or not a number themselves y is what it should be.  Whole calls: one such token of 64 in 8 of 128 experts 204 -> 269 us, one
// of 2048 in 6 of 64 322 -> 541, all 2048 of them 21 ms.
__device__ __noinline__ void gc_redo(const GcParams& p, const GcTable& tab, int items, int width) {
  __shared__ unsigned lost[GC_ROWS / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, pair = blockIdx.x >> 1, pairs = gridDim.x >> 1, K = p.K;
  const float inf = __int_as_float(0x7f800000);
  float* const y = static_cast<float*>(p.y);
  auto load8 = [](const __half* at, float (&v)[8]) {
    const uint4 q = __ldg(reinterpret_cast<const uint4*>(at));
    const __half2* e = reinterpret_cast<const __half2*>(&q);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = __half22float2(e[j]);
      v[2 * j] = f.x;
      v[2 * j + 1] = f.y;
    }
  };
  int e = 0;
  for (int item = pair; item < items; item += pairs) {
    const GcItem it = gc_item(tab, item, e);
    const int col0 = (it.block * 2 + static_cast<int>(tc::cluster_rank())) * width, cols = min(width, p.N - col0);
    __syncthreads();
    if (threadIdx.x < GC_ROWS / 32) lost[threadIdx.x] = 0;
    __syncthreads();
    for (int r = warp; r < it.rows && cols > 0; r += GC_THREADS / 32) {
      const int64_t row = it.row0 + r;
      if (fabsf(__ldcg(y + row * p.N + col0)) < inf) continue;
      bool mine = false;
      for (int k = lane; k < K; k += 32)
        if (!(fabsf(__half2float(p.xp[row * K + k])) <= 65504.f)) mine |= fabsf(p.x_wide[row * K + k]) < inf;
      if (__any_sync(0xffffffffu, mine) && lane == 0) atomicOr(&lost[r >> 5], 1u << (r & 31));
    }
    __syncthreads();
    for (int r = 0; r < it.rows; ++r) {
      if (!(lost[r >> 5] >> (r & 31) & 1u)) continue;
      const int64_t row = it.row0 + r;
      const __half *x = p.xp + row * K, *w = p.wp + (static_cast<int64_t>(it.e) * p.N + col0) * K;
      for (int c0 = 4 * warp; c0 < cols; c0 += 4 * (GC_THREADS / 32)) {
        float sum[4] = {};
#pragma unroll 2
        for (int k = 8 * lane; k < K; k += 256) {
          float f[8], q[4][8];
          load8(x + k, f);
#pragma unroll
          for (int c = 0; c < 4; ++c) load8(w + static_cast<int64_t>(min(c0 + c, cols - 1)) * K + k, q[c]);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (!(fabsf(f[j]) <= 65504.f)) f[j] = p.x_wide[row * K + k + j];
#pragma unroll
            for (int c = 0; c < 4; ++c) sum[c] = fmaf(q[c][j], f[j], sum[c]);
          }
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) sum[c] += __shfl_xor_sync(0xffffffffu, sum[c], o);
          if (lane == c && c0 + c < cols) y[row * p.N + col0 + c0 + c] = sum[c];
        }
      }
    }
  }
}

// F32: y is fp32 (no gated pair).  GATHER: rows of x by index.
template <bool GLU, bool GATHER, bool F32, bool BF16>
__global__ void __launch_bounds__(GC_THREADS, 1) grouped_tc_kernel(const __grid_constant__ GcParams p) {
  extern __shared__ unsigned char gc_raw[];
  __shared__ __align__(8) uint64_t full[GC_MAX_STAGES], empty[GC_MAX_STAGES], acc_full[2], acc_empty[2], drained;
  __shared__ int gave_up;                  // a wait of either CTA ran out
  __shared__ int not_finite;               // a sum of this CTA is not
  __shared__ int issued[4];                // stages that either CTA's producers (2 rank, 2 rank + 1) have issued
  __shared__ uint32_t tmem_slot;
  __shared__ int longest;
  __shared__ int4 rows4[32];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(gc_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  unsigned char* const turn = smem + GC_RING;
  int* const t_first = reinterpret_cast<int*>(turn + GC_EPI_WARPS * GC_TURN_BYTES);
  int *const t_start = t_first + p.E + 1, *const t_count = t_start + p.E;
  const int warp = tc::warp_index(), lane = threadIdx.x & 31;
  const uint32_t rank = tc::cluster_rank();
  if (threadIdx.x == 0) {
    for (int i = 0; i < GC_MAX_STAGES; ++i) {
      tc::mbar_init(&full[i], 1);
      tc::mbar_init(&empty[i], 1);
    }
    gave_up = p.guard.limit_ns == 0;
    not_finite = 0;
    tc::mbar_init(&drained, 1);
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&acc_full[i], 1);
      tc::mbar_init(&acc_empty[i], 2 * GC_EPI_WARPS);
    }
    tc::mbar_init_fence();
  }
  if (threadIdx.x == 32) {
    auto prefetch = [](const CUtensorMap* m) { asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(m)) : "memory"); };
    prefetch(&p.x);
    prefetch(&p.w32);
    if (!GATHER) prefetch(&p.x8);
    if (!GLU || p.whole) prefetch(&p.w);
  }
  __syncthreads();
  tc::cluster_arrive();
  grid_wait();
  if (p.may_be_empty && __ldg(p.offsets + p.E) == 0) {
    tc::cluster_wait();
    gc_places(p.slots, warp, lane);
    return;
  }
  for (int e = threadIdx.x; e < p.E; e += GC_THREADS) {
    const int2 r = group_rows(p.offsets, e, p.rows);
    t_start[e] = r.x;
    t_count[e] = r.y - r.x;
  }
  tc::cluster_wait();                          // both CTAs run and their barriers are set up
  if (warp == 2) {
    tc::tmem_alloc_pair(&tmem_slot, 512);
    // not before: a launch that came to this SM ahead of the allocation could take tensor memory and then wait for this one
    grid_launch_dependents();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem_base = tmem_slot;
  if (warp == 0) {
    int before = 0, most = 16;
    for (int e0 = 0; e0 < p.E; e0 += 32) {
      const int e = e0 + lane, n = e < p.E ? t_count[e] : 0;
      most = max(most, gc_piece(n));
      int incl = (n + GC_ROWS - 1) / GC_ROWS;
      const int mine = incl;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      if (e < p.E) t_first[e] = before + incl - mine;
      before += __shfl_sync(0xffffffffu, incl, 31);
    }
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0) {
      t_first[p.E] = before;
      longest = most;
    }
  }
  __syncthreads();
  const int pieces = t_first[p.E], pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  constexpr int QUARTER = GLU ? 32 : 64;       // columns of y of a pair's quarter
  const int cols1 = (p.N + QUARTER - 1) / QUARTER, quarters = static_cast<int64_t>(pieces) * cols1 <= pairs ? 1 : static_cast<int64_t>(pieces) * ((cols1 + 1) / 2) <= pairs ? 2 : 4;
  const GcTable tab{t_first, t_start, t_count, (cols1 + quarters - 1) / quarters};
  const int items = pieces * tab.blocks, a_bytes = quarters * (GC_A_BYTES / 4);
  // a stage's barriers, waits and commit cost 0.2 us: small slices share them
  const int slice = a_bytes + longest / 2 * GC_K * 2, sub = slice <= GC_RING / 32 ? 4 : slice <= GC_RING / 10 ? 2 : 1;
  const int stages = min(GC_RING / (slice * sub), GC_MAX_STAGES);
  bool ok = true;
  auto wait = [&](uint64_t* bar, uint32_t parity) { return tc::mbar_wait_limit(bar, parity, p.guard.limit_ns); };
  auto to_both = [&](int* what, int v) {
    for (uint32_t r = 0; r < 2; ++r) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(tc::cluster_map(tc::smem_u32(what), r)), "r"(v) : "memory");
  };

  if (warp == 0) {
    // ------------------------------------------------------------------ weight rows
    uint32_t st = 0, ph = 0;
    int e = 0, n = 0;
    for (int item = pair; item < items && ok; item += pairs) {
      const GcItem it = gc_item(tab, item, e);
      const uint32_t bytes = 2 * (a_bytes + (it.n() >> 1) * GC_K * 2);      // of both CTAs' slices
      const int col0 = (it.block * 2 + static_cast<int>(rank)) * quarters * (QUARTER / 2);
      for (int k0 = 0; k0 < p.slices; k0 += sub) {
        if (!(ok = wait(&empty[st], ph ^ 1))) break;
        if (tc::elect_one()) {
          const int cnt = min(sub, p.slices - k0);
          const uint32_t bar = tc::cluster_map(tc::smem_u32(&full[st]), 0);
          if (rank == 0) tc::mbar_expect_tx(&full[st], cnt * bytes);
          for (int j = 0; j < cnt; ++j) {
            unsigned char* sa = smem + (st * sub + j) * slice;
            const int k = (k0 + j) * GC_K;
            if (GLU) {
              if (quarters == 4 && p.whole) tma_load_5d_pair(sa, &p.w, k, 0, 0, col0 / 16, it.e, bar);
              else
                for (int b = 0; b < quarters; ++b) tma_load_4d_pair(sa + b * (GC_A_BYTES / 4), &p.w32, k, col0 + 16 * b, 0, it.e, bar);
            } else if (quarters == 4) {
              tma_load_3d_pair(sa, &p.w, k, col0, it.e, bar);
            } else {
              for (int b = 0; b < quarters; ++b) tma_load_3d_pair(sa + b * (GC_A_BYTES / 4), &p.w32, k, col0 + 32 * b, it.e, bar);
            }
          }
        }
        __syncwarp();
        ++n;
        if (++st == stages) { st = 0; ph ^= 1; }
      }
    }
    if (lane == 0) to_both(&issued[2 * rank + (warp != 0)], n);
  } else if (warp == 3) {
    // ------------------------------------------------------------------ rows of x
    uint32_t st = 0, ph = 0;
    int e = 0, n = 0;
    for (int item = pair; item < items && ok; item += pairs) {
      const GcItem it = gc_item(tab, item, e);
      const int half = it.n() >> 1, first = it.row0 + static_cast<int>(rank) * half;
      if (GATHER) {
        int id[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          // columns past the item's rows are not used: they repeat its last row
          id[j] = __ldg(p.index + min(first + 4 * lane + j, it.row0 + it.rows - 1));
          if (id[j] < 0 || id[j] >= p.x_rows) id[j] = p.x_rows;       // outside the matrix: zeros
        }
        __syncwarp();
        rows4[lane] = make_int4(id[0], id[1], id[2], id[3]);
        __syncwarp();
      }
      for (int k0 = 0; k0 < p.slices; k0 += sub) {
        if (!(ok = wait(&empty[st], ph ^ 1))) break;
        if (tc::elect_one()) {
          const int cnt = min(sub, p.slices - k0);
          const uint32_t bar = tc::cluster_map(tc::smem_u32(&full[st]), 0);
          for (int j = 0; j < cnt; ++j) {
            unsigned char* const sb = smem + (st * sub + j) * slice + a_bytes;
            const int k = (k0 + j) * GC_K;
            if (GATHER) {
#pragma unroll 4
              for (int r = 0; r < half; r += 4) tma_gather4_pair(sb + r * (GC_K * 2), &p.x, k, rows4[r / 4], bar);
            } else {
              int r = 0;
              for (; r + GC_BOX <= half; r += GC_BOX) tma_load_2d_pair(sb + r * (GC_K * 2), &p.x, k, first + r, bar);
              for (; r < half; r += 8) tma_load_2d_pair(sb + r * (GC_K * 2), &p.x8, k, first + r, bar);
            }
          }
        }
        __syncwarp();
        ++n;
        if (++st == stages) { st = 0; ph ^= 1; }
      }
    }
    if (lane == 0) to_both(&issued[2 * rank + (warp != 0)], n);
  } else if (warp == 1 && rank == 0) {
    // ------------------------------------------------------------------ MMA issue
    uint32_t st = 0, ph = 0, ti = 0;
    int e = 0;
    for (int item = pair; item < items && ok; item += pairs, ++ti) {
      const GcItem it = gc_item(tab, item, e);
      const uint32_t ab = ti & 1u, idesc = BF16 ? tc::idesc_bf16(256, it.n()) : tc::idesc_f16(256, it.n()), parts = it.parts(), apart = GC_ROWS / parts;
      if (ti >= 2 && !(ok = tc::mbar_wait_limit<true>(&acc_empty[ab], ((ti >> 1) - 1) & 1, p.guard.limit_ns))) break;    // read out two items ago
      tc::fence_after_sync();
      for (int k0 = 0; k0 < p.slices; k0 += sub) {
        if (!(ok = wait(&full[st], ph))) break;
        tc::fence_after_sync();
        if (tc::elect_one()) {
          const int cnt = min(sub, p.slices - k0);
          for (int j = 0; j < cnt; ++j) {
            const uint32_t sa = tc::smem_u32(smem + (st * sub + j) * slice);
            const uint64_t ad = gc_desc(sa), bd = gc_desc(sa + a_bytes);
#pragma unroll
            for (int kk = 0; kk < GC_K / 16; ++kk)
              tc::mma_f16_pair(tmem_base + ab * GC_ROWS + (kk & (parts - 1)) * apart, ad + 2 * kk, bd + 2 * kk, idesc, k0 + j > 0 || kk >= parts ? 1u : 0u);
          }
          tc::mma_commit_pair(&empty[st]);
        }
        __syncwarp();
        if (++st == stages) { st = 0; ph ^= 1; }
      }
      if (ok && tc::elect_one()) tc::mma_commit_pair(&acc_full[ab]);
      __syncwarp();
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------------ places of the slots, for whoever sums over a token's experts
    gc_places(p.slots, 0, lane);
  } else if (warp >= GC_EPI0) {
    // ------------------------------------------------------------------ epilogue: lane quarter q, every other block of 32 rows
    const int q = warp & 3, half = (warp - GC_EPI0) >> 2;
    gc_places(p.slots, warp - GC_EPI0 + 1, lane);
    constexpr int WIDE = GLU ? 16 : 32, PITCH = GLU ? 48 : GC_TURN_PITCH, PIECES = WIDE / 8;      // columns of y a warp has, bytes between rows, 16-byte pieces
    unsigned char* const mine = turn + (warp - GC_EPI0) * GC_TURN_BYTES;
    uint32_t ti = 0;
    int e = 0;
    for (int item = pair; item < items && ok; item += pairs, ++ti) {
      const GcItem it = gc_item(tab, item, e);
      const uint32_t ab = ti & 1u;
      if (!(ok = wait(&acc_full[ab], (ti >> 1) & 1))) break;
      tc::fence_after_sync();
      const uint32_t acc = tmem_base + (static_cast<uint32_t>(32 * q) << 16) + ab * GC_ROWS;
      const int col0 = (it.block * 2 + static_cast<int>(rank)) * quarters * (QUARTER / 2) + WIDE * q, parts = it.parts();
#pragma unroll 1
      for (int c0 = q < quarters ? 32 * half : it.rows; c0 < it.rows; c0 += 64) {
        if (F32) {
          // a lane owns a column: a warp's store is 128 bytes of a row of y
          float v[32];
          tc::tmem_ld32(acc + c0, v);
          for (int i = 1; i < parts; ++i) {
            float w[32];
            tc::tmem_ld32(acc + c0 + i * (GC_ROWS / parts), w);
#pragma unroll
            for (int c = 0; c < 32; ++c) v[c] += w[c];
          }
          if (!BF16 && p.x_wide) {
            float s = 0.f;
#pragma unroll
            for (int c = 0; c < 32; ++c) s += v[c];
            if (!(fabsf(s) < __int_as_float(0x7f800000))) not_finite = 1;
          }
          float* out = static_cast<float*>(p.y) + static_cast<int64_t>(it.row0 + c0) * p.N + col0 + lane;
          if (col0 + lane < p.N)
#pragma unroll
            for (int c = 0; c < 32; ++c)
              if (c0 + c < it.rows) out[static_cast<int64_t>(c) * p.N] = v[c];
          continue;
        }
        uint32_t lo[16], hi[16];
        tc::tmem_ld_frag32(acc + c0, lo);
        tc::tmem_ld_frag32(acc + (16u << 16) + c0, hi);
        tc::tmem_ld_wait(lo, hi);
        for (int i = 1; i < parts; ++i) {
          uint32_t l2[16], h2[16];
          tc::tmem_ld_frag32(acc + c0 + i * (GC_ROWS / parts), l2);
          tc::tmem_ld_frag32(acc + (16u << 16) + c0 + i * (GC_ROWS / parts), h2);
          tc::tmem_ld_wait(l2, h2);
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            lo[j] = __float_as_uint(__uint_as_float(lo[j]) + __uint_as_float(l2[j]));
            hi[j] = __float_as_uint(__uint_as_float(hi[j]) + __uint_as_float(h2[j]));
          }
        }
        const uint32_t at = tc::smem_u32(mine) + ((lane & 7) + 8 * (lane >> 4)) * PITCH + 16 * ((lane >> 3) & 1);
        if (GLU) {
#pragma unroll
          for (int i = 0; i < 16; ++i) lo[i] = __float_as_uint(silu_mul(__uint_as_float(lo[i]), __uint_as_float(hi[i])));
          if (!BF16 && p.wide) {
            bool fits = true;
#pragma unroll
            for (int i = 0; i < 16; ++i) fits &= fits_fp16(__uint_as_float(lo[i]));
            if (!fits)
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const int r = c0 + 8 * (i >> 2) + 2 * (lane & 3) + (i & 1), col = col0 + (lane >> 2) + 8 * ((i >> 1) & 1);
                if (!fits_fp16(__uint_as_float(lo[i])) && r < it.rows && col < p.N) p.wide[static_cast<int64_t>(it.row0 + r) * p.N + col] = __uint_as_float(lo[i]);
              }
          }
        }
#pragma unroll
        for (int h = 0; h < (GLU ? 1 : 2); ++h) {
          uint32_t m[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) m[i] = gc_pack<BF16>(__uint_as_float(h ? hi[2 * i] : lo[2 * i]), __uint_as_float(h ? hi[2 * i + 1] : lo[2 * i + 1]));
          stmatrix_x4_trans(at + 32 * h, m[0], m[1], m[2], m[3]);
          stmatrix_x4_trans(at + 32 * h + 16 * PITCH, m[4], m[5], m[6], m[7]);
        }
        __syncwarp();
        uint16_t* out = static_cast<uint16_t*>(p.y) + static_cast<int64_t>(it.row0 + c0) * p.N + col0;
        if (p.vec) {
#pragma unroll
          for (int u = 0; u < PIECES; ++u) {
            const int r = (32 / PIECES) * u + lane / PIECES, pc = lane % PIECES;
            if (c0 + r < it.rows && col0 + 8 * pc < p.N)
              *reinterpret_cast<uint4*>(out + static_cast<int64_t>(r) * p.N + 8 * pc) = *reinterpret_cast<const uint4*>(mine + r * PITCH + 16 * pc);
          }
        } else {
          const int c = lane % WIDE;
#pragma unroll 4
          for (int r = lane / WIDE; r < 32; r += 32 / WIDE)
            if (c0 + r < it.rows && col0 + c < p.N) out[static_cast<int64_t>(r) * p.N + c] = *reinterpret_cast<const uint16_t*>(mine + r * PITCH + 2 * c);
        }
        __syncwarp();
      }
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive_release_cluster(tc::cluster_map(tc::smem_u32(&acc_empty[ab]), 0));
    }
  }
  if (!ok && lane == 0) to_both(&gave_up, 1);
  tc::fence_before_sync();
  __syncthreads();
  tc::cluster_arrive();
  tc::cluster_wait();                          // nothing of the other CTA reaches into this one any more, but for copies and products where a wait gave up
  if (gave_up) {
    // Stages that one producer has issued and another has not would never be full: the others' bytes are made up, for at most a ring of
    // stages, since nobody is a ring ahead of a stage that is not full.  Then the last copies into every stage are waited for, and the products.
    const int upto = max(max(issued[0], issued[1]), max(issued[2], issued[3]));
    if ((warp == 0 || warp == 3) && tc::elect_one()) {
      int k = 0, e = 0;
      for (int item = pair; item < items && k < upto; item += pairs) {
        const GcItem it = gc_item(tab, item, e);
        const uint32_t of_x = (it.n() >> 1) * GC_K * 2;
        for (int k0 = 0; k0 < p.slices && k < upto; k0 += sub, ++k) {
          if (k < issued[2 * rank + (warp != 0)]) continue;
          const int cnt = min(sub, p.slices - k0);
          if (warp == 0 && rank == 0) tc::mbar_expect_tx(&full[k % stages], cnt * 2 * (a_bytes + of_x));
          tc::mbar_complete_tx(tc::cluster_map(tc::smem_u32(&full[k % stages]), 0), cnt * (warp == 0 ? a_bytes : of_x));
        }
      }
    }
    __syncwarp();
    if (warp == 0 && rank == 0)
      for (int k = max(0, upto - stages); k < upto; ++k) tc::mbar_wait(&full[k % stages], (k / stages) & 1);
    if (warp == 1) {
      if (rank == 0 && tc::elect_one()) tc::mma_commit_pair(&drained);
      __syncwarp();
      tc::mbar_wait(&drained, 0);
    }
    if (threadIdx.x == 0) atomicExch(p.guard.status, BM_ERR_TIMEOUT);
    __syncthreads();
    tc::cluster_arrive();
    tc::cluster_wait();
  }
  if (warp == 2) tc::tmem_dealloc_pair(tmem_base, 512);
  if (F32 && !BF16 && p.x_wide && not_finite) gc_redo(p, tab, items, quarters * 32);
}

static void (*const GC_KERNELS[])(const GcParams) = {
    grouped_tc_kernel<false, false, false, false>, grouped_tc_kernel<false, false, false, true>, grouped_tc_kernel<false, true, false, false>,
    grouped_tc_kernel<false, true, false, true>,   grouped_tc_kernel<true, false, false, false>, grouped_tc_kernel<true, false, false, true>,
    grouped_tc_kernel<true, true, false, false>,   grouped_tc_kernel<true, true, false, true>,   grouped_tc_kernel<false, false, true, false>,
    grouped_tc_kernel<false, false, true, true>};

int launch_grouped_tc(const GroupedArgs& a, cudaStream_t st) {
  const int64_t quarters = (a.N + (a.glu ? 31 : 63)) / (a.glu ? 32 : 64);
  // pieces there can be: every group that has rows ends in one of its own
  const int64_t most = (static_cast<int64_t>(a.rows) / GC_ROWS + (a.E < a.rows ? a.E : a.rows)) * quarters;
  if (a.K % 8 != 0 || a.x_rows == 0 || a.E > GC_MAX_E || !aligned16(a.x, a.w) || most > 0x3fffffff) return BM_ERR_UNSUPPORTED;
  GcParams p;
  memset(&p, 0, sizeof(p));
  const cuuint64_t K = a.K, N = a.N, E = a.E;
  {
    const cuuint64_t dims[2] = {K, static_cast<cuuint64_t>(a.x_rows)}, strides[1] = {K * 2};
    const cuuint32_t box[2] = {GC_K, a.index ? 1u : static_cast<cuuint32_t>(GC_BOX)}, box8[2] = {GC_K, 8};
    if (!encode_map16(&p.x, a.x, 2, dims, strides, box) || (!a.index && !encode_map16(&p.x8, a.x, 2, dims, strides, box8))) return BM_ERR_UNSUPPORTED;
  }
  if (a.glu) {
    const cuuint64_t dims[4] = {K, N, 2, E}, strides[3] = {K * 2, N * K * 2, 2 * N * K * 2};
    const cuuint32_t box[4] = {GC_K, 16, 2, 1};
    if (!encode_map16(&p.w32, a.w, 4, dims, strides, box)) return BM_ERR_UNSUPPORTED;
    if (N % 16 == 0) {
      // 16 rows, gate or up, block of 16 rows: a CTA's 128 operand rows in one copy
      const cuuint64_t dims5[5] = {K, 16, 2, N / 16, E}, strides5[4] = {K * 2, N * K * 2, 16 * K * 2, 2 * N * K * 2};
      const cuuint32_t box5[5] = {GC_K, 16, 2, 4, 1};
      p.whole = encode_map16(&p.w, a.w, 5, dims5, strides5, box5);
    }
  } else {
    const cuuint64_t dims[3] = {K, N, E}, strides[2] = {K * 2, N * K * 2};
    const cuuint32_t box[3] = {GC_K, 128, 1}, box32[3] = {GC_K, 32, 1};
    if (!encode_map16(&p.w, a.w, 3, dims, strides, box) || !encode_map16(&p.w32, a.w, 3, dims, strides, box32)) return BM_ERR_UNSUPPORTED;
  }
  p.offsets = a.offsets; p.index = a.index; p.y = a.y; p.wide = a.wide;
  p.x_wide = a.x_wide; p.xp = static_cast<const __half*>(a.x); p.wp = static_cast<const __half*>(a.w); p.K = a.K;
  p.x_rows = a.x_rows; p.rows = a.rows; p.N = a.N; p.E = a.E;
  p.slices = (a.K + GC_K - 1) / GC_K;
  p.vec = a.N % 8 == 0 && aligned16(a.y);
  p.slots = a.slots;
  p.may_be_empty = a.may_be_empty;
  const bool f32 = a.y_dtype == BM_F32;
  if (f32 && (a.glu || a.index)) return BM_ERR_UNSUPPORTED;
  static PerDeviceOnce once;
  static int grids[MAX_DEVICES];
  int dev = -1;
  BM_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= MAX_DEVICES) return BM_ERR_UNSUPPORTED;
  const int rc = dense_guard(&p.guard);
  if (rc) return rc;
  if (!once.is_done(dev)) {
    for (auto& k : GC_KERNELS) BM_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, gc_smem_bytes(GC_MAX_E)));
    BM_CUDA(cudaDeviceGetAttribute(&grids[dev], cudaDevAttrMultiProcessorCount, dev));
    grids[dev] &= ~1;
    once.mark(dev);
  }
  const int grid = most * 2 < grids[dev] ? static_cast<int>(most) * 2 : grids[dev];
  const int which = (f32 ? 4 : (a.glu ? 2 : 0) + (a.index ? 1 : 0)) * 2 + (a.dtype == BM_BF16);
  BM_CUDA(launch_after(a.after, 2, GC_KERNELS[which], dim3(grid), GC_THREADS, gc_smem_bytes(a.E), st, p));
  BM_LAUNCH_CHECK("grouped_tc_kernel");
  return BM_OK;
}

}  // namespace bm
