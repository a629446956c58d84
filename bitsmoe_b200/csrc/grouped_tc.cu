// Products of rows grouped by expert on tcgen05, for groups of any size: y[i] = x[row(i)] . W[e(i)]^T, or silu(gate) * up of it.
//
// The weights are the M operand and the rows the N operand: N goes in steps of 16, so that a group of 130 rows costs 144 columns
// where tiles of 128 rows would cost 256, and a group of one row costs 16.  A pair of CTAs (cluster of two, cta_group::2) takes an item =
// (expert, up to 256 of its rows, 256 weight rows): each CTA loads 128 weight rows and half of the item's rows, and the tensor cores
// read both halves, so that an SM fetches 32 KB per 64 columns of K for 128 x 256 sums (a lone CTA would need 48, which is more than an SM gets
// from L2 while its tensor core multiplies them).
//   warp 0      producer: weight rows as tiled copies, the rows of x by tile::gather4 (a lane names four of them), all onto the even CTA's barrier
//   warp 1      MMA issue, in the even CTA for both: four tcgen05.mma (M = 256, N = the item's rows, K = 16) per stage
//   warps 4-11  epilogue: tensor memory -> registers -> y.  A lane owns an output column (weight row), so that a warp's store is one
//               contiguous piece of a row of y and needs no alignment.  With a gated pair a quarter of the accumulator's lanes holds
//               16 gate rows and the 16 up rows that belong to them; lanes l and l + 16 exchange every other row's sums and each
//               finishes one of two rows.
// The accumulator alternates between two halves of tensor memory.  Items are handed out round robin; which expert an item belongs
// to every CTA works out from the offsets, so that the host never reads them.  Waits are bounded.
#include <cuda.h>

#include <cstring>

#include "grouped.cuh"
#include "tc05.cuh"

namespace bm {

bool encode_map16(CUtensorMap* map, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box);

constexpr int GC_THREADS = 384, GC_EPI0 = 4, GC_EPI_WARPS = 8, GC_K = 64, GC_ROWS = 256, GC_STAGES = 6, GC_MAX_E = 1024;
constexpr int GC_A_BYTES = 128 * GC_K * 2, GC_B_BYTES = 128 * GC_K * 2, GC_STAGE = GC_A_BYTES + GC_B_BYTES;
constexpr int gc_smem_bytes(int E) { return GC_STAGES * GC_STAGE + 1024 + (3 * E + 1) * 4; }

struct GcParams {
  CUtensorMap x, w;
  const int32_t* offsets;
  const int32_t* index;
  void* y;
  int x_rows, rows, N, E, slices, blocks, y_dtype, bf16;     // blocks: items along the weight rows
};

// 2-D gather of four rows / 3-D and 4-D tiles into this CTA's shared memory, signalled on `bar` (shared::cluster address)
__device__ __forceinline__ void tma_gather4_pair(void* dst, const CUtensorMap* map, int x, int4 r, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(
          tc::smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(r.x), "r"(r.y), "r"(r.z), "r"(r.w), "r"(bar)
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
// K-major operand tile of 128-byte rows, 8-row groups 1024 bytes apart, 128-byte swizzle
__device__ __forceinline__ uint64_t gc_desc(uint32_t saddr) {
  return static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4) | (1ull << 16) | (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// The items of the groups: group e has ceil(rows / 256) pieces of (nearly) equal size, each with `blocks` items.
struct GcTable {
  const int *first, *start, *count;     // [E + 1] items before the group; its first row; its rows
};
struct GcItem {
  int e, row0, rows, block;
};
__device__ __forceinline__ GcItem gc_item(const GcTable& tab, int item, int blocks, int& e) {
  while (item >= tab.first[e + 1]) ++e;
  const int local = item - tab.first[e], piece = local / blocks, n = tab.count[e], pieces = (n + GC_ROWS - 1) / GC_ROWS;
  const int size = ((n + pieces - 1) / pieces + 15) & ~15;
  GcItem it;
  it.e = e;
  it.block = local - piece * blocks;
  it.row0 = tab.start[e] + piece * size;
  it.rows = min(size, n - piece * size);       // at least one: size < 256 only where 16 (pieces - 1) < n / pieces
  return it;
}

template <bool GLU>
__global__ void __launch_bounds__(GC_THREADS, 1) grouped_tc_kernel(const __grid_constant__ GcParams p) {
  extern __shared__ unsigned char gc_raw[];
  __shared__ __align__(8) uint64_t full[GC_STAGES], empty[GC_STAGES], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_slot;
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(gc_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  int* const t_first = reinterpret_cast<int*>(smem + GC_STAGES * GC_STAGE);
  int *const t_start = t_first + p.E + 1, *const t_count = t_start + p.E;
  const int warp = tc::warp_index(), lane = threadIdx.x & 31;
  const uint32_t rank = tc::cluster_rank();
  if (threadIdx.x == 0) {
    for (int i = 0; i < GC_STAGES; ++i) {
      tc::mbar_init(&full[i], 1);
      tc::mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&acc_full[i], 1);
      tc::mbar_init(&acc_empty[i], 2 * GC_EPI_WARPS);
    }
    tc::mbar_init_fence();
  }
  __syncthreads();
  tc::cluster_arrive();
  tc::cluster_wait();                          // both CTAs run and their barriers are set up
  if (warp == 2) tc::tmem_alloc_pair(&tmem_slot, 512);
  grid_launch_dependents();
  grid_wait();
  for (int e = threadIdx.x; e < p.E; e += GC_THREADS) {
    const int2 r = group_rows(p.offsets, e, p.rows);
    t_start[e] = r.x;
    t_count[e] = r.y - r.x;
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem_base = tmem_slot;
  if (warp == 0) {
    int before = 0;
    for (int e0 = 0; e0 < p.E; e0 += 32) {
      const int e = e0 + lane;
      int incl = e < p.E ? (t_count[e] + GC_ROWS - 1) / GC_ROWS * p.blocks : 0;
      const int mine = incl;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      if (e < p.E) t_first[e] = before + incl - mine;
      before += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) t_first[p.E] = before;
  }
  __syncthreads();
  const GcTable tab{t_first, t_start, t_count};
  const int items = t_first[p.E], pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  bool ok = true;

  if (warp == 0) {
    // ------------------------------------------------------------------ producer
    uint32_t st = 0, ph = 0;
    int e = 0;
    for (int item = pair; item < items && ok; item += pairs) {
      const GcItem it = gc_item(tab, item, p.blocks, e);
      const int half = ((it.rows + 15) & ~15) >> 1;
      int4 src;
      int* s = reinterpret_cast<int*>(&src);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        // columns past the item's rows are not used: they repeat its last row
        const int r = it.row0 + min(static_cast<int>(rank) * half + 4 * lane + j, it.rows - 1);
        const int id = p.index ? __ldg(p.index + r) : r;
        s[j] = id >= 0 && id < p.x_rows ? id : p.x_rows;       // outside the matrix: zeros
      }
      const uint32_t bytes = 2 * (GC_A_BYTES + half * GC_K * 2);
      for (int k = 0; k < p.slices; ++k) {
        if (!(ok = tc::mbar_wait(&empty[st], ph ^ 1))) break;
        unsigned char* sa = smem + st * GC_STAGE;
        const uint32_t bar = tc::cluster_map(tc::smem_u32(&full[st]), 0);
        if (tc::elect_one()) {
          if (rank == 0) tc::mbar_expect_tx(&full[st], bytes);
          if (GLU) {
#pragma unroll
            for (int b = 0; b < 4; ++b)
              tma_load_4d_pair(sa + b * (GC_A_BYTES / 4), &p.w, k * GC_K, it.block * 128 + static_cast<int>(rank) * 64 + 16 * b, 0, it.e, bar);
          } else {
            tma_load_3d_pair(sa, &p.w, k * GC_K, it.block * 256 + static_cast<int>(rank) * 128, it.e, bar);
          }
        }
        __syncwarp();
        if (4 * lane < half) tma_gather4_pair(sa + GC_A_BYTES + lane * 512, &p.x, k * GC_K, src, bar);
        __syncwarp();
        if (++st == GC_STAGES) { st = 0; ph ^= 1; }
      }
    }
  } else if (warp == 1 && rank == 0) {
    // ------------------------------------------------------------------ MMA issue
    uint32_t st = 0, ph = 0, ti = 0;
    int e = 0;
    for (int item = pair; item < items && ok; item += pairs, ++ti) {
      const GcItem it = gc_item(tab, item, p.blocks, e);
      const uint32_t ab = ti & 1u, n = (it.rows + 15) & ~15, idesc = p.bf16 ? tc::idesc_bf16(256, n) : tc::idesc_f16(256, n);
      if (ti >= 2 && !(ok = tc::mbar_wait(&acc_empty[ab], ((ti >> 1) - 1) & 1))) break;    // read out two items ago
      tc::fence_after_sync();
      for (int k = 0; k < p.slices; ++k) {
        if (!(ok = tc::mbar_wait(&full[st], ph))) break;
        tc::fence_after_sync();
        if (tc::elect_one()) {
          const uint32_t sa = tc::smem_u32(smem + st * GC_STAGE);
          const uint64_t ad = gc_desc(sa), bd = gc_desc(sa + GC_A_BYTES);
#pragma unroll
          for (int kk = 0; kk < GC_K / 16; ++kk)
            tc::mma_f16_pair(tmem_base + ab * GC_ROWS, ad + 2 * kk, bd + 2 * kk, idesc, (k > 0 || kk > 0) ? 1u : 0u);
          tc::mma_commit_pair(&empty[st]);
        }
        __syncwarp();
        if (++st == GC_STAGES) { st = 0; ph ^= 1; }
      }
      if (ok && tc::elect_one()) tc::mma_commit_pair(&acc_full[ab]);
      __syncwarp();
    }
  } else if (warp >= GC_EPI0) {
    // ------------------------------------------------------------------ epilogue: lane quarter q, every other block of 32 rows
    const int q = warp & 3, half = (warp - GC_EPI0) >> 2;
    uint32_t ti = 0;
    int e = 0;
    for (int item = pair; item < items && ok; item += pairs, ++ti) {
      const GcItem it = gc_item(tab, item, p.blocks, e);
      const uint32_t ab = ti & 1u;
      if (!(ok = tc::mbar_wait(&acc_full[ab], (ti >> 1) & 1))) break;
      tc::fence_after_sync();
      const uint32_t acc = tmem_base + (static_cast<uint32_t>(32 * q) << 16) + ab * GC_ROWS;
      const int col = GLU ? it.block * 128 + static_cast<int>(rank) * 64 + 16 * q + (lane & 15) : it.block * 256 + static_cast<int>(rank) * 128 + 32 * q + lane;
#pragma unroll 1
      for (int c0 = 32 * half; c0 < it.rows; c0 += 64) {
        float v[32];
        tc::tmem_ld32(acc + c0, v);
        if (GLU) {
          const int up = lane >> 4;
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            const float other = __shfl_xor_sync(0xffffffffu, up ? v[c] : v[c + 1], 16);
            const int row = c0 + c + up;
            if (row < it.rows && col < p.N)
              store_act(p.y, p.y_dtype, static_cast<int64_t>(it.row0 + row) * p.N + col, up ? silu_mul(other, v[c + 1]) : silu_mul(v[c], other));
          }
        } else if (col < p.N) {
#pragma unroll
          for (int c = 0; c < 32; ++c)
            if (c0 + c < it.rows) store_act(p.y, p.y_dtype, static_cast<int64_t>(it.row0 + c0 + c) * p.N + col, v[c]);
        }
      }
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0)
        asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(tc::cluster_map(tc::smem_u32(&acc_empty[ab]), 0)) : "memory");
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::cluster_arrive();
  tc::cluster_wait();                          // nothing of the other CTA reaches into this one any more
  if (warp == 2) tc::tmem_dealloc_pair(tmem_base, 512);
}

int launch_grouped_tc(const GroupedArgs& a, cudaStream_t st) {
  const int64_t blocks = (a.N + (a.glu ? 127 : 255)) / (a.glu ? 128 : 256);
  if (a.K % 8 != 0 || a.x_rows == 0 || a.E > GC_MAX_E || !aligned16(a.x, a.w) || (static_cast<int64_t>(a.rows) / GC_ROWS + a.E + 1) * blocks > 0x7fffffff)
    return BM_ERR_UNSUPPORTED;
  GcParams p;
  memset(&p, 0, sizeof(p));
  const cuuint64_t K = a.K, N = a.N, E = a.E;
  {
    const cuuint64_t dims[2] = {K, static_cast<cuuint64_t>(a.x_rows)}, strides[1] = {K * 2};
    const cuuint32_t box[2] = {GC_K, 1};
    if (!encode_map16(&p.x, a.x, 2, dims, strides, box)) return BM_ERR_UNSUPPORTED;
  }
  if (a.glu) {
    const cuuint64_t dims[4] = {K, N, 2, E}, strides[3] = {K * 2, N * K * 2, 2 * N * K * 2};
    const cuuint32_t box[4] = {GC_K, 16, 2, 1};
    if (!encode_map16(&p.w, a.w, 4, dims, strides, box)) return BM_ERR_UNSUPPORTED;
  } else {
    const cuuint64_t dims[3] = {K, N, E}, strides[2] = {K * 2, N * K * 2};
    const cuuint32_t box[3] = {GC_K, 128, 1};
    if (!encode_map16(&p.w, a.w, 3, dims, strides, box)) return BM_ERR_UNSUPPORTED;
  }
  p.offsets = a.offsets; p.index = a.index; p.y = a.y;
  p.x_rows = a.x_rows; p.rows = a.rows; p.N = a.N; p.E = a.E;
  p.slices = (a.K + GC_K - 1) / GC_K; p.blocks = static_cast<int>(blocks);
  p.y_dtype = a.y_dtype; p.bf16 = a.dtype == BM_BF16;
  static PerDeviceOnce once;
  static int grids[MAX_DEVICES];
  int dev = -1;
  BM_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= MAX_DEVICES) return BM_ERR_UNSUPPORTED;
  if (!once.is_done(dev)) {
    for (auto* kernel : {grouped_tc_kernel<true>, grouped_tc_kernel<false>})
      BM_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, gc_smem_bytes(GC_MAX_E)));
    BM_CUDA(cudaDeviceGetAttribute(&grids[dev], cudaDevAttrMultiProcessorCount, dev));
    grids[dev] &= ~1;
    once.mark(dev);
  }
  // items there can be: every group that has rows ends in a piece of its own
  const int64_t most = (static_cast<int64_t>(a.rows) / GC_ROWS + (a.E < a.rows ? a.E : a.rows)) * blocks;
  const int grid = most * 2 < grids[dev] ? static_cast<int>(most) * 2 : grids[dev];
  BM_CUDA(launch_after(a.after, 2, a.glu ? grouped_tc_kernel<true> : grouped_tc_kernel<false>, dim3(grid), GC_THREADS, gc_smem_bytes(a.E), st, p));
  BM_LAUNCH_CHECK("grouped_tc_kernel");
  return BM_OK;
}

}  // namespace bm
