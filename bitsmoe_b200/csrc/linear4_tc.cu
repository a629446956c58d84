// Products with 4-bit weights and group scales for more tokens than linear4_kernel streams the weights for, on tcgen05:
//   y[t][n] = sum over groups of scale[n][g] * (sum over the group's columns of x[t][k] * q[n][k]),  q = code - 8
//
// The weights are the M operand (128 rows), the tokens the N operand (up to 128, in steps of 16).  Codes become exact 16-bit numbers of
// x's type in shared memory; a group's products are summed by the tensor core into a tensor memory buffer of its own, and the epilogue
// warps multiply each by the row's scale in fp32 as they add it to the sums they hold in registers -- a lane owns a row, so that its
// scale is one value.  Nothing but y is rounded; weights rounded to 16 bits after scaling would put the result of an MLP twice as
// far from the exact one as the rounding of its output does.
//   warps 0, 3   producers: codes (64 columns of 128 rows, 4 KB) twelve slices ahead; rows of x six to twelve, as tiled copies
//   warps 12-19  converters, two groups that take the slices in turn: codes -> pairs by mask and subtraction -> 128-byte swizzled rows
//   warp 1       MMA issue: M = 128, N = the tile's tokens, K = 16; a commit per group of columns hands its buffer to the epilogue
//   warps 4-11   epilogue: lane quarter, every other block of 16 tokens
// Where there are few tiles, clusters of CTAs share a tile's columns and add their sums up in the first one's shared memory, in order.
// With a gated pair the rows alternate between 16 gate rows and the 16 up rows that belong to them; lanes l and l + 16 exchange every
// other token's sums at the end.  Waits are bounded; one that gives up raises the status word, and the CTA leaves once its copies and
// products are done.
//
// Measured (bf16, groups of 128): 4096 x 4096 at 64 / 256 / 1024 tokens 19 / 27 / 76 us (0.11 / 0.31 / 0.45 PFLOP/s).  A slice of 64 columns costs 0.45 us of waits, four
// products and commits whatever the tile's width, a launch 8 to 10 us of start, first data, exchange and end.
#include <cuda.h>

#include <cstring>

#include "linear4.cuh"
#include "tc05.cuh"

namespace bm {

bool encode_map16(CUtensorMap* map, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box);
bool encode_map_bytes(CUtensorMap* map, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box);

constexpr int LT_THREADS = 640, LT_EPI0 = 4, LT_EPI_WARPS = 8, LT_CONV0 = 12, LT_CONV_WARPS = 8, LT_ROWS = 128, LT_TOK = 128, LT_K = 64;
constexpr int LT_P_BYTES = LT_ROWS * LT_K / 2, LT_A_BYTES = LT_ROWS * LT_K * 2, LT_B_BYTES = LT_TOK * LT_K * 2;
constexpr int LT_PS = 12, LT_AS = 4, LT_BS = 12, LT_ACC = 4, LT_BOX = 32;       // slots of codes, stages of weights and (at most) of x, accumulators; rows of x a copy
constexpr int LT_B_RING = 6 * LT_B_BYTES;
constexpr int LT_SMEM = LT_PS * LT_P_BYTES + LT_AS * LT_A_BYTES + LT_B_RING + 1024;

struct LtParams {
  CUtensorMap x, x8, p[2];     // x: 32 tokens or 8
  Linear4Args a;
  DenseGuard guard;
  int splits, slices, row_tiles, tok_tiles, tok_piece, per_group;      // splits: CTAs that share a tile's columns; per_group: products of K = 16
};

__device__ __forceinline__ void lt_load_2d(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(tc::smem_u32(dst)),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(tc::smem_u32(bar))
               : "memory");
}
// K-major operand tile of 128-byte rows, 8-row groups 1024 bytes apart, 128-byte swizzle
__device__ __forceinline__ uint64_t lt_desc(uint32_t saddr) {
  return static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4) | (1ull << 16) | (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

template <int XD, bool GLU>
__global__ void __launch_bounds__(LT_THREADS, 1) linear4_tc_kernel(const __grid_constant__ LtParams p) {
  extern __shared__ unsigned char lt_raw[];
  __shared__ __align__(8) uint64_t p_full[LT_PS], p_empty[LT_PS], b_full[LT_BS], b_empty[LT_BS], a_ready[LT_AS], a_empty[LT_AS], acc_full[LT_ACC], acc_empty[LT_ACC], drained;
  __shared__ uint32_t tmem_slot;
  __shared__ int left_out;                 // linear4_finish
  __shared__ int gave_up;                  // a wait of this CTA ran out
  unsigned char* const smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(lt_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  unsigned char *const b_ring = smem + LT_AS * LT_A_BYTES, *const codes = b_ring + LT_B_RING;
  const int warp = tc::warp_index(), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    left_out = 0;
    gave_up = p.guard.limit_ns == 0;
    tc::mbar_init(&drained, 1);
    for (int i = 0; i < LT_PS; ++i) {
      tc::mbar_init(&p_full[i], 1);
      tc::mbar_init(&p_empty[i], LT_CONV_WARPS / 2);
    }
    for (int i = 0; i < LT_BS; ++i) {
      tc::mbar_init(&b_full[i], 1);
      tc::mbar_init(&b_empty[i], 1);
    }
    for (int i = 0; i < LT_AS; ++i) {
      tc::mbar_init(&a_ready[i], LT_CONV_WARPS / 2);
      tc::mbar_init(&a_empty[i], 1);
    }
    for (int i = 0; i < LT_ACC; ++i) {
      tc::mbar_init(&acc_full[i], 1);
      tc::mbar_init(&acc_empty[i], LT_EPI_WARPS);
    }
    tc::mbar_init_fence();
  }
  if (threadIdx.x == 96)
    for (const CUtensorMap* m : {&p.x, &p.x8, &p.p[0], &p.p[1]}) asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(m)) : "memory");
  if (warp == 2) tc::tmem_alloc(&tmem_slot, 512);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem_base = tmem_slot;
  if (!p.a.lead) grid_launch_dependents();
  if (!p.a.beside) grid_wait();
  if (p.a.lead) grid_launch_dependents();
  // tiles of this CTA (neighbours share weight rows), and its slices of their columns: all, or a share that starts with a group
  const int rank = blockIdx.x % p.splits, first = blockIdx.x / p.splits, grid = gridDim.x / p.splits, tiles = p.row_tiles * p.tok_tiles;
  const int mine = tiles > first ? (tiles - first + grid - 1) / grid : 0;
  const int k_first = p.slices * rank / p.splits & ~1, k_end = rank + 1 < p.splits ? p.slices * (rank + 1) / p.splits & ~1 : p.slices;
  const int slices = k_end - k_first, total = mine * slices;
  auto tile_of = [&](int i, int& row0, int& tok0, int& n) {
    const int tile = first + i * grid, rt = tile / p.tok_tiles;
    row0 = rt * (GLU ? LT_ROWS / 2 : LT_ROWS);
    tok0 = (tile - rt * p.tok_tiles) * p.tok_piece;
    n = (min(p.tok_piece, p.a.T - tok0) + 15) & ~15;
  };
  const int b_bytes = p.tok_piece * LT_K * 2, b_stages = min(LT_B_RING / b_bytes, LT_BS);
  bool ok = true;
  int issued = 0;                          // stages of copies under way or done (warps 0 and 3)
  auto wait = [&](uint64_t* bar, uint32_t parity) { return tc::mbar_wait_limit(bar, parity, p.guard.limit_ns); };

  if (warp == 0) {
    // ------------------------------------------------------------------ codes, as far ahead as there are slots
    int slot = 0, ph = 1;
    for (int i = 0; i < mine && ok; ++i) {
      int row0, tok0, n;
      tile_of(i, row0, tok0, n);
      for (int k = k_first; k < k_end; ++k) {
        if (!(ok = wait(&p_empty[slot], ph))) break;
        if (tc::elect_one()) {
          unsigned char* to = codes + slot * LT_P_BYTES;
          tc::mbar_expect_tx(&p_full[slot], LT_P_BYTES);
          lt_load_2d(to, &p.p[0], k * (LT_K / 2), row0, &p_full[slot]);
          lt_load_2d(to + LT_P_BYTES / 2, &p.p[GLU], k * (LT_K / 2), GLU ? row0 : row0 + LT_ROWS / 2, &p_full[slot]);
        }
        __syncwarp();
        ++issued;
        if (++slot == LT_PS) { slot = 0; ph ^= 1; }
      }
    }
  } else if (warp == 3) {
    // ------------------------------------------------------------------ rows of x
    int st = 0, ph = 1;
    for (int i = 0; i < mine && ok; ++i) {
      int row0, tok0, n;
      tile_of(i, row0, tok0, n);
      for (int k = k_first; k < k_end; ++k) {
        if (!(ok = wait(&b_empty[st], ph))) break;
        if (tc::elect_one()) {
          unsigned char* to = b_ring + st * b_bytes;
          tc::mbar_expect_tx(&b_full[st], n * LT_K * 2);
          int r = 0;
          for (; r + LT_BOX <= n; r += LT_BOX) lt_load_2d(to + r * (LT_K * 2), &p.x, k * LT_K, tok0 + r, &b_full[st]);
          for (; r < n; r += 8) lt_load_2d(to + r * (LT_K * 2), &p.x8, k * LT_K, tok0 + r, &b_full[st]);
        }
        __syncwarp();
        ++issued;
        if (++st == b_stages) { st = 0; ph ^= 1; }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issue
    uint32_t acc = 0;                          // groups so far: buffer acc % LT_ACC
    const bool two = p.per_group == 2;
    int s = 0, bs = 0, b_ph = 0;
    for (int i = 0; i < mine && ok; ++i) {
      int row0, tok0, n;
      tile_of(i, row0, tok0, n);
      const uint32_t idesc = XD == BM_F16 ? tc::idesc_f16(LT_ROWS, n) : tc::idesc_bf16(LT_ROWS, n);
      int in_group = 0;
      for (int k = 0; k < slices && ok; ++k, ++s) {
        const int st = s % LT_AS;
        if (!(ok = wait(&b_full[bs], b_ph) && wait(&a_ready[st], (s / LT_AS) & 1))) break;
        tc::fence_after_sync();
        const uint64_t ad = lt_desc(tc::smem_u32(smem + st * LT_A_BYTES)), bd = lt_desc(tc::smem_u32(b_ring + bs * b_bytes));
        // the slice's products of one group at a time: four, or two and two
        const bool end = k + 1 == slices;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (h == 1 && !two) break;
          const uint32_t buf = acc % LT_ACC, d = tmem_base + buf * LT_TOK;
          if (in_group == 0) {
            if (acc >= LT_ACC && !(ok = wait(&acc_empty[buf], (acc / LT_ACC - 1) & 1))) break;
            tc::fence_after_sync();
          }
          const bool last = two || in_group + 4 == p.per_group || end;
          if (tc::elect_one()) {
            tc::mma_f16(d, ad + 4 * h, bd + 4 * h, idesc, in_group > 0 ? 1u : 0u);
            tc::mma_f16(d, ad + 4 * h + 2, bd + 4 * h + 2, idesc, 1u);
            if (!two) {
              tc::mma_f16(d, ad + 4, bd + 4, idesc, 1u);
              tc::mma_f16(d, ad + 6, bd + 6, idesc, 1u);
            }
            if (last) tc::mma_commit(&acc_full[buf]);
            if (h == 1 || !two) {
              tc::mma_commit(&a_empty[st]);
              tc::mma_commit(&b_empty[bs]);
            }
          }
          __syncwarp();
          in_group = last ? 0 : in_group + 4;
          acc += last;
        }
        if (++bs == b_stages) { bs = 0; b_ph ^= 1; }
      }
    }
  } else if (warp >= LT_CONV0) {
    // ------------------------------------------------------------------ converters: a piece is 32 codes of a row
    const int grp = (warp - LT_CONV0) / (LT_CONV_WARPS / 2), i = threadIdx.x - 32 * LT_CONV0 - grp * (16 * LT_CONV_WARPS);
    for (int s = grp; s < total; s += 2) {
      const int slot = s % LT_PS, st = s % LT_AS;
      if (!(ok = wait(&p_full[slot], (s / LT_PS) & 1))) break;
      uint4 w[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int piece = i + u * (16 * LT_CONV_WARPS), m = piece >> 1;
        // row m of the operand: of a gated pair the gate rows come first among the codes
        const int src = GLU ? ((m & 16) ? LT_ROWS / 2 : 0) + 16 * (m >> 5) + (m & 15) : m;
        w[u] = *reinterpret_cast<const uint4*>(codes + slot * LT_P_BYTES + src * (LT_K / 2) + (piece & 1) * 16);
      }
      if (s >= LT_AS && !(ok = wait(&a_empty[st], (s / LT_AS - 1) & 1))) break;
      unsigned char* const to = smem + st * LT_A_BYTES;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int piece = i + u * (16 * LT_CONV_WARPS), m = piece >> 1;
        const uint32_t words[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t q[4];
          codes_to_pairs<XD>(words[j], q);     // (0, 4) (1, 5) (2, 6) (3, 7) -> in order
          *reinterpret_cast<uint4*>(to + m * 128 + (((4 * (piece & 1) + j) ^ (m & 7)) << 4)) =
              make_uint4(__byte_perm(q[0], q[1], 0x5410), __byte_perm(q[2], q[3], 0x5410), __byte_perm(q[0], q[1], 0x7632), __byte_perm(q[2], q[3], 0x7632));
        }
      }
      tc::fence_async_smem();
      __syncwarp();
      // the codes' slot is given back here, where what was read of it has been stored: the compiler may move the loads down to their use,
      // past an arrival that stands between the two (it did: rows of the slice twelve later, once the epilogue was fast enough to wait)
      if (lane == 0) {
        tc::mbar_arrive(&p_empty[slot]);
        tc::mbar_arrive(&a_ready[st]);
      }
    }
  } else if (warp >= LT_EPI0) {
    // ------------------------------------------------------------------ epilogue
    const int q = warp & 3, half = (warp - LT_EPI0) >> 2, up = GLU ? lane >> 4 : 0;
    uint32_t acc = 0;
    for (int i = 0; i < mine && ok; ++i) {
      int row0, tok0, n;
      tile_of(i, row0, tok0, n);
      const int row = row0 + (GLU ? 16 * q + (lane & 15) : 32 * q + lane);
      const __half* sc = p.a.s[up] + static_cast<int64_t>(min(row, p.a.N - 1)) * p.a.groups;
      float sum[4][16] = {};
      // scales four groups ahead; columns behind the matrix are zeros of x, what they are scaled by must only be finite
      uint32_t ahead[4];
      auto load_scales = [&](int g0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) ahead[j] = g0 + j < p.a.groups ? __ldg(reinterpret_cast<const unsigned short*>(sc) + g0 + j) : 0u;
      };
      const int g_first = k_first * (LT_K / 16) / p.per_group, g_end = g_first + (slices * (LT_K / 16) + p.per_group - 1) / p.per_group;
      load_scales(g_first);
      for (int g0 = g_first; g0 < g_end && ok; g0 += 4) {
        const uint32_t now[4] = {ahead[0], ahead[1], ahead[2], ahead[3]};
        load_scales(g0 + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (g0 + j >= g_end) break;
          const uint32_t buf = acc % LT_ACC;
          if (!(ok = wait(&acc_full[buf], (acc / LT_ACC) & 1))) break;
          tc::fence_after_sync();
          const uint32_t at = tmem_base + (static_cast<uint32_t>(32 * q) << 16) + buf * LT_TOK;
          const float f = __half2float(__ushort_as_half(static_cast<unsigned short>(now[j])));
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const int c0 = 16 * (half + 2 * b);
            if (c0 >= n) break;
            float v[16];
            tc::tmem_ld16(at + c0, v);
#pragma unroll
            for (int c = 0; c < 16; ++c) sum[b][c] = fmaf(v[c], f, sum[b][c]);
          }
          tc::fence_before_sync();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(&acc_empty[buf]);
          ++acc;
        }
      }
      if (p.splits > 1) {
        // (one tile a CTA) the sums meet in the first CTA's shared memory, whose rings nothing uses any more behind the first barrier
        const int me = threadIdx.x - 32 * LT_EPI0;
        tc::cluster_arrive();
        tc::cluster_wait();
        if (rank > 0)
#pragma unroll
          for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int c = 0; c < 16; c += 4)
              asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(tc::cluster_map(tc::smem_u32(smem) + (((rank - 1) * 16 + 4 * b + c / 4) * 32 * LT_EPI_WARPS + me) * 16, 0)),
                           "f"(sum[b][c]), "f"(sum[b][c + 1]), "f"(sum[b][c + 2]), "f"(sum[b][c + 3])
                           : "memory");
        tc::cluster_arrive();
        tc::cluster_wait();
        if (rank > 0) break;
        for (int r = 1; r < p.splits; ++r)
#pragma unroll
          for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int c = 0; c < 16; c += 4) {
              const float4 v = *reinterpret_cast<const float4*>(smem + (((r - 1) * 16 + 4 * b + c / 4) * 32 * LT_EPI_WARPS + me) * 16);
              sum[b][c] += v.x; sum[b][c + 1] += v.y; sum[b][c + 2] += v.z; sum[b][c + 3] += v.w;
            }
      }
      if (!ok) break;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int c0 = 16 * (half + 2 * b);
        if (c0 >= n) break;
        if (GLU) {
          float z[8];
#pragma unroll
          for (int j = 0; j < 16; j += 2) {
            const float other = __shfl_xor_sync(0xffffffffu, up ? sum[b][j] : sum[b][j + 1], 16);
            z[j / 2] = up ? silu_mul(other, sum[b][j + 1]) : silu_mul(sum[b][j], other);
          }
          linear4_finish<XD, XD == BM_F16>(p.a, row, z, left_out, [&](int j) { return tok0 + c0 + 2 * j + up < p.a.T && row < p.a.N ? tok0 + c0 + 2 * j + up : -1; });
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = sum[b][8 * h + j];
            linear4_finish<XD, XD == BM_F16>(p.a, row, v, left_out, [&](int j) { return tok0 + c0 + 8 * h + j < p.a.T && row < p.a.N ? tok0 + c0 + 8 * h + j : -1; });
          }
        }
      }
    }
  }
  if (p.splits > 1 && (warp < LT_EPI0 || warp >= LT_CONV0))
    for (int i = 0; i < 2; ++i) {
      tc::cluster_arrive();
      tc::cluster_wait();
    }
  if (!ok && lane == 0) gave_up = 1;
  if (p.a.beside) grid_wait();
  tc::fence_before_sync();
  __syncthreads();
  if (gave_up) {
    // nothing may be under way when the CTA leaves: the last copies into every slot and stage, and the products
    if (warp == 0)
      for (int k = max(0, issued - LT_PS); k < issued; ++k) tc::mbar_wait(&p_full[k % LT_PS], (k / LT_PS) & 1);
    if (warp == 3)
      for (int k = max(0, issued - b_stages); k < issued; ++k) tc::mbar_wait(&b_full[k % b_stages], (k / b_stages) & 1);
    if (warp == 1) {
      if (tc::elect_one()) tc::mma_commit(&drained);
      __syncwarp();
      tc::mbar_wait(&drained, 0);
    }
    if (threadIdx.x == 0) atomicExch(p.guard.status, BM_ERR_TIMEOUT);
    __syncthreads();
  }
  if (XD == BM_F16 && !GLU && p.a.x_wide && left_out)
    for (int i = 0; i < mine; ++i) {
      int row0, tok0, n;
      tile_of(i, row0, tok0, n);
      linear4_redo(p.a, row0, LT_ROWS, tok0, min(p.tok_piece, p.a.T - tok0));
    }
  if (warp == 2) tc::tmem_dealloc(tmem_base, 512);
}

// CTAs that share a tile's columns where there are few tiles (a cluster of four leaves a few SMs of a group unused).
static int lt_splits(int64_t tiles, int slices, int sms) { return tiles * 4 <= sms * 7 / 8 && slices >= 8 ? 4 : tiles * 2 <= sms && slices >= 4 ? 2 : 1; }

double linear4_tc_us(const Linear4Args& a, int sms) {
  const int rows = a.glu ? LT_ROWS / 2 : LT_ROWS, slices = (a.K + LT_K - 1) / LT_K;
  const int64_t tiles = static_cast<int64_t>((a.N + rows - 1) / rows) * ((a.T + LT_TOK - 1) / LT_TOK);
  const int splits = lt_splits(tiles, slices, sms);
  return 9.0 + 0.45 * ((slices + splits - 1) / splits) * ((tiles * splits + sms - 1) / sms);
}

int launch_linear4_tc(const Linear4Args& args, int x_dtype, int group, LaunchAfter after, cudaStream_t st) {
  const Linear4Args& a = args;
  if (a.ldx % 8 != 0 || !aligned16(a.x, a.p[0], a.p[1])) return BM_ERR_UNSUPPORTED;
  LtParams p;
  memset(&p, 0, sizeof(p));
  p.a = a;
  {
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(a.K), static_cast<cuuint64_t>(a.T)}, strides[1] = {static_cast<cuuint64_t>(a.ldx) * 2};
    const cuuint32_t box[2] = {LT_K, LT_BOX}, box8[2] = {LT_K, 8};
    if (!encode_map16(&p.x, a.x, 2, dims, strides, box) || !encode_map16(&p.x8, a.x, 2, dims, strides, box8)) return BM_ERR_UNSUPPORTED;
  }
  for (int i = 0; i < 2; ++i) {
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(a.words) * 4, static_cast<cuuint64_t>(a.N)}, strides[1] = {static_cast<cuuint64_t>(a.words) * 4};
    const cuuint32_t box[2] = {LT_K / 2, LT_ROWS / 2};
    if (!encode_map_bytes(&p.p[i], a.p[a.glu ? i : 0], 2, dims, strides, box)) return BM_ERR_UNSUPPORTED;
  }
  p.slices = (a.K + LT_K - 1) / LT_K;
  p.per_group = group / 16;
  p.row_tiles = (a.N + (a.glu ? LT_ROWS / 2 : LT_ROWS) - 1) / (a.glu ? LT_ROWS / 2 : LT_ROWS);
  const int pieces = (a.T + LT_TOK - 1) / LT_TOK;
  p.tok_piece = ((a.T + pieces - 1) / pieces + 15) & ~15;
  p.tok_tiles = (a.T + p.tok_piece - 1) / p.tok_piece;
  if (static_cast<int64_t>(p.row_tiles) * p.tok_tiles * p.slices > 0x3fffffff) return BM_ERR_UNSUPPORTED;
  static PerDeviceOnce once;
  static int sms[MAX_DEVICES];
  int dev = -1;
  BM_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= MAX_DEVICES) return BM_ERR_UNSUPPORTED;
  const int rc = dense_guard(&p.guard);
  if (rc) return rc;
  if (!once.is_done(dev)) {
    for (auto* kernel : {linear4_tc_kernel<BM_F16, false>, linear4_tc_kernel<BM_F16, true>, linear4_tc_kernel<BM_BF16, false>, linear4_tc_kernel<BM_BF16, true>})
      BM_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, LT_SMEM));
    BM_CUDA(cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev));
    once.mark(dev);
  }
  const int tiles = p.row_tiles * p.tok_tiles;
  p.splits = lt_splits(tiles, p.slices, sms[dev]);
  const int grid = p.splits > 1 ? tiles * p.splits : tiles < sms[dev] ? tiles : sms[dev];
  auto* kernel = x_dtype == BM_F16 ? (a.glu ? linear4_tc_kernel<BM_F16, true> : linear4_tc_kernel<BM_F16, false>)
                                   : (a.glu ? linear4_tc_kernel<BM_BF16, true> : linear4_tc_kernel<BM_BF16, false>);
  BM_CUDA(launch_after(after, p.splits, kernel, dim3(grid), LT_THREADS, LT_SMEM, st, p));
  BM_LAUNCH_CHECK("linear4_tc_kernel");
  return BM_OK;
}

}  // namespace bm
