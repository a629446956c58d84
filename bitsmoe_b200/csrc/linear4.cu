// Products with 4-bit weights and one fp16 scale for every 32, 64 or 128 columns of a row:
//   y[t][n] = sum_k x[t][k] * scale[n][k / group] * (code[n][k] - 8)   (+ residual[t][n])
// The code of column 8 j + i is in bits 4 i .. 4 i + 3 of word j of the row; rows are padded to whole 16 bytes.
//
// linear4_kernel streams the weights once per 16 tokens.  A warp takes 16 rows; lane (g, t) of it holds, for rows g and g + 8, the words of
// group / 4 neighbouring columns, so that one mma.sync m16n8k16 never crosses a group: contraction position is whatever order both
// operands agree on, and x is put into that order once per CTA (shared memory, 16 bytes per lane and word).  Codes become exact
// 16-bit numbers -8 .. 7 of x's type by mask and subtraction of a constant; products of a group are summed in fp32 by the tensor
// core and multiplied by the group's scale in fp32, so nothing but the output is rounded.  Few rows: the eight warps of a CTA and the
// CTAs of a cluster share a row's columns and meet in shared memory, in a fixed order.
//
// Measured (groups of 128): K 2048, N 100003, 4 tokens 35.6 us in bf16 and 32 in fp16 (3.0 and 3.3 TB/s; floor 16.3): latency, since the
// 40 instructions for 512 codes use 39 % of the issue slots: four warps a scheduler, each one chain of loads, unpacking, products and scale.  K 2048, N 4096, one token 4.5 us inside a graph, 8192 x 8192 at 1 / 8 / 16 tokens 15 / 20 / 29 (floor 5.3).
#include <cooperative_groups.h>

#include <algorithm>

#include "linear4.cuh"

namespace cg = cooperative_groups;

namespace bm {

int launch_row_gate(const void* x, int x_dtype, const uint16_t* w, int w_dtype, int T, int H, float* gate, LaunchAfter after, cudaStream_t st, bool lead);

constexpr int L4_THREADS = 256, L4_WARPS = 8, L4_CHUNK = 128;
__host__ __device__ constexpr int l4_batch(int nt) { return 4; }      // chunks in flight a warp and buffer
__host__ __device__ constexpr int l4_ctas(int nt) { return 2; }       // CTAs an SM
constexpr size_t L4_SMEM = 110 * 1024, L4_SMEM_MOST = 220 * 1024;          // two CTAs an SM, one

template <int XD>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float c0, float c1, float c2, float c3) {
  if (XD == BM_F16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}

// Place of word kw (eight columns of x) among the words of a CTA: the words that a quad's lanes use together are neighbours.
template <int WPL>
__device__ __forceinline__ int l4_place(int kw) { return (kw / (4 * WPL)) * (4 * WPL) + (kw % WPL) * 4 + (kw / WPL) % 4; }
// Byte offset of token n's piece: NT pieces of 16 bytes a word, swapped so that eight neighbouring lanes (two tokens, four words) hit
// eight different bank groups.
template <int NT>
__device__ __forceinline__ int l4_piece(int place, int n) {
  const int t = place & 3, sw = NT >= 8 ? 2 * t : 0;
  return (place * NT + (n ^ sw)) * 16;
}

// Weights are read once: past the first-level cache.
__device__ __forceinline__ uint4 l4_stream(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// WIDE: one of the two products of an fp16 MLP, whose middle may pass fp16's range; its few instructions on the way out cost products that have
// no need of them 2 to 7 %.
template <int NT, int XD, int WPL, bool WIDE>
__global__ void __launch_bounds__(L4_THREADS, l4_ctas(NT)) linear4_kernel(const __grid_constant__ Linear4Args a) {
  constexpr int NB = NT < 8 ? 1 : NT / 8, GPC = 4 / WPL, L4_BATCH = l4_batch(NT), SPR = (L4_BATCH * GPC + 3) / 4;     // groups a chunk, scale loads per row and batch
  extern __shared__ __align__(16) unsigned char l4_smem[];
  __shared__ int left_out;                 // linear4_finish
  if (WIDE && threadIdx.x == 0) left_out = 0;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int split = blockIdx.x % a.splits, kw = warp % a.kwarps, rw = warp / a.kwarps, rws = L4_WARPS / a.kwarps;
  const int chunks = (a.K + L4_CHUNK - 1) / L4_CHUNK;
  const int c_first = chunks * split / a.splits, c_end = chunks * (split + 1) / a.splits;           // this CTA's chunks of 128 columns
  const int n0 = blockIdx.y * NT, nn = min(NT, a.T - n0);
  float* const recv = reinterpret_cast<float*>(l4_smem + static_cast<size_t>((chunks + a.splits - 1) / a.splits) * (L4_CHUNK / 8) * NT * 16);
  const int wc = c_end - c_first, w_first = wc * kw / a.kwarps, w_end = wc * (kw + 1) / a.kwarps;      // this warp's chunks, CTA-relative
  const int per = a.glu ? 8 : 16, cluster_id = blockIdx.x / a.splits, clusters = gridDim.x / a.splits;
  // ---- the weights travel a batch ahead of the products, across the ends of units too: where the next batch starts
  int f_rb = cluster_id, f_c = w_first;
  const uint32_t *pa, *pc;
  const __half *sa, *sc;
  auto rows_of = [&](int rb) {
    const int r0 = (rb * rws + rw) * per, ra = min(r0 + g, a.N - 1), rc = a.glu ? ra : min(r0 + 8 + g, a.N - 1);
    pa = a.p[0] + static_cast<int64_t>(ra) * a.words;
    pc = (a.glu ? a.p[1] : a.p[0]) + static_cast<int64_t>(rc) * a.words;
    sa = a.s[0] + static_cast<int64_t>(ra) * a.groups;
    sc = (a.glu ? a.s[1] : a.s[0]) + static_cast<int64_t>(rc) * a.groups;
  };
  rows_of(f_rb);
  auto fetch = [&](uint32_t (&wd)[2][L4_BATCH][4], float (&sd)[2][SPR]) {
    if (f_rb >= a.row_blocks) return;
    // codes behind the matrix meet zeros of x, chunks behind the warp's are not multiplied: any word of the row will do there
    const int first = (c_first + f_c) * (L4_CHUNK / 8) + t * WPL, last = a.words - WPL;
    auto load = [&](int u, int j, const uint32_t* sa_, const uint32_t* sc_) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint32_t* src = r ? sc_ : sa_;
        if (WPL == 4) {
          const uint4 v = l4_stream(reinterpret_cast<const uint4*>(src));
          wd[r][u][0] = v.x; wd[r][u][1] = v.y; wd[r][u][2] = v.z; wd[r][u][3] = v.w;
        } else if (WPL == 2) {
          const uint2 v = __ldg(reinterpret_cast<const uint2*>(src));
          wd[r][u][2 * j] = v.x; wd[r][u][2 * j + 1] = v.y;
        } else {
          wd[r][u][j] = __ldg(src);
        }
      }
    };
    if (first + (L4_BATCH * L4_CHUNK / 8 - 4 * WPL) <= last) {       // the whole batch lies inside the row: one address a row
      const uint32_t *qa = pa + first, *qc = pc + first;
#pragma unroll
      for (int u = 0; u < L4_BATCH; ++u)
#pragma unroll
        for (int j = 0; j < GPC; ++j) load(u, j, qa + u * (L4_CHUNK / 8) + j * 4 * WPL, qc + u * (L4_CHUNK / 8) + j * 4 * WPL);
    } else {
#pragma unroll
      for (int u = 0; u < L4_BATCH; ++u)
#pragma unroll
        for (int j = 0; j < GPC; ++j) {
          const int at = min(first + u * (L4_CHUNK / 8) + j * 4 * WPL, last);
          load(u, j, pa + at, pc + at);
        }
    }
#pragma unroll
    for (int i = 0; i < SPR; ++i) {
      const int grp = (c_first + f_c) * GPC + 4 * i + t;
      const bool in = grp < a.groups && f_c + (4 * i + t) / GPC < w_end;
      sd[0][i] = in ? __half2float(sa[grp]) : 0.f;
      sd[1][i] = in ? __half2float(sc[grp]) : 0.f;
    }
    f_c += L4_BATCH;
    if (f_c >= w_end) {
      f_c = w_first;
      f_rb += clusters;
      if (f_rb < a.row_blocks) rows_of(f_rb);
    }
  };
  uint32_t w[2][2][L4_BATCH][4];           // [buffer][row][chunk][word]
  float sv[2][2][SPR];                     // lane t: scale of group 4 i + t of the batch
  if (!a.lead) grid_launch_dependents();
  if (!a.early && !a.beside) grid_wait();
  if (a.lead) grid_launch_dependents();
  fetch(w[0], sv[0]);
  if (a.early) grid_wait();
  // ---- x of this CTA's columns, in the order of the products
  {
    const int words = wc * (L4_CHUNK / 8);
    constexpr int U = NT >= 16 ? 8 : 4;
    for (int i0 = threadIdx.x; i0 < words * nn; i0 += U * L4_THREADS) {
      uint4 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * L4_THREADS, n = i / words, k = c_first * L4_CHUNK + 8 * (i - n * words);
        v[u] = make_uint4(0u, 0u, 0u, 0u);
        if (i < words * nn) {
          const uint16_t* src = static_cast<const uint16_t*>(a.x) + static_cast<int64_t>(n0 + n) * a.ldx + k;
          if (a.vec_x && k + 8 <= a.K) v[u] = *reinterpret_cast<const uint4*>(src);
          else {
            uint16_t* e = reinterpret_cast<uint16_t*>(&v[u]);
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (k + j < a.K) e[j] = src[j];
          }
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * L4_THREADS, n = i / words;
        if (i < words * nn)
          *reinterpret_cast<uint4*>(l4_smem + l4_piece<NT>(l4_place<WPL>(i - n * words), n)) =
              make_uint4(__byte_perm(v[u].x, v[u].z, 0x5410), __byte_perm(v[u].x, v[u].z, 0x7632), __byte_perm(v[u].y, v[u].w, 0x5410),
                         __byte_perm(v[u].y, v[u].w, 0x7632));
      }
    }
  }
  __syncthreads();
  float acc[NB][4] = {};
  // where this lane's tokens' pieces start; columns of tokens that are not there may hold anything, they are not looked at
  const unsigned char* xs[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) xs[b] = l4_smem + l4_piece<NT>(t, NT < 8 ? g % NT : 8 * b + g);
  auto multiply = [&](int c, const uint32_t (&wd)[2][L4_BATCH][4], const float (&sd)[2][SPR]) {
    const int base = c * (L4_CHUNK / 8) * NT * 16;
#pragma unroll
    for (int u = 0; u < L4_BATCH; ++u) {
      if (c + u >= w_end) break;
#pragma unroll
      for (int j = 0; j < GPC; ++j) {
        float part[NB][4];
#pragma unroll
        for (int v = 0; v < WPL; ++v) {
          uint32_t qa[4], qc[4];
          codes_to_pairs<XD>(wd[0][u][j * WPL + v], qa);
          codes_to_pairs<XD>(wd[1][u][j * WPL + v], qc);
          const uint32_t first[4] = {qa[0], qc[0], qa[1], qc[1]}, second[4] = {qa[2], qc[2], qa[3], qc[3]};
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            const uint4 xv = *reinterpret_cast<const uint4*>(xs[b] + base + (u * (L4_CHUNK / 8) + (j * WPL + v) * 4) * NT * 16);
            float (&p)[4] = part[b];
            if (v == 0) mma_16816<XD>(p, first, xv.x, xv.y, 0.f, 0.f, 0.f, 0.f);
            else mma_16816<XD>(p, first, xv.x, xv.y, p[0], p[1], p[2], p[3]);
            mma_16816<XD>(p, second, xv.z, xv.w, p[0], p[1], p[2], p[3]);
          }
        }
        const int q = u * GPC + j;
        const float f0 = __shfl_sync(0xffffffffu, sd[0][q / 4], (lane & ~3) + q % 4), f1 = __shfl_sync(0xffffffffu, sd[1][q / 4], (lane & ~3) + q % 4);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          acc[b][0] = fmaf(part[b][0], f0, acc[b][0]);
          acc[b][1] = fmaf(part[b][1], f0, acc[b][1]);
          acc[b][2] = fmaf(part[b][2], f1, acc[b][2]);
          acc[b][3] = fmaf(part[b][3], f1, acc[b][3]);
        }
      }
    }
  };
  // ---- sums of the warps (and CTAs) that share the rows, then out
  auto finish_unit = [&](int rb) {
    const int ra = (rb * rws + rw) * per + g, rc = ra + 8;
    if (a.kwarps == 1 && a.splits == 1) {
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        auto token = [&](int row, int i) { return 8 * b + 2 * t + i < nn && row < a.N ? n0 + 8 * b + 2 * t + i : -1; };
        if (a.glu) {
          const float z[2] = {silu_mul(acc[b][0], acc[b][2]), silu_mul(acc[b][1], acc[b][3])};
          linear4_finish<XD, WIDE>(a, ra, z, left_out, [&](int i) { return token(ra, i); });
        } else {
          const float lo[2] = {acc[b][0], acc[b][1]}, hi[2] = {acc[b][2], acc[b][3]};
          linear4_finish<XD, WIDE>(a, ra, lo, left_out, [&](int i) { return token(ra, i); });
          linear4_finish<XD, WIDE>(a, rc, hi, left_out, [&](int i) { return token(rc, i); });
        }
      }
      return;
    }
    constexpr int COLS = 8 * NB, PART = 16 * COLS;       // floats of one warp's part: [row][token]
    float* mine = recv + (split * L4_WARPS + warp) * PART;
    if (a.splits > 1) {
      cg::this_cluster().sync();                         // the first CTA runs, and has read the parts of the rows before
      mine = cg::this_cluster().map_shared_rank(mine, 0);
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      *reinterpret_cast<float2*>(mine + g * COLS + 8 * b + 2 * t) = make_float2(acc[b][0], acc[b][1]);
      *reinterpret_cast<float2*>(mine + (g + 8) * COLS + 8 * b + 2 * t) = make_float2(acc[b][2], acc[b][3]);
    }
    if (a.splits > 1) cg::this_cluster().sync();
    else __syncthreads();
    if (split == 0) {
      const int outs = per * rws;
      for (int o = threadIdx.x; o < outs * nn; o += L4_THREADS) {
        const int n = o / outs, r = o - n * outs, wr = r / per, row = r - wr * per, out_row = (rb * rws + wr) * per + row;
        if (out_row >= a.N) continue;
        float v = 0.f, u = 0.f;
        for (int s = 0; s < a.splits; ++s)
          for (int k = 0; k < a.kwarps; ++k) {
            const float* part = recv + (s * L4_WARPS + wr * a.kwarps + k) * PART + n;
            v += part[row * COLS];
            if (a.glu) u += part[(row + 8) * COLS];
          }
        const float out[1] = {a.glu ? silu_mul(v, u) : v};
        linear4_finish<XD, WIDE>(a, out_row, out, left_out, [&](int) { return n0 + n; });
      }
    }
    if (a.splits == 1) __syncthreads();                  // the parts may be overwritten
  };
  int rb = cluster_id, c = w_first;
  auto step = [&](uint32_t (&now)[2][L4_BATCH][4], float (&snow)[2][SPR], uint32_t (&next)[2][L4_BATCH][4], float (&snext)[2][SPR]) {
    fetch(next, snext);
    multiply(c, now, snow);
    c += L4_BATCH;
    if (c >= w_end) {
      finish_unit(rb);
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[b][i] = 0.f;
      c = w_first;
      rb += clusters;
    }
    return rb < a.row_blocks;
  };
  while (step(w[0], sv[0], w[1], sv[1]) && step(w[1], sv[1], w[0], sv[0])) {
  }
  if (WIDE && a.x_wide) {
    __syncthreads();
    if (left_out)
      for (rb = cluster_id; rb < a.row_blocks; rb += clusters) linear4_redo(a, rb * rws * 16, rws * 16, n0, nn);
  }
  if (a.beside) grid_wait();
}

// Any size and alignment: a warp takes a row of the matrix (of each of a gated pair) and eight tokens, element loads, fp32 FMA.  For rows whose columns of
// x fit no CTA's shared memory and that tiled copies cannot describe.
constexpr int LA_TOKENS = 8;
template <int XD, bool GLU>
__global__ void __launch_bounds__(L4_THREADS) linear4_any_kernel(const __grid_constant__ Linear4Args a) {
  constexpr int M = GLU ? 2 : 1;
  const int lane = threadIdx.x & 31, row = blockIdx.x * L4_WARPS + (threadIdx.x >> 5);
  if (!a.lead) grid_launch_dependents();
  grid_wait();
  if (a.lead) grid_launch_dependents();
  if (row >= a.N) return;
  for (int64_t n0 = static_cast<int64_t>(blockIdx.y) * LA_TOKENS; n0 < a.T; n0 += static_cast<int64_t>(gridDim.y) * LA_TOKENS) {
    float acc[M][LA_TOKENS] = {};
    for (int w = lane; 8 * w < a.K; w += 32) {
      float part[M][LA_TOKENS] = {};
      uint32_t code[M];
#pragma unroll
      for (int m = 0; m < M; ++m) code[m] = __ldg(a.p[m] + static_cast<int64_t>(row) * a.words + w);
      for (int j = 0; j < 8 && 8 * w + j < a.K; ++j)
#pragma unroll
        for (int n = 0; n < LA_TOKENS; ++n) {
          if (n0 + n >= a.T) break;
          const int64_t o = (n0 + n) * a.ldx + 8 * w + j;
          float v = load_x<XD>(a.x, o);
          if (XD == BM_F16 && a.x_wide && !(fabsf(v) <= 65504.f)) v = a.x_wide[o];
#pragma unroll
          for (int m = 0; m < M; ++m) part[m][n] = fmaf(v, static_cast<float>(static_cast<int>(code[m] >> (4 * j) & 15u) - 8), part[m][n]);
        }
#pragma unroll
      for (int m = 0; m < M; ++m) {
        const float f = __half2float(a.s[m][static_cast<int64_t>(row) * a.groups + 8 * w / a.group]);
#pragma unroll
        for (int n = 0; n < LA_TOKENS; ++n) acc[m][n] = fmaf(part[m][n], f, acc[m][n]);
      }
    }
#pragma unroll
    for (int n = 0; n < LA_TOKENS; ++n) {
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) acc[m][n] += __shfl_xor_sync(0xffffffffu, acc[m][n], o);
      const int64_t t = n0 + n;
      if (lane != n || t >= a.T) continue;
      const float v = GLU ? silu_mul(acc[0][n], acc[M - 1][n]) : acc[0][n];
      store_x<XD>(a.y, t * a.ldy + row, fmaf(v, a.row_gate ? a.row_gate[t] : 1.f, a.residual ? load_x<XD>(a.residual, t * a.N + row) : 0.f));
      if (XD == BM_F16 && a.wide && !fits_fp16(v)) a.wide[t * a.ldy + row] = v;
    }
  }
}

static size_t l4_smem_bytes(int nt, int K, int splits, bool shared_rows) {
  const int chunks = (K + L4_CHUNK - 1) / L4_CHUNK, cols = nt < 8 ? 8 : nt;
  return static_cast<size_t>((chunks + splits - 1) / splits) * (L4_CHUNK / 8) * nt * 16 + (shared_rows ? static_cast<size_t>(splits) * L4_WARPS * 16 * cols * 4 : 0);
}

template <int NT, int XD, int WPL, bool WIDE>
static int l4_launch_one(const Linear4Args& a, dim3 grid, size_t smem, LaunchAfter after, cudaStream_t st) {
  static PerDeviceOnce once;
  int dev = -1;
  BM_CUDA(cudaGetDevice(&dev));
  if (!once.is_done(dev)) {
    BM_CUDA(cudaFuncSetAttribute(linear4_kernel<NT, XD, WPL, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(L4_SMEM_MOST)));
    once.mark(dev);
  }
  BM_CUDA(launch_after(after, a.splits, linear4_kernel<NT, XD, WPL, WIDE>, grid, L4_THREADS, smem, st, a));
  BM_LAUNCH_CHECK("linear4_kernel");
  return BM_OK;
}
template <int NT, int XD, bool WIDE>
static int l4_launch_group(const Linear4Args& a, int group, dim3 grid, size_t smem, LaunchAfter after, cudaStream_t st) {
  return group == 128 ? l4_launch_one<NT, XD, 4, WIDE>(a, grid, smem, after, st) : group == 64 ? l4_launch_one<NT, XD, 2, WIDE>(a, grid, smem, after, st)
                                                                                       : l4_launch_one<NT, XD, 1, WIDE>(a, grid, smem, after, st);
}
template <int NT>
static int l4_launch(const Linear4Args& a, int x_dtype, int group, dim3 grid, size_t smem, LaunchAfter after, cudaStream_t st) {
  if (x_dtype == BM_BF16) return l4_launch_group<NT, BM_BF16, false>(a, group, grid, smem, after, st);
  return a.wide || a.x_wide ? l4_launch_group<NT, BM_F16, true>(a, group, grid, smem, after, st) : l4_launch_group<NT, BM_F16, false>(a, group, grid, smem, after, st);
}

// y = x . W^T, or with glu z = silu(x . Wg^T) * (x . Wu^T).
static int linear4(Linear4Args a, int x_dtype, int group, LaunchAfter after, cudaStream_t st) {
  a.words = (a.K + 31) / 32 * 4;
  a.groups = (a.K + group - 1) / group;
  a.group = group;
  a.vec_x = aligned16(a.x) && a.ldx % 8 == 0;
  static PerDeviceOnce once;
  static int sm_counts[MAX_DEVICES];
  int dev = -1;
  BM_CUDA(cudaGetDevice(&dev));
  BM_REQUIRE(dev >= 0 && dev < MAX_DEVICES, BM_ERR_UNSUPPORTED, "linear4: device ordinal %d out of range", dev);
  if (!once.is_done(dev)) {
    BM_CUDA(cudaDeviceGetAttribute(&sm_counts[dev], cudaDevAttrMultiProcessorCount, dev));
    once.mark(dev);
  }
  const int sms = sm_counts[dev];
  const int chunks = (a.K + L4_CHUNK - 1) / L4_CHUNK, units = (a.N + (a.glu ? 7 : 15)) / (a.glu ? 8 : 16);
  int nt = a.T <= 2 ? 2 : a.T <= 8 ? 8 : 16;
  a.kwarps = 1; a.splits = 1;
  while (nt > 8 && l4_smem_bytes(nt, a.K, 8, true) > L4_SMEM_MOST) nt /= 2;
  while (a.splits < 8 && l4_smem_bytes(nt, a.K, a.splits, true) > L4_SMEM) a.splits *= 2;
  // Warps of a CTA that share a row's columns: what leaves the fewest chunks one after the other.  A barrier and the pass over the parts cost a chunk and
  // a half per row block, a cluster's barriers three: 100003 rows of 2048 columns with one, two, four and eight warps 36, 38, 44 and 59 us.
  const int most = sms * l4_ctas(nt) / a.splits, per_split = (chunks + a.splits - 1) / a.splits;
  double best = 1e30, round = 0.0;
  for (int kw = 1; kw <= 8 && (kw == 1 || kw * a.splits <= chunks); kw *= 2) {
    const int blocks = (units + L4_WARPS / kw - 1) / (L4_WARPS / kw), rounds = (blocks + most - 1) / most;
    const double one = (per_split + kw - 1) / kw + (kw > 1 ? 1.5 : 0.3) + (a.splits > 1 ? 3.0 : 0.0);
    if (rounds * one < best) { best = rounds * one; round = one; a.kwarps = kw; }
  }
  const int rws = L4_WARPS / a.kwarps;
  a.row_blocks = (units + rws - 1) / rws;
  const int64_t passes = (a.T + nt - 1) / nt;
  const bool fits = l4_smem_bytes(nt, a.K, a.splits, true) <= L4_SMEM_MOST && passes <= 65535;
  // More tokens than 16: passes over the weights side by side, or the tensor core's kernel, whichever has the smaller estimate (a wave of CTAs takes its
  // chunks and some four us).  us in passes / on the tensor core, bf16, groups of 128: K 512, N 2048, 64 tokens 6 / 11; 2048 x 2048, 32 tokens 9 / 13 and
  // 48 tokens 14 / 14; K 2048, N 4096, 20 tokens 13 / 14 and 32 tokens 16 / 14; 4096 x 4096, 20 tokens 19 / 17; K 2048, N 16384, 20 tokens 25 / 19.  Where
  // the two are close the rule may take the slower (K 8192, N 2048, 20 tokens 21 / 24: estimates 25 / 23), and a gated pair's estimate is low (300 tokens,
  // 2048 columns, 512 rows of each: 13, with a profiler 21).
  const double stream_us = ((a.row_blocks * a.splits * passes + sms * l4_ctas(nt) - 1) / (sms * l4_ctas(nt))) * (round + 4.0);
  if (!fits || (a.T > 16 && linear4_tc_us(a, sms) < stream_us)) {
    const int rc = launch_linear4_tc(a, x_dtype, group, after, st);
    if (rc != BM_ERR_UNSUPPORTED) return rc;
  }
  if (!fits) {
    const dim3 any((a.N + L4_WARPS - 1) / L4_WARPS, std::min((a.T + LA_TOKENS - 1) / LA_TOKENS, 65535));
    auto* kernel = x_dtype == BM_F16 ? (a.glu ? linear4_any_kernel<BM_F16, true> : linear4_any_kernel<BM_F16, false>)
                                     : (a.glu ? linear4_any_kernel<BM_BF16, true> : linear4_any_kernel<BM_BF16, false>);
    BM_CUDA(launch_after(after, 1, kernel, any, L4_THREADS, 0, st, a));
    BM_LAUNCH_CHECK("linear4_any_kernel");
    return BM_OK;
  }
  const int grid = std::min(a.row_blocks, std::max(most, 1)) * a.splits;
  const dim3 g(grid, static_cast<unsigned>(passes));
  const size_t smem = l4_smem_bytes(nt, a.K, a.splits, a.kwarps > 1 || a.splits > 1);
  return nt == 2 ? l4_launch<2>(a, x_dtype, group, g, smem, after, st) : nt == 8 ? l4_launch<8>(a, x_dtype, group, g, smem, after, st)
                                                                               : l4_launch<16>(a, x_dtype, group, g, smem, after, st);
}

}  // namespace bm

using namespace bm;

static int l4_check(const char* what, int dtype, int32_t T, int32_t group, std::initializer_list<int32_t> sizes) {
  BM_REQUIRE(T >= 0, BM_ERR_INVALID_ARG, "%s: bad sizes", what);
  for (int32_t v : sizes) {
    BM_REQUIRE(v > 0, BM_ERR_INVALID_ARG, "%s: bad sizes", what);
    BM_REQUIRE(v < (1 << 30), BM_ERR_UNSUPPORTED, "%s: size %d is too large", what, v);
  }
  BM_REQUIRE(dtype == BM_F16 || dtype == BM_BF16, BM_ERR_INVALID_ARG, "%s: x must be fp16 or bf16", what);
  BM_REQUIRE(group == 32 || group == 64 || group == 128, BM_ERR_UNSUPPORTED, "%s: groups of %d columns; 32, 64 and 128 are supported", what, group);
  return BM_OK;
}

extern "C" int bm_linear4(const void* x, int dtype, const uint32_t* payload, const uint16_t* scale, int32_t T, int32_t K, int32_t N, int32_t group,
                          const void* residual, void* y, void* stream) {
  bm::NvtxRange nvtx_range("bm_linear4");
  const int rc = l4_check("linear4", dtype, T, group, {K, N});
  if (rc) return rc;
  if (T == 0) return BM_OK;
  BM_REQUIRE(x && payload && scale && y, BM_ERR_INVALID_ARG, "linear4: null pointer");
  BM_REQUIRE(aligned16(payload), BM_ERR_INVALID_ARG, "linear4: the codes must start on a 16-byte boundary");
  Linear4Args a{};
  a.p[0] = payload; a.s[0] = reinterpret_cast<const __half*>(scale);
  a.x = x; a.residual = residual; a.y = y;
  a.T = T; a.K = K; a.N = N; a.ldx = K; a.ldy = N;
  return linear4(a, dtype, group, AFTER_READS, static_cast<cudaStream_t>(stream));
}

extern "C" size_t bm_dense_mlp4_workspace_bytes(int32_t T, int32_t intermediate) {
  if (T <= 0 || intermediate <= 0) return 0;
  // z [T, intermediate], rows of whole 16 bytes, its values that fp16 does not hold, and the per-token gate
  const size_t z = static_cast<size_t>(T) * align_up(intermediate, 8);
  return align_up(z * 2, 256) + align_up(z * 4, 256) + align_up(static_cast<size_t>(T) * 4, 256);
}

extern "C" int bm_dense_mlp4_forward(const void* x, int dtype, const uint32_t* gate_payload, const uint16_t* gate_scale, const uint32_t* up_payload,
                                     const uint16_t* up_scale, const uint32_t* down_payload, const uint16_t* down_scale, const uint16_t* token_gate_w,
                                     int32_t T, int32_t hidden, int32_t intermediate, int32_t group, const void* residual, void* y, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  bm::NvtxRange nvtx_range("bm_dense_mlp4_forward");
  int rc = l4_check("dense_mlp4", dtype, T, group, {hidden, intermediate});
  if (rc) return rc;
  if (T == 0) return BM_OK;
  BM_REQUIRE(x && gate_payload && gate_scale && up_payload && up_scale && down_payload && down_scale && y, BM_ERR_INVALID_ARG, "dense_mlp4: null pointer");
  BM_REQUIRE(aligned16(gate_payload, up_payload, down_payload), BM_ERR_INVALID_ARG, "dense_mlp4: the codes must start on a 16-byte boundary");
  const size_t need = bm_dense_mlp4_workspace_bytes(T, intermediate);
  BM_REQUIRE(workspace && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 255u) == 0, BM_ERR_WORKSPACE,
             "dense_mlp4: workspace must be 256-byte aligned and hold %zu bytes (%zu given)", need, workspace_bytes);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int ldz = static_cast<int>(align_up(intermediate, 8));
  void* z = workspace;
  const size_t nz = static_cast<size_t>(T) * ldz;
  float* wide = reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) + align_up(nz * 2, 256));
  float* gate = reinterpret_cast<float*>(reinterpret_cast<unsigned char*>(wide) + align_up(nz * 4, 256));
  if (dtype != BM_F16) wide = nullptr;
  if (token_gate_w && (rc = launch_row_gate(x, dtype, token_gate_w, BM_F16, T, hidden, gate, AFTER_READS, st, true))) return rc;
  Linear4Args a{};
  a.p[0] = gate_payload; a.p[1] = up_payload;
  a.s[0] = reinterpret_cast<const __half*>(gate_scale); a.s[1] = reinterpret_cast<const __half*>(up_scale);
  a.x = x; a.y = z; a.T = T; a.K = hidden; a.N = intermediate; a.ldx = hidden; a.ldy = ldz; a.glu = 1; a.lead = 1; a.beside = token_gate_w != nullptr;
  a.wide = wide;
  if ((rc = linear4(a, dtype, group, AFTER_READS, st))) return rc;
  Linear4Args d{};
  d.p[0] = down_payload; d.s[0] = reinterpret_cast<const __half*>(down_scale);
  d.x = z; d.residual = residual; d.row_gate = token_gate_w ? gate : nullptr; d.y = y;
  d.T = T; d.K = intermediate; d.N = hidden; d.ldx = ldz; d.ldy = hidden; d.early = 1;
  d.x_wide = wide;
  return linear4(d, dtype, group, AFTER_READS, st);
}
