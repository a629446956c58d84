// Products with 4-bit weights (linear4.cu, linear4_tc.cu).
#pragma once

#include "grouped.cuh"

namespace bm {

struct Linear4Args {
  const uint32_t* p[2];        // codes [N, words]; GLU: gate and up
  const __half* s[2];          // scales [N, groups]
  const void* x;               // [T, ldx]
  const void* residual;        // [T, N] of y's type, or null
  const float* row_gate;       // factor per token, or null
  void* y;                     // [T, ldy]
  float* wide;                 // GLU with fp16 y: [T, ldy], gets the values that fp16 does not hold (their y is infinite); or null
  const float* x_wide;         // [T, ldx], such values of x; or null
  int T, K, N, ldx, ldy, words, groups, group;
  int glu, vec_x, kwarps, splits, row_blocks;
  // early: fetches weights before it waits.  Everything that may have written them has to be over when it starts, so the launch before is a `lead` one.
  // lead: lets the next launch start once what came before itself is over, not as soon as it runs.  beside: does not wait before its end,
  // since the launch before is a lead one that wrote nothing that this one reads.
  int early, lead, beside;
};

// Eight codes -> four pairs (code i, code i + 4), i = 0 .. 3, as exact numbers -8 .. 7 of the type.
template <int XD>
__device__ __forceinline__ void codes_to_pairs(uint32_t w, uint32_t (&q)[4]) {
  if (XD == BM_F16) {
    // 1024 + u and 1024 + 16 u are fp16 numbers with u in their low mantissa bits
    const __half2 off = __float2half2_rn(1032.f), sixteenth = __float2half2_rn(0.0625f), minus72 = __float2half2_rn(-72.f);
#pragma unroll
    for (int h = 0; h < 2; ++h, w >>= 8) {
      const uint32_t lo = (w & 0x000F000Fu) | 0x64006400u, hi = (w & 0x00F000F0u) | 0x64006400u;
      const __half2 a = __hsub2(*reinterpret_cast<const __half2*>(&lo), off), b = __hfma2(*reinterpret_cast<const __half2*>(&hi), sixteenth, minus72);
      q[2 * h] = *reinterpret_cast<const uint32_t*>(&a);
      q[2 * h + 1] = *reinterpret_cast<const uint32_t*>(&b);
    }
  } else {
    const __nv_bfloat162 off = __float2bfloat162_rn(136.f);       // 128 + u
#pragma unroll
    for (int i = 0; i < 4; ++i, w >>= 4) {
      const uint32_t v = (w & 0x000F000Fu) | 0x43004300u;
      const __nv_bfloat162 a = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), off);
      q[i] = *reinterpret_cast<const uint32_t*>(&a);
    }
  }
}

template <int XD>
__device__ __forceinline__ float load_x(const void* p, int64_t i) {
  return XD == BM_F16 ? __half2float(static_cast<const __half*>(p)[i]) : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
template <int XD>
__device__ __forceinline__ void store_x(void* p, int64_t i, float v) {
  if (XD == BM_F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}
// x is the product between the two matrices of an MLP, which may pass fp16's range although the sums over it do not: x is infinite there, and with it
// every sum of that token.  Sums that are not finite are left out by linear4_finish, and the CTA works them out here, once it is
// through with everything else, from x's values before their rounding: a warp a sum.  One such token of five
// behind 2816 columns 12.4 -> 27 us, one of 300 behind 512 44 -> 72, all 300 1400.
static __device__ __noinline__ void linear4_redo(const Linear4Args& a, int row0, int rows, int tok0, int toks) {      // toks <= 128
  __shared__ unsigned odd[4], odd_scale;      // tokens with values that are not finite; any such scale
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const float inf = __int_as_float(0x7f800000);
  __syncthreads();
  if (threadIdx.x < 4) odd[threadIdx.x] = 0;
  if (threadIdx.x == 4) odd_scale = 0;
  __syncthreads();
  for (int t = warp; t < toks; t += warps) {
    const __half* x = static_cast<const __half*>(a.x) + static_cast<int64_t>(tok0 + t) * a.ldx;
    bool any = false;
    for (int k = lane; k < a.K; k += 32) any |= !(fabsf(__half2float(x[k])) < inf);
    if (__any_sync(0xffffffffu, any) && lane == 0) atomicOr(&odd[t >> 5], 1u << (t & 31));
  }
  for (int r = warp; r < rows && row0 + r < a.N; r += warps)
    for (int g = lane; g < a.groups; g += 32)
      if (!(fabsf(__half2float(a.s[0][static_cast<int64_t>(row0 + r) * a.groups + g])) < inf)) odd_scale = 1;
  __syncthreads();
  for (int t = 0; t < toks; ++t) {
    const bool of_x = odd[t >> 5] >> (t & 31) & 1u;
    if (!of_x && !odd_scale) continue;
    const int64_t token = tok0 + t;
    const __half* x = static_cast<const __half*>(a.x) + token * a.ldx;
    const float* wide = a.x_wide + token * a.ldx;
    for (int r = warp; r < rows && row0 + r < a.N; r += warps) {
      const int64_t row = row0 + r;
      const uint32_t* codes = a.p[0] + row * a.words;
      float sum = 0.f;
#pragma unroll 2
      for (int w = lane; 8 * w < a.K; w += 32) {
        const uint32_t code = codes[w];
        float part = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int k = 8 * w + j;
          float v = k < a.K ? __half2float(x[k]) : 0.f;
          if (!(fabsf(v) < inf)) v = wide[k];
          part = fmaf(v, static_cast<float>(static_cast<int>(code >> (4 * j) & 15u) - 8), part);
        }
        sum = fmaf(part, __half2float(a.s[0][row * a.groups + 8 * w / a.group]), sum);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      // with x finite a sum is not where a scale is not, here as there
      if (lane == 0 && (of_x || !(fabsf(sum) < inf))) {
        const float f = a.row_gate ? a.row_gate[token] : 1.f, res = a.residual ? load_x<BM_F16>(a.residual, token * a.N + row) : 0.f;
        store_x<BM_F16>(a.y, token * a.ldy + row, fmaf(sum, f, res));
      }
    }
  }
}
// Finished sums of one row and up to C tokens: times the tokens' gates, plus the residual, out.  All loads are in flight before the
// first store (one by one a product of 300 tokens, 512 x 2048, with a residual took 22 us instead of 17).
template <int XD, bool WIDE, int C, typename Token>      // WIDE: a.wide and a.x_wide are looked at
__device__ __forceinline__ void linear4_finish(const Linear4Args& a, int row, const float (&v)[C], int& left_out, Token token) {      // token(i) < 0: none
  float f[C], r[C];
#pragma unroll
  for (int i = 0; i < C; ++i) {
    f[i] = 1.f;
    r[i] = 0.f;
  }
  if (a.row_gate)
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (token(i) >= 0) f[i] = __ldg(a.row_gate + token(i));
  if (a.residual)
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (token(i) >= 0) r[i] = load_x<XD>(a.residual, static_cast<int64_t>(token(i)) * a.N + row);
#pragma unroll
  for (int i = 0; i < C; ++i)
    if (token(i) >= 0) {
      if (WIDE && a.x_wide && !(fabsf(v[i]) < __int_as_float(0x7f800000))) {
        left_out = 1;
        continue;
      }
      const int64_t o = static_cast<int64_t>(token(i)) * a.ldy + row;
      store_x<XD>(a.y, o, fmaf(v[i], f[i], r[i]));
      if (WIDE && a.wide && !fits_fp16(v[i])) a.wide[o] = v[i];
    }
}

// BM_ERR_UNSUPPORTED, with nothing launched, when a shape or pointer does not suit tiled copies.
double linear4_tc_us(const Linear4Args& a, int sms);       // its time, roughly
int launch_linear4_tc(const Linear4Args& a, int x_dtype, int group, LaunchAfter after, cudaStream_t st);

}  // namespace bm
