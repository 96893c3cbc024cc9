// q3_q4.cuh -- Q4_0 GEMV for sm_100a: y[r][n] = sum_k w[n][k] x[r][k], a few rows of x.
//
// Weights are 18-byte Q4_0 blocks of 32 values in [N][K/32] order, as a GGUF file holds them: an f16
// scale d, then 16 bytes; byte j holds value j in its low nibble and value j + 16 in its high one, and
// a value is w = d * (q - 8).  Weights are read once and dominate: 0.5625 bytes each, 2 R flops.
//
// The dot products run on the tensor pipe (m16n8k16: 16 weight rows, up to 8 rows of x, f32 sums),
// because unpacking already takes most of the issue slots: per block of 32 and row, f32 FMAs would
// add 32 R / 32 lanes, the MMA adds 2 / 16.  q - 8 is an exact f16, so the products are exact; a
// block's sum is scaled by d in f32, in this order: within a block the MMA's, then a warp's blocks in
// order, then the warps.  One rounding to f16 at the end.
//
// MMA operands need no shuffle.  A lane (g = lane / 4, t = lane % 4) reads the 4 bytes 4t..4t+3 of a
// block of rows g and g + 8.  Low nibbles are values 4t..4t+3, high nibbles 16+4t..16+4t+3: one MMA
// takes the low ones as its 16 k, one the high ones, and x is read in that same order.
#pragma once

#include "q3_common.cuh"

namespace q3 {

constexpr int kQ4Bytes = 18;
constexpr int kQ4MaxK = 16384;
constexpr int kQ4MaxRows = 16;
constexpr int kQ4Warps = 8;

struct Q4GemvArgs {
  const uint8_t* w;
  const uint16_t* x;  // [R][K]
  uint16_t* y;        // [R][N]
  int N, K, R;
  int pitch;          // bytes between weight rows in shared memory
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool take) {
  const int n = take ? 16 : 0;  // 0: the 16 bytes are filled with zeros, src is not read
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n)
               : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// c += A . B, one m16n8k16 MMA, f16 in, f32 sums.
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                          uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// One word of nibbles -> q - 8 as exact f16 pairs: (values 0, 2), (1, 3), (16, 18), (17, 19) of the
// lane's eight.  0x6400 | n is the f16 1024 + n; a high nibble arrives as 1024 + 16 q.
__device__ __forceinline__ void q4_unpack(uint32_t w, uint32_t (&h)[4]) {
  const uint32_t u = w >> 8;
  const __half2 k1032 = __half2half2(__ushort_as_half(0x6408));
  const __half2 k16th = __half2half2(__ushort_as_half(0x2c00));
  const __half2 km72 = __half2half2(__ushort_as_half(0xd480));
  const uint32_t l0 = (w & 0x000f000fu) | 0x64006400u, l1 = (u & 0x000f000fu) | 0x64006400u;
  const uint32_t h0 = (w & 0x00f000f0u) | 0x64006400u, h1 = (u & 0x00f000f0u) | 0x64006400u;
  __half2 r[4] = {__hsub2(*(const __half2*)&l0, k1032), __hsub2(*(const __half2*)&l1, k1032),
                  __hfma2(*(const __half2*)&h0, k16th, km72),
                  __hfma2(*(const __half2*)&h1, k16th, km72)};
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = *(uint32_t*)&r[i];
}

// x values of one block for the MMAs: (4t, 4t+2), (4t+1, 4t+3) and the same 16 higher.
__device__ __forceinline__ void q4_load_x(const uint16_t* xb, int t, uint32_t (&b)[4]) {
  const uint2 lo = __ldg(reinterpret_cast<const uint2*>(xb + 4 * t));
  const uint2 hi = __ldg(reinterpret_cast<const uint2*>(xb + 16 + 4 * t));
  b[0] = __byte_perm(lo.x, lo.y, 0x5410);
  b[1] = __byte_perm(lo.x, lo.y, 0x7632);
  b[2] = __byte_perm(hi.x, hi.y, 0x5410);
  b[3] = __byte_perm(hi.x, hi.y, 0x7632);
}

// Two neighbouring blocks (36 bytes at shared address `a` of row g, `a8` of row g + 8) times NT
// groups of 8 rows of x.
template <int NT>
__device__ __forceinline__ void q4_pair(uint32_t a, uint32_t a8, int t, const uint32_t (&b)[NT][2][4],
                                        float (&acc)[NT][4]) {
  uint32_t w0[2], w1[2];  // the lane's word of blocks 0 and 1
  w0[0] = __byte_perm(lds32(a + 4 * t), lds32(a + 4 * t + 4), 0x5432);
  w1[0] = __byte_perm(lds32(a8 + 4 * t), lds32(a8 + 4 * t + 4), 0x5432);
  w0[1] = lds32(a + 4 * t + 20);
  w1[1] = lds32(a8 + 4 * t + 20);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const float d0 = h2f(lds16(a + 18 * j)), d1 = h2f(lds16(a8 + 18 * j));
    uint32_t h0[4], h1[4];
    q4_unpack(w0[j], h0);
    q4_unpack(w1[j], h1);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      mma_16816(c, h0[0], h1[0], h0[1], h1[1], b[n][j][0], b[n][j][1]);
      mma_16816(c, h0[2], h1[2], h0[3], h1[3], b[n][j][2], b[n][j][3]);
      acc[n][0] = __fmaf_rn(d0, c[0], acc[n][0]);
      acc[n][1] = __fmaf_rn(d0, c[1], acc[n][1]);
      acc[n][2] = __fmaf_rn(d1, c[2], acc[n][2]);
      acc[n][3] = __fmaf_rn(d1, c[3], acc[n][3]);
    }
  }
}

constexpr int kQ4PartPitch = 20;  // floats between x rows of a warp's partial sums: no bank conflict

// One CTA per 16 weight rows; its 8 warps take the row's pairs of blocks in turn.  The rows arrive
// by cp.async while the warps load their x.
template <int NT>
__global__ void __launch_bounds__(kQ4Warps * 32) k_gemv_q4(const Q4GemvArgs a) {
  extern __shared__ __align__(128) uint8_t smem[];
  float* part = reinterpret_cast<float*>(smem);  // [warp][8 NT][pitch]
  uint8_t* ws = smem + sizeof(float) * kQ4Warps * 8 * NT * kQ4PartPitch;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int row0 = blockIdx.x * 16;
  const int nrow = min(16, a.N - row0);
  const int rb = a.K / 32 * kQ4Bytes, chunks = rb / 16;
  const uint8_t* src = a.w + (int64_t)row0 * rb;
  for (int i = threadIdx.x; i < nrow * chunks; i += blockDim.x) {
    const int r = i / chunks;
    cp_async16(smem_u32(ws) + r * a.pitch + (i - r * chunks) * 16, src + (int64_t)i * 16, true);
  }
  cp_commit();
  const int npair = a.K / 64;
  const uint32_t wa = smem_u32(ws) + g * a.pitch, wa8 = wa + 8 * a.pitch;
  float acc[NT][4] = {};
  uint32_t b[NT][2][4] = {};
  auto load = [&](int p) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
      if (8 * n + g < a.R) {
        const uint16_t* xr = a.x + (int64_t)(8 * n + g) * a.K + 64 * p;
        q4_load_x(xr, t, b[n][0]);
        q4_load_x(xr + 32, t, b[n][1]);
      }
  };
  if (warp < npair) load(warp);
  cp_wait<0>();
  __syncthreads();
  for (int p = warp; p < npair; p += kQ4Warps) {
    if (p != warp) load(p);
    q4_pair<NT>(wa + 36 * p, wa8 + 36 * p, t, b, acc);
  }
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      part[(warp * 8 * NT + 8 * n + 2 * t + (e & 1)) * kQ4PartPitch + g + 8 * (e >> 1)] = acc[n][e];
  __syncthreads();
  const int r = threadIdx.x >> 4, n = threadIdx.x & 15;
  if (r < a.R && n < nrow) {
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < kQ4Warps; ++k) s = __fadd_rn(s, part[(k * 8 * NT + r) * kQ4PartPitch + n]);
    a.y[(int64_t)r * a.N + row0 + n] = f2h(s);
  }
}

}  // namespace q3
