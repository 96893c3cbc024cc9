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

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// c += A . B, one m16n8k16 MMA, f16 in, f32 sums.  Not volatile: the compiler overlaps it with loads.
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                          uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// c = A . B.
__device__ __forceinline__ void mma_16816_zero(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                               uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

// One word of nibbles -> q - 8 as exact f16 pairs: (values 0, 2), (1, 3), (16, 18), (17, 19) of the
// lane's eight.  0x6400 | n is the f16 1024 + n; a high nibble arrives as 1024 + 16 q.
// (As C expressions, with the masks and 0x6400 as immediates, this compiled to twice the instructions.)
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t mask, uint32_t bits) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(d) : "r"(a), "r"(mask), "r"(bits));
  return d;
}
__device__ __forceinline__ uint32_t hfma2_u32(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ void q4_unpack(uint32_t w, uint32_t (&h)[4]) {
  const uint32_t u = w >> 8;
  h[0] = hsub2_u32(and_or(w, 0x000f000fu, 0x64006400u), 0x64086408u);               // - 1032
  h[1] = hsub2_u32(and_or(u, 0x000f000fu, 0x64006400u), 0x64086408u);
  h[2] = hfma2_u32(and_or(w, 0x00f000f0u, 0x64006400u), 0x2c002c00u, 0xd480d480u);  // / 16 - 72
  h[3] = hfma2_u32(and_or(u, 0x00f000f0u, 0x64006400u), 0x2c002c00u, 0xd480d480u);
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

template <int OFF>
__device__ __forceinline__ uint32_t lds32_at(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1+%2];" : "=r"(v) : "r"(a), "n"(OFF));
  return v;
}
template <int OFF>
__device__ __forceinline__ float lds_scale_at(uint32_t a) {
  uint16_t v;
  asm volatile("ld.shared.b16 %0, [%1+%2];" : "=h"(v) : "r"(a), "n"(OFF));
  return h2f(v);
}
template <int OFF>
__device__ __forceinline__ void lds128_at(uint32_t a, uint32_t (&v)[4]) {
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4+%5];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
               : "r"(a), "n"(OFF));
}

// The pair PAIR of neighbouring blocks (36 bytes) of row g (shared address a) and of row g + 8 (a8),
// times NT groups of 8 rows of x.  at, a8t: the same addresses + 4 t.  Addresses differ by constants
// from pair to pair, so a pair is 66 instructions: 12 loads, 38 to unpack, 4 MMAs, 12 to scale and add.
template <int NT, int PAIR>
__device__ __forceinline__ void q4_pair(uint32_t a, uint32_t a8, uint32_t at, uint32_t a8t,
                                        const uint32_t (&b)[NT][2][4], float (&acc)[NT][4]) {
  constexpr int O = 36 * PAIR;
  uint32_t w0[2], w1[2];  // the lane's word of blocks 0 and 1
  w0[0] = __byte_perm(lds32_at<O>(at), lds32_at<O + 4>(at), 0x5432);
  w1[0] = __byte_perm(lds32_at<O>(a8t), lds32_at<O + 4>(a8t), 0x5432);
  w0[1] = lds32_at<O + 20>(at);
  w1[1] = lds32_at<O + 20>(a8t);
  const float d0[2] = {lds_scale_at<O>(a), lds_scale_at<O + 18>(a)};
  const float d1[2] = {lds_scale_at<O>(a8), lds_scale_at<O + 18>(a8)};
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    uint32_t h0[4], h1[4];
    q4_unpack(w0[j], h0);
    q4_unpack(w1[j], h1);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float c[4];
      mma_16816_zero(c, h0[0], h1[0], h0[1], h1[1], b[n][j][0], b[n][j][1]);
      mma_16816(c, h0[2], h1[2], h0[3], h1[3], b[n][j][2], b[n][j][3]);
      acc[n][0] = __fmaf_rn(d0[j], c[0], acc[n][0]);
      acc[n][1] = __fmaf_rn(d0[j], c[1], acc[n][1]);
      acc[n][2] = __fmaf_rn(d1[j], c[2], acc[n][2]);
      acc[n][3] = __fmaf_rn(d1[j], c[3], acc[n][3]);
    }
  }
}

constexpr int kQ4PartPitch = 20;  // floats between x rows of a warp's partial sums: no bank conflict

// One CTA per 16 weight rows; its 8 warps take the row's pairs of blocks in turn.  Bound by the launch
// and one memory round trip: 2048 x 1024, one row, 2.6 us; 6007 x 1280, three rows, 3.7 us.  The rows arrive
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
    cp_async16(smem_u32(ws) + r * a.pitch + (i - r * chunks) * 16, src + (int64_t)i * 16);
  }
  cp_commit();
  const int npair = a.K / 64;
  const uint32_t wa = smem_u32(ws) + g * a.pitch, wa8 = wa + 8 * a.pitch;
  float acc[NT][4] = {};
  uint32_t b[NT][2][4];
  auto load = [&](int p) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const uint16_t* xr = a.x + (int64_t)min(8 * n + g, a.R - 1) * a.K + 64 * p;
      q4_load_x(xr, t, b[n][0]);
      q4_load_x(xr + 32, t, b[n][1]);
    }
  };
  if (warp < npair) load(warp);
  cp_wait<0>();
  __syncthreads();
  for (int p = warp; p < npair; p += kQ4Warps) {
    if (p != warp) load(p);
    q4_pair<NT, 0>(wa + 36 * p, wa8 + 36 * p, wa + 36 * p + 4 * t, wa8 + 36 * p + 4 * t, b, acc);
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

// Many rows: a persistent CTA an SM.  A group of KW warps streams tiles of 16 rows through a ring of
// its own and splits their K between them; the first warp adds the others' sums to its own in order.
// No barrier between groups after x is laid out in shared memory, in the order of the B fragments
// ([block][8 NT rows][t], 16 bytes each; rows behind R stay unset, their columns are not stored).
//
// A bulk copy takes the SM's copy engine about 30 cycles whatever its size (151936 x 1024 in copies of
// 288 bytes: 37 us, of 1152: 25), so a copy is as many rows as keep the fragment loads free of bank
// conflicts: rows are 36 K/256 words apart, so 8 / gcd(8, K/256) neighbouring rows fall into different
// banks, and 16 bytes between the copies shift the next ones.  151936 x 1024, 8 rows: 24.4 us, 3.6
// TB/s (16 rows 35); the copies alone take 18, the arithmetic alone 19.
constexpr int kQ4StreamSplit = 2;       // KW
constexpr int kQ4StreamMaxGroups = 10;
constexpr int kQ4StreamStages = 2;

struct Q4StreamArgs {
  Q4GemvArgs g;
  int copy_rows;  // rows a copy: 1, 2, 4 or 16
  int stage;      // bytes of a tile in shared memory
  int ntiles;
};

// x fragments of two pairs of blocks.
template <int NT>
__device__ __forceinline__ void lds_x(uint32_t xb, uint32_t (&b)[2][NT][2][4]) {
  lds128_at<0>(xb, b[0][0][0]);
  lds128_at<512 * NT>(xb, b[0][0][1]);
  lds128_at<1024 * NT>(xb, b[1][0][0]);
  lds128_at<1536 * NT>(xb, b[1][0][1]);
  if (NT == 2) {
    lds128_at<512>(xb, b[0][NT - 1][0]);
    lds128_at<512 * NT + 512>(xb, b[0][NT - 1][1]);
    lds128_at<1024 * NT + 512>(xb, b[1][NT - 1][0]);
    lds128_at<1536 * NT + 512>(xb, b[1][NT - 1][1]);
  }
}

__device__ __forceinline__ void bulk_g2s_plain(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

template <int NT>
__global__ void __launch_bounds__(kQ4StreamMaxGroups * kQ4StreamSplit * 32, 1) k_gemv_q4_stream(const Q4StreamArgs s) {
  constexpr int KW = kQ4StreamSplit;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t full[kQ4StreamMaxGroups][kQ4StreamStages];
  __shared__ __align__(8) uint64_t done[kQ4StreamMaxGroups][kQ4StreamStages];
  const Q4GemvArgs& a = s.g;
  const int groups = blockDim.x / (32 * KW), grp = threadIdx.x / (32 * KW), part = (threadIdx.x >> 5) % KW;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + grp * kQ4StreamStages * s.stage;
  const uint32_t rg = smem_u32(ring);
  // sums of the group's other warps, per stage: [stage][KW - 1][4 NT][32]
  float* sums = reinterpret_cast<float*>(smem + groups * kQ4StreamStages * s.stage) + grp * kQ4StreamStages * (KW - 1) * NT * 128;
  uint4* xs = reinterpret_cast<uint4*>(smem + groups * kQ4StreamStages * (s.stage + (KW - 1) * NT * 512));
  const int rb = a.K / 32 * kQ4Bytes, ub = s.copy_rows * rb;  // bytes of a row, of a copy
  // this CTA's tiles, dealt to its groups in turn
  const int t0 = (int)((int64_t)s.ntiles * blockIdx.x / gridDim.x) + grp;
  const int t1 = (int)((int64_t)s.ntiles * (blockIdx.x + 1) / gridDim.x);
  auto issue = [&](int tile, int st) {  // by the first warp
    const int rows = min(16, a.N - tile * 16), r = lane * s.copy_rows;
    uint64_t* bar = &full[grp][st];
    if (lane == 0) mbar_expect_tx(bar, rows * rb);
    __syncwarp();
    if (r < rows)
      bulk_g2s_plain(rg + st * s.stage + lane * (ub + 16), a.w + (int64_t)(tile * 16 + r) * rb,
                     min(s.copy_rows, rows - r) * rb, bar);
  };
  if (part == 0) {
    if (lane == 0) {
      for (int i = 0; i < kQ4StreamStages; ++i) mbar_init(&full[grp][i], 1), mbar_init(&done[grp][i], KW - 1);
      fence_mbar_init();
    }
    __syncwarp();
    for (int i = 0; i < kQ4StreamStages; ++i)
      if (t0 + i * groups < t1) issue(t0 + i * groups, i);
  }
  const int frags = a.K / 32 * a.R * 4;
  for (int i = threadIdx.x; i < frags; i += blockDim.x) {
    const int blk = i / (4 * a.R), n = i / 4 - blk * a.R;
    uint32_t b[4];
    q4_load_x(a.x + (int64_t)n * a.K + blk * 32, i & 3, b);
    xs[(blk * 8 * NT + n) * 4 + (i & 3)] = make_uint4(b[0], b[1], b[2], b[3]);
  }
  __syncthreads();
  const int g8 = g + 8, lg = __ffs(s.copy_rows) - 1;
  const int at = (g >> lg) * (ub + 16) + (g & (s.copy_rows - 1)) * rb;
  const int at8 = (g8 >> lg) * (ub + 16) + (g8 & (s.copy_rows - 1)) * rb;
  const int np = a.K / 64 / KW, p0 = part * np;  // even: K is a multiple of 256
  int st = 0, tile = t0;
  uint32_t ph = 0;
  bool ok = true;
  for (; tile < t1; tile += groups) {
    ok = mbar_wait_own(&full[grp][st], ph, nullptr, kErrTimeoutFull);
    if (!__all_sync(0xffffffffu, ok)) break;
    uint32_t w0 = rg + st * s.stage + at + 36 * p0, w1 = rg + st * s.stage + at8 + 36 * p0;
    uint32_t xb = smem_u32(xs) + lane * 16 + p0 * (NT * 1024);
    float acc[NT][4] = {};
    for (int p = 0; p < np; p += 2) {
      uint32_t b[2][NT][2][4];
      lds_x<NT>(xb, b);
      q4_pair<NT, 0>(w0, w1, w0 + 4 * t, w1 + 4 * t, b[0], acc);
      q4_pair<NT, 1>(w0, w1, w0 + 4 * t, w1 + 4 * t, b[1], acc);
      w0 += 72, w1 += 72, xb += NT * 2048;
    }
    // the other warps run on, up to a ring ahead: their sums go to a place per stage, and they reach
    // the same stage again only after a copy that the first warp has begun after reading them
    float* at_sums = sums + st * (KW - 1) * NT * 128 + lane;
    if (part) {
#pragma unroll
      for (int i = 0; i < 4 * NT; ++i) at_sums[((part - 1) * 4 * NT + i) * 32] = acc[i >> 2][i & 3];
      __syncwarp();
      if (lane == 0) mbar_arrive(&done[grp][st]);
    } else {
      ok = mbar_wait_own(&done[grp][st], ph, nullptr, kErrTimeoutFull);
      if (!__all_sync(0xffffffffu, ok)) break;
#pragma unroll
      for (int k = 0; k < KW - 1; ++k)
#pragma unroll
        for (int i = 0; i < 4 * NT; ++i)
          acc[i >> 2][i & 3] = __fadd_rn(acc[i >> 2][i & 3], at_sums[(k * 4 * NT + i) * 32]);
      __syncwarp();  // all are done with the stage and the sums have been read
      if (tile + kQ4StreamStages * groups < t1) issue(tile + kQ4StreamStages * groups, st);
      const int row = tile * 16 + g;
#pragma unroll
      for (int i = 0; i < 4 * NT; ++i) {
        const int r = 8 * (i >> 2) + 2 * t + (i & 1), w = row + 4 * (i & 2);
        if (r < a.R && w < a.N) a.y[(int64_t)r * a.N + w] = f2h(acc[i >> 2][i & 3]);
      }
    }
    if (++st == kQ4StreamStages) st = 0, ph ^= 1;
  }
  // a wait gave up: there is no error word here, so the rows without a sum become NaN
  if (part == 0 && tile < t1) {
    for (int i = 0; i < kQ4StreamStages && tile + i * groups < t1; ++i) {  // copies under way land first
      mbar_wait_own(&full[grp][st], ph, nullptr, kErrTimeoutFull);
      if (++st == kQ4StreamStages) st = 0, ph ^= 1;
    }
    for (; tile < t1; tile += groups)
      for (int i = lane; i < 16 * a.R; i += 32) {
        const int w = tile * 16 + (i & 15);
        if (w < a.N) a.y[(int64_t)(i >> 4) * a.N + w] = 0x7fff;
      }
  }
}

}  // namespace q3
