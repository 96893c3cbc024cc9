// q3_tree.cuh -- attention of several drafted tokens (a tree) over a KV cache, the single-token form
// that also accumulates every slot's attention weight, and the move of an accepted path.
//
// For sequence b with m cached slots, drafted token i (parent p_i < i, or -1: the last cached token)
// has depth = its number of ancestors and sits at RoPE position pos + depth.  With q, k after
// QK-RMSNorm and RoPE (each rounded to f16, the bits the one-token engines put into the cache):
//   out_i = sum_j softmax_j(q_i . k_j / sqrt(128)) v_j,   j over slots 0..m-1, i's ancestors and i.
// The new K/V rows go to slots m + i.
//
// What it has to move is 512 bytes per (slot, kv head), once, for all 2 T query rows of that head, so
// the work is split over the keys: a thread-block cluster of up to 16 CTAs owns a (sequence, kv head)
// and each CTA a contiguous run of 64-key tiles, streamed by cp.async into a ring.  The softmax runs
// online in registers; the CTAs' partial (max, sum, output) meet over distributed shared memory, so
// there is no workspace, no counter and no second launch.
#pragma once

#include "q3_attn.cuh"
#include "q3_common.cuh"
#include "q3_q4.cuh"

namespace q3 {

constexpr int kTreeMaxTokens = 64;
constexpr int kTreeThreads = 128;
constexpr int kTreeTile = 64;                       // keys per ring stage
constexpr int kTreeStages = 3;
constexpr int kTreeStageBytes = 2 * kTreeTile * kHD * 2;  // K then V
constexpr int kTreeOPitch = kHD + 4;                // floats between partial output rows

struct TreeArgs {
  const uint16_t* qkv;  // [B][T][(q_heads + 2 kv_heads) * 128]
  const uint16_t* q_norm;
  const uint16_t* k_norm;
  const float* rope_cos;  // [rope_rows][64]
  const float* rope_sin;
  int64_t rope_rows;
  uint16_t* k;  // the layer's cache of sequence 0
  uint16_t* v;
  int64_t seq_stride, slot_stride, head_stride;
  int64_t S;
  int T, q_heads, kv_heads, group_log2;
  const int32_t* parents;   // [B][T]
  const int32_t* n_tokens;  // [B], or null: T each
  const int64_t* len;       // [B] cached slots
  const int64_t* pos;       // [B] RoPE position of a token of depth 0
  uint16_t* out;            // [B][T][q_heads * 128]
  int* err;
  const float* w_in;  // scored form: [B][..][kv_heads][S] of this layer
  float* w_out;
  int32_t* slot_pos;
  int64_t w_stride;  // elements between sequences of w_in, w_out, slot_pos
  int score_cap;     // keys a CTA can hold scores for
};

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *(const uint32_t*)&h;
}
__device__ __forceinline__ float4 ld_dsmem_f4(uint32_t local_addr, uint32_t rank) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(dsmem_map(local_addr, rank))
               : "memory");
  return v;
}

// Byte offset of 16-byte chunk c of row r in a tile of 256-byte rows: the low three chunk bits are
// xored with the row, so that the 8 rows of an ldmatrix fall into different banks.
__device__ __forceinline__ uint32_t tile_at(int r, int c) { return r * 256 + ((c ^ (r & 7)) << 4); }

// One head vector through RMSNorm and RoPE by a warp into row `row` of a swizzled tile; returns this
// lane's values (dims lane + 32 i).  The operations and roundings of norm_rope_vals.
__device__ __forceinline__ void norm_rope_row(const float (&v)[4], const uint16_t (&gv)[4], float c0,
                                              float s0, float c1, float s1, int lane, uint8_t* tile,
                                              int row, uint16_t (&o)[4]) {
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) ss = __fmaf_rn(v[i], v[i], ss);
  ss = warp_sum(ss);
  const float r = __fsqrt_rn(__fadd_rn(__fdiv_rn(ss, 128.0f), kEps));
  float n[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) n[i] = h2f(f2h(__fmul_rn(__fdiv_rn(v[i], r), h2f(gv[i]))));
  o[0] = f2h(__fsub_rn(__fmul_rn(n[0], c0), __fmul_rn(n[2], s0)));
  o[2] = f2h(__fadd_rn(__fmul_rn(n[0], s0), __fmul_rn(n[2], c0)));
  o[1] = f2h(__fsub_rn(__fmul_rn(n[1], c1), __fmul_rn(n[3], s1)));
  o[3] = f2h(__fadd_rn(__fmul_rn(n[1], s1), __fmul_rn(n[3], c1)));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = lane + 32 * i;
    *reinterpret_cast<uint16_t*>(tile + tile_at(row, d >> 3) + (d & 7) * 2) = o[i];
  }
}

// Rows of q: r = token * group + j.  A warp owns MT * 16 of them and 64 / WK keys of a tile; WR warps
// cover the rows, WK the keys (WR * WK = 4).
template <int MT, int WR, int WK, bool SCORED>
__global__ void __launch_bounds__(kTreeThreads, MT * WR * 16 <= 64 ? 2 : 1) k_tree_attn(const TreeArgs a) {
  constexpr int RP = MT * WR * 16;       // rows, padded
  constexpr int KW = kTreeTile / WK;     // keys of a tile per warp
  constexpr int KS = KW < 32 ? KW : 32;  // keys per softmax step
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* qs = smem;                                   // [RP][128] f16
  uint8_t* ring = qs + RP * 256;                        // kTreeStages stages; then the partial outputs
  float2* mlw = reinterpret_cast<float2*>(ring + kTreeStages * kTreeStageBytes);  // [WK][RP]
  float2* ml = mlw + WK * RP;                           // [RP] this CTA's (max, sum)
  unsigned long long* anc = reinterpret_cast<unsigned long long*>(ml + RP);  // [64] ancestors and self
  int* up = reinterpret_cast<int*>(anc + kTreeMaxTokens);                    // [64]
  float* score = reinterpret_cast<float*>(up + kTreeMaxTokens);              // [group][score_cap]
  float* op = reinterpret_cast<float*>(ring);           // [WK][RP][kTreeOPitch]

  const int C = gridDim.x, rank = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int wr = warp / WK, wk = warp % WK;
  const int gl = a.group_log2, G = 1 << gl;

  const int n = SCORED ? 1 : (a.n_tokens ? a.n_tokens[b] : a.T);
  const int64_t len = a.len[b], pos = a.pos[b];
  // every CTA of the cluster sees the same values and leaves together
  if (SCORED ? len == -1 : n == 0) return;
  bool bad = n < 0 || n > a.T || len < 0 || len > a.S - n || pos < 0 || pos >= a.rope_rows;
  if (bad) {
    if (tid == 0 && a.err) atomicCAS(a.err, 0, kErrBadPos);
    return;
  }
  const int R = n << gl;
  const int nct = (int)((len + kTreeTile - 1) / kTreeTile), nt = nct + 1;  // the last tile: the new tokens
  const int lo = (int)((int64_t)rank * nt / C), hi = (int)((int64_t)(rank + 1) * nt / C);
  uint16_t* kb = a.k + b * a.seq_stride + h * a.head_stride;
  uint16_t* vb = a.v + b * a.seq_stride + h * a.head_stride;

  // cached tiles stream while the queries are prepared
  auto issue_cached = [&](int i) {
    const int64_t base = (int64_t)i * kTreeTile;
    const int r0 = tid >> 4, c = tid & 15;
    const uint32_t dst = smem_u32(ring) + ((i - lo) % kTreeStages) * kTreeStageBytes + tile_at(r0, c);
    const uint16_t* ks = kb + (base + r0) * a.slot_stride + c * 8;
    const uint16_t* vs = vb + (base + r0) * a.slot_stride + c * 8;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const bool in = base + r0 + 8 * k < len;
      cp_async16(dst + k * 2048, in ? ks : kb, in);
      ks += 8 * a.slot_stride;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const bool in = base + r0 + 8 * k < len;
      cp_async16(dst + kTreeStageBytes / 2 + k * 2048, in ? vs : vb, in);
      vs += 8 * a.slot_stride;
    }
  };
#pragma unroll
  for (int i = 0; i < kTreeStages - 1; ++i) {
    if (lo + i < hi && lo + i < nct) issue_cached(lo + i);
    cp_commit();
  }

  // ancestors by doubling: after step k a token knows 2^k of them
  if (!SCORED) {
    bool ok = true;
    if (tid < n) {
      const int p = a.parents[(int64_t)b * a.T + tid];
      ok = p >= -1 && p < tid;
      up[tid] = ok ? p : -1;
      anc[tid] = 1ull << tid;
    }
    if (__syncthreads_or(!ok)) {
      if (tid == 0 && a.err) atomicCAS(a.err, 0, kErrBadTree);
      cp_wait<0>();
      return;
    }
    for (int s = 1; s < n; s <<= 1) {
      unsigned long long m = 0;
      int u = -1;
      if (tid < n && up[tid] >= 0) m = anc[up[tid]], u = up[up[tid]];
      __syncthreads();
      if (tid < n) anc[tid] |= m, up[tid] = u;
      __syncthreads();
    }
    const bool far = tid < n && pos + __popcll(anc[tid]) - 1 >= a.rope_rows;
    if (__syncthreads_or(far)) {
      if (tid == 0 && a.err) atomicCAS(a.err, 0, kErrBadPos);
      cp_wait<0>();
      return;
    }
  }
  const int row_el = (a.q_heads + 2 * a.kv_heads) * kHD;
  const uint16_t* qkv = a.qkv + (int64_t)b * a.T * row_el;
  auto rope_at = [&](int tok, float& c0, float& s0, float& c1, float& s1) {
    const int64_t p = (pos + (SCORED ? 0 : __popcll(anc[tok]) - 1)) * 64;
    c0 = a.rope_cos[p + lane], c1 = a.rope_cos[p + lane + 32];
    s0 = a.rope_sin[p + lane], s1 = a.rope_sin[p + lane + 32];
  };
  {
    uint16_t gq[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) gq[i] = a.q_norm[lane + 32 * i];
#pragma unroll 2
    for (int r = warp; r < RP; r += 4) {
      if (r < R) {
        const int tok = r >> gl;
        const uint16_t* x = qkv + (int64_t)tok * row_el + ((h << gl) + (r & (G - 1))) * kHD;
        float v[4], c0, s0, c1, s1;
        uint16_t o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = h2f(x[lane + 32 * i]);
        rope_at(tok, c0, s0, c1, s1);
        norm_rope_row(v, gq, c0, s0, c1, s1, lane, qs, r, o);
      } else {
        *reinterpret_cast<uint2*>(qs + r * 256 + lane * 8) = make_uint2(0u, 0u);
      }
    }
  }
  // the new tokens' tile: K rows normed and roped, V rows as they are, both also into the cache
  auto issue_new = [&](int i) {
    uint8_t* st = ring + ((i - lo) % kTreeStages) * kTreeStageBytes;
    uint16_t gk[4];
#pragma unroll
    for (int i2 = 0; i2 < 4; ++i2) gk[i2] = a.k_norm[lane + 32 * i2];
    const int np = (n + 31) & ~31;  // a step of up to 32 keys reads no further
    for (int r = warp; r < np; r += 4) {
      uint2* vd = reinterpret_cast<uint2*>(st + kTreeStageBytes / 2 + tile_at(r, lane >> 1) + (lane & 1) * 8);
      if (r < n) {
        const uint16_t* x = qkv + (int64_t)r * row_el + (a.q_heads + h) * kHD;
        float v[4], c0, s0, c1, s1;
        uint16_t o[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = h2f(x[lane + 32 * k]);
        const uint2 vv = *reinterpret_cast<const uint2*>(x + a.kv_heads * kHD + lane * 4);
        rope_at(r, c0, s0, c1, s1);
        norm_rope_row(v, gk, c0, s0, c1, s1, lane, st, r, o);
        uint16_t* kd = kb + (len + r) * a.slot_stride;
#pragma unroll
        for (int k = 0; k < 4; ++k) kd[lane + 32 * k] = o[k];
        *vd = vv;
        *reinterpret_cast<uint2*>(vb + (len + r) * a.slot_stride + lane * 4) = vv;
      } else {
        *reinterpret_cast<uint2*>(st + r * 256 + lane * 8) = make_uint2(0u, 0u);
        *vd = make_uint2(0u, 0u);
      }
    }
  };
#pragma unroll
  for (int i = 0; i < kTreeStages - 1; ++i)
    if (lo + i < hi && lo + i == nct) issue_new(nct);

  constexpr float kC = kAttnScale * 1.44269504088896341f;  // scores in powers of two
  float o[MT][16][4] = {}, m[MT][2], l[MT][2] = {};
#pragma unroll
  for (int i = 0; i < MT; ++i) m[i][0] = m[i][1] = -INFINITY;
  uint32_t qf[8][4];
  const int qrow = wr * MT * 16 + (lane & 7) + ((lane >> 3) & 1) * 8;
  if (MT == 1) {
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) ldsm4(qf[kk], smem_u32(qs) + tile_at(qrow, 2 * kk + (lane >> 4)));
  }

  for (int it = lo; it < hi; ++it) {
    cp_wait<kTreeStages - 2>();
    __syncthreads();
    const int ahead = it + kTreeStages - 1;
    if (ahead < hi) {
      if (ahead < nct) issue_cached(ahead);
      else issue_new(nct);
    }
    cp_commit();
    const uint32_t st = smem_u32(ring) + ((it - lo) % kTreeStages) * kTreeStageBytes;
    const bool fresh = it == nct;
    const int nv = fresh ? n : (int)(len - (int64_t)it * kTreeTile < kTreeTile ? len - (int64_t)it * kTreeTile : kTreeTile);
#pragma unroll 1
    for (int k0 = wk * KW; k0 < wk * KW + KW && k0 < nv; k0 += KS) {
      float s[MT][KS / 8][4] = {};
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) {
        uint32_t af[MT][4];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          if (MT == 1) {
#pragma unroll
            for (int e = 0; e < 4; ++e) af[i][e] = qf[kk][e];
          } else {
            ldsm4(af[i], smem_u32(qs) + tile_at(qrow + 16 * i, 2 * kk + (lane >> 4)));
          }
        }
#pragma unroll
        for (int j = 0; j < KS / 16; ++j) {
          uint32_t bf[4];
          ldsm4(bf, st + tile_at(k0 + 16 * j + (lane & 7) + (lane >> 4) * 8, 2 * kk + ((lane >> 3) & 1)));
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            mma_16816(s[i][2 * j], af[i][0], af[i][1], af[i][2], af[i][3], bf[0], bf[1]);
            mma_16816(s[i][2 * j + 1], af[i][0], af[i][1], af[i][2], af[i][3], bf[2], bf[3]);
          }
        }
      }
      if (fresh || nv < kTreeTile) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int row = wr * MT * 16 + 16 * i + g + 8 * e;
            unsigned long long see = nv >= 64 ? ~0ull : (1ull << nv) - 1;
            if (fresh && !SCORED) see = row < R ? anc[row >> gl] : 0ull;
#pragma unroll
            for (int j = 0; j < KS / 8; ++j)
#pragma unroll
              for (int c = 0; c < 2; ++c)
                if (!((see >> (k0 + 8 * j + 2 * t + c)) & 1)) s[i][j][2 * e + c] = -INFINITY;
          }
      }
      if (SCORED && g < G) {
#pragma unroll
        for (int j = 0; j < KS / 8; ++j)
          *reinterpret_cast<float2*>(score + g * a.score_cap + (it - lo) * kTreeTile + k0 + 8 * j + 2 * t) =
              make_float2(s[0][j][0], s[0][j][1]);
      }
      uint32_t pf[MT][KS / 8][2];
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mx = -INFINITY;
#pragma unroll
          for (int j = 0; j < KS / 8; ++j) mx = fmaxf(mx, fmaxf(s[i][j][2 * e], s[i][j][2 * e + 1]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          const float mn = fmaxf(m[i][e], __fmul_rn(mx, kC));
          const float mu = mn == -INFINITY ? 0.0f : mn;  // a row that sees no key yet
          const float al = ex2(__fsub_rn(m[i][e], mu));
          m[i][e] = mn;
          float sum = 0.0f;
#pragma unroll
          for (int j = 0; j < KS / 8; ++j) {
            const float p0 = ex2(__fmaf_rn(s[i][j][2 * e], kC, -mu));
            const float p1 = ex2(__fmaf_rn(s[i][j][2 * e + 1], kC, -mu));
            sum = __fadd_rn(sum, __fadd_rn(p0, p1));
            pf[i][j][e] = pack_h2(p0, p1);
          }
          l[i][e] = __fmaf_rn(l[i][e], al, sum);
#pragma unroll
          for (int d = 0; d < 16; ++d) {
            o[i][d][2 * e] = __fmul_rn(o[i][d][2 * e], al);
            o[i][d][2 * e + 1] = __fmul_rn(o[i][d][2 * e + 1], al);
          }
        }
      const uint32_t sv = st + kTreeStageBytes / 2;
#pragma unroll
      for (int j = 0; j < KS / 16; ++j)
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          uint32_t bf[4];
          ldsm4_t(bf, sv + tile_at(k0 + 16 * j + (lane & 7) + ((lane >> 3) & 1) * 8, 2 * d + (lane >> 4)));
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            mma_16816(o[i][2 * d], pf[i][2 * j][0], pf[i][2 * j][1], pf[i][2 * j + 1][0], pf[i][2 * j + 1][1],
                      bf[0], bf[1]);
            mma_16816(o[i][2 * d + 1], pf[i][2 * j][0], pf[i][2 * j][1], pf[i][2 * j + 1][0],
                      pf[i][2 * j + 1][1], bf[2], bf[3]);
          }
        }
    }
  }
  cp_wait<0>();
  __syncthreads();  // the ring becomes the partial outputs

#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int row = wr * MT * 16 + 16 * i + g + 8 * e;
      float s = l[i][e];
      s = __fadd_rn(s, __shfl_xor_sync(0xffffffffu, s, 1));
      s = __fadd_rn(s, __shfl_xor_sync(0xffffffffu, s, 2));
      if (t == 0) mlw[wk * RP + row] = make_float2(m[i][e], s);
#pragma unroll
      for (int d = 0; d < 16; ++d)
        *reinterpret_cast<float2*>(op + (wk * RP + row) * kTreeOPitch + 8 * d + 2 * t) =
            make_float2(o[i][d][2 * e], o[i][d][2 * e + 1]);
    }
  __syncthreads();
  // the key warps' partials into one per row: a warp a row, four dims a lane
  for (int r = warp; r < R; r += 4) {
    float M = -INFINITY, L = 0.0f;
#pragma unroll
    for (int k = 0; k < WK; ++k) M = fmaxf(M, mlw[k * RP + r].x);
    const float mu = M == -INFINITY ? 0.0f : M;
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int k = 0; k < WK; ++k) {
      const float2 q = mlw[k * RP + r];
      const float f = ex2(__fsub_rn(q.x, mu));
      const float4 x = *reinterpret_cast<const float4*>(op + (k * RP + r) * kTreeOPitch + 4 * lane);
      L = __fmaf_rn(q.y, f, L);
      s.x = __fmaf_rn(x.x, f, s.x), s.y = __fmaf_rn(x.y, f, s.y);
      s.z = __fmaf_rn(x.z, f, s.z), s.w = __fmaf_rn(x.w, f, s.w);
    }
    if (WK > 1) *reinterpret_cast<float4*>(op + r * kTreeOPitch + 4 * lane) = s;
    if (lane == 0) ml[r] = make_float2(M, L);
  }
  cluster_sync_all();

  // the cluster's partials into the output: rank c takes rows c, c + C, ...
  auto row_total = [&](int r, float& M, float& L, float& f) {  // f: lane c's factor for rank c
    float2 q = make_float2(-INFINITY, 0.0f);
    if (lane < C) {
      q.x = ld_dsmem_f32(smem_u32(ml + r), lane);
      q.y = ld_dsmem_f32(smem_u32(ml + r) + 4, lane);
    }
    M = warp_max(q.x);
    f = ex2(__fsub_rn(q.x, M == -INFINITY ? 0.0f : M));
    L = warp_sum(__fmul_rn(q.y, f));
  };
  for (int r = rank + C * warp; r < R; r += C * 4) {
    float M, L, f;
    row_total(r, M, L, f);
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int c = 0; c < C; ++c) {
      const float fc = __shfl_sync(0xffffffffu, f, c);
      const float4 x = ld_dsmem_f4(smem_u32(op + r * kTreeOPitch + 4 * lane), c);
      s.x = __fmaf_rn(x.x, fc, s.x), s.y = __fmaf_rn(x.y, fc, s.y);
      s.z = __fmaf_rn(x.z, fc, s.z), s.w = __fmaf_rn(x.w, fc, s.w);
    }
    const float inv = L == 0.0f ? 0.0f : __fdiv_rn(1.0f, L);  // a row that sees nothing is zero
    const uint2 w = make_uint2(pack_h2(__fmul_rn(s.x, inv), __fmul_rn(s.y, inv)),
                               pack_h2(__fmul_rn(s.z, inv), __fmul_rn(s.w, inv)));
    const int tok = r >> gl;
    *reinterpret_cast<uint2*>(a.out + ((int64_t)b * a.T + tok) * a.q_heads * kHD +
                              ((h << gl) + (r & (G - 1))) * kHD + lane * 4) = w;
  }
  if (SCORED) {
    // each slot's softmax weights of the group's heads join its accumulator, in f32
    float M[8], I[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < G) {
        float L, f;
        row_total(j, M[j], L, f);
        if (M[j] == -INFINITY) M[j] = 0.0f;
        I[j] = L == 0.0f ? 0.0f : __fdiv_rn(1.0f, L);
      }
    const int64_t w0 = b * a.w_stride + (int64_t)h * a.S, s0 = (int64_t)lo * kTreeTile;
    const int64_t left = len - s0;
    const int held = (int)(left < 0 ? 0 : left < (int64_t)(hi - lo) * kTreeTile ? left : (int64_t)(hi - lo) * kTreeTile);
    for (int i = tid; i < held; i += kTreeThreads) {
      float w = a.w_in[w0 + s0 + i];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < G) w = __fmaf_rn(ex2(__fmaf_rn(score[j * a.score_cap + i], kC, -M[j])), I[j], w);
      a.w_out[w0 + s0 + i] = w;
    }
    if (hi == nt && tid == 0) {  // the new slot starts with its own weight
      float w = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < G)
          w = __fmaf_rn(ex2(__fmaf_rn(score[j * a.score_cap + (nct - lo) * kTreeTile], kC, -M[j])), I[j], w);
      a.w_out[w0 + len] = w;
      a.slot_pos[w0 + len] = (int32_t)pos;
    }
  }
  cluster_sync_all();  // peers read this CTA's shared memory until here
}

// The accepted path's K/V rows from slots len + a_i to len + i, in n_layers layers.  A warp owns a
// (sequence, layer, kv head): lanes 0-15 hold its K row's 16-byte chunks, lanes 16-31 its V row's.
// a_i ascends, so a_i >= i and a row is read before anything is written over it: eight rows are read,
// then written, and what later rows read lies behind what was written.
struct CommitArgs {
  uint16_t* k;  // layer0 of sequence 0
  uint16_t* v;
  int64_t seq_stride, layer_stride, slot_stride, head_stride;
  int64_t S;
  int n_layers, kv_heads, A, B;
  const int32_t* accepted;    // [B][A]
  const int32_t* n_accepted;  // [B]
  const int64_t* len;
  int64_t* new_len;
  const int64_t* pos;  // null: no accumulators
  float* w;            // layer0 of sequence 0: [B][layers][kv_heads][S]
  int32_t* slot_pos;
  int64_t w_stride;
  int* err;
};

__global__ void __launch_bounds__(128) k_tree_commit(const CommitArgs a) {
  const int lane = threadIdx.x & 31, b = blockIdx.y;
  const int unit = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (unit >= a.n_layers * a.kv_heads) return;
  const int layer = unit / a.kv_heads, h = unit - layer * a.kv_heads;
  const int n = a.n_accepted[b];
  const int64_t len = a.len[b];
  bool bad = n < 0 || n > a.A || len < 0 || len > a.S - n;
  const int32_t* acc = a.accepted + (int64_t)b * a.A;
  if (!bad) {
    for (int i = lane; i < n; i += 32) {
      const int x = acc[i], before = i ? acc[i - 1] : -1;
      bad |= x <= before || x >= kTreeMaxTokens || len + x >= a.S;
    }
  }
  bad = __any_sync(0xffffffffu, bad);
  if (unit == 0 && lane == 0) {
    if (bad && a.err) atomicCAS(a.err, 0, kErrBadTree);
    a.new_len[b] = bad ? len : len + n;
  }
  if (bad) return;
  if (a.pos != nullptr) {
    const int64_t w0 = b * a.w_stride + (int64_t)unit * a.S + len;
    for (int i = lane; i < n; i += 32) a.w[w0 + i] = 0.0f, a.slot_pos[w0 + i] = (int32_t)(a.pos[b] + i);
  }
  uint16_t* base = (lane < 16 ? a.k : a.v) + b * a.seq_stride + layer * a.layer_stride +
                   h * a.head_stride + len * a.slot_stride + (lane & 15) * 8;
  for (int i0 = 0; i0 < n; i0 += 8) {
    uint4 x[8];
    int src[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      src[i] = i0 + i < n ? acc[i0 + i] : i0 + i;
      if (src[i] != i0 + i) x[i] = *reinterpret_cast<const uint4*>(base + src[i] * a.slot_stride);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (src[i] != i0 + i) *reinterpret_cast<uint4*>(base + (i0 + i) * a.slot_stride) = x[i];
  }
}

}  // namespace q3
