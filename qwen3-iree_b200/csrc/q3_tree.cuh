// q3_tree.cuh -- attention of several drafted tokens (a tree) over a KV cache, the single-token form
// that also accumulates every slot's attention weight, and the move of an accepted path.
//
// For sequence b with m cached slots, drafted token i (parent p_i < i, or -1: the last cached token)
// has depth = its number of ancestors and sits at RoPE position pos + depth.  With q, k after
// QK-RMSNorm and RoPE (each rounded to f16, the bits the one-token engines put into the cache):
//   out_i = sum_j softmax_j(q_i . k_j / sqrt(128)) v_j,   j over slots 0..m-1, i's ancestors and i.
// The new K/V rows go to slots m + i.
//
// What it has to move is 512 bytes per (slot, kv head), once, for all group x T query rows of that
// head, so the work is split over the keys: a thread-block cluster of up to 16 CTAs owns a (sequence,
// kv head) and each CTA a contiguous run of 64-key tiles, streamed by tensor TMA into a ring.  (With
// cp.async instead, 64 warp instructions a tile, the copies took 840 cycles of an SM a tile by
// themselves, and 4800 when one warp issued them.)  The softmax runs online; the CTAs' partial (max,
// sum, output) meet over distributed shared memory, so there is no workspace, no counter and no second
// launch.
//
// Two kernels: up to 16 rows the products run as mma.sync, a warp taking 16 keys of each tile
// (k_tree_attn); above that as tcgen05.mma on 128 rows, a thread taking one row (k_tree_tc).
#pragma once

#include "q3_attn.cuh"
#include "q3_common.cuh"
#include "q3_q4.cuh"
#include "q3_tc.cuh"

namespace q3 {

constexpr int kTreeMaxTokens = 64;
constexpr int kTreeThreads = 160;                         // four computing warps, a copying warp
constexpr int kTreeTile = 64;                             // keys per ring stage
constexpr int kTreeHalf = kTreeTile * kHD * 2;            // a stage: K, then V
constexpr int kTreeStageBytes = 2 * kTreeHalf;
constexpr int kTreeOPitch = kHD + 4;                      // floats between partial output rows
constexpr int kTreeMaxCluster = 16;
constexpr int kTreeMaxDepth = 3;                          // tiles a ring of k_tree_attn holds, two or three
constexpr int kTreeSmallRows = 16;                        // rows of k_tree_attn
constexpr float kTreeLog2Scale = kAttnScale * 1.44269504088896341f;  // scores in powers of two
// The softmax weights go to P V as f16, relative to a reference that puts the largest near 2^15, the top
// of that type: then a weight down to 2^-29 of the largest keeps half a step of 2^-11 of itself, and a
// smaller one is off by at most 2^-40 of the largest.  (With the largest at 1 these were 2^-14 and 2^-25:
// over a cache whose first slots draw nearly everything, as they do in trained models, the others' share
// lost digits or vanished.)  Where an output is rescaled late, by kTreeLazy powers of two at most, the
// reference starts that much lower: 2^-23 and 2^-34 (64 tokens over 32749 slots: 48.2 us with 8, 48.4
// with 6, 50.1 with 4).  Sums share the reference, so quotients do not change.
constexpr float kTreeTop = 15.0f, kTreeLazy = 6.0f;

struct TreeArgs {
  CUtensorMap km, vm;   // the layer's K and V: {dim, slot, head, sequence}, boxes of 64 dims x 64 slots
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
// The reference that puts a score of `top` at 2^exponent.  Steps of f32 above 2^20 are too coarse for it.
__device__ __forceinline__ float tree_ref(float top, float exponent) {
  return fabsf(top) < 1048576.0f ? __fsub_rn(top, exponent) : top;
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
__device__ __forceinline__ void st_dsmem_u16(uint32_t local_addr, uint32_t rank, uint16_t v) {
  asm volatile("st.shared::cluster.b16 [%0], %1;" ::"r"(dsmem_map(local_addr, rank)), "h"(v) : "memory");
}
__device__ __forceinline__ void st_dsmem_v2(uint32_t local_addr, uint32_t rank, uint2 v) {
  asm volatile("st.shared::cluster.v2.b32 [%0], {%1, %2};" ::"r"(dsmem_map(local_addr, rank)), "r"(v.x),
               "r"(v.y)
               : "memory");
}

__device__ __forceinline__ void st_dsmem_u8(uint32_t local_addr, uint32_t rank, uint32_t v) {
  asm volatile("st.shared::cluster.b8 [%0], %1;" ::"r"(dsmem_map(local_addr, rank)), "r"(v) : "memory");
}

// Byte offset of 16-byte chunk c (0..15) of row r in a tile of ROWS 256-byte rows: two halves of 64
// dims, each in the SWIZZLE_128B layout (128-byte rows, the chunk xored with the row).  The 8 rows of
// an ldmatrix fall into different banks, and the tensor core reads it K-major (rows along N) or
// MN-major (rows along K).
template <int ROWS>
__device__ __forceinline__ uint32_t tile_at(int r, int c) {
  return (c >> 3) * (ROWS * 128) + r * 128 + (((c ^ r) & 7) << 4);
}

// What a CTA works on.
struct TreeCta {
  int C, rank, h, b, tid, warp, lane;
  int n, R, nct, lo, tiles, fresh;  // tokens, rows, cached tiles; this CTA's first tile and tile count
  int64_t len, pos;                 // fresh: 1 in the last CTA, whose tile 0 holds the new tokens
  uint16_t *kb, *vb;
  int parent;                       // of token `tid`
};

__device__ __forceinline__ void tree_place(TreeCta& c) {
  c.C = gridDim.x, c.rank = blockIdx.x, c.h = blockIdx.y, c.b = blockIdx.z;
  c.fresh = c.rank == c.C - 1;
  c.tid = threadIdx.x, c.lane = c.tid & 31;
  c.warp = __shfl_sync(0xffffffffu, c.tid >> 5, 0);  // uniform for the compiler too
}
// Reads and checks the sequence's values; false: nothing to do (the same in all CTAs of a cluster).
template <bool SCORED>
__device__ __forceinline__ bool tree_begin(const TreeArgs& a, TreeCta& c) {
  c.n = SCORED ? 1 : (a.n_tokens ? a.n_tokens[c.b] : a.T);
  c.len = a.len[c.b], c.pos = a.pos[c.b];
  c.parent = !SCORED && c.tid < a.T ? a.parents[(int64_t)c.b * a.T + c.tid] : -1;
  if (SCORED ? c.len == -1 : c.n == 0) return false;
  if (c.n < 0 || c.n > a.T || c.len < 0 || c.len > a.S - c.n || c.pos < 0 || c.pos >= a.rope_rows) {
    if (c.tid == 0 && a.err) atomicCAS(a.err, 0, kErrBadPos);
    return false;
  }
  c.R = c.n << a.group_log2;
  c.nct = (int)((c.len + kTreeTile - 1) / kTreeTile);
  const int nt = c.nct + 1;  // the new tokens count as a last tile
  c.lo = (int)((int64_t)c.rank * nt / c.C);
  c.tiles = (int)((int64_t)(c.rank + 1) * nt / c.C) - c.lo;
  c.kb = a.k + c.b * a.seq_stride + c.h * a.head_stride;
  c.vb = a.v + c.b * a.seq_stride + c.h * a.head_stride;
  return true;
}

// Cached keys of this CTA's tile j (at most 64 count).
__device__ __forceinline__ int64_t tree_left(const TreeCta& c, int j) {
  return c.len - (int64_t)(c.lo + j - c.fresh) * kTreeTile;
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z,
                                            int w, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}
// K or V of tile j (not the new tokens'), two boxes of 64 dims; slots behind the layer arrive as zeros.
__device__ __forceinline__ void tree_copy(const TreeCta& c, const CUtensorMap* map, uint32_t dst, int j,
                                          uint64_t* bar) {
  const int slot = (c.lo + j - c.fresh) * kTreeTile;
  tma_load_4d(dst, map, 0, slot, c.h, c.b, bar);
  tma_load_4d(dst + kTreeHalf / 2, map, 64, slot, c.h, c.b, bar);
}

// Ancestors by doubling, until the deepest token has met the root: after each step a token knows twice
// as many.  anc[i]: ancestors of i and i itself; up: scratch.  false: a bad tree, or a token beyond the
// RoPE tables.
__device__ __forceinline__ bool tree_ancestors(const TreeArgs& a, const TreeCta& c,
                                               unsigned long long* anc, int* up) {
  const bool mine = c.tid < c.n;
  int u = c.parent;
  unsigned long long m = 1ull << (c.tid & 63);
  if (mine) up[c.tid] = u, anc[c.tid] = m;
  if (__syncthreads_or(mine && (u < -1 || u >= c.tid))) {
    if (c.tid == 0 && a.err) atomicCAS(a.err, 0, kErrBadTree);
    return false;
  }
  while (true) {
    const bool more = mine && u >= 0;
    if (more) m |= anc[u], u = up[u];
    if (!__syncthreads_or(more)) break;
    if (more) anc[c.tid] = m, up[c.tid] = u;
    __syncthreads();
  }
  if (__syncthreads_or(mine && c.pos + __popcll(m) - 1 >= a.rope_rows)) {
    if (c.tid == 0 && a.err) atomicCAS(a.err, 0, kErrBadPos);
    return false;
  }
  return true;
}

// v / r, correctly rounded, from y = 1 / r correctly rounded (Markstein, IBM J. Res. Dev. 34, 1990):
// q = v y is within an ulp, its remainder v - q r is exact in one fma, and one more fma rounds the
// corrected quotient as a division would.  Where r is infinite (y = 0) q itself is the answer.  Needs
// no underflow: here |v| >= 2^-24 or 0, and 2^-10 <= r <= 2^16.
__device__ __forceinline__ float div_by(float v, float r, float y) {
  const float q = __fmul_rn(v, y);
  const float c = __fmaf_rn(__fmaf_rn(-q, r, v), y, q);
  return y == 0.0f ? q : c;
}

// Two f16 with zeros for infinities and NaNs.
__device__ __forceinline__ uint32_t finite_h2(uint32_t h) {
  uint32_t m = 0;
  if ((h & 0x00007c00u) != 0x00007c00u) m |= 0x0000ffffu;
  if ((h & 0x7c000000u) != 0x7c000000u) m |= 0xffff0000u;
  return h & m;
}

// Raw rows a warp prepares at a time: one dim of each quarter a lane, and four dims of the V row.
template <int E>
struct TreeRaw {
  uint16_t x[E][4];
  uint2 v[E];
};

// The rows to prepare are numbered over all T tokens, so that the first can be read before the number
// of tokens is known: query rows token * group + j, then the new K rows.  SHARE: dealt out to the
// cluster's CTAs (above 16 rows; below, pushing a row to the others costs more than preparing it).
template <int WARPS, bool SHARE>
struct TreeUnits {
  int first, step, queries, units;
  __device__ __forceinline__ TreeUnits(const TreeArgs& a, const TreeCta& c) {
    queries = a.T << a.group_log2;
    units = SHARE || c.fresh ? queries + a.T : queries;
    first = SHARE ? c.rank + c.C * c.warp : c.warp;
    step = SHARE ? WARPS * c.C : WARPS;
  }
};
template <int WARPS, int E, bool SHARE>
__device__ __forceinline__ void tree_load(const TreeArgs& a, const TreeCta& c,
                                          const TreeUnits<WARPS, SHARE>& n, int u0, TreeRaw<E>& raw) {
  const int gl = a.group_log2;
  const int64_t row_el = (int64_t)(a.q_heads + 2 * a.kv_heads) * kHD;
  const uint16_t* qkv = a.qkv + (int64_t)c.b * a.T * row_el;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int u = min(u0 + e * n.step, n.units - 1);  // a repeated row is computed and dropped
    const bool isq = u < n.queries;
    const int tok = isq ? u >> gl : u - n.queries;
    const uint16_t* x = qkv + tok * row_el + (isq ? (c.h << gl) + (u & ((1 << gl) - 1)) : a.q_heads + c.h) * kHD;
#pragma unroll
    for (int i = 0; i < 4; ++i) raw.x[e][i] = x[c.lane + 32 * i];
    if (!isq) raw.v[e] = *reinterpret_cast<const uint2*>(x + a.kv_heads * kHD + c.lane * 4);
  }
}

// QK-RMSNorm and RoPE of the query rows into the tile `qs` (ROWS rows), of every CTA with SHARE (the
// caller has waited until all CTAs run, and follows with a cluster barrier), and of the new K rows,
// with the V rows as they are, into the first tile of the last CTA and into the cache.  The operations
// and roundings of norm_rope_vals, a warp per row, E rows at a time without branches between them (its
// divisions branch, and took most of 0.35 us a row).  `raw`: the first rows, as tree_load read them.
// An infinity or NaN of a V row must not reach the tokens that do not see it (0 * inf is a NaN), so the
// tile gets zeros for them, and odd[k] says that token k has some: tree_add_odd gives them to those that
// do see them.
template <int ROWS, int WARPS, int E, bool SHARE, bool SCORED>
__device__ __forceinline__ void tree_rows(const TreeArgs& a, const TreeCta& c,
                                          const TreeUnits<WARPS, SHARE>& n, TreeRaw<E>& raw,
                                          const unsigned long long* anc, uint8_t* qs, uint8_t* knew,
                                          uint8_t* vnew, uint8_t* odd) {
  const int gl = a.group_log2, lane = c.lane;
  float gq[4], gk[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) gq[i] = h2f(a.q_norm[lane + 32 * i]), gk[i] = h2f(a.k_norm[lane + 32 * i]);
  const int last = c.C - 1;
  for (int u0 = n.first; u0 < n.units; u0 += E * n.step) {
    float v[E][4], cs[E][4];
    uint2 vv[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int u = min(u0 + e * n.step, n.units - 1);
      const int tok = min(u < n.queries ? u >> gl : u - n.queries, c.n - 1);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[e][i] = h2f(raw.x[e][i]);
      vv[e] = raw.v[e];
      const int64_t p = (c.pos + (SCORED ? 0 : __popcll(anc[tok]) - 1)) * 64 + lane;
      cs[e][0] = a.rope_cos[p], cs[e][1] = a.rope_cos[p + 32];
      cs[e][2] = a.rope_sin[p], cs[e][3] = a.rope_sin[p + 32];
    }
    if (u0 + E * n.step < n.units) tree_load(a, c, n, u0 + E * n.step, raw);
    float ss[E] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < E; ++e) ss[e] = __fmaf_rn(v[e][i], v[e][i], ss[e]);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1)
#pragma unroll
      for (int e = 0; e < E; ++e) ss[e] = __fadd_rn(ss[e], __shfl_xor_sync(0xffffffffu, ss[e], off));
    uint16_t o[E][4];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const bool isq = u0 + e * n.step < n.queries;
      const float r = __fsqrt_rn(__fadd_rn(__fmul_rn(ss[e], 0.0078125f), kEps));
      const float y = __frcp_rn(r);
      float x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = h2f(f2h(__fmul_rn(div_by(v[e][i], r, y), isq ? gq[i] : gk[i])));
      o[e][0] = f2h(__fsub_rn(__fmul_rn(x[0], cs[e][0]), __fmul_rn(x[2], cs[e][2])));
      o[e][2] = f2h(__fadd_rn(__fmul_rn(x[0], cs[e][2]), __fmul_rn(x[2], cs[e][0])));
      o[e][1] = f2h(__fsub_rn(__fmul_rn(x[1], cs[e][1]), __fmul_rn(x[3], cs[e][3])));
      o[e][3] = f2h(__fadd_rn(__fmul_rn(x[1], cs[e][3]), __fmul_rn(x[3], cs[e][1])));
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int u = u0 + e * n.step;
      if (u >= n.units) break;
      const bool isq = u < n.queries;
      if ((isq ? u >> gl : u - n.queries) >= c.n) continue;  // tokens that the sequence does not have
      if (isq) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d = lane + 32 * i;
          *reinterpret_cast<uint16_t*>(qs + tile_at<ROWS>(u, d >> 3) + (d & 7) * 2) = o[e][i];
        }
        if (SHARE) {  // half a warp a peer
          __syncwarp();
          const uint8_t* at = qs + tile_at<ROWS>(u, lane & 15);
          const uint4 row = *reinterpret_cast<const uint4*>(at);
          for (int p = lane >> 4; p < c.C; p += 2)
            if (p != c.rank) st_dsmem_v4(smem_u32(at), p, row);
        }
      } else {
        const int k = u - n.queries;
        uint16_t* kd = c.kb + (c.len + k) * a.slot_stride;
        *reinterpret_cast<uint2*>(c.vb + (c.len + k) * a.slot_stride + lane * 4) = vv[e];
        uint2 fin = make_uint2(finite_h2(vv[e].x), finite_h2(vv[e].y));
        const bool any = __any_sync(0xffffffffu, fin.x != vv[e].x || fin.y != vv[e].y);
        if (SCORED) fin = vv[e];  // one token, which sees itself
        else if (lane == 0) st_dsmem_u8(smem_u32(odd + k), last, any);
        st_dsmem_v2(smem_u32(vnew) + tile_at<kTreeTile>(k, lane >> 1) + (lane & 1) * 8, last, fin);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d = lane + 32 * i;
          kd[d] = o[e][i];
          st_dsmem_u16(smem_u32(knew) + tile_at<kTreeTile>(k, d >> 3) + (d & 7) * 2, last, o[e][i]);
        }
      }
    }
  }
}

// V rows nv..63 of a tile become zeros, by a warp: no weight falls on rows behind the cached slots, or
// behind the new tokens, but 0 * NaN would.
__device__ __forceinline__ void tree_zero_tail(uint8_t* v, int nv, int lane) {
  for (int i = nv * 16 + lane; i < kTreeTile * 16; i += 32)
    *reinterpret_cast<uint4*>(v + tile_at<kTreeTile>(i >> 4, i & 15)) = make_uint4(0u, 0u, 0u, 0u);
}

// Tokens whose V rows hold infinities or NaNs (by a whole warp).
__device__ __forceinline__ unsigned long long tree_odd(const TreeCta& c, const uint8_t* odd) {
  const uint32_t lo = __ballot_sync(0xffffffffu, c.lane < c.n && odd[c.lane]);
  const uint32_t hi = __ballot_sync(0xffffffffu, c.lane + 32 < c.n && odd[c.lane + 32]);
  return (unsigned long long)hi << 32 | lo;
}
// Adds dim d's infinities and NaNs of the tokens in `from` to x.
__device__ __forceinline__ float tree_add_odd(const TreeArgs& a, const TreeCta& c, unsigned long long from, int d,
                                              float x) {
  const int64_t row_el = (int64_t)(a.q_heads + 2 * a.kv_heads) * kHD;
  const uint16_t* v = a.qkv + (int64_t)c.b * a.T * row_el + (int64_t)(a.q_heads + a.kv_heads + c.h) * kHD + d;
  for (; from; from &= from - 1) {
    const uint16_t h = v[(__ffsll((long long)from) - 1) * row_el];
    if ((h & 0x7c00u) == 0x7c00u) x = __fadd_rn(x, h2f(h));
  }
  return x;
}

// Keys of tile j that row `row` sees, as bits; `nv`: keys the tile holds.
__device__ __forceinline__ unsigned long long tree_seen(const TreeCta& c, const unsigned long long* anc,
                                                        bool tree, int row, int nv, int gl) {
  if (tree) return row < c.R ? anc[row >> gl] : 0ull;
  return nv >= 64 ? ~0ull : (1ull << nv) - 1;
}

// This lane's factor for rank `lane`, and the row's max and sum over the cluster.
__device__ __forceinline__ void tree_row_total(const TreeCta& c, const float2* ml, int r, float& M,
                                               float& L, float& f) {
  float2 q = make_float2(-INFINITY, 0.0f);
  if (c.lane < c.C) {
    q.x = ld_dsmem_f32(smem_u32(ml + r), c.lane);
    q.y = ld_dsmem_f32(smem_u32(ml + r) + 4, c.lane);
  }
  M = warp_max(q.x);
  f = ex2(__fsub_rn(q.x, M == -INFINITY ? 0.0f : M));
  L = warp_sum(__fmul_rn(q.y, f));
}

// The cluster's partials (max and sum in ml, outputs in op) into the output: rank c takes rows c,
// c + C, ..., a warp a row, four dims a lane.
__device__ __forceinline__ void tree_output(const TreeArgs& a, const TreeCta& c, const float2* ml,
                                            const float* op) {
  const int gl = a.group_log2, G = 1 << gl, warps = blockDim.x >> 5;
  for (int r = c.rank + c.C * c.warp; r < c.R; r += c.C * warps) {
    float4 x[kTreeMaxCluster];  // all under way before the factors are known
#pragma unroll
    for (int k = 0; k < kTreeMaxCluster; ++k)
      if (k < c.C) x[k] = ld_dsmem_f4(smem_u32(op + r * kTreeOPitch + 4 * c.lane), k);
    float M, L, f;
    tree_row_total(c, ml, r, M, L, f);
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int k = 0; k < kTreeMaxCluster; ++k) {
      if (k >= c.C) break;
      const float fk = __shfl_sync(0xffffffffu, f, k);
      s.x = __fmaf_rn(x[k].x, fk, s.x), s.y = __fmaf_rn(x[k].y, fk, s.y);
      s.z = __fmaf_rn(x[k].z, fk, s.z), s.w = __fmaf_rn(x[k].w, fk, s.w);
    }
    const float inv = L == 0.0f ? 0.0f : __fdiv_rn(1.0f, L);  // a row that sees nothing is zero
    const uint2 w = make_uint2(pack_h2(__fmul_rn(s.x, inv), __fmul_rn(s.y, inv)),
                               pack_h2(__fmul_rn(s.z, inv), __fmul_rn(s.w, inv)));
    const int tok = r >> gl;
    *reinterpret_cast<uint2*>(a.out + ((int64_t)c.b * a.T + tok) * a.q_heads * kHD +
                              ((c.h << gl) + (r & (G - 1))) * kHD + c.lane * 4) = w;
  }
}

// Up to 16 query rows: r = token * group + j.  Each warp takes 16 keys of every tile, with a softmax
// state of its own, so a tile costs it 16 + 16 MMAs and one pass over its K and V fragments.  Bound by
// the copies where there is work for all SMs (scored, four sequences of 8000: 28.8 us, 4.6 TB/s; 32 of
// 2000: 50 us, 5.3 TB/s), by a chain of round trips (lengths, rows, tiles, merge) where there is little
// (8 tokens over 500 slots: 9.2 us).
struct TreeSmallSmem {  // behind the ring
  uint8_t q[kTreeSmallRows * 256];
  float2 mlw[4][kTreeSmallRows];  // the warps' (max, sum)
  float2 ml[kTreeSmallRows];      // this CTA's
  unsigned long long anc[kTreeMaxTokens];
  int up[kTreeMaxTokens];
  uint8_t odd[kTreeMaxTokens];
  uint64_t full[kTreeMaxDepth], empty[kTreeMaxDepth], tail;
};
constexpr size_t tree_small_bytes(int depth) {
  return 1024 + (size_t)depth * kTreeStageBytes + sizeof(TreeSmallSmem);
}
template <bool SCORED>
__global__ void __launch_bounds__(kTreeThreads, 3)
    k_tree_attn(const __grid_constant__ TreeArgs a, const int depth) {
  constexpr int RP = kTreeSmallRows;
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* ring = smem + ((1024u - (smem_u32(smem) & 1023u)) & 1023u);  // stages; then the partial outputs
  TreeSmallSmem& sm = *reinterpret_cast<TreeSmallSmem*>(ring + depth * kTreeStageBytes);
  float* score = reinterpret_cast<float*>(&sm + 1);                    // [group][score_cap]
  float* op = reinterpret_cast<float*>(ring);                          // [4][RP][kTreeOPitch]

  if (threadIdx.x == 128) prefetch_tmap(&a.km), prefetch_tmap(&a.vm);
  TreeCta c;
  tree_place(c);
  const TreeUnits<5, false> units(a, c);
  TreeRaw<SCORED ? 1 : 5> raw;
  if (units.first < units.units) tree_load(a, c, units, units.first, raw);
  if (!tree_begin<SCORED>(a, c)) return;
  const int warp = c.warp, lane = c.lane, g = lane >> 2, t = lane & 3;
  const int gl = a.group_log2, G = 1 << gl;
  cluster_arrive();
  const uint32_t rg = smem_u32(ring);
  // one thread copies; a tile with rows behind the cached slots is announced after its V rows there
  // have been zeroed
  auto copy = [&](int j) {
    if (j < c.fresh) return;
    const int s = j % depth;
    uint64_t* bar = tree_left(c, j) < kTreeTile ? &sm.tail : &sm.full[s];
    mbar_expect_tx(bar, kTreeStageBytes);
    tree_copy(c, &a.km, rg + s * kTreeStageBytes, j, bar);
    tree_copy(c, &a.vm, rg + s * kTreeStageBytes + kTreeHalf, j, bar);
  };
  if (c.tid == 128) {
    for (int i = 0; i < depth; ++i) {
      mbar_init(&sm.full[i], 1);
      mbar_init(&sm.empty[i], 4);
    }
    mbar_init(&sm.tail, 1);
    fence_mbar_init();
    for (int j = 0; j < depth && j < c.tiles; ++j) copy(j);
  }
  const bool ok = SCORED || tree_ancestors(a, c, sm.anc, sm.up);
  cluster_wait();  // every CTA of the cluster runs
  if (ok)
    tree_rows<RP, 5, SCORED ? 1 : 5, false, SCORED>(a, c, units, raw, sm.anc, sm.q, ring, ring + kTreeHalf,
                                                         sm.odd);
  if (ok && warp == 4 && c.fresh) tree_zero_tail(ring + kTreeHalf, c.n, lane);
  __syncthreads();
  if (!ok) {  // nothing but the first copies is under way
    if (c.tid == 128)
      for (int j = c.fresh; j < depth && j < c.tiles; ++j)
        mbar_wait_own(tree_left(c, j) < kTreeTile ? &sm.tail : &sm.full[j], 0, a.err, kErrTimeoutFull);
    return;
  }

  const unsigned long long odd = !SCORED && c.fresh ? tree_odd(c, sm.odd) : 0ull;
  float o[16][4] = {}, m[2] = {-INFINITY, -INFINITY}, l[2] = {};
  if (warp == 4) {
    fence_async_smem();  // the new tokens' stage was written by threads, later by copies
    bool run = true;
    int j = 0;
    for (; j < c.tiles; ++j) {
      const int s = j % depth;
      if (j >= depth) {
        run &= mbar_wait_own(&sm.empty[s], (j / depth - 1) & 1, a.err, kErrTimeoutEmpty);
        if (!__all_sync(0xffffffffu, run)) break;
        if (lane == 0) copy(j);
      }
      if (j < c.fresh) {
        if (lane == 0) mbar_arrive(&sm.full[s]);
      } else if (tree_left(c, j) < kTreeTile) {
        mbar_wait_own(&sm.tail, 0, a.err, kErrTimeoutFull);
        tree_zero_tail(ring + s * kTreeStageBytes + kTreeHalf, (int)tree_left(c, j), lane);
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.full[s]);
      }
    }
    // the copies under way land before the memory is used again
    for (int i = j > depth ? j - depth : 0; i < j; ++i)
      mbar_wait_own(&sm.full[i % depth], (i / depth) & 1, a.err, kErrTimeoutFull);
  } else {
    uint32_t qf[8][4];
#pragma unroll
    for (int kk = 0; kk < 8; ++kk)
      ldsm4(qf[kk], smem_u32(sm.q) + tile_at<RP>((lane & 7) + ((lane >> 3) & 1) * 8, 2 * kk + (lane >> 4)));

    bool run = true;
    for (int j = 0; j < c.tiles; ++j) {
      const int sl = j % depth;
      const uint32_t st = rg + sl * kTreeStageBytes;
      const bool fresh = j < c.fresh;
      const int64_t left = tree_left(c, j);
      const int nv = fresh ? c.n : (int)(left < kTreeTile ? left : kTreeTile);
      run &= mbar_wait_own(&sm.full[sl], (j / depth) & 1, a.err, kErrTimeoutFull);
      if (!__all_sync(0xffffffffu, run)) break;
      const int k0 = warp * 16;
      if (k0 < nv) {
        float s[2][4] = {};
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          uint32_t bf[4];
          ldsm4(bf, st + tile_at<kTreeTile>(k0 + (lane & 7) + (lane >> 4) * 8, 2 * kk + ((lane >> 3) & 1)));
          mma_16816(s[0], qf[kk][0], qf[kk][1], qf[kk][2], qf[kk][3], bf[0], bf[1]);
          mma_16816(s[1], qf[kk][0], qf[kk][1], qf[kk][2], qf[kk][3], bf[2], bf[3]);
        }
        if (fresh || nv < kTreeTile) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const unsigned long long see = tree_seen(c, sm.anc, fresh && !SCORED, g + 8 * e, nv, gl);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (!((see >> (k0 + 8 * (i >> 1) + 2 * t + (i & 1))) & 1)) s[i >> 1][2 * e + (i & 1)] = -INFINITY;
          }
        }
        if (SCORED && g < G) {
#pragma unroll
          for (int i = 0; i < 2; ++i)
            *reinterpret_cast<float2*>(score + g * a.score_cap + j * kTreeTile + k0 + 8 * i + 2 * t) =
                make_float2(s[i][0], s[i][1]);
        }
        uint32_t pf[2][2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mx = fmaxf(fmaxf(s[0][2 * e], s[0][2 * e + 1]), fmaxf(s[1][2 * e], s[1][2 * e + 1]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          const float mn = fmaxf(m[e], tree_ref(__fmul_rn(mx, kTreeLog2Scale), kTreeTop));
          const float mu = mn == -INFINITY ? 0.0f : mn;  // a row that sees no key yet
          const float al = ex2(__fsub_rn(m[e], mu));
          m[e] = mn;
          float sum = 0.0f;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float p0 = ex2(__fmaf_rn(s[i][2 * e], kTreeLog2Scale, -mu));
            const float p1 = ex2(__fmaf_rn(s[i][2 * e + 1], kTreeLog2Scale, -mu));
            sum = __fadd_rn(sum, __fadd_rn(p0, p1));
            pf[i][e] = pack_h2(p0, p1);
          }
          l[e] = __fmaf_rn(l[e], al, sum);
#pragma unroll
          for (int d = 0; d < 16; ++d) {
            o[d][2 * e] = __fmul_rn(o[d][2 * e], al);
            o[d][2 * e + 1] = __fmul_rn(o[d][2 * e + 1], al);
          }
        }
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          uint32_t bf[4];
          ldsm4_t(bf, st + kTreeHalf +
                          tile_at<kTreeTile>(k0 + (lane & 7) + ((lane >> 3) & 1) * 8, 2 * d + (lane >> 4)));
          mma_16816(o[2 * d], pf[0][0], pf[0][1], pf[1][0], pf[1][1], bf[0], bf[1]);
          mma_16816(o[2 * d + 1], pf[0][0], pf[0][1], pf[1][0], pf[1][1], bf[2], bf[3]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.empty[sl]);
    }
  }
  __syncthreads();  // the ring becomes the partial outputs

  if (warp < 4) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int row = g + 8 * e;
      float s = l[e];
      s = __fadd_rn(s, __shfl_xor_sync(0xffffffffu, s, 1));
      s = __fadd_rn(s, __shfl_xor_sync(0xffffffffu, s, 2));
      if (t == 0) sm.mlw[warp][row] = make_float2(m[e], s);
#pragma unroll
      for (int d = 0; d < 16; ++d)
        *reinterpret_cast<float2*>(op + (warp * RP + row) * kTreeOPitch + 8 * d + 2 * t) =
            make_float2(o[d][2 * e], o[d][2 * e + 1]);
    }
  }
  __syncthreads();
  // the warps' partials into one per row: a warp a row, four dims a lane
  for (int r = warp; r < c.R && warp < 4; r += 4) {
    float M = -INFINITY, L = 0.0f;
#pragma unroll
    for (int k = 0; k < 4; ++k) M = fmaxf(M, sm.mlw[k][r].x);
    const float mu = M == -INFINITY ? 0.0f : M;
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 q = sm.mlw[k][r];
      const float f = ex2(__fsub_rn(q.x, mu));
      const float4 x = *reinterpret_cast<const float4*>(op + (k * RP + r) * kTreeOPitch + 4 * lane);
      L = __fmaf_rn(q.y, f, L);
      s.x = __fmaf_rn(x.x, f, s.x), s.y = __fmaf_rn(x.y, f, s.y);
      s.z = __fmaf_rn(x.z, f, s.z), s.w = __fmaf_rn(x.w, f, s.w);
    }
    if (odd) {
      const unsigned long long from = odd & sm.anc[r >> gl];
      s.x = tree_add_odd(a, c, from, 4 * lane, s.x), s.y = tree_add_odd(a, c, from, 4 * lane + 1, s.y);
      s.z = tree_add_odd(a, c, from, 4 * lane + 2, s.z), s.w = tree_add_odd(a, c, from, 4 * lane + 3, s.w);
    }
    *reinterpret_cast<float4*>(op + r * kTreeOPitch + 4 * lane) = s;
    if (lane == 0) sm.ml[r] = make_float2(M, L);
  }
  cluster_sync_all();
  tree_output(a, c, sm.ml, op);
  if (SCORED) {
    // each slot's softmax weights of the group's heads join its accumulator, in f32
    float M[8], I[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < G) {
        float L, f;
        tree_row_total(c, sm.ml, j, M[j], L, f);
        if (M[j] == -INFINITY) M[j] = 0.0f;
        I[j] = L == 0.0f ? 0.0f : __fdiv_rn(1.0f, L);
      }
    const int64_t w0 = c.b * a.w_stride + (int64_t)c.h * a.S, s0 = (int64_t)c.lo * kTreeTile;
    const int64_t span = (int64_t)(c.tiles - c.fresh) * kTreeTile, left = c.len - s0;
    const int held = (int)(left < span ? left : span), first = c.fresh * kTreeTile;
    for (int i0 = c.tid; i0 < held; i0 += 8 * kTreeThreads) {
      float w[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int i = i0 + k * kTreeThreads;
        if (i < held) w[k] = a.w_in[w0 + s0 + i];
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int i = i0 + k * kTreeThreads;
        if (i >= held) break;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j < G)
            w[k] = __fmaf_rn(ex2(__fmaf_rn(score[j * a.score_cap + first + i], kTreeLog2Scale, -M[j])), I[j], w[k]);
        a.w_out[w0 + s0 + i] = w[k];
      }
    }
    if (c.fresh && c.tid == 0) {  // the new slot starts with its own weight
      float w = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < G) w = __fmaf_rn(ex2(__fmaf_rn(score[j * a.score_cap], kTreeLog2Scale, -M[j])), I[j], w);
      a.w_out[w0 + c.len] = w;
      a.slot_pos[w0 + c.len] = (int32_t)c.pos;
    }
  }
  cluster_sync_all();  // peers read this CTA's shared memory until here
}

// ---------------------------------------------------------------- above 16 rows: tcgen05
// D[tmem] (+)= A[tmem] x B[smem desc], kind::f16 (f16 x f16 -> f32).
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc,
                                            uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t e;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
  return e != 0;
}
// 32 consecutive columns of this thread's TMEM lane to / from registers.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
      "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
      "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// V as the B operand: rows are keys (the contraction), 64 dims a 128-byte row, MN-major.  8 keys are
// 1024 bytes (the stride offset), the second 64 dims lie kTreeHalf / 2 behind (the leading offset).
__device__ __forceinline__ uint64_t tree_v_desc(uint32_t saddr) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr >> 4) & 0x3FFFu);
  d |= (uint64_t)((kTreeHalf / 2) >> 4) << 16;
  d |= (uint64_t)(1024u >> 4) << 32;
  d |= (uint64_t)1u << 46;
  d |= (uint64_t)2u << 61;
  return d;
}

// TMEM columns: S of even and of odd tiles (f32; the first half then holds the weights as f16 pairs,
// the A operand of O += P V), and O.  256 in all: two CTAs an SM.
constexpr uint32_t kTreeTmemCols = 256, kTreeTmemO = 128;
constexpr int kTreeTcThreads = 192;  // four softmax warps, a copying warp, an MMA warp
constexpr int kTreeMaxSlots = 3;     // K or V halves of tiles in flight
// Two CTAs an SM leave 113 KB each: the queries (ROWS rows, 64 or 128) and five or six halves.
template <int ROWS>
struct TreeTc {
  static constexpr int kSlots = 3, vSlots = ROWS == 64 ? 3 : 2;
  static constexpr int q_bytes = ROWS * 256;
  static constexpr int op_bytes = ROWS * kTreeOPitch * 4;  // partial outputs, over all of it at the end
  static constexpr int ring_bytes = (kSlots + vSlots) * kTreeHalf;
  static_assert(op_bytes + ROWS * 8 <= q_bytes + ring_bytes, "");
};

struct TreeTcSmem {  // behind the ring
  unsigned long long anc[kTreeMaxTokens];
  int up[kTreeMaxTokens];
  uint8_t odd[kTreeMaxTokens];
  uint64_t k_full[kTreeMaxSlots], k_empty[kTreeMaxSlots], v_full[kTreeMaxSlots], v_empty[kTreeMaxSlots];
  uint64_t s_full[2], p_full[2], o_done, tail;
  uint32_t tmem;
};
template <int ROWS>
constexpr size_t tree_tc_bytes() {
  return TreeTc<ROWS>::q_bytes + TreeTc<ROWS>::ring_bytes + sizeof(TreeTcSmem);
}
static_assert(tree_tc_bytes<128>() <= 233472 / 2 - 1024 && tree_tc_bytes<64>() <= 233472 / 2 - 1024, "two CTAs an SM");

// Up to 128 rows, M = 128 whatever the number (padding rows cost nothing that bounds it).  Roles:
//   copying warp  one thread streams the K and V halves of the tiles into the ring
//   MMA warp      one thread: S(j) = Q K^T (8 MMAs of 128 x 64 x 16) into one of two S buffers, then,
//                 when the weights of tile j - 1 are written, O += P V (4 of 128 x 128 x 16); so S(j)
//                 runs during the softmax of tile j - 1
//   softmax warps thread r holds row r: one TMEM lane, no shuffles.  O stays in TMEM; it is rescaled
//                 only when a row's maximum has grown by more than kTreeLazy since the last time (each
//                 time costs a pass over its 128 columns; sum and output share the reference)
// Measured: 64 tokens over 32749 slots 48.4 us (2.8 TB/s, 355 TFLOP/s).  128 CTAs on 114 SMs: preparation
// 7 to 9, then 33 tiles in 26 on an SM of its own (0.78 a tile) and in 31 beside another CTA (0.94), which
// 28 of them are and all wait for; merge and output 9 to 10 (time stamps, which add about 4 in all).
// 17 tokens x 16 sequences to 4001: 39.7 us (3.7 TB/s).
template <int ROWS>
__global__ void __launch_bounds__(kTreeTcThreads, 2) k_tree_tc(const __grid_constant__ TreeArgs a) {
  using L = TreeTc<ROWS>;
  constexpr int KD = L::kSlots, VD = L::vSlots;
  extern __shared__ __align__(1024) uint8_t smem_tc[];
  uint8_t* qs = smem_tc;  // [ROWS][128] f16; an A operand of 128 rows reads on into the ring
  uint8_t* kring = qs + L::q_bytes;
  uint8_t* vring = kring + KD * kTreeHalf;
  TreeTcSmem& sm = *reinterpret_cast<TreeTcSmem*>(vring + VD * kTreeHalf);
  float* op = reinterpret_cast<float*>(qs);                    // [ROWS][kTreeOPitch], at the end
  float2* ml = reinterpret_cast<float2*>(qs + L::op_bytes);    // [ROWS]
  if (smem_u32(smem_tc) & 1023u) {  // the swizzle goes by address bits; no launch here breaks it
    if (threadIdx.x == 0 && a.err) atomicCAS(a.err, 0, kErrTimeoutFull);
    return;
  }

  if (threadIdx.x == 128) prefetch_tmap(&a.km), prefetch_tmap(&a.vm);
  TreeCta c;
  tree_place(c);
  const TreeUnits<6, true> units(a, c);
  TreeRaw<4> raw;
  if (units.first < units.units) tree_load(a, c, units, units.first, raw);
  if (!tree_begin<false>(a, c)) return;
  const int gl = a.group_log2, row = c.tid, warp = c.warp, lane = c.lane;
  const uint32_t kr = smem_u32(kring), vr = smem_u32(vring);
  cluster_arrive();
  auto copy_k = [&](int j) {
    if (j < c.fresh) return;
    mbar_expect_tx(&sm.k_full[j % KD], kTreeHalf);
    tree_copy(c, &a.km, kr + (j % KD) * kTreeHalf, j, &sm.k_full[j % KD]);
  };
  auto copy_v = [&](int j) {  // with rows behind the cached slots: announced after these are zeroed
    if (j < c.fresh) return;
    uint64_t* bar = tree_left(c, j) < kTreeTile ? &sm.tail : &sm.v_full[j % VD];
    mbar_expect_tx(bar, kTreeHalf);
    tree_copy(c, &a.vm, vr + (j % VD) * kTreeHalf, j, bar);
  };
  if (c.tid == 128) {
    for (int i = 0; i < kTreeMaxSlots; ++i) {
      mbar_init(&sm.k_full[i], 1);
      mbar_init(&sm.k_empty[i], 1);
      mbar_init(&sm.v_full[i], 1);
      mbar_init(&sm.v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.s_full[i], 1);
      mbar_init(&sm.p_full[i], (c.R + 31) / 32);
    }
    mbar_init(&sm.o_done, 1);
    mbar_init(&sm.tail, 1);
    fence_mbar_init();
    for (int j = 0; j < KD && j < c.tiles; ++j) {
      copy_k(j);
      if (j < VD) copy_v(j);
    }
  }
  const bool tree_ok = tree_ancestors(a, c, sm.anc, sm.up);
  cluster_wait();
  if (!tree_ok) {
    if (c.tid == 128)
      for (int j = c.fresh; j < KD && j < c.tiles; ++j) {
        mbar_wait_own(&sm.k_full[j], 0, a.err, kErrTimeoutFull);
        if (j < VD) mbar_wait_own(tree_left(c, j) < kTreeTile ? &sm.tail : &sm.v_full[j], 0, a.err, kErrTimeoutFull);
      }
    return;
  }
  if (warp == 5) {
    __syncwarp();
    tmem_alloc(&sm.tmem, kTreeTmemCols);
    tmem_relinquish();
  }
  tree_rows<ROWS, 6, 4, true, false>(a, c, units, raw, sm.anc, qs, kring, vring, sm.odd);
  if (warp == 4 && c.fresh) tree_zero_tail(vring, c.n, lane);
  asm volatile("fence.proxy.async;" ::: "memory");  // queries and new rows, here or in a peer, go to MMAs
  tc_fence_before();
  if (c.C > 1) cluster_sync_all();
  else __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem;
  const bool live = warp * 32 < c.R;  // softmax warps of padding rows have nothing to do
  float m = -INFINITY, l = 0.0f, limit = -INFINITY;  // reference, sum, the score from which it is moved

  if (warp == 4) {
    // K runs KD - VD tiles ahead of V, whose slots are freed later
    fence_async_smem();
    bool ok = true;
    int j = 0, kj = KD;  // V tiles and K tiles begun
    for (; j < c.tiles; ++j) {
      if (j >= VD) {
        if (kj < c.tiles) {
          ok &= mbar_wait_own(&sm.k_empty[kj % KD], (kj / KD - 1) & 1, a.err, kErrTimeoutEmpty);
          if (!__all_sync(0xffffffffu, ok)) break;
          if (lane == 0) copy_k(kj);
          ++kj;
        }
        ok &= mbar_wait_own(&sm.v_empty[j % VD], (j / VD - 1) & 1, a.err, kErrTimeoutEmpty);
        if (!__all_sync(0xffffffffu, ok)) break;
        if (lane == 0) copy_v(j);
      }
      if (j < c.fresh) {
        if (lane == 0) {
          mbar_arrive(&sm.k_full[0]);
          mbar_arrive(&sm.v_full[0]);
        }
      } else if (tree_left(c, j) < kTreeTile) {
        mbar_wait_own(&sm.tail, 0, a.err, kErrTimeoutFull);
        tree_zero_tail(vring + (j % VD) * kTreeHalf, (int)tree_left(c, j), lane);
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.v_full[j % VD]);
      }
    }
    // the copies under way land before the memory is used again
    kj = min(kj, c.tiles);
    for (int i = max(kj - KD, 0); i < kj; ++i)
      mbar_wait_own(&sm.k_full[i % KD], (i / KD) & 1, a.err, kErrTimeoutFull);
    for (int i = max(j - VD, 0); i < j; ++i)
      mbar_wait_own(&sm.v_full[i % VD], (i / VD) & 1, a.err, kErrTimeoutFull);
  } else if (warp == 5) {
    // the whole warp runs the loop, so that descriptors stay in uniform registers (with one lane in
    // the loop, moving them there took 80 cycles an MMA); one lane issues
    constexpr uint32_t kIdS = idesc_f16_f32(128, kTreeTile);
    constexpr uint32_t kIdO = idesc_f16_f32(128, kHD) | (1u << 16);  // B is MN-major
    const uint64_t qd = sw128_desc(smem_u32(qs)), kd = sw128_desc(kr), vd = tree_v_desc(vr);
    const bool leader = elect_one();
    bool ok = true;
    int s = 0, sp = 0;            // slots of K of tile j and of V of tile j - 1
    uint32_t ph = 0, php = 0;     // their phases
    for (int j = 0; j <= c.tiles; ++j) {
      // the weights of tile j - 2 share the S buffer; and o_done may have one phase open at most, in the
      // last round too: a wait by parity takes a phase two behind for the one it is for
      if (j >= 2) ok &= mbar_wait_own(&sm.o_done, j & 1, a.err, kErrTimeoutFull);
      if (j < c.tiles) {
        ok &= mbar_wait_own(&sm.k_full[s], ph, a.err, kErrTimeoutFull);
        if (!__all_sync(0xffffffffu, ok)) break;
        tc_fence_after();
        if (leader) {
          const uint64_t kj = kd + (uint64_t)(s * (kTreeHalf >> 4));
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            umma_f16(tmem + (j & 1) * 64, qd + ((kk >> 2) * (ROWS * 128) + (kk & 3) * 32) / 16,
                     kj + ((kk >> 2) * (kTreeHalf / 2) + (kk & 3) * 32) / 16, kIdS, kk != 0);
          umma_commit(&sm.s_full[j & 1]);
          umma_commit(&sm.k_empty[s]);
        }
        __syncwarp();
      }
      if (j > 0) {
        const int i = j - 1;
        ok &= mbar_wait_own(&sm.v_full[sp], php, a.err, kErrTimeoutFull);
        ok &= mbar_wait_own(&sm.p_full[i & 1], (i >> 1) & 1, a.err, kErrTimeoutFull);
        if (!__all_sync(0xffffffffu, ok)) break;
        tc_fence_after();
        if (leader) {
          const uint64_t vi = vd + (uint64_t)(sp * (kTreeHalf >> 4));
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            umma_f16_ts(tmem + kTreeTmemO, tmem + (i & 1) * 64 + 8 * ks, vi + 2048 * ks / 16, kIdO, (i | ks) != 0);
          umma_commit(&sm.o_done);
          umma_commit(&sm.v_empty[sp]);
        }
        __syncwarp();
        if (++sp == VD) sp = 0, php ^= 1;
      }
      if (++s == KD) s = 0, ph ^= 1;
    }
    // nothing may be in flight when the TMEM goes
    if (c.tiles > 0) mbar_wait_own(&sm.o_done, (c.tiles - 1) & 1, a.err, kErrTimeoutFull);
    __syncwarp();
  } else if (live) {
    const uint32_t lane_base = tmem + ((uint32_t)(warp * 32) << 16);
    bool ok = true;
    for (int j = 0; j < c.tiles; ++j) {
      const uint32_t sa = lane_base + (j & 1) * 64;
      ok &= mbar_wait_own(&sm.s_full[j & 1], (j >> 1) & 1, a.err, kErrTimeoutFull);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      const bool fresh = j < c.fresh;
      const int64_t left = tree_left(c, j);
      const int nv = fresh ? c.n : (int)(left < kTreeTile ? left : kTreeTile);
      uint32_t u[64];
      tmem_ld32(sa, u);
      tmem_ld32(sa + 32, u + 32);
      tmem_wait_ld();
      if (fresh || nv < kTreeTile) {
        const unsigned long long see = tree_seen(c, sm.anc, fresh, row, nv, gl);
#pragma unroll
        for (int i = 0; i < 64; ++i)
          if (!((see >> i) & 1)) u[i] = 0xff800000u;
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < 64; ++i) mx[i & 3] = fmaxf(mx[i & 3], __uint_as_float(u[i]));
      const float top = __fmul_rn(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), kTreeLog2Scale);
      const bool grow = row < c.R && top > limit;  // from -inf: the first key that counts
      const float mn = grow ? tree_ref(top, kTreeTop - kTreeLazy) : m;
      if (grow) limit = __fadd_rn(top, kTreeLazy);
      const float mu = mn == -INFINITY ? 0.0f : mn;
      if (j > 0 && __any_sync(0xffffffffu, grow)) {
        ok &= mbar_wait_own(&sm.o_done, (j - 1) & 1, a.err, kErrTimeoutFull);
        if (!__all_sync(0xffffffffu, ok)) break;
        tc_fence_after();
        const float al = grow ? ex2(__fsub_rn(m, mu)) : 1.0f;
        l = __fmul_rn(l, al);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t x[32];
          tmem_ld32(lane_base + kTreeTmemO + 32 * i, x);
          tmem_wait_ld();
#pragma unroll
          for (int k = 0; k < 32; ++k) x[k] = __float_as_uint(__fmul_rn(__uint_as_float(x[k]), al));
          tmem_st32(lane_base + kTreeTmemO + 32 * i, x);
        }
      }
      m = mn;
      float sum[4] = {};
      uint32_t p[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const float p0 = ex2(__fmaf_rn(__uint_as_float(u[2 * i]), kTreeLog2Scale, -mu));
        const float p1 = ex2(__fmaf_rn(__uint_as_float(u[2 * i + 1]), kTreeLog2Scale, -mu));
        sum[i & 3] = __fadd_rn(sum[i & 3], __fadd_rn(p0, p1));
        p[i] = pack_h2(p0, p1);
      }
      l = __fadd_rn(l, __fadd_rn(__fadd_rn(sum[0], sum[1]), __fadd_rn(sum[2], sum[3])));
      tmem_st32(sa, p);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.p_full[j & 1]);
    }
  }
  __syncthreads();  // all MMAs and copies are done: the operands' memory becomes the partial outputs
  tc_fence_after();
  if (warp < 4 && live) {
    const uint32_t lane_base = tmem + ((uint32_t)(warp * 32) << 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t x[32];
      tmem_ld32(lane_base + kTreeTmemO + 32 * i, x);
      tmem_wait_ld();
      if (row < c.R) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          *reinterpret_cast<uint4*>(op + row * kTreeOPitch + 32 * i + 4 * k) =
              c.tiles > 0 ? make_uint4(x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3]) : make_uint4(0, 0, 0, 0);
      }
    }
    const unsigned long long odd = c.fresh ? tree_odd(c, sm.odd) : 0ull;
    if (row < c.R) {
      if (odd & sm.anc[row >> gl])
        for (int d = 0; d < kHD; ++d)
          op[row * kTreeOPitch + d] = tree_add_odd(a, c, odd & sm.anc[row >> gl], d, op[row * kTreeOPitch + d]);
      ml[row] = make_float2(m, l);
    }
  }
  tc_fence_before();
  cluster_sync_all();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem, kTreeTmemCols);
  }
  tree_output(a, c, ml, op);
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
  if (a.pos != nullptr) bad |= a.pos[b] < 0 || a.pos[b] > INT32_MAX - kTreeMaxTokens;  // slot_pos holds 32 bits
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
