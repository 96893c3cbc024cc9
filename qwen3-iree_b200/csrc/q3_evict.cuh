// q3_evict.cuh -- eviction from a KV cache by accumulated attention weight.
//
// Per (sequence, layer, kv head) with `len` cached slots and a budget M < len, the slots kept are the
// ones whose position is among the newest (position >= pos - recent), then those of the largest
// accumulated weight, ties going to the lower slot; M in all.  Attention does not depend on the order
// of the slots (RoPE is in the K rows), so nothing is compacted: the i-th kept slot at or behind M
// moves into the i-th hole below M.  Sources and destinations are disjoint, and the weights and
// positions go to arrays of their own, so no CTA ever waits for another.
//
// Bound: the moved rows, 512 bytes read and 512 written each.  Every CTA selects for itself (the
// weights of one head are a few KB, from L2) and moves its share of the rows.
//
// Selection: keys are the weights' bits in an order-preserving form, above them all the newest.  A
// histogram of their top 11 bits gives the bin of the M-th largest; its keys, some tens, are ranked by
// counting, or by two more histograms where there are many.  Ballots then give each slot's fate and its
// rank in slot order.  28 layers of 1024 slots, 512 kept: selection 8 us, moves 8 (at the copy rate).
// Small CTAs, many to an SM, so that some select while others move.
#pragma once

#include "q3_common.cuh"

namespace q3 {

constexpr int kEvictThreads = 256;
constexpr int kEvictWarps = kEvictThreads / 32;
constexpr int kEvictBins = 2048;
constexpr int kEvictWindow = 512;  // moves listed in shared memory at a time, or candidates ranked
constexpr int64_t kEvictMaxSlots = 524288;
constexpr int kEvictKeySlots = 32768;  // up to here the keys are held in shared memory

struct EvictArgs {
  uint16_t* k;  // layer0 of sequence 0
  uint16_t* v;
  int64_t seq_stride, layer_stride, slot_stride, head_stride;
  int64_t S;
  int kv_heads;
  int64_t budget, recent;
  const int64_t* len;
  const int64_t* pos;
  const float* w;  // layer0 of sequence 0: [B][layers][kv_heads][S]
  const int32_t* sp;
  int64_t w_stride;  // between sequences
  int64_t* new_len;
  float* new_w;
  int32_t* new_sp;
  int* err;
};

struct EvictSmem {
  uint32_t hist[kEvictBins];
  uint32_t warp_sum[kEvictWarps + 1];
  uint32_t digit, above, count, listed;
  int src[kEvictWindow], dst[kEvictWindow];
};

__host__ __device__ inline size_t evict_smem_bytes(int64_t S) {
  const size_t words = (size_t)((S + 31) / 32);
  return sizeof(EvictSmem) + 8 * words + (S <= kEvictKeySlots ? 4 * (size_t)S : 0);
}

// Order-preserving bits: larger key, more worth keeping.  0 is a NaN, all ones a newest slot.
__device__ __forceinline__ uint32_t evict_key(float w, int32_t p, int64_t newest) {
  if (p >= newest) return 0xffffffffu;
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(__fadd_rn(w, 0.0f));  // -0 ties with 0
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Exclusive prefix of v over the CTA's threads; *total: the sum.  `s` holds kEvictWarps + 1 words.
__device__ __forceinline__ uint32_t evict_scan(uint32_t v, uint32_t* s, uint32_t* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) s[warp] = x;
  __syncthreads();
  if (warp == 0) {
    uint32_t y = lane < kEvictWarps ? s[lane] : 0u;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t z = __shfl_up_sync(0xffffffffu, y, o);
      if (lane >= o) y += z;
    }
    if (lane < kEvictWarps) s[lane] = y;
  }
  __syncthreads();
  const uint32_t r = x - v + (warp ? s[warp - 1] : 0u);
  *total = s[kEvictWarps - 1];
  __syncthreads();
  return r;
}

__global__ void __launch_bounds__(kEvictThreads, 6) k_cache_evict(const EvictArgs a) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  EvictSmem& sm = *reinterpret_cast<EvictSmem*>(smem_raw);
  const int words_max = (int)((a.S + 31) / 32);
  uint32_t* bits = reinterpret_cast<uint32_t*>(smem_raw + sizeof(EvictSmem));  // holes and movers
  uint32_t* pre = bits + words_max;                                           // their rank per word
  uint32_t* keys = pre + words_max;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.z, layer = blockIdx.y / a.kv_heads, h = blockIdx.y - layer * a.kv_heads;
  const int64_t len64 = a.len[b];
  const int64_t pos = a.pos[b], newest = pos - a.recent;
  const bool bad = len64 < 0 || len64 > a.S || pos < 0;
  const int len = bad ? 0 : (int)len64;
  const int M = (int)a.budget, held = len < M ? len : M;
  if (blockIdx.x == 0 && blockIdx.y == 0 && tid == 0) {
    a.new_len[b] = bad ? len64 : held;
    if (bad && a.err) atomicCAS(a.err, 0, kErrBadPos);
  }
  if (bad) return;
  const int64_t w0 = b * a.w_stride + ((int64_t)layer * a.kv_heads + h) * a.S;
  const float* w = a.w + w0;
  const int32_t* sp = a.sp + w0;
  float* nw = a.new_w + w0;
  int32_t* np = a.new_sp + w0;
  const int X = gridDim.x, x = blockIdx.x;
  const int c0 = (int)((int64_t)held * x / X), c1 = (int)((int64_t)held * (x + 1) / X);
  if (len <= M) {
    for (int j = c0 + tid; j < c1; j += kEvictThreads) nw[j] = w[j], np[j] = sp[j];
    return;
  }
  const bool stored = a.S <= kEvictKeySlots;
  auto key_at = [&](int j) { return stored ? keys[j] : evict_key(w[j], sp[j], newest); };

  // the M-th largest key: digits of 11, 11 and 10 bits, from the top
  constexpr int kPer = kEvictBins / kEvictThreads;
  uint32_t prefix = 0, want = (uint32_t)M, ties = 0;
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const uint32_t mask = pass == 2 ? 1023u : 2047u;
    for (int i = tid; i < kEvictBins; i += kEvictThreads) sm.hist[i] = 0;
    if (tid == 0) sm.listed = 0;
    __syncthreads();
    if (pass == 0) {
      for (int j0 = tid; j0 < len; j0 += 4 * kEvictThreads) {
        float wv[4];
        int32_t pv[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int j = min(j0 + k * kEvictThreads, len - 1);
          wv[k] = w[j], pv[k] = sp[j];
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int j = j0 + k * kEvictThreads;
          if (j >= len) break;
          const uint32_t key = evict_key(wv[k], pv[k], newest);
          if (stored) keys[j] = key;
          atomicAdd(&sm.hist[key >> 21], 1u);
        }
      }
    } else {
      for (int j = tid; j < len; j += kEvictThreads) {
        const uint32_t key = key_at(j);
        if ((pass == 1 ? key >> 21 : key >> 10) == prefix) atomicAdd(&sm.hist[(key >> shift) & mask], 1u);
      }
    }
    __syncthreads();
    // thread i: kPer bins from the top; the bin where the count from above reaches `want`
    const int top = kEvictBins - 1 - kPer * tid;
    uint32_t c[kPer], s = 0, total;
#pragma unroll
    for (int i = 0; i < kPer; ++i) c[i] = sm.hist[top - i], s += c[i];
    uint32_t over = evict_scan(s, sm.warp_sum, &total);
    if (over < want && want <= over + s) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        if (over < want && want <= over + c[i]) sm.digit = top - i, sm.above = over, sm.count = c[i];
        over += c[i];
      }
    }
    __syncthreads();
    prefix = (prefix << (pass == 2 ? 10 : 11)) | sm.digit;
    want -= sm.above;
    ties = sm.count;
    __syncthreads();
    if (pass == 0 && ties <= (uint32_t)kEvictWindow) {
      // few keys in the bin: list them, and count for each the larger and the equal ones
      uint32_t* cand = reinterpret_cast<uint32_t*>(sm.src);
      for (int j = tid; j < len; j += kEvictThreads) {
        const uint32_t key = key_at(j);
        if (key >> 21 == prefix) cand[atomicAdd(&sm.listed, 1u)] = key;
      }
      __syncthreads();
      const uint32_t n = ties;
      for (uint32_t i = tid; i < n; i += kEvictThreads) {
        const uint32_t mine = cand[i];
        uint32_t more = 0, same = 0;
#pragma unroll 4
        for (uint32_t k = 0; k < n; ++k) more += cand[k] > mine, same += cand[k] == mine;
        if (more < want && want <= more + same) sm.digit = mine, sm.above = more, sm.count = same;  // all ties alike
      }
      __syncthreads();
      prefix = sm.digit;
      want -= sm.above;
      ties = sm.count;
      __syncthreads();
      break;
    }
  }
  const uint32_t kth = prefix;  // `want` of its `ties` slots stay

  // each warp owns a run of 32-slot words: count ties, then fates and ranks
  const int words = (len + 31) / 32, per = (words + kEvictWarps - 1) / kEvictWarps;
  const int wa = min(words, warp * per), wb = min(words, wa + per);
  uint32_t tie_rank = 0, total;
  if (want < ties) {
    uint32_t mine = 0;
    for (int q = wa; q < wb; ++q) {
      const int j = q * 32 + lane;
      mine += __popc(__ballot_sync(0xffffffffu, j < len && key_at(j) == kth));
    }
    tie_rank = evict_scan(lane == 0 ? mine : 0u, sm.warp_sum, &total);
    tie_rank = __shfl_sync(0xffffffffu, tie_rank, 0);
  }
  uint32_t mine = 0;
  const bool partly = want < ties;  // some of the ties go: their order counts
  for (int q = wa; q < wb; ++q) {
    const int j = q * 32 + lane;
    const uint32_t key = j < len ? key_at(j) : 0u;
    bool keep = key >= kth;
    if (partly) {
      const uint32_t eqs = __ballot_sync(0xffffffffu, j < len && key == kth);
      keep = key > kth || (key == kth && tie_rank + __popc(eqs & ((1u << lane) - 1)) < want);
      tie_rank += __popc(eqs);
    }
    const uint32_t sel = __ballot_sync(0xffffffffu, j < len && (j < M) != keep);
    if (lane == 0) bits[q] = sel, pre[q] = mine;
    mine += __popc(sel);
  }
  uint32_t base = evict_scan(lane == 0 ? mine : 0u, sm.warp_sum, &total);
  base = __shfl_sync(0xffffffffu, base, 0);
  for (int q = wa + lane; q < wb; q += 32) pre[q] += base;
  __syncthreads();
  const int H = (int)(total / 2);  // holes below M, and as many kept slots behind

  for (int j0 = c0 + tid; j0 < c1; j0 += 4 * kEvictThreads) {
    float wv[4];
    int32_t pv[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int j = min(j0 + k * kEvictThreads, c1 - 1);
      wv[k] = w[j], pv[k] = sp[j];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int j = j0 + k * kEvictThreads;
      if (j < c1 && !((bits[j >> 5] >> (j & 31)) & 1)) nw[j] = wv[k], np[j] = pv[k];
    }
  }

  const int m0 = (int)((int64_t)H * x / X), m1 = (int)((int64_t)H * (x + 1) / X);
  const int64_t off = b * a.seq_stride + layer * a.layer_stride + h * a.head_stride + (lane & 15) * 8;
  uint16_t* row = (lane < 16 ? a.k : a.v) + off;
  for (int r0 = m0; r0 < m1; r0 += kEvictWindow) {
    const int r1 = min(m1, r0 + kEvictWindow);
    for (int j = tid; j < len; j += kEvictThreads) {
      const uint32_t f = bits[j >> 5] >> (j & 31);
      if (!(f & 1)) continue;
      const int rank = (int)pre[j >> 5] + __popc(bits[j >> 5] & ((1u << (j & 31)) - 1));
      const int r = j < M ? rank : rank - H;
      if (r >= r0 && r < r1) (j < M ? sm.dst : sm.src)[r - r0] = j;
    }
    __syncthreads();
    const int n = r1 - r0;
    for (int i0 = warp * 4; i0 < n; i0 += kEvictWarps * 4) {
      uint4 val[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i0 + i < n) val[i] = __ldcs(reinterpret_cast<const uint4*>(row + sm.src[i0 + i] * a.slot_stride));
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i0 + i < n) __stcs(reinterpret_cast<uint4*>(row + sm.dst[i0 + i] * a.slot_stride), val[i]);
    }
    for (int i = tid; i < n; i += kEvictThreads) nw[sm.dst[i]] = w[sm.src[i]], np[sm.dst[i]] = sp[sm.src[i]];
    __syncthreads();
  }
}

}  // namespace q3
