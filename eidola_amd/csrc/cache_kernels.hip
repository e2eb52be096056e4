// gfx950 kernels that thin a paged cache out: attention weight received per cached key, choice of
// the rows that stay, move of the rows that stay.
#include "eid_cache_params.h"
#include "eid_device.h"

namespace eid {

namespace {

typedef const __attribute__((address_space(4))) int32_t *const_i32_ptr;
__device__ __forceinline__ const_i32_ptr as_constant(const int32_t *p) { return (const_i32_ptr)(uintptr_t)p; }
__device__ __forceinline__ int clamp_id(const int id, const int last) { return min(max(id, 0), last); }

struct ScoreSeq {
  int row0, qlen, len;
};
__device__ __forceinline__ ScoreSeq score_seq(const ScoreParams &p, const int s) {
  ScoreSeq v;
  const const_i32_ptr cu = as_constant(p.cu_seqlens_q), sl = as_constant(p.seq_lens);
  v.row0 = cu[s];
  v.qlen = cu[s + 1] - v.row0;
  v.len = min(sl[s], p.max_blocks_per_seq * kBlock);
  if (v.qlen < 0 || v.len < v.qlen || v.row0 < 0 || v.row0 + v.qlen > p.num_q_tokens) v.qlen = 0;
  return v;
}

// K operand of 16 keys (one page) of a head: lane (key i16, segment g) holds elements 16 g .. 16 g + 15
template <bool FP8>
__device__ __forceinline__ void load_k(const uint8_t *base, const uint32_t row_bytes, Frag8 (&kf)[2]) {
  const int lane = threadIdx.x & 63, i16 = lane & 15, g = lane >> 4;
  const uint8_t *src = base + (uint32_t)i16 * row_bytes + g * (FP8 ? 16 : 32);
  if constexpr (FP8) {
    const u32x4 r = *(const u32x4 *)src;
    fp8x8_to_bf16x8(r[0], r[1], kf[0].w);
    fp8x8_to_bf16x8(r[2], r[3], kf[1].w);
  } else {
    kf[0].u = *(const u32x4 *)src;
    kf[1].u = *(const u32x4 *)(src + 16);
  }
}

// 16 rows of q (two tokens x 8 heads) from token `tok` of the sequence on, and what the rows'
// exponents take off: lse in log2 units; +inf where there is no row (its weights are then 0).
__device__ __forceinline__ void load_rows(const ScoreParams &p, const ScoreSeq &v, const int kvh, const int tok,
                                          Frag8 (&qf)[2], f32x4 &off) {
  const int lane = threadIdx.x & 63, i16 = lane & 15, g = lane >> 4;
  const int tq = tok + (i16 >> 3), tl = tok + (g >> 1);
  qf[0].u = qf[1].u = u32x4{0, 0, 0, 0};
  if (tq < v.qlen) {
    const uint16_t *src = p.q + ((size_t)(v.row0 + tq) * p.num_q_heads + kvh * kGroup + (i16 & 7)) * kHeadDim + 16 * g;
    qf[0].u = *(const u32x4 *)src;
    qf[1].u = *(const u32x4 *)(src + 8);
  }
  off = f32x4{INFINITY, INFINITY, INFINITY, INFINITY};
  if (tl < v.qlen) {
    const f32x4 e = *(const f32x4 *)(p.lse + (size_t)(v.row0 + tl) * p.num_q_heads + kvh * kGroup + 4 * (g & 1));
#pragma unroll
    for (int r = 0; r < 4; ++r) off[r] = e[r] == -INFINITY ? INFINITY : e[r] * kLog2e;  // (a row that saw nothing)
  }
}

// Weights of 16 keys from 16 rows, summed over the lane's four rows.  D of Q K^T: lane (key i16,
// rows 4 g + r); rows 8 and up belong to the second token.
__device__ __forceinline__ float weights(const Frag8 (&qf)[2], const Frag8 (&kf)[2], const f32x4 off, const float c2,
                                         const bool see) {
  f32x4 S = mfma16x32(qf[0], kf[0], f32x4{0.f, 0.f, 0.f, 0.f});
  S = mfma16x32(qf[1], kf[1], S);
  float w = 0.f;
#pragma unroll
  for (int r = 0; r < 4; ++r) w += fast_exp2(__builtin_fmaf(S[r], c2, -off[r]));
  return see ? w : 0.f;
}

constexpr int kScoreFewRows = 2;  // q_len that the few-rows kernel takes

// ---------------------------------------------------------------------------------------
// score[j] = (key j is new ? 0 : score[j]) + sum over rows i and the group's heads of
// vis(i, j) e^(c q.k_j - lse_i).
//
// Sequences of one or two rows: bound by reading K.  A wave takes 64 keys of one KV head; the
// workgroup's waves take neighbouring heads of the same keys, so that whole pages are read at
// once.  grid = (chunks, sequences, head groups).
// ---------------------------------------------------------------------------------------
template <bool FP8>
__global__ __launch_bounds__(512) void score_few_kernel(const ScoreParams p) {
  const int lane = threadIdx.x & 63, i16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int s = blockIdx.y, kvh = blockIdx.z * (blockDim.x >> 6) + wave;
  const ScoreSeq v = score_seq(p, s);
  const int tc = blockIdx.x * kChunk;
  if (v.qlen < 1 || v.qlen > kScoreFewRows || tc >= v.len || kvh >= p.num_kv_heads) return;
  const int prefix = v.len - v.qlen;
  const const_i32_ptr bt = as_constant(p.block_table + (size_t)s * p.max_blocks_per_seq);
  const int last_page = (v.len - 1) / kBlock;
  const uint32_t row_bytes = (uint32_t)p.num_kv_heads * kHeadDim * (FP8 ? 1 : 2);
  const float c2 = p.softmax_scale * kLog2e * (FP8 ? p.k_scale[kvh] : 1.0f);
  Frag8 qf[2], kf[4][2];
  f32x4 off;
  int page[4];
#pragma unroll
  for (int b = 0; b < 4; ++b) page[b] = clamp_id(bt[min(tc / kBlock + b, last_page)], p.last_block);
#pragma unroll
  for (int b = 0; b < 4; ++b)
    load_k<FP8>(p.k_cache + (size_t)page[b] * kBlock * row_bytes + (size_t)kvh * kHeadDim * (FP8 ? 1 : 2), row_bytes, kf[b]);
  load_rows(p, v, kvh, 0, qf, off);
  float mine = 0.f;
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    const int j = tc + b * kBlock + i16, pos = prefix + (g >> 1);
    const bool see = j <= pos && (p.window <= 0 || pos - j < p.window);
    const float w = rowgroup_sum(weights(qf, kf[b], off, c2, see));
    mine = g == b ? w : mine;  // lane (i16, g) keeps key i16 of page g
  }
  const int j = tc + g * kBlock + i16;
  if (j < v.len) {
    const int pg = g == 0 ? page[0] : g == 1 ? page[1] : g == 2 ? page[2] : page[3];
    float *dst = p.scores + ((size_t)pg * p.num_kv_heads + kvh) * kBlock + i16;
    *dst = (j >= prefix ? 0.f : *dst) + mine;
  }
}

// ---------------------------------------------------------------------------------------
// Sequences of more rows: bound by the products and exponentials.  A workgroup owns 64 KT keys of
// one KV head (held as operands by every wave) and its waves share out the rows; no two
// workgroups touch one key, so the sums need no atomics and have one order.
// ---------------------------------------------------------------------------------------
constexpr int kScoreWaves = 8;
constexpr int kScorePages = 8;  // pages of keys per workgroup
template <bool FP8>
__global__ __launch_bounds__(kScoreWaves * 64) void score_rows_kernel(const ScoreParams p) {
  const int lane = threadIdx.x & 63, i16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kvh = blockIdx.x % p.num_kv_heads, tc = blockIdx.x / p.num_kv_heads * (kScorePages * kBlock);
  const int s = blockIdx.y;
  const ScoreSeq v = score_seq(p, s);
  if (v.qlen <= kScoreFewRows || tc >= v.len) return;
  __shared__ float part[kScoreWaves][kScorePages * kBlock];
  const int prefix = v.len - v.qlen;
  const const_i32_ptr bt = as_constant(p.block_table + (size_t)s * p.max_blocks_per_seq);
  const int last_page = (v.len - 1) / kBlock;
  const uint32_t row_bytes = (uint32_t)p.num_kv_heads * kHeadDim * (FP8 ? 1 : 2);
  const float c2 = p.softmax_scale * kLog2e * (FP8 ? p.k_scale[kvh] : 1.0f);
  Frag8 kf[kScorePages][2];
#pragma unroll
  for (int b = 0; b < kScorePages; ++b) {
    const int page = clamp_id(bt[min(tc / kBlock + b, last_page)], p.last_block);
    load_k<FP8>(p.k_cache + (size_t)page * kBlock * row_bytes + (size_t)kvh * kHeadDim * (FP8 ? 1 : 2), row_bytes, kf[b]);
  }
  const int key_end = min(tc + kScorePages * kBlock, v.len);
  // rows that see any of these keys: positions tc .. key_end - 1 + window - 1
  int i0 = max(0, tc - prefix) & ~1;
  int i1 = v.qlen;
  if (p.window > 0) i1 = (int)min((long long)i1, (long long)key_end - 1 + p.window - prefix);
  float sum[kScorePages];
#pragma unroll
  for (int b = 0; b < kScorePages; ++b) sum[b] = 0.f;
  for (int i = i0 + 2 * wave; i < i1; i += 2 * kScoreWaves) {
    Frag8 qf[2];
    f32x4 off;
    load_rows(p, v, kvh, i, qf, off);
    const int pos = prefix + i + (g >> 1);
    const bool edge = prefix + i < key_end - 1 || (p.window > 0 && prefix + i + 1 - tc >= p.window);
    if (edge) {
#pragma unroll
      for (int b = 0; b < kScorePages; ++b) {
        const int j = tc + b * kBlock + i16;
        sum[b] += weights(qf, kf[b], off, c2, j <= pos && (p.window <= 0 || pos - j < p.window));
      }
    } else {
#pragma unroll
      for (int b = 0; b < kScorePages; ++b) sum[b] += weights(qf, kf[b], off, c2, true);
    }
  }
#pragma unroll
  for (int b = 0; b < kScorePages; ++b) {
    const float w = rowgroup_sum(sum[b]);
    if (g == 0) part[wave][b * kBlock + i16] = w;
  }
  __syncthreads();
  const int x = threadIdx.x;
  if (x < kScorePages * kBlock && tc + x < v.len) {
    float w = 0.f;
#pragma unroll
    for (int k = 0; k < kScoreWaves; ++k) w += part[k][x];
    const int page = clamp_id(p.block_table[(size_t)s * p.max_blocks_per_seq + (tc + x) / kBlock], p.last_block);
    float *dst = p.scores + ((size_t)page * p.num_kv_heads + kvh) * kBlock + (x & 15);
    *dst = (tc + x >= prefix ? 0.f : *dst) + w;
  }
}

// ---------------------------------------------------------------------------------------
// Rows to keep.  A workgroup per (sequence, KV head) finds the score of the last row that stays
// by radix selection over order-preserving keys, 8 bits a pass, then writes the rows in order: a
// thread counts a run of consecutive rows, one scan over the workgroup gives it its places.
//
// Sequences of up to 32 rows per thread are read once, into LDS (four words of padding after every
// 32 keep the threads' runs on different banks), and all passes work there; longer ones are read
// again by every pass.  Eight copies of the histogram: lanes with equal digits, the usual case in
// the first pass, do not queue on one address.
// ---------------------------------------------------------------------------------------
// larger = kept first; NaN lowest, -0 = +0
__device__ __forceinline__ uint32_t order_key(const float x) {
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x == 0.f ? 0.f : x);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
constexpr int kSelRun = 32;  // rows per thread of the LDS path
constexpr int kSelCopies = 8;

template <int THREADS>
__global__ __launch_bounds__(THREADS) void select_kernel(const SelectParams p) {
  constexpr int kWaves = THREADS / 64, kCap = THREADS * kSelRun;
  __shared__ __align__(16) uint32_t keys[kCap + kCap / 32 * 4];
  __shared__ uint32_t hist[256 * kSelCopies];
  __shared__ uint32_t wave_sum[kWaves];
  __shared__ uint32_t found[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int s = blockIdx.x / p.num_kv_heads, kvh = blockIdx.x % p.num_kv_heads;
  const int len = max(0, min(p.seq_lens[s], p.max_blocks_per_seq * kBlock));
  const int budget = p.budget;
  int32_t *keep = p.keep + (size_t)blockIdx.x * budget;
  if (kvh == 0 && tid == 0) p.counts[s] = min(len, budget);
  if (len <= budget) {
    for (int i = tid; i < budget; i += THREADS) keep[i] = i < len ? i : -1;
    return;
  }
  const int32_t *bt = p.block_table + (size_t)s * p.max_blocks_per_seq;
  const int lo = p.keep_first, hi = len - p.keep_last;  // candidates: lo <= j < hi
  const int quads = (len + 3) / 4;                      // four rows of one page
  const bool in_lds = len <= kCap;
  auto page_of = [&](const int q) { return clamp_id(bt[min(q, quads - 1) >> 2], p.last_block); };
  auto quad_at = [&](const int page, const int q) {
    return *(const f32x4 *)(p.scores + ((size_t)page * p.num_kv_heads + kvh) * kBlock + 4 * (q & 3));
  };
  auto slot = [](const int q) { return 4 * q + (q >> 3) * 4; };
  // f(j, key) for the rows of all quads q = tid, tid + THREADS, ... (any order of the workgroup)
  auto for_rows = [&](auto f) {
    if (in_lds) {
      for (int q = tid; q < quads; q += THREADS) {
        const u32x4 k = *(const u32x4 *)&keys[slot(q)];
#pragma unroll
        for (int e = 0; e < 4; ++e) f(4 * q + e, k[e]);
      }
    } else {
      for (int q0 = tid; q0 < quads; q0 += 4 * THREADS) {
        int page[4];
        f32x4 x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) page[i] = page_of(q0 + i * THREADS);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = quad_at(page[i], q0 + i * THREADS);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (q0 + i * THREADS < quads)
#pragma unroll
            for (int e = 0; e < 4; ++e) f(4 * (q0 + i * THREADS) + e, order_key(x[i][e]));
      }
    }
  };
  if (in_lds) {
    constexpr int kQ = kSelRun / 4;
    int page[kQ];
    f32x4 x[kQ];
#pragma unroll
    for (int i = 0; i < kQ; ++i)
      if (i * THREADS < quads) page[i] = page_of(tid + i * THREADS);
#pragma unroll
    for (int i = 0; i < kQ; ++i)
      if (i * THREADS < quads) x[i] = quad_at(page[i], tid + i * THREADS);
#pragma unroll
    for (int i = 0; i < kQ; ++i)
      if (tid + i * THREADS < quads) {
        u32x4 k;
#pragma unroll
        for (int e = 0; e < 4; ++e) k[e] = order_key(x[i][e]);
        *(u32x4 *)&keys[slot(tid + i * THREADS)] = k;
      }
  }
  for (int i = tid; i < 256 * kSelCopies; i += THREADS) hist[i] = 0;
  __syncthreads();

  uint32_t want = (uint32_t)(budget - p.keep_first - p.keep_last);  // candidates to keep
  uint32_t prefix = 0;
  if (want > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      for_rows([&](const int j, const uint32_t k) {
        if (j >= lo && j < hi && (shift == 24 || ((k ^ prefix) >> (shift + 8)) == 0))
          atomicAdd(&hist[(k >> shift & 255) * kSelCopies + (lane & (kSelCopies - 1))], 1u);
      });
      __syncthreads();
      // counts of the digits from the highest down: thread d holds digit 255 - d
      uint32_t n = 0;
      if (tid < 256) {
        uint32_t *h = &hist[(255 - tid) * kSelCopies];
#pragma unroll
        for (int c = 0; c < kSelCopies; ++c) {
          n += h[c];
          h[c] = 0;  // for the next pass
        }
      }
      uint32_t incl = n;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const uint32_t o = __shfl_up(incl, d);
        if (lane >= d) incl += o;
      }
      if (tid < 256 && lane == 63) wave_sum[wave] = incl;
      __syncthreads();
      if (tid < 256) {
        for (int w = 0; w < wave; ++w) incl += wave_sum[w];
        if (incl >= want && incl - n < want) {
          found[0] = (uint32_t)(255 - tid);
          found[1] = incl - n;  // candidates above this digit
        }
      }
      __syncthreads();
      prefix |= found[0] << shift;
      want -= found[1];
    }
  }
  for (int i = tid; i < p.keep_first; i += THREADS) keep[i] = i;
  for (int i = tid; i < p.keep_last; i += THREADS) keep[budget - p.keep_last + i] = hi + i;
  if (budget == p.keep_first + p.keep_last) return;
  // keys above `prefix` stay, and the first `want` of those equal to it.  Blocks of kCap rows (one,
  // where the rows are in LDS), a run of consecutive rows per thread.
  uint32_t base = (uint32_t)p.keep_first, ties = 0;  // rows written, ties passed
  for (int q_base = 0; q_base < quads; q_base += kCap / 4) {
    const int here = min(quads - q_base, kCap / 4);
    const int run = (here + THREADS - 1) / THREADS;  // quads per thread
    const int q0 = min(tid * run, here), q1 = min(q0 + run, here);
    auto keys_of = [&](const int q) {
      u32x4 k;
      if (in_lds) {
        k = *(const u32x4 *)&keys[slot(q)];
      } else {
        const f32x4 x = quad_at(page_of(q_base + q), q_base + q);
#pragma unroll
        for (int e = 0; e < 4; ++e) k[e] = order_key(x[e]);
      }
      return k;
    };
    uint32_t count = 0;  // rows above in the low half, ties in the high half (at most kCap <= 32768 each)
    for (int q = q0; q < q1; ++q) {
      const u32x4 k = keys_of(q);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = 4 * (q_base + q) + e;
        if (j >= lo && j < hi) count += k[e] > prefix ? 1u : k[e] == prefix ? 0x10000u : 0u;
      }
    }
    uint32_t incl = count;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t o = __shfl_up(incl, d);
      if (lane >= d) incl += o;
    }
    __syncthreads();  // (the last use of wave_sum)
    if (lane == 63) wave_sum[wave] = incl;
    __syncthreads();
    uint32_t mine = incl - count, all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      if (w < wave) mine += wave_sum[w];
      all += wave_sum[w];
    }
    uint32_t t = ties + (mine >> 16);  // ties before this thread's run
    uint32_t at = base + (mine & 0xFFFFu) + (min(t, want) - min(ties, want));
    for (int q = q0; q < q1; ++q) {
      const u32x4 k = keys_of(q);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = 4 * (q_base + q) + e;
        if (j < lo || j >= hi) continue;
        if (k[e] > prefix || (k[e] == prefix && t < want)) keep[at++] = j;
        t += k[e] == prefix ? 1u : 0u;
      }
    }
    base += (all & 0xFFFFu) + (min(ties + (all >> 16), want) - min(ties, want));
    ties += all >> 16;
  }
}

// ---------------------------------------------------------------------------------------
// row start + i <- row keep[i], i ascending, keep[i] >= start + i.  In place: a workgroup owns a
// column of the sequence (one KV head, or eight where all heads keep the same rows) in one tensor
// of one layer and moves it in steps; a step's rows are all in registers before its first
// store, and later steps read only rows behind everything that this one overwrites.
// ---------------------------------------------------------------------------------------
__device__ __forceinline__ void step_loaded() {
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's rows are in registers
  __syncthreads();                     // ... and every wave's
}

template <int THREADS>
__global__ __launch_bounds__(THREADS) void compact_kernel(const CompactParams p, const int heads) {
  constexpr int R = 8;
  const int tid = threadIdx.x;
  const int groups = p.num_kv_heads / heads;
  const int tensors = p.has_scores ? 3 : 2;
  int b = blockIdx.x;
  const int hg = b % groups;
  b /= groups;
  const int what = b % tensors, s = b / tensors, layer = blockIdx.y;
  const int start = p.starts ? p.starts[s] : 0;
  const int len = max(0, min(p.seq_lens[s], p.max_blocks_per_seq * kBlock));
  const int n = min(min(p.counts[s], p.max_rows), len - start);
  if (start < 0 || n <= 0) return;
  const int32_t *keep = p.keep + (size_t)layer * p.keep_layer + (size_t)s * p.keep_seq + (size_t)hg * heads * p.keep_head;
  const int32_t *bt = p.block_table + (size_t)s * p.max_blocks_per_seq;
  if (what < 2) {
    uint8_t *base = what ? p.v[layer] : p.k[layer];
    const int lanes = heads * kHeadDim * p.elt / 16;  // 16-byte lanes of a row: 4 .. 64
    const uint32_t row_bytes = (uint32_t)p.num_kv_heads * kHeadDim * p.elt;
    const uint32_t col = (uint32_t)hg * heads * kHeadDim * p.elt + (tid % lanes) * 16;
    const int per = THREADS / lanes, r0 = tid / lanes;
    auto addr = [&](const int row) {
      const int page = clamp_id(bt[row / kBlock], p.last_block);
      return (size_t)page * kBlock * row_bytes + (size_t)(row & 15) * row_bytes + col;
    };
    for (int i0 = 0; i0 < n; i0 += per * R) {
      u32x4 x[R];
      bool move[R];
#pragma unroll
      for (int k = 0; k < R; ++k) {
        const int i = i0 + k * per + r0;
        const int src = i < n ? keep[i] : -1;
        move[k] = src > start + i && src < len;  // (a row that stays in place is not touched)
        if (move[k]) x[k] = *(const u32x4 *)(base + addr(src));
      }
      step_loaded();
#pragma unroll
      for (int k = 0; k < R; ++k)
        if (move[k]) *(u32x4 *)(base + addr(start + i0 + k * per + r0)) = x[k];
    }
  } else {
    float *base = p.scores[layer];
    for (int i0 = 0; i0 < n; i0 += THREADS / heads * R) {
      const int per = THREADS / heads, h = hg * heads + tid % heads, r0 = tid / heads;
      auto addr = [&](const int row) {
        return ((size_t)clamp_id(bt[row / kBlock], p.last_block) * p.num_kv_heads + h) * kBlock + (row & 15);
      };
      float x[R];
      bool move[R];
#pragma unroll
      for (int k = 0; k < R; ++k) {
        const int i = i0 + k * per + r0;
        const int src = i < n ? keep[i] : -1;
        move[k] = src > start + i && src < len;
        if (move[k]) x[k] = base[addr(src)];
      }
      step_loaded();
#pragma unroll
      for (int k = 0; k < R; ++k)
        if (move[k]) base[addr(start + i0 + k * per + r0)] = x[k];
    }
  }
}

}  // namespace

hipError_t launch_score(const ScoreParams &p, const bool fp8, const bool few, const bool many, hipStream_t st) {
  if (few) {
    const int waves = p.num_kv_heads < 8 ? p.num_kv_heads : 8;
    const dim3 grid((unsigned)((p.max_kv_len + kChunk - 1) / kChunk), (unsigned)p.num_seqs,
                    (unsigned)((p.num_kv_heads + waves - 1) / waves));
    if (fp8) score_few_kernel<true><<<grid, waves * 64, 0, st>>>(p);
    else score_few_kernel<false><<<grid, waves * 64, 0, st>>>(p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (many) {
    constexpr int keys = kScorePages * kBlock;
    const dim3 grid((unsigned)((p.max_kv_len + keys - 1) / keys) * (unsigned)p.num_kv_heads, (unsigned)p.num_seqs);
    if (fp8) score_rows_kernel<true><<<grid, kScoreWaves * 64, 0, st>>>(p);
    else score_rows_kernel<false><<<grid, kScoreWaves * 64, 0, st>>>(p);
    return hipGetLastError();
  }
  return hipSuccess;
}

int score_few_rows() { return kScoreFewRows; }

hipError_t launch_select(const SelectParams &p, hipStream_t st) {
  // small workgroups while the longest sequence fits them: three share a CU's LDS
  const unsigned grid = (unsigned)(p.num_seqs * p.num_kv_heads);
  if (p.max_kv_len <= 256 * kSelRun) select_kernel<256><<<grid, 256, 0, st>>>(p);
  else select_kernel<1024><<<grid, 1024, 0, st>>>(p);
  return hipGetLastError();
}

hipError_t launch_compact(const CompactParams &p, const int num_layers, hipStream_t st) {
  const int heads = p.keep_head != 0 ? 1 : p.num_kv_heads < 8 ? p.num_kv_heads : 8;
  const unsigned x = (unsigned)(p.num_seqs * (p.num_kv_heads / heads) * (p.has_scores ? 3 : 2));
  const dim3 grid(x, (unsigned)num_layers);
  if ((long long)p.max_rows * heads * kHeadDim * p.elt > 64 * 1024) compact_kernel<1024><<<grid, 1024, 0, st>>>(p, heads);
  else compact_kernel<256><<<grid, 256, 0, st>>>(p, heads);
  return hipGetLastError();
}

}  // namespace eid
