// gfx950 kernels that thin a paged cache out: attention weight received per cached key, choice of
// the rows that stay, move of the rows that stay.
#include "eid_cache_params.h"
#include "eid_device.h"

#include <type_traits>

namespace eid {

namespace {

struct ScoreSeq {
  int row0, qlen, len;
};
__device__ __forceinline__ ScoreSeq score_seq(const ScoreParams &p, const int s) {
  ScoreSeq v;
  const const_i32_ptr cu = as_constant(p.cu_seqlens_q), sl = as_constant(p.seq_lens);
  v.row0 = cu[s];
  v.qlen = cu[s + 1] - v.row0;
  v.len = min(sl[s], p.max_kv_len);
  if (v.qlen < 0 || v.len < v.qlen || v.row0 < 0 || v.row0 + v.qlen > p.num_q_tokens) v.qlen = 0;
  return v;
}

// K operand of 16 keys (one page) of a head: lane (key i16, segment g) holds elements 8 g .. 8 g + 7
// and 32 + 8 g .. 32 + 8 g + 7: a load instruction covers 64 consecutive bytes of each row.  An fp8
// row is half as long, one load: elements 16 g .. 16 g + 15.  q is read in the same order.  Through the
// caches, as lines are picked up in halves: with the non-temporal hint 8 x 37 rows behind 8k bf16 keys take
// 49.7 us (47), 4 heads of 64 fp8 sequences of one row 37 (34); 4 heads of bf16 58.5 on both sides.
template <bool FP8>
__device__ __forceinline__ void load_k(const uint8_t *base, const uint32_t row_bytes, Frag8 (&kf)[2]) {
  const int lane = threadIdx.x & 63, i16 = lane & 15, g = lane >> 4;
  const uint8_t *src = base + (uint32_t)i16 * row_bytes + g * 16;
  if constexpr (FP8) {
    const u32x4 r = *(const u32x4 *)src;
    fp8x8_to_bf16x8(r[0], r[1], kf[0].w);
    fp8x8_to_bf16x8(r[2], r[3], kf[1].w);
  } else {
    kf[0].u = *(const u32x4 *)src;
    kf[1].u = *(const u32x4 *)(src + 64);
  }
}

// 16 rows of q (two tokens x 8 heads) from token `tok` of the sequence on, and what the rows'
// exponents take off: lse in log2 units; -inf where there is no row, or one that saw nothing.
template <bool FP8>
__device__ __forceinline__ void load_rows(const ScoreParams &p, const ScoreSeq &v, const int kvh, const int tok,
                                          Frag8 (&qf)[2], f32x4 &off) {
  const int lane = threadIdx.x & 63, i16 = lane & 15, g = lane >> 4;
  const int tq = tok + (i16 >> 3), tl = tok + (g >> 1);
  qf[0].u = qf[1].u = u32x4{0, 0, 0, 0};
  if (tq < v.qlen) {
    const uint16_t *src = p.q + ((size_t)(v.row0 + tq) * p.num_q_heads + kvh * kGroup + (i16 & 7)) * kHeadDim + (FP8 ? 16 : 8) * g;
    qf[0].u = *(const u32x4 *)src;
    qf[1].u = *(const u32x4 *)(src + (FP8 ? 8 : 32));
  }
  off = f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
  if (tl < v.qlen) {
    const f32x4 e = *(const f32x4 *)(p.lse + (size_t)(v.row0 + tl) * p.num_q_heads + kvh * kGroup + 4 * (g & 1));
#pragma unroll
    for (int r = 0; r < 4; ++r) off[r] = e[r] * kLog2e;
  }
}

// Weights of 16 keys from 16 rows, summed over the lane's four rows.  D of Q K^T: lane (key i16,
// rows 4 g + r); rows 8 and up belong to the second token.  Rows without an offset add nothing, to keys
// that are not finite either (whose scores are NaN there: 0 x inf).
__device__ __forceinline__ float weights(const Frag8 (&qf)[2], const Frag8 (&kf)[2], const f32x4 off, const float c2,
                                         const bool see) {
  f32x4 S = mfma16x32(qf[0], kf[0], f32x4{0.f, 0.f, 0.f, 0.f});
  S = mfma16x32(qf[1], kf[1], S);
  float w = 0.f;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const float x = fast_exp2(__builtin_fmaf(S[r], c2, -off[r]));
    w += off[r] == -INFINITY ? 0.f : x;
  }
  return see ? w : 0.f;
}

// score of key j, new from `prefix` on
__device__ __forceinline__ void add_score(const ScoreParams &p, const int s, const int kvh, const int j,
                                          const int prefix, const float w) {
  const int page = clamp_id(p.block_table[(size_t)s * p.max_blocks_per_seq + j / kBlock], p.last_block);
  float *dst = p.scores + ((size_t)page * p.num_kv_heads + kvh) * kBlock + (j & 15);
  *dst = (j >= prefix ? 0.f : *dst) + w;
}


// Keys below `key_end` that no row of the sequence has in its window, none of them new: their scores stay.
__device__ __forceinline__ bool below_window(const ScoreParams &p, const int prefix, const int key_end) {
  return p.window > 0 && key_end <= prefix - p.window + 1;
}

// ---------------------------------------------------------------------------------------
// score[j] = (key j is new ? 0 : score[j]) + sum over rows i and the group's heads of
// vis(i, j) e^(c q.k_j - lse_i).
//
// Sequences of one or two rows: bound by reading K.  A wave takes 64 keys of one KV head; the
// workgroup's waves are the heads of the same keys, so that whole pages are read at once.  grid = (chunks,
// sequences).  For 1, 2 and 4 heads, which the stream below does not take: at 4 heads 64 sequences of one
// row behind 8192 bf16 keys are 58.5 us, 4.6 TB/s, fp8 34 us, 3.9 TB/s.
// ---------------------------------------------------------------------------------------
template <bool FP8>
__global__ __launch_bounds__(256) void score_few_kernel(const ScoreParams p) {
  const int lane = threadIdx.x & 63, i16 = lane & 15, g = lane >> 4;
  const int s = blockIdx.y, kvh = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const ScoreSeq v = score_seq(p, s);
  const int tc = blockIdx.x * kChunk;
  if (v.qlen < 1 || v.qlen > kScoreFewRows || tc >= v.len) return;
  const int prefix = v.len - v.qlen;
  if (below_window(p, prefix, tc + kChunk)) return;
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
  load_rows<FP8>(p, v, kvh, 0, qf, off);
  // lane (i16, g) keeps key i16 of page g
  const int mine = tc + g * kBlock + i16;
  const int pg = g == 0 ? page[0] : g == 1 ? page[1] : g == 2 ? page[2] : page[3];
  float *dst = p.scores + ((size_t)pg * p.num_kv_heads + kvh) * kBlock + i16;
  const float old = mine < prefix ? *dst : 0.f;
  float sum = 0.f;
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    const int j = tc + b * kBlock + i16, pos = prefix + (g >> 1);
    const bool see = j <= pos && (p.window <= 0 || pos - j < p.window);
    const float w = rowgroup_sum(weights(qf, kf[b], off, c2, see));
    sum = g == b ? w : sum;
  }
  if (mine < v.len) *dst = old + sum;
}

// ---------------------------------------------------------------------------------------
// The same with KV heads in groups of eight, as a stream.  The launch's 64-key chunks (from the first a
// window reaches) stand in a line, cut into equal ranges, and a wave walks a range for one head (two of
// an fp8 cache, whose rows are half a line) with two chunks under way through direct global -> LDS
// loads, whole 128-byte rows at a time, without barriers: its tiles are its own.
// 64 sequences of one row behind 8192 bf16 keys, 8 KV heads: 102 us, 5.6 TB/s (117 us in the form of the kernel
// above, which picks every row up in halves; 116 us here without the non-temporal hint); fp8 63 us
// (72).  A window of 128 behind 128 x 4096 keys: 8.4 us (47: most workgroups of a grid over all
// chunks find nothing to do).  One sequence of 500: 4.1 us (4.7); fp8 8 x 8192 alone loses, 13.1 (12.3).
// ---------------------------------------------------------------------------------------
constexpr int kStreamTile = kChunk * 128;      // K rows of a chunk

// One cursor of a stream: a chunk of a sequence.
struct StreamPos {
  int s, chunk, chunks, begin;
  ScoreSeq v;
};
struct Pages {
  int a, b, c, d;
};
__device__ __forceinline__ int stream_chunks(const ScoreParams &p, const ScoreSeq &v, int &begin) {
  begin = p.window > 0 ? max(0, v.len - v.qlen - p.window + 1) & ~(kChunk - 1) : 0;
  return v.qlen >= 1 && v.qlen <= kScoreFewRows ? (v.len - begin + kChunk - 1) / kChunk : 0;
}

template <bool FP8>
__global__ __launch_bounds__(FP8 ? 256 : 512, 2) void score_stream_kernel(const ScoreParams p) {
  constexpr int kHeads = FP8 ? 2 : 1, kWaves = 8 / kHeads;
  constexpr int kWave = kStreamTile + kHeads * 256;  // a wave's tile: the rows, and the old scores
  __shared__ __align__(1024) uint8_t tile0[kWaves * kWave], tile1[kWaves * kWave];
  const int lane = threadIdx.x & 63, i16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int groups = p.num_kv_heads / 8;
  const int kvh = blockIdx.x % groups * 8 + wave * kHeads, range = blockIdx.x / groups;
  const uint32_t row_bytes = (uint32_t)p.num_kv_heads * (128 / kHeads);
  const size_t page_bytes = (size_t)kBlock * row_bytes;
  float c2[kHeads];
#pragma unroll
  for (int h = 0; h < kHeads; ++h) c2[h] = p.softmax_scale * kLog2e * (FP8 ? p.k_scale[kvh + h] : 1.0f);

  // this range of the line
  int total = 0;
  auto units_at = [&](const int s) {
    ScoreSeq v;
    v.row0 = v.qlen = v.len = 0;
    if (s < p.num_seqs) {
      v.row0 = p.cu_seqlens_q[s];
      v.qlen = p.cu_seqlens_q[s + 1] - v.row0;
      v.len = min(p.seq_lens[s], p.max_kv_len);
      if (v.qlen < 0 || v.len < v.qlen || v.row0 < 0 || v.row0 + v.qlen > p.num_q_tokens) v.qlen = 0;
    }
    int begin;
    return stream_chunks(p, v, begin);
  };
  int n = 0, incl = 0;
  for (int s0 = 0; s0 < p.num_seqs; s0 += 64) {
    n = units_at(s0 + lane);
    incl = wave_inclusive_scan(n);
    total += __builtin_amdgcn_readlane(incl, 63);
  }
  const int per = (total + p.ranges - 1) / p.ranges;
  int left = min(total - range * per, per);  // units of this range (per > 0 where total > 0)
  if (left <= 0) return;
  StreamPos at;  // the next chunk to be requested
  for (int s0 = 0, base = 0;; s0 += 64) {
    if (p.num_seqs > 64) {
      n = units_at(s0 + lane);
      incl = wave_inclusive_scan(n);
    }
    const int sum = __builtin_amdgcn_readlane(incl, 63);
    if (base + sum > range * per) {  // (the unit exists: some batch holds it)
      const int i = __builtin_ctzll(__ballot(base + incl > range * per));
      at.s = s0 + i;
      at.chunk = range * per - (base + __builtin_amdgcn_readlane(incl, i) - __builtin_amdgcn_readlane(n, i));
      break;
    }
    base += sum;
  }
  at.v = score_seq(p, at.s);
  at.chunks = stream_chunks(p, at.v, at.begin);
  auto advance = [&](StreamPos &c) {  // (called only while units are left in the range)
    if (++c.chunk < c.chunks) return;
    c.chunk = 0;
    do {
      c.v = score_seq(p, ++c.s);
      c.chunks = stream_chunks(p, c.v, c.begin);
    } while (c.chunks == 0);
  };
  auto pages_of = [&](const StreamPos &c, Pages &pg) {
    const const_i32_ptr bt = as_constant(p.block_table + (size_t)c.s * p.max_blocks_per_seq);
    const int first = (c.begin + c.chunk * kChunk) / kBlock, last = (c.v.len - 1) / kBlock;
    pg.a = clamp_id(bt[min(first, last)], p.last_block);
    pg.b = clamp_id(bt[min(first + 1, last)], p.last_block);
    pg.c = clamp_id(bt[min(first + 2, last)], p.last_block);
    pg.d = clamp_id(bt[min(first + 3, last)], p.last_block);
  };
  // the lane's page of four
  const int m1 = g == 1 ? -1 : 0, m2 = g == 2 ? -1 : 0, m3 = g == 3 ? -1 : 0, m0 = ~(m1 | m2 | m3);
  auto of_lane = [&](const Pages &pg) {
    return (uint32_t)((pg.a & m0) | (pg.b & m1) | (pg.c & m2) | (pg.d & m3));
  };
  const int dr = lane >> 3, sl = lane & 7;
  auto request = [&](const Pages &pg, uint8_t *tile) {
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const int page = b == 0 ? pg.a : b == 1 ? pg.b : b == 2 ? pg.c : pg.d;
      const uint8_t *base = p.k_cache + (size_t)page * page_bytes + (uint32_t)kvh * (128 / kHeads);
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // (rows past the end are some page's rows: their weights are not stored)
        const uint32_t off = (uint32_t)(8 * h + dr) * row_bytes + (uint32_t)(sl ^ (4 * h + (dr >> 1))) * 16;
        __builtin_amdgcn_global_load_lds((gptr_t *)(base + off), (lptr_t *)(tile + (2 * b + h) * 1024), 16, 0, 2);
      }
    }
    const float *src = p.scores + ((size_t)of_lane(pg) * p.num_kv_heads + kvh) * kBlock + i16;
#pragma unroll
    for (int h = 0; h < kHeads; ++h)
      __builtin_amdgcn_global_load_lds((gptr_t *)(src + h * kBlock), (lptr_t *)(tile + kStreamTile + h * 256), 4, 0, 0);
  };
  uint8_t *t0 = tile0 + wave * kWave, *t1 = tile1 + wave * kWave;
  const uint32_t k_off = (uint32_t)i16 * 128 + (uint32_t)(g ^ ((i16 >> 1) & 7)) * 16;

  StreamPos cur = at;  // the chunk that is computed
  int asked = 1;       // chunks requested so far
  Pages pg0, pg1;
  pages_of(at, pg0);
  request(pg0, t0);
  if (asked < left) {
    advance(at);
    pages_of(at, pg1);
    request(pg1, t1);
    ++asked;
  }
  Frag8 qf[kHeads][2];
  f32x4 off[kHeads];
  int have = -1;  // sequence of qf and off
  auto step = [&](uint8_t *tile, Pages &pg, const int u) {
    if (have != cur.s) {
#pragma unroll
      for (int h = 0; h < kHeads; ++h) load_rows<FP8>(p, cur.v, kvh + h, 0, qf[h], off[h]);
      __builtin_amdgcn_s_waitcnt(0xF70);  // vmcnt(0): no wait for them below
      have = cur.s;
    }
    // younger than this chunk's loads: the next one's, and the stores of the last one
    if (u + 1 >= left) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    else if (u > 0) asm volatile("s_waitcnt vmcnt(%0)" ::"i"(8 + 2 * kHeads) : "memory");
    else asm volatile("s_waitcnt vmcnt(%0)" ::"i"(8 + kHeads) : "memory");
    // (read by hand: the compiler would wait for every load under way before it reads a tile)
    u32x4 raw[4][2];
    float old[kHeads];
    const uint32_t lo = (uint32_t)(uintptr_t)(lptr_t *)tile + k_off, hi = lo ^ 64;
    const uint32_t at_old = (uint32_t)(uintptr_t)(lptr_t *)tile + kStreamTile + 4 * lane;
    asm volatile(
        "ds_read_b128 %0, %10\n ds_read_b128 %1, %11\n ds_read_b128 %2, %10 offset:2048\n"
        "ds_read_b128 %3, %11 offset:2048\n ds_read_b128 %4, %10 offset:4096\n"
        "ds_read_b128 %5, %11 offset:4096\n ds_read_b128 %6, %10 offset:6144\n"
        "ds_read_b128 %7, %11 offset:6144\n ds_read_b32 %8, %12\n ds_read_b32 %9, %12 offset:%13\n"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(raw[0][0]), "=&v"(raw[0][1]), "=&v"(raw[1][0]), "=&v"(raw[1][1]), "=&v"(raw[2][0]),
          "=&v"(raw[2][1]), "=&v"(raw[3][0]), "=&v"(raw[3][1]), "=&v"(old[0]), "=&v"(old[kHeads - 1])
        : "v"(lo), "v"(hi), "v"(at_old), "i"((kHeads - 1) * 256)
        : "memory");  // the operands are in registers: the tile is free
    const int prefix = cur.v.len - cur.v.qlen, tc = cur.begin + cur.chunk * kChunk;
    const int mine = tc + g * kBlock + i16;
    float *dst = p.scores + ((size_t)of_lane(pg) * p.num_kv_heads + kvh) * kBlock + i16;
    if (asked < left) {
      advance(at);
      pages_of(at, pg);
      request(pg, tile);
      ++asked;
    }
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      float sum = 0.f;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        Frag8 kf[2];
        if constexpr (FP8) {
          fp8x8_to_bf16x8(raw[b][h][0], raw[b][h][1], kf[0].w);
          fp8x8_to_bf16x8(raw[b][h][2], raw[b][h][3], kf[1].w);
        } else {
          kf[0].u = raw[b][0];
          kf[1].u = raw[b][1];
        }
        const int j = tc + b * kBlock + i16, pos = prefix + (g >> 1);
        const bool see = j <= pos && (p.window <= 0 || pos - j < p.window);
        const float w = rowgroup_sum(weights(qf[h], kf, off[h], c2[h], see));
        sum = g == b ? w : sum;
      }
      if (mine < cur.v.len) dst[h * kBlock] = (mine < prefix ? old[h] : 0.f) + sum;
    }
    if (u + 1 < left) advance(cur);
  };
  for (int u = 0; u < left; u += 2) {
    step(t0, pg0, u);
    if (u + 1 < left) step(t1, pg1, u + 1);
  }
}

// First tile of sequence s in the workspace: behind those of the sequences before it.  -1 where the
// workspace has no room for its tiles (a batch of more keys than its descriptor says): its rows are not
// shared out then.  To be called by whole waves.
__device__ __forceinline__ int first_ws_tile(const ScoreParams &p, const int s, const int len) {
  int base = 0;
  for (int s0 = 0; s0 < s; s0 += 64) {
    const int i = s0 + (threadIdx.x & 63);
    const int keys = i < s ? max(0, min(p.seq_lens[i], p.max_kv_len)) : 0;
    base += __builtin_amdgcn_readlane(wave_inclusive_scan((keys + kScoreTile - 1) / kScoreTile), 63);
  }
  return base + (len + kScoreTile - 1) / kScoreTile <= p.ws_tiles ? base : -1;
}

// ---------------------------------------------------------------------------------------
// Sequences of more rows: bound by the exponentials and products.  A wave holds 128 keys of one KV
// head as operands and walks row pairs; one lane adds up one key's weights, so the sums need no
// atomics and have one order.  The four waves of a workgroup hold neighbouring keys and walk the
// same rows, which the CU's cache then reads once.  With parts > 1 a workgroup takes every
// parts-th row pair, its sums go to the workspace and score_join_kernel adds the parts up: a few key
// tiles alone do not fill the device, and the tiles that see the causal edge have less to do.
//
// A stage is one 16-key page: its two matrix instructions are issued a stage ahead of its four
// (multiply-add, exponential, add) per lane, which is what bounds the kernel: 2048 rows of one sequence
// behind 4k keys, 8 KV heads, 0.4 G weights, 102 us with the join, 4.0 weights per ns (51 GFLOP of
// products, 0.51 PFLOP/s); 8 x 37 rows behind 8k fp8 keys 33 us.
// ---------------------------------------------------------------------------------------
template <bool FP8>
__global__ __launch_bounds__(kScoreWaves * 64, 3) void score_rows_kernel(const ScoreParams p) {
  const int lane = threadIdx.x & 63, i16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kvh = blockIdx.x % p.num_kv_heads;
  const int tc = blockIdx.x / p.num_kv_heads * kScoreTile + wave * kScoreKeys;
  const int s = blockIdx.y, part = blockIdx.z;
  const ScoreSeq v = score_seq(p, s);
  const int prefix = v.len - v.qlen;
  const bool few = v.qlen <= kScoreFewRows;  // one row pair: no parts
  if (v.qlen < 1 || (few && (part > 0 || !p.all_rows)) || tc >= v.len || below_window(p, prefix, tc + kScoreKeys)) return;
  const const_i32_ptr bt = as_constant(p.block_table + (size_t)s * p.max_blocks_per_seq);
  const int last_page = (v.len - 1) / kBlock;
  const uint32_t row_bytes = (uint32_t)p.num_kv_heads * kHeadDim * (FP8 ? 1 : 2);
  const float c2 = p.softmax_scale * kLog2e * (FP8 ? p.k_scale[kvh] : 1.0f);
  constexpr int kPages = kScoreKeys / kBlock;
  // rows that see any of these keys: positions tc .. key_end - 1 + window - 1
  const int key_end = min(tc + kScoreKeys, v.len);
  const int i0 = max(0, tc - prefix) & ~1;
  int i1 = v.qlen;
  if (p.window > 0) i1 = (int)min((long long)i1, (long long)key_end - 1 + p.window - prefix);
  const int first = i0 + 2 * part;

  Frag8 kf[kPages][2], qf[2], qn[2];
  f32x4 e, en;  // lse of the rows, as they stand
#pragma unroll
  for (int b = 0; b < kPages; ++b) {
    const int page = clamp_id(bt[min(tc / kBlock + b, last_page)], p.last_block);
    load_k<FP8>(p.k_cache + (size_t)page * kBlock * row_bytes + (size_t)kvh * kHeadDim * (FP8 ? 1 : 2), row_bytes, kf[b]);
  }
  // row pair from token i on; tokens past the end repeat the last (their weights are dropped)
  const uint16_t *q_lane = p.q + ((size_t)v.row0 * p.num_q_heads + kvh * kGroup + (i16 & 7)) * kHeadDim + (FP8 ? 16 : 8) * g;
  const float *e_lane = p.lse + (size_t)v.row0 * p.num_q_heads + kvh * kGroup + 4 * (g & 1);
  auto fetch = [&](const int i, Frag8 (&q)[2], f32x4 &x) {
    const uint16_t *src = q_lane + (size_t)min(i + (i16 >> 3), v.qlen - 1) * p.num_q_heads * kHeadDim;
    q[0].u = *(const u32x4 *)src;
    q[1].u = *(const u32x4 *)(src + (FP8 ? 8 : 32));
    x = *(const f32x4 *)(e_lane + (size_t)min(i + (g >> 1), v.qlen - 1) * p.num_q_heads);
  };
  float sum[kPages];
#pragma unroll
  for (int b = 0; b < kPages; ++b) sum[b] = 0.f;
  // EDGE: some row of the pair does not see all keys, or is none.  DROP: a row saw nothing (its lse is -inf)
  // and adds nothing, to keys that are not finite either.
  auto pair = [&](auto edge_c, auto drop_c, const int i) {
    constexpr bool EDGE = decltype(edge_c)::value, DROP = decltype(drop_c)::value;
    // what the exponents take off, in log2 units
    f32x4 off;
#pragma unroll
    for (int r = 0; r < 4; ++r) off[r] = -kLog2e * e[r];
    const int pos = prefix + i + (g >> 1);
    const bool real = !EDGE || i + (g >> 1) < v.qlen;
    auto weight = [&](const float S, const int r) {
      const float x = fast_exp2(__builtin_fmaf(S, c2, off[r]));
      return !DROP || e[r] != -INFINITY ? x : 0.f;
    };
    f32x4 S[3];
    auto first_half = [&](const int b) { S[b % 3] = mfma16x32(qf[0], kf[b][0], f32x4{0.f, 0.f, 0.f, 0.f}); };
    auto second_half = [&](const int b) { S[b % 3] = mfma16x32(qf[1], kf[b][1], S[b % 3]); };
    first_half(0);
    first_half(1);
    second_half(0);
#pragma unroll
    for (int b = 0; b < kPages; ++b) {
      float w[4];
      __builtin_amdgcn_sched_barrier(0);
      if (b + 1 < kPages) second_half(b + 1);
#pragma unroll
      for (int r = 0; r < 2; ++r) w[r] = weight(S[b % 3][r], r);
      __builtin_amdgcn_sched_barrier(0);
      if (b + 2 < kPages) first_half(b + 2);
#pragma unroll
      for (int r = 2; r < 4; ++r) w[r] = weight(S[b % 3][r], r);
      float add = (w[0] + w[1]) + (w[2] + w[3]);
      if constexpr (EDGE) {
        const int j = tc + b * kBlock + i16;
        add = real && j <= pos && (p.window <= 0 || pos - j < p.window) ? add : 0.f;
      }
      sum[b] += add;
    }
  };
  if (first < i1) fetch(first, qf, e);
  const int ws_tile = p.parts > 1 && !few ? first_ws_tile(p, s, v.len) : -1;  // (while keys and rows arrive)
  const bool shared = ws_tile >= 0;
  if (part > 0 && !shared) return;
  const int stride = shared ? 2 * p.parts : 2;
  for (int i = first; i < i1; i += stride) {
    fetch(i + stride, qn, en);
    const bool edge = prefix + i < key_end - 1 || (p.window > 0 && prefix + i + 1 - tc >= p.window) || i + 1 >= v.qlen;
    if (__any(fminf(fminf(e[0], e[1]), fminf(e[2], e[3])) == -INFINITY)) pair(std::true_type{}, std::true_type{}, i);
    else if (edge) pair(std::true_type{}, std::false_type{}, i);
    else pair(std::false_type{}, std::false_type{}, i);
    qf[0] = qn[0];
    qf[1] = qn[1];
    e = en;
  }
  // lane (i16, g) keeps key i16 of pages g and 4 + g
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float w = 0.f;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const float x = rowgroup_sum(sum[4 * h + b]);
      w = g == b ? x : w;
    }
    const int j = tc + (4 * h + g) * kBlock + i16;
    if (j >= v.len) continue;
    if (shared) p.ws[(((size_t)part * p.num_kv_heads + kvh) * p.ws_tiles + ws_tile) * kScoreTile + j] = w;
    else add_score(p, s, kvh, j, prefix, w);
  }
}

// Adds the parts of the rows kernel up, part after part.  grid = (keys / 256, KV heads, sequences).
__global__ __launch_bounds__(256) void score_join_kernel(const ScoreParams p) {
  const int s = blockIdx.z, kvh = blockIdx.y, j = blockIdx.x * 256 + threadIdx.x;
  const ScoreSeq v = score_seq(p, s);
  if (v.qlen <= kScoreFewRows || (int)blockIdx.x * 256 >= v.len) return;
  const int ws_tile = first_ws_tile(p, s, v.len);
  if (ws_tile < 0 || j >= v.len || below_window(p, v.len - v.qlen, j + 1)) return;
  const float *src = p.ws + ((size_t)kvh * p.ws_tiles + ws_tile) * kScoreTile + j;
  const size_t step = (size_t)p.num_kv_heads * p.ws_tiles * kScoreTile;
  float w = 0.f;
  for (int part = 0; part < p.parts; part += 8) {  // eight loads under way, added in order
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = src[min(part + i, p.parts - 1) * step];
#pragma unroll
    for (int i = 0; i < 8; ++i) w += part + i < p.parts ? x[i] : 0.f;
  }
  add_score(p, s, kvh, j, v.len - v.qlen, w);
}

// Workgroups are dealt to the 8 XCDs in turn: the item of this one, so that neighbouring items
// (heads of a sequence, whose rows lie beside each other) run on one XCD.
__device__ __forceinline__ int xcd_order() {
  const int n8 = gridDim.x >> 3, b = blockIdx.x;
  return b < 8 * n8 ? (b & 7) * n8 + (b >> 3) : b;
}

// ---------------------------------------------------------------------------------------
// Rows to keep.  A workgroup per (sequence, KV head) finds the score of the last row that stays
// by radix selection over order-preserving keys, eleven bits a pass, then writes the rows in
// order.  A thread holds RUN rows as keys in its registers: the scores are read once, every pass
// works on registers, and ballots give each row its place.  Sequences beyond 32 rows per thread are
// walked in blocks of that size and read again by every pass.  A wave reads whole pages, four lanes
// each; workgroups of neighbouring heads, which share cache lines of scores, run on one XCD (32
// sequences of 32k rows: 24 us against 28).  Four copies of the histogram: lanes with equal digits,
// the usual case in the first pass, queue less on one address (8 and 16 copies cost more to clear
// than they save: 31 and 44 us against 28).  A pass whose digit is kept whole ends the search.
// 32 sequences of up to 32k rows to 4096, 28 MB: 21 us, the second and third pass 4 of them; one of
// 3000: 6.4 us, a chain of passes in one workgroup.
// ---------------------------------------------------------------------------------------
// larger = kept first, -0 = +0; NaN ranks lowest, as 1: 0 stands for rows that are no candidates, which
// are therefore never reached (the candidates are at least as many as the rows wanted)
__device__ __forceinline__ uint32_t order_key(const float x) {
  const uint32_t u = __float_as_uint(x + 0.f);  // (-0 + 0 = +0)
  const uint32_t k = u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
  return x != x ? 1u : k;
}
constexpr int kSelThreads = 1024;
constexpr int kSelBins = 2048, kSelCopies = 4;

template <int RUN>
__global__ __launch_bounds__(kSelThreads) void select_kernel(const SelectParams p) {
  constexpr int THREADS = kSelThreads, kWaves = THREADS / 64, kCap = THREADS * RUN, kBins = kSelBins / THREADS;
  __shared__ __align__(16) uint32_t hist[kSelBins * kSelCopies];
  __shared__ uint32_t wave_sum[kWaves];
  __shared__ uint32_t found[3];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int id = xcd_order();
  const int s = id / p.num_kv_heads, kvh = id % p.num_kv_heads;
  const int len = max(0, min(p.seq_lens[s], p.max_blocks_per_seq * kBlock));
  const int budget = p.budget;
  int32_t *keep = p.keep + (size_t)id * budget;
  if (kvh == 0 && tid == 0) p.counts[s] = min(len, budget);
  if (len <= budget) {
    for (int i = tid; i < budget; i += THREADS) keep[i] = i < len ? i : -1;
    return;
  }
  const int32_t *bt = p.block_table + (size_t)s * p.max_blocks_per_seq;
  const int lo = p.keep_first, hi = len - p.keep_last;  // candidates: lo <= j < hi
  const int last_page = (len - 1) / kBlock;
  uint32_t key[RUN];
  // row of key[0] in the block that starts at j0; key[4 k + e] is 256 k + e rows behind
  const int mine = wave * (64 * RUN) + 4 * lane;
  auto load = [&](const int j0) {
    const int j = j0 + mine;
#pragma unroll
    for (int i = 0; i < RUN; ++i) key[i] = 0;
    const int first = j0 + wave * (64 * RUN);  // the wave's rows
    if (first >= hi) return;
    f32x4 x[RUN / 4];
    int page[RUN / 4];
#pragma unroll
    for (int k = 0; k < RUN / 4; ++k) page[k] = bt[min((j + 256 * k) / kBlock, last_page)];
#pragma unroll
    for (int k = 0; k < RUN / 4; ++k)
      x[k] = *(const f32x4 *)(p.scores + ((size_t)clamp_id(page[k], p.last_block) * p.num_kv_heads + kvh) * kBlock + j % kBlock);
#pragma unroll
    for (int i = 0; i < RUN; ++i) {
      key[i] = order_key(x[i / 4][i % 4]);
    }
    if (first < lo || first + 64 * RUN > hi) {
#pragma unroll
      for (int i = 0; i < RUN; ++i)
        if ((uint32_t)(j + 256 * (i / 4) + i % 4 - lo) >= (uint32_t)(hi - lo)) key[i] = 0;
    }
  };
  const bool once = len <= kCap;
  if (once) load(0);
  for (int i = tid; i < kSelBins * kSelCopies; i += THREADS) hist[i] = 0;
  __syncthreads();

  uint32_t want = (uint32_t)(budget - p.keep_first - p.keep_last);  // candidates to keep
  uint32_t cut = 0;    // the digits found so far
  bool whole = false;  // every key equal to `cut` in the bits searched stays
  int shift = 21;
  if (want > 0) {
    for (int pass = 0; pass < 3; ++pass) {
      shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
      const uint32_t digits = pass < 2 ? 2047u : 1023u;
      for (int j0 = 0; j0 < len; j0 += kCap) {
        if (!once) load(j0);
#pragma unroll
        for (int i = 0; i < RUN; ++i)
          if (pass == 0 ? key[i] != 0 : (key[i] ^ cut) >> shift <= digits)
            atomicAdd(&hist[(key[i] >> shift & digits) * kSelCopies + (lane & (kSelCopies - 1))], 1u);
      }
      __syncthreads();
      // counts from the highest digit down: thread d holds digits (last - d kBins) .. of kBins bins
      uint32_t n[kBins], sum = 0;
#pragma unroll
      for (int c = 0; c < kBins; ++c) {
        u32x4 *h = (u32x4 *)&hist[(kSelBins - 1 - (tid * kBins + c)) * kSelCopies];
        n[c] = 0;
#pragma unroll
        for (int v = 0; v < kSelCopies / 4; ++v) {
          const u32x4 x = h[v];
          h[v] = u32x4{0, 0, 0, 0};  // for the next pass
          n[c] += x[0] + x[1] + x[2] + x[3];
        }
        sum += n[c];
      }
      uint32_t incl = (uint32_t)wave_inclusive_scan((int)sum);
      if (lane == 63) wave_sum[wave] = incl;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kWaves; ++w)
        if (w < wave) incl += wave_sum[w];
      uint32_t above = incl - sum;  // candidates with a higher digit
#pragma unroll
      for (int c = 0; c < kBins; ++c) {
        if (above < want && above + n[c] >= want) {
          found[0] = (uint32_t)(kSelBins - 1 - (tid * kBins + c));
          found[1] = above;
          found[2] = n[c];
        }
        above += n[c];
      }
      __syncthreads();
      cut |= found[0] << shift;
      want -= found[1];
      whole = found[2] == want;
      if (whole) break;
      __syncthreads();  // (found is read before the next pass writes it)
    }
  }
  for (int i = tid; i < p.keep_first; i += THREADS) keep[i] = i;
  for (int i = tid; i < p.keep_last; i += THREADS) keep[budget - p.keep_last + i] = hi + i;
  if (budget == p.keep_first + p.keep_last) return;
  // Keys from `least` on stay: those whose searched bits are above those of `cut`, and those equal to it
  // if it is kept whole; else the first `want` of the latter stay as well.  In a wave's share of a
  // block, the rows before (k, lane, e) are those of a lower k, and of the same k in a lower lane or in
  // the same lane with a lower e.
  const uint32_t least = whole ? max(cut, 1u) : cut + 1;
  uint32_t base = (uint32_t)p.keep_first, ties = 0;  // rows written, ties passed
  // sum over the workgroup's waves (`all`), and over those before this one
  auto before = [&](const uint32_t n, uint32_t &all) {
    __syncthreads();  // (the last use of wave_sum)
    if (lane == 0) wave_sum[wave] = n;
    __syncthreads();
    uint32_t sum = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      if (w < wave) sum += wave_sum[w];
      all += wave_sum[w];
    }
    return sum;
  };
  // rows of the wave among its four-key groups k that pass `test`; calls take(k, rows of the group in
  // lower lanes) on the way
  auto ranks = [&](auto test, auto take) {
    uint32_t n = 0;
#pragma unroll
    for (int k = 0; k < RUN / 4; ++k) {
      uint32_t below = n;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint64_t m = __ballot(test(key[4 * k + e]));
        below = __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, below));
        n += (uint32_t)__popcll(m);
      }
      take(k, below);
    }
    return n;
  };
  auto stays = [&](const uint32_t k) { return k >= least; };
  auto is_tie = [&](const uint32_t k) { return k == cut; };
  auto nothing = [](int, uint32_t) {};
  const uint32_t room = (uint32_t)(budget - p.keep_last);  // (also if scores change under a long selection)
  for (int j0 = 0; j0 < len; j0 += kCap) {
    if (!once) load(j0);
    uint32_t all;
    if (!whole) {  // (all bits are searched)
      const uint32_t t = ties + before(ranks(is_tie, nothing), all);
      ties += all;
      ranks(is_tie, [&](const int k, uint32_t at) {
        at += t;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (is_tie(key[4 * k + e]) && at++ < want) key[4 * k + e] = ~0u;
      });
    }
    const uint32_t row = base + before(ranks(stays, nothing), all);
    base += all;
    ranks(stays, [&](const int k, uint32_t at) {
      at += row;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (stays(key[4 * k + e]) && at < room) keep[at++] = j0 + mine + 256 * k + e;
    });
  }
}

// ---------------------------------------------------------------------------------------
// row start + i <- row keep[i], i ascending, keep[i] >= start + i.  In place: a workgroup owns a
// column of the sequence (one KV head, or eight where all heads keep the same rows) in one tensor
// of one layer and moves it in steps; a step's rows are all in registers before its first
// store, and later steps read only rows behind everything that this one overwrites.  What bounds
// long moves is that order: a column's loads, drain and stores follow one another four times over with
// nothing in flight during the stores, on as many CUs as there are columns (8 sequences cut from 16k to 4k:
// 39 us in the kernel for 137 MB, 3.5 TB/s, 128 workgroups for K and V and 64 for scores).  A head's rows are lone
// lines of 128 bytes of a token's 1 KiB, which alone do not cost that much: a kernel that only loads one head's
// rows runs at 5.4 TB/s and more; two workgroups per column, 64 bytes of a row each, 49 us.  Neighbouring
// heads on one XCD: 45.5 us the call against 47.
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
  int b = xcd_order();
  const int hg = b % groups;
  b /= groups;
  const int what = b % tensors, s = b / tensors, layer = blockIdx.y;
  const int start = p.starts ? p.starts[s] : 0;
  const int len = max(0, min(p.seq_lens[s], p.max_blocks_per_seq * kBlock));
  const int n = min(min(p.counts[s], p.max_rows), len - start);
  if (start < 0 || n <= 0) return;
  const int32_t *keep = p.keep + (size_t)layer * p.keep_layer + (size_t)s * p.keep_seq + (size_t)hg * heads * p.keep_head;
  const int32_t *bt = p.block_table + (size_t)s * p.max_blocks_per_seq;
  auto page_of = [&](const int row) { return clamp_id(bt[row / kBlock], p.last_block); };
  // Addresses are found a step ahead, and loads are issued for all R rows of a lane at once (one
  // that does not move loads the sequence's row `start` and stores nothing).
  auto move_all = [&](auto zero, auto *base, const int lanes, auto at) {
    using T = decltype(zero);
    const int per = THREADS / lanes, r0 = tid / lanes;
    int src[R], from[R], to[R];  // source row (its own place: no move), pages of both
    auto find = [&](const int i0) {
#pragma unroll
      for (int k = 0; k < R; ++k) {
        const int i = i0 + k * per + r0, row = start + min(i, n - 1);
        const int x = keep[min(i, n - 1)];
        src[k] = i < n && x > row && x < len ? x : row;
      }
#pragma unroll
      for (int k = 0; k < R; ++k) {
        from[k] = page_of(src[k]);
        to[k] = page_of(start + min(i0 + k * per + r0, n - 1));
      }
    };
    find(0);
    for (int i0 = 0; i0 < n; i0 += per * R) {
      T x[R];
      T *dst[R];
      bool move[R];
#pragma unroll
      for (int k = 0; k < R; ++k) {
        const int row = start + min(i0 + k * per + r0, n - 1);
        move[k] = i0 + k * per + r0 < n && src[k] != row;
        x[k] = *(const T *)at(base, from[k], src[k]);
        dst[k] = (T *)at(base, to[k], row);
      }
      if (i0 + per * R < n) find(i0 + per * R);
      step_loaded();
#pragma unroll
      for (int k = 0; k < R; ++k)
        if (move[k]) *dst[k] = x[k];
    }
  };
  if (what < 2) {
    const int lanes = heads * kHeadDim * p.elt / 16;  // 16-byte lanes of a row: 4 .. 64
    const uint32_t row_bytes = (uint32_t)p.num_kv_heads * kHeadDim * p.elt;
    const uint32_t col = (uint32_t)hg * heads * kHeadDim * p.elt + (tid % lanes) * 16;
    move_all(u32x4{}, what ? p.v[layer] : p.k[layer], lanes, [=](uint8_t *base, const int page, const int row) {
      return base + (size_t)page * kBlock * row_bytes + (uint32_t)(row & 15) * row_bytes + col;
    });
  } else {
    const int h = hg * heads + tid % heads, Hkv = p.num_kv_heads;
    move_all(0.f, p.scores[layer], heads, [=](float *base, const int page, const int row) {
      return base + ((size_t)page * Hkv + h) * kBlock + (row & 15);
    });
  }
}

}  // namespace

hipError_t launch_score(const ScoreParams &p, const bool fp8, const bool many, hipStream_t st) {
  const bool few = !many || !p.all_rows;
  if (few && p.num_kv_heads % 8 == 0) {
    const unsigned grid = (unsigned)(p.ranges * (p.num_kv_heads / 8));
    if (fp8) score_stream_kernel<true><<<grid, 256, 0, st>>>(p);
    else score_stream_kernel<false><<<grid, 512, 0, st>>>(p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  } else if (few) {
    const dim3 grid((unsigned)((p.max_kv_len + kChunk - 1) / kChunk), (unsigned)p.num_seqs);
    const unsigned threads = (unsigned)p.num_kv_heads * 64;  // (1, 2 or 4 heads)
    if (fp8) score_few_kernel<true><<<grid, threads, 0, st>>>(p);
    else score_few_kernel<false><<<grid, threads, 0, st>>>(p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (many) {
    const dim3 grid((unsigned)(p.tile_keys / kScoreTile) * (unsigned)p.num_kv_heads, (unsigned)p.num_seqs,
                    (unsigned)p.parts);
    if (fp8) score_rows_kernel<true><<<grid, kScoreWaves * 64, 0, st>>>(p);
    else score_rows_kernel<false><<<grid, kScoreWaves * 64, 0, st>>>(p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.parts == 1) return e;
    score_join_kernel<<<dim3((unsigned)(p.max_kv_len + 255) / 256, (unsigned)p.num_kv_heads, (unsigned)p.num_seqs), 256, 0, st>>>(p);
    return hipGetLastError();
  }
  return hipSuccess;
}

hipError_t launch_select(const SelectParams &p, hipStream_t st) {
  // rows per thread: as few as hold the longest sequence (8 of 3000: 6.8 us with 4, 10.0 with 16, 14.5
  // with 32; 8 of 12000: 11.4 with 16, 16.4 with 32)
  const unsigned grid = (unsigned)(p.num_seqs * p.num_kv_heads);
  if (p.max_kv_len <= kSelThreads * 4) select_kernel<4><<<grid, kSelThreads, 0, st>>>(p);
  else if (p.max_kv_len <= kSelThreads * 16) select_kernel<16><<<grid, kSelThreads, 0, st>>>(p);
  else select_kernel<32><<<grid, kSelThreads, 0, st>>>(p);
  return hipGetLastError();
}

hipError_t launch_compact(const CompactParams &p, const int num_layers, hipStream_t st) {
  const int heads = p.keep_head != 0 ? 1 : p.num_kv_heads < 8 ? p.num_kv_heads : 8;
  const unsigned x = (unsigned)(p.num_seqs * (p.num_kv_heads / heads) * (p.has_scores ? 3 : 2));
  const dim3 grid(x, (unsigned)num_layers);
  // A column's rows in one step of the larger workgroup or a few of the smaller: a commit of 36 layers
  // 9.0 us with 256 threads, 25 with 1024; 8 sequences cut from 16k to 4k rows 55 and 47.
  if ((long long)p.max_rows * heads * kHeadDim * p.elt > 64 * 1024) compact_kernel<1024><<<grid, 1024, 0, st>>>(p, heads);
  else compact_kernel<256><<<grid, 256, 0, st>>>(p, heads);
  return hipGetLastError();
}

}  // namespace eid
