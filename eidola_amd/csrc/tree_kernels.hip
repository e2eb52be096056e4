// gfx950 kernels of the attention for trees of drafted tokens over the paged cache.
#include "eid_cache_params.h"
#include "eid_device.h"

#include <utility>

namespace eid {

namespace {

constexpr float kLazyLog2 = 8.0f;  // a row's reference moves when a score outgrows it by this
constexpr float kRowSumGuard = 1152921504606846976.0f;  // 2^60

// What one sequence gives the kernel: `chunks` 64-key chunks from key `begin` on for each of
// `tiles` tiles of drafted tokens.
struct TreeSeq {
  int row0, qlen, len, begin, chunks, tiles;
};

// The rows at and behind prefix = len - qlen stand for the drafted tokens.  A token's position is
// prefix + (ancestors it sees) >= prefix - 1, so no row sees keys below prefix - window.
__device__ __forceinline__ TreeSeq tree_seq(const TreeParams &p, const int row0, const int row1, const int len,
                                            const int tile_tok) {
  TreeSeq v;
  v.row0 = row0;
  v.qlen = row1 - row0;
  v.len = min(len, p.max_kv_len);
  // (junk lengths: nothing of the sequence is computed, nothing is read)
  if (row0 < 0 || row1 < row0 || row1 > p.num_q_tokens || v.qlen > p.max_q_len || v.len < v.qlen) v.qlen = 0;
  v.begin = p.window > 0 ? max(0, v.len - v.qlen - p.window) & ~(kBlock - 1) : 0;
  v.tiles = (v.qlen + tile_tok - 1) / tile_tok;
  v.chunks = v.qlen > 0 ? (v.len - v.begin + kChunk - 1) / kChunk : 0;
  return v;
}

// Place of one workgroup's range in the line of units.  Batches of up to 64 sequences are looked at
// once, a lane per sequence; `lane_*` stay with the lanes.
struct TreePlace {
  int lane_row0, lane_row1, lane_len;
  int per, u, u_end;  // units per range; this range's
  int seq, before;    // the sequence that holds unit u, and the units before it
};
__device__ __forceinline__ TreePlace find_place(const TreeParams &p, const int range, const int tile_tok) {
  const int lane = threadIdx.x & 63;
  TreePlace w;
  int total = 0, incl = 0, n = 0;
  auto load = [&](const int s) {
    w.lane_row0 = w.lane_row1 = w.lane_len = 0;
    if (s < p.num_seqs) {
      w.lane_row0 = p.cu_seqlens_q[s];
      w.lane_row1 = p.cu_seqlens_q[s + 1];
      w.lane_len = p.seq_lens[s];
    }
    const TreeSeq v = tree_seq(p, w.lane_row0, w.lane_row1, w.lane_len, tile_tok);
    n = v.tiles * v.chunks;
    incl = wave_inclusive_scan(n);
    return __builtin_amdgcn_readlane(incl, 63);
  };
  for (int s0 = 0; s0 < p.num_seqs; s0 += 64) total += load(s0 + lane);
  w.per = max((total + p.ranges - 1) / p.ranges, p.min_chunks);
  w.u = range < (total + w.per - 1) / w.per ? range * w.per : total;
  w.u_end = min(total - w.u, w.per) + w.u;
  w.seq = w.before = 0;
  for (int s0 = 0, base = 0; w.u < w.u_end; s0 += 64) {  // (the unit exists: some batch holds it)
    const int sum = p.num_seqs <= 64 ? total : load(s0 + lane);
    if (base + sum > w.u) {
      const int i = __builtin_ctzll(__ballot(base + incl > w.u));
      w.seq = s0 + i;
      w.before = base + __builtin_amdgcn_readlane(incl, i) - __builtin_amdgcn_readlane(n, i);
      break;
    }
    base += sum;
  }
  return w;
}
__device__ __forceinline__ TreeSeq seq_at(const TreeParams &p, const TreePlace &w, const int s, const int tile_tok) {
  if (!p.whole && p.num_seqs <= 64)
    return tree_seq(p, __builtin_amdgcn_readlane(w.lane_row0, s), __builtin_amdgcn_readlane(w.lane_row1, s),
                    __builtin_amdgcn_readlane(w.lane_len, s), tile_tok);
  const const_i32_ptr cu = as_constant(p.cu_seqlens_q), sl = as_constant(p.seq_lens);
  return tree_seq(p, cu[s], cu[s + 1], sl[s], tile_tok);
}

// 64 visibility bits of one drafted token for the keys tc .. tc + 63.
__device__ __forceinline__ uint64_t chunk_bits(const uint64_t *mask, const int lo, const int prefix, const int tc) {
  const int d = tc - prefix;
  uint64_t w;
  if (d >= 0) {
    const int i = d >> 6, sh = d & 63;
    w = i < kTreeWordsMax ? mask[i] >> sh : 0;
    if (sh && i + 1 < kTreeWordsMax) w |= mask[i + 1] << (64 - sh);
  } else if (d <= -64) {
    w = ~0ull;
  } else {
    w = ((1ull << -d) - 1) | mask[0] << -d;
  }
  // context keys below the window (lo is far below 0 in a window near 2^31)
  const int cut = min(min(max(lo, 0), prefix) - tc, 64);
  if (cut >= 64) w = 0;
  else if (cut > 0) w &= ~((1ull << cut) - 1);
  return w;
}

// ---------------------------------------------------------------------------------------
// out[i] = sum_j vis(i, j) e^(c q_i.k_j) v_j / (sum_j vis(i, j) e^(c q_i.k_j) + e^sink), with
// vis(i, j) = j < prefix, or bit j - prefix of row i's mask; one pass with a running reference.
//
// A workgroup of four waves owns up to 8 NT drafted tokens x the 8 query heads of one KV head:
// 16 NT rows per wave.  The launch's (sequence, tile) pairs,
// 64 keys at a time, are laid out in a line and cut into `ranges` equal pieces, one per workgroup,
// so that a batch of unequal contexts loads every CU alike; a range that ends inside a sequence
// leaves (o, m, l) for tree_merge_kernel.
//
// K and V chunks stand in LDS as 64 rows of 128 bytes, read by all four waves; 16-byte segments
// are permuted by the row (K: segment ^ (row / 2) % 8, V: pairs of segments by (row / 2) % 4),
// which keeps the operand reads off each other's banks without padding.  bf16 caches: direct
// global -> LDS loads, up to three chunks under way while one is computed.  fp8 caches:
// through registers, where the bytes are widened once for the four waves, two stages.
//
// Chunks that some row does not see whole (the drafted tokens' own, a window's edge) differ in
// two ways: scores are masked, and values that are not finite are taken out of the operands
// (0 x inf would be NaN in rows that do not see the key); if there were any, their terms are added
// afterwards, row by row, where they are seen.
//
// Roundings: a row's weights enter the value product as bf16 (the matrix unit takes both operands in one type,
// and V is bf16; fp16 would hold neither V's range nor weights of 2^60; the weights' low halves in a
// second product would be 8 more matrix instructions per chunk and 16-row tile beside 18, and their
// subtractions and packings).  Against 64 bits an answer is off by 0.0022 - 0.0024 of its size, of which
// 0.0017 are the rounding of the answer itself.  Sums and statistics are fp32.
//
// What bounds it, 8 KV heads.  4 x 64 behind 32k, 137 GFLOP, 176 us, 0.78 PFLOP/s: a 64-key chunk of a
// 16-row tile takes 16 exponentials, 16 multiply-adds and 8 packings per lane and 18 matrix instructions;
// vector units are 60 % and matrix units 36 % busy, which mostly add up instead of overlapping.  Small trees:
// no unit, but latency and what every piece repeats (lengths, pages, q and masks one after the other, a drain,
// the join): 16 trees of up to 16 tokens behind up to 8k keys, 199 MB, 54 us, 3.7 TB/s, matrix units 14 %
// busy, vector units 36 %.  8 x 17 .. 32 tokens behind 16k fp8, 86 us: 23 % of its tiles' rows are nobody's (the
// longest tree chooses the tile for all), and one chunk is requested ahead; vector units 43 % busy, matrix units
// 23 %.  32 x 24 in a window of 128, 19 MB, 15 us: three chunks, the third requested when the first is done.
// 1 x 8 behind 500, 11.5 us: eight chunks one after the other in one workgroup per head.
// ---------------------------------------------------------------------------------------
constexpr int kTileBytes = kChunk * 128;

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
// e with |x| in [2^(e-1), 2^e); 0 for 0
__device__ __forceinline__ int top_exponent(const float x) {
  return x > 0.f ? __builtin_amdgcn_frexp_expf(x) : 0;
}

template <int... Is, typename F>
__device__ __forceinline__ void static_for_impl(std::integer_sequence<int, Is...>, F &&f) {
  (f(std::integral_constant<int, Is>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void static_for(F &&f) {
  static_for_impl(std::make_integer_sequence<int, N>{}, f);
}
template <int I>
using IC = std::integral_constant<int, I>;
#define EID_SB() __builtin_amdgcn_sched_barrier(0)

template <int NT, bool FP8, bool LSE>
__global__ __launch_bounds__(kTreeWaves * 64, 2) void tree_kernel(const TreeParams p) {
  constexpr int kTok = 2 * NT * kTreeWaves;  // tokens of a tile
  constexpr int kRows = kTok * kGroup;
  constexpr int kElt = FP8 ? 1 : 2;
  // Q operands of three and four tiles do not fit the registers beside the rest: LDS, in place of
  // more stages.
  constexpr bool QLDS = NT >= 3;
  constexpr int ST = FP8 || QLDS ? 2 : 4;  // K/V stages
  constexpr bool DEEP8 = NT <= 3;          // fp8: two chunks under way
  // (separate arrays: the compiler can then tell the stage being filled from the one being read)
  // Up to 16 tokens are one tile: every chunk is read once, past the caches (non-temporal): 16 x 16 behind
  // 8k keys 72 us against 75.  Larger trees may be cut, and a chunk then serves several tiles: 4 x 200
  // behind 4k 98 us from the caches, 109 past them (16 x 24, one tile, 90 and 89).
  constexpr int kAux = NT <= 2 ? 2 : 0;
  constexpr int kMore = ST == 4 ? kTileBytes : 16;
  __shared__ __align__(1024) uint8_t k_st0[kTileBytes], k_st1[kTileBytes], k_st2[kMore], k_st3[kMore];
  __shared__ __align__(1024) uint8_t v_st0[kTileBytes], v_st1[kTileBytes], v_st2[kMore], v_st3[kMore];
  __shared__ __align__(16) uint8_t lds_q[QLDS ? kTreeWaves * 2 * NT * 1024 : 16];
  __shared__ uint64_t lds_mask[kTok][kTreeWordsMax];
  __shared__ int lds_lo[kTok];
  __shared__ int lds_depth[kTreeMax];
  static_assert(kTreeMax == kTreeWaves * 64, "a thread per token of the longest tree");
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i16 = lane & 15, g = lane >> 4;
  const int Hkv = p.num_kv_heads;
  const int kvh = blockIdx.x % Hkv, range = blockIdx.x / Hkv;
  const float c2 = p.softmax_scale * kLog2e * (FP8 ? p.k_scale[kvh] : 1.0f);
  const float vs = FP8 ? p.v_scale[kvh] : 1.0f;

  TreePlace place;
  if (p.whole) {  // a range is one tile of one sequence
    place.seq = range / p.max_tiles;
    place.per = 0x7fffffff;
    const TreeSeq v = seq_at(p, place, place.seq, kTok);
    place.before = 0;
    place.u = range % p.max_tiles * v.chunks;
    place.u_end = range % p.max_tiles < v.tiles ? place.u + v.chunks : place.u;
  } else {
    place = find_place(p, range, kTok);
  }
  Frag8 ones;
  ones.u = u32x4{0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};
  asm volatile("" : "+v"(ones.u));  // (kept in registers)
  int u = place.u, s = place.seq, before = place.before;

  const uint32_t row_bytes = (uint32_t)Hkv * kHeadDim * kElt;
  const size_t page_bytes = (size_t)kBlock * row_bytes;
  // operand reads (see above): K row i16 of a page, V rows 4 g + i16 / 4 (transposing read)
  const int sw_k = (i16 >> 1) & 7;
  const uint32_t k_off = (uint32_t)i16 * 128 + (uint32_t)((2 * g) ^ sw_k) * 16;
  const int v_row = 4 * g + (i16 >> 2);
  const uint32_t v_off = (uint32_t)v_row * 128 + 8 * (i16 & 3);
  const int v_sw = 32 * ((v_row >> 1) & 3);

  while (u < place.u_end) {
    const TreeSeq v = seq_at(p, place, s, kTok);
    const int units = v.tiles * v.chunks;
    if (u - before >= units) {  // next sequence (those without rows have no units)
      before += units;
      ++s;
      continue;
    }
    const int tile = (u - before) / v.chunks, c0 = (u - before) - tile * v.chunks;
    const int n = min(v.chunks - c0, place.u_end - u);
    const int prefix = v.len - v.qlen;
    const int tok0 = tile * kTok;                   // first token of the tile, in the sequence
    const int ntok = min(kTok, v.qlen - tok0);
    const int wtok = wave * 2 * NT;                 // the wave's first token in the tile
    const bool wave_active = wtok < ntok;
    const int t_begin = v.begin + c0 * kChunk;
    const int t_end = min(v.len, t_begin + n * kChunk);
    const const_i32_ptr bt = as_constant(p.block_table + (size_t)s * p.max_blocks_per_seq);
    const int last_page = (v.len + kBlock - 1) / kBlock - 1;
    auto page_at = [&](const int tc) { return clamp_id(bt[min(tc / kBlock + wave, last_page)], p.last_block); };
    auto masked = [&](const int tc) {
      return tc + kChunk > prefix || (p.window > 0 && tc < prefix + v.qlen - p.window);
    };

    // ---- loaders: wave w brings page w of a chunk.  Rows past the end of the sequence repeat its
    // last row: nobody sees them, and the memory behind may never have been written.
    auto dma = [&](uint8_t *kbuf, uint8_t *vbuf, const int tc, const int page) {
      const int dr = lane >> 3, sl = lane & 7;
      const uint8_t *kp = p.k_cache + (size_t)page * page_bytes + (uint32_t)kvh * 128;
      const uint8_t *vp = p.v_cache + (size_t)page * page_bytes + (uint32_t)kvh * 128;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int tok = min(tc + 16 * wave + 8 * h + dr, v.len - 1);
        const uint32_t off = (uint32_t)(tok & 15) * row_bytes;
        const int kseg = sl ^ (4 * h + (dr >> 1)), vseg = sl ^ ((dr >> 1) << 1);
        __builtin_amdgcn_global_load_lds((gptr_t *)(kp + off + kseg * 16), (lptr_t *)(kbuf + (2 * wave + h) * 1024), 16, 0, kAux);
        __builtin_amdgcn_global_load_lds((gptr_t *)(vp + off + vseg * 16), (lptr_t *)(vbuf + (2 * wave + h) * 1024), 16, 0, kAux);
      }
    };
    const int fr = lane >> 2, fs = lane & 3;  // fp8: row of the page, 16-element segment
    auto fetch8 = [&](const int tc, const int page, u32x4 &kr, u32x4 &vr) {
      const int tok = min(tc + 16 * wave + fr, v.len - 1);
      const size_t off = (size_t)page * page_bytes + (uint32_t)(tok & 15) * row_bytes + (uint32_t)kvh * 64 + fs * 16;
      kr = *(const u32x4 *)(p.k_cache + off);
      vr = *(const u32x4 *)(p.v_cache + off);
    };
    auto stash8 = [&](uint8_t *kbuf, uint8_t *vbuf, const u32x4 kr, const u32x4 vr) {
      const int row = 16 * wave + fr, ks = (row >> 1) & 7, vsw = ((row >> 1) & 3) << 1;
      Frag8 x;
      fp8x8_to_bf16x8(kr[0], kr[1], x.w);
      *(u32x4 *)(kbuf + row * 128 + ((2 * fs) ^ ks) * 16) = x.u;
      fp8x8_to_bf16x8(kr[2], kr[3], x.w);
      *(u32x4 *)(kbuf + row * 128 + ((2 * fs + 1) ^ ks) * 16) = x.u;
      fp8x8_to_bf16x8(vr[0], vr[1], x.w);
      *(u32x4 *)(vbuf + row * 128 + ((2 * fs) ^ vsw) * 16) = x.u;
      fp8x8_to_bf16x8(vr[2], vr[3], x.w);
      *(u32x4 *)(vbuf + row * 128 + ((2 * fs + 1) ^ vsw) * 16) = x.u;
    };

    __syncthreads();  // (the last piece's readers are done)
    // Requested together: the first chunks' pages, the rows of q (row i16 of 16-row tile t is token
    // 2 t + i16 / 8, head i16 % 8; tokens past the end repeat the last), the masks; then the chunks.
    int pages[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) pages[i] = page_at(t_begin + i * kChunk);
    Frag8 qx[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int tok = tok0 + min(wtok + 2 * t + (i16 >> 3), ntok - 1);
      const uint16_t *src = p.q + ((size_t)(v.row0 + tok) * p.num_q_heads + kvh * kGroup + (i16 & 7)) * kHeadDim + 16 * g;
      qx[t][0].u = *(const u32x4 *)src;
      qx[t][1].u = *(const u32x4 *)(src + 8);
    }
    // bits of tokens of this sequence in word w of a row's mask
    auto mask_word = [&](const int tok, const int w) {
      const uint64_t m = p.mask[(size_t)(v.row0 + min(tok, v.qlen - 1)) * p.mask_words + min(w, p.mask_words - 1)];
      const int left = tok < v.qlen ? v.qlen - 64 * w : 0;
      return left <= 0 ? 0 : left < 64 ? m & ((1ull << left) - 1) : m;
    };
    uint64_t mine[kTreeWordsMax];
    if (tid < kTok) {
#pragma unroll
      for (int w = 0; w < kTreeWordsMax; ++w) mine[w] = mask_word(tok0 + tid, w);
    }
    u32x4 ka, va, kb, vb;  // fp8: two chunks under way
    int page = pages[0];
    if constexpr (FP8) {
      fetch8(t_begin, pages[0], ka, va);
      if (DEEP8 && t_begin + kChunk < t_end) fetch8(t_begin + kChunk, pages[1], kb, vb);
    } else {
      dma(k_st0, v_st0, t_begin, pages[0]);
      if constexpr (ST == 4) {
        if (t_begin + kChunk < t_end) dma(k_st1, v_st1, t_begin + kChunk, pages[1]);
        if (t_begin + 2 * kChunk < t_end) dma(k_st2, v_st2, t_begin + 2 * kChunk, pages[2]);
      }
    }
    Frag8 qf[QLDS ? 2 : NT][2];
    uint8_t *q_lds = lds_q + (QLDS ? wave * (2 * NT * 1024) + lane * 16 : 0);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if constexpr (QLDS) *(u32x4 *)(q_lds + (2 * t + h) * 1024) = qx[t][h].u;  // (read by this lane alone)
        else qf[t][h] = qx[t][h];
      }
    if (tid < kTok) {
      int depth = -1;
#pragma unroll
      for (int w = 0; w < kTreeWordsMax; ++w) {
        lds_mask[tid][w] = mine[w];
        depth += __popcll(mine[w]);
      }
      lds_lo[tid] = p.window > 0 ? prefix + depth - p.window + 1 : 0;
    }
    // A drafted token may lie outside a row's window: depths go from -1 (an empty mask) to qlen - 1.
    if (p.window > 0 && p.window <= v.qlen) {
      int depth = -1;  // of token tid of the tree
      for (int w = 0; w < p.mask_words; ++w) depth += __popcll(mask_word(tid, w));
      lds_depth[tid] = depth;
      __syncthreads();
      uint64_t keep = 0;
      const int tl = tid / kTreeWordsMax, w = tid % kTreeWordsMax;
      if (tl < kTok) {
        uint64_t m = lds_mask[tl][w];
        keep = m;
        while (m) {
          const int b = __builtin_ctzll(m);
          m &= m - 1;
          if (prefix + lds_depth[64 * w + b] < lds_lo[tl]) keep &= ~(1ull << b);
        }
      }
      __syncthreads();
      if (tl < kTok) lds_mask[tl][w] = keep;
    }

    float m[NT], l[NT];
    f32x4 acc[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      m[t] = kNegBig;
      l[t] = 0.f;
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) acc[t][mt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    bool fresh = true;  // no row has a reference from a chunk that it sees whole
    bool odd = false;  // this lane took a value that is not finite out of a masked chunk

    // One chunk.  Its tiles overlap: while tile t's exponentials run, the matrix unit works on the
    // scores of tile t + 1 and the output of tile t - 1.  A row's reference is the maximum of its first
    // chunks (those that are masked and the first that is not) and then stays: a weight may grow far
    // beyond 1, which costs nothing in fp32 and bf16 until its row's sum reaches 2^60 (see guard).
    // Row sums: products of the rounded weights with ones; exact fp32 sums where lse is asked for.
    auto step = [&](const uint8_t *kbuf, const uint8_t *vbuf, const int tc) {
      const bool need_mask = masked(tc);  // (one stream for both kinds: two would not share registers)
      const bool track = need_mask || fresh;
      Frag8 kf[4][2], vf[4][2];
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        kf[b][0].u = *(const u32x4 *)(kbuf + k_off + b * (kBlock * 128));
        kf[b][1].u = *(const u32x4 *)(kbuf + (k_off ^ 16) + b * (kBlock * 128));
      }
#pragma unroll
      for (int mt = 0; mt < 4; ++mt)
#pragma unroll
        for (int pr = 0; pr < 2; ++pr) {
          const uint8_t *src = vbuf + v_off + ((32 * mt) ^ v_sw);
          const u32x2 a = lds_read_tr16(src + (2 * pr) * (kBlock * 128));
          const u32x2 b = lds_read_tr16(src + (2 * pr + 1) * (kBlock * 128));
          vf[mt][pr].w[0] = a[0];
          vf[mt][pr].w[1] = a[1];
          vf[mt][pr].w[2] = b[0];
          vf[mt][pr].w[3] = b[1];
        }
      if (need_mask) {
#pragma unroll
        for (int mt = 0; mt < 4; ++mt)
#pragma unroll
          for (int pr = 0; pr < 2; ++pr)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t &x = vf[mt][pr].w[i];
              const bool hi = (x & 0x7F800000u) == 0x7F800000u, lo = (x & 0x7F80u) == 0x7F80u;
              odd |= hi | lo;
              x &= (hi ? 0xFFFFu : ~0u) & (lo ? 0xFFFF0000u : ~0u);
            }
      }
      f32x4 S[2][4], lt;
      Frag8 P[2][2];
      float sum = 0.f;  // LSE: of a tile's weights, this lane's keys
      auto load_q = [&](auto t_c) {
        constexpr int t = t_c;
        if constexpr (QLDS && t < NT) {
          qf[t & 1][0].u = *(const u32x4 *)(q_lds + (2 * t) * 1024);
          qf[t & 1][1].u = *(const u32x4 *)(q_lds + (2 * t + 1) * 1024);
        }
      };
      // matrix instruction j of 8: scores of tile t / output of tile t
      auto score = [&](auto t_c, auto j_c) {
        constexpr int t = t_c, j = j_c, b = j & 3, x = QLDS ? t & 1 : t;
        if constexpr (j < 4) S[t & 1][b] = mfma16x32(kf[b][0], qf[x][0], f32x4{0.f, 0.f, 0.f, 0.f});
        else S[t & 1][b] = mfma16x32(kf[b][1], qf[x][1], S[t & 1][b]);
      };
      auto value = [&](auto t_c, auto j_c) {
        constexpr int t = t_c, j = j_c, mt = j & 3, pr = j >> 2;
        acc[t][mt] = mfma16x32(vf[mt][pr], P[t & 1][pr], acc[t][mt]);
      };
      auto row_sum = [&](auto t_c, auto j_c) {  // every lane of a row receives its sum over the chunk
        constexpr int t = t_c, j = j_c;
        if constexpr (j == 0) lt = mfma16x32(ones, P[t & 1][0], f32x4{0.f, 0.f, 0.f, 0.f});
        else lt = mfma16x32(ones, P[t & 1][1], lt);
      };
      auto lane_max = [&](const f32x4(&Sx)[4]) {
        float mx = max3(Sx[0][0], Sx[0][1], Sx[0][2]);
#pragma unroll
        for (int o = 1; o < 7; ++o)
          mx = max3(mx, Sx[(2 * o + 1) >> 2][(2 * o + 1) & 3], Sx[(2 * o + 2) >> 2][(2 * o + 2) & 3]);
        return max2(mx, Sx[3][3]) * c2;
      };
      auto move_ref = [&](auto t_c, const float m_new) {
        constexpr int t = t_c;
        const float alpha = fast_exp2(m[t] - m_new);
        l[t] *= alpha;
#pragma unroll
        for (int mt = 0; mt < 4; ++mt)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[t][mt][r] *= alpha;
        m[t] = m_new;
      };
      // After tile t's weights: a row whose sum is not below 2^60 (inf and NaN among that) has outgrown
      // its reference.  Its scores are computed again and the reference moves to their maximum.  (In a
      // masked chunk the reference has just followed the maximum: only a NaN could be found there.)
      auto guard = [&](auto t_c) {
        constexpr int t = t_c;
        float got = LSE ? sum : lt[0];
        if (!need_mask && __any(!(got < kRowSumGuard))) {
          f32x4(&Sx)[4] = S[t & 1];
          Frag8 q2[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if constexpr (QLDS) q2[h].u = *(const u32x4 *)(q_lds + (2 * t + h) * 1024);
            else q2[h] = qf[QLDS ? 0 : t][h];
          }
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            Sx[b] = mfma16x32(kf[b][0], q2[0], f32x4{0.f, 0.f, 0.f, 0.f});
            Sx[b] = mfma16x32(kf[b][1], q2[1], Sx[b]);
          }
          move_ref(t_c, max2(m[t], rowgroup_max(lane_max(Sx))));  // (a plain chunk: every key is seen)
          got = 0.f;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float p0 = fast_exp2(__builtin_fmaf(Sx[(2 * k) >> 2][(2 * k) & 3], c2, -m[t]));
            const float p1 = fast_exp2(__builtin_fmaf(Sx[(2 * k + 1) >> 2][(2 * k + 1) & 3], c2, -m[t]));
            got += p0 + p1;
            P[t & 1][k >> 2].w[k & 3] = pack_bf16(p0, p1);
          }
          if constexpr (!LSE) got = rowgroup_sum(got);
        }
        l[t] += got;
      };
      load_q(IC<0>{});
      load_q(IC<1>{});
      static_for<8>([&](auto j) { score(IC<0>{}, j); });
      static_for<NT>([&](auto t_c) {
        constexpr int t = t_c;
        f32x4(&Sx)[4] = S[t & 1];
        if constexpr (t > 0) guard(IC<t - 1>{});
        if (track) {
          if (need_mask) {
            const int tl = wtok + 2 * t + (i16 >> 3);
            const uint64_t w = chunk_bits(lds_mask[tl], lds_lo[tl], prefix, tc) >> (4 * g);
#pragma unroll
            for (int b = 0; b < 4; ++b)
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (!((w >> (16 * b + r)) & 1)) Sx[b][r] = -INFINITY;
          }
          const float mx = lane_max(Sx);
          if (__any(mx > m[t] + kLazyLog2)) {
            const float mrow = rowgroup_max(mx);
            move_ref(t_c, mrow > m[t] + kLazyLog2 ? mrow : m[t]);
          }
        }
        EID_SB();
        // The stage: output of tile t - 1, scores of tile t + 1, and between them the 16 scores of a
        // lane; the row sums two matrix instructions before the end, so that they are there for the guard.
        constexpr int n_value = t > 0 ? 8 : 0, n_score = t + 1 < NT ? 8 : 0, n_mfma = n_value + n_score;
        constexpr int slots = n_mfma > 0 ? n_mfma : 1, spread = n_mfma > 2 ? n_mfma - 2 : 1;
        static_for<slots>([&](auto i_c) {
          constexpr int i = i_c;
          if constexpr (!LSE && i == spread) {
            row_sum(t_c, IC<0>{});
            row_sum(t_c, IC<1>{});
          }
          if constexpr (i < n_value) value(IC<(t > 0 ? t - 1 : 0)>{}, i_c);
          else if constexpr (i < n_mfma) score(IC<(t + 1 < NT ? t + 1 : 0)>{}, IC<i - n_value>{});
          if constexpr (i == n_mfma - 1) load_q(IC<t + 2>{});
          static_for<16>([&](auto e_c) {
            constexpr int e = e_c;
            if constexpr (e * spread / 16 == i) {
              const float x = fast_exp2(__builtin_fmaf(Sx[e >> 2][e & 3], c2, -m[t]));
              Sx[e >> 2][e & 3] = x;
              if constexpr (e % 2 == 1) {
                const float y = Sx[(e - 1) >> 2][(e - 1) & 3];
                uint32_t w = pack_bf16(y, x);
                // (pinned here: they would be sunk to where they are used)
                if constexpr (LSE) {
                  sum = e == 1 ? y + x : sum + y + x;
                  asm volatile("" : "+v"(w), "+v"(sum));
                } else {
                  asm volatile("" : "+v"(w));
                }
                P[t & 1][e >> 3].w[(e >> 1) & 3] = w;
              }
            }
          });
          EID_SB();
        });
        if constexpr (!LSE && spread >= slots) {
          row_sum(t_c, IC<0>{});
          row_sum(t_c, IC<1>{});
        }
      });
      guard(IC<NT - 1>{});
      static_for<8>([&](auto j) { value(IC<NT - 1>{}, j); });
      if (!need_mask) fresh = false;
    };

    if constexpr (FP8) {
      // chunk c is in stage c % 2, chunk c + 1 in registers; with registers to spare chunk c + 2 is
      // requested as well
      stash8(k_st0, v_st0, ka, va);
      __syncthreads();
      auto iter = [&](const uint8_t *kcur, const uint8_t *vcur, uint8_t *knxt, uint8_t *vnxt, u32x4 &k1, u32x4 &v1,
                      u32x4 &k2, u32x4 &v2, const int tc) {
        if constexpr (DEEP8) {
          if (tc + 2 * kChunk < t_end) fetch8(tc + 2 * kChunk, page_at(tc + 2 * kChunk), k2, v2);
        } else {
          if (tc + kChunk < t_end) fetch8(tc + kChunk, page_at(tc + kChunk), k1, v1);
        }
        if (wave_active) step(kcur, vcur, tc);
        if (tc + kChunk < t_end) stash8(knxt, vnxt, k1, v1);
        __syncthreads();
      };
      for (int tc = t_begin; tc < t_end; tc += 2 * kChunk) {
        iter(k_st0, v_st0, k_st1, v_st1, DEEP8 ? kb : ka, DEEP8 ? vb : va, ka, va, tc);
        if (tc + kChunk < t_end) iter(k_st1, v_st1, k_st0, v_st0, ka, va, kb, vb, tc + kChunk);
      }
    } else {
      page = ST == 2 ? pages[1] : page_at(t_begin + (ST - 1) * kChunk);
      // (the first chunk's loads are the oldest; the rows of q behind them have to be here as well)
      __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
      __syncthreads();
      auto iter = [&](const uint8_t *kcur, const uint8_t *vcur, uint8_t *kfar, uint8_t *vfar, const int tc) {
        const bool more = tc + (ST - 1) * kChunk < t_end;
        if (more) {
          dma(kfar, vfar, tc + (ST - 1) * kChunk, page);
          page = page_at(tc + ST * kChunk);
        }
        if (wave_active) step(kcur, vcur, tc);
        // The next chunk has landed: its four loads are older than those of the chunks behind it.
        // Not __syncthreads(): it would wait for all of them.
        if (ST == 4 && tc + 3 * kChunk < t_end) asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)" ::: "memory");
        else if (ST == 4 && tc + 2 * kChunk < t_end) asm volatile("s_waitcnt vmcnt(4) lgkmcnt(0)" ::: "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
      };
      for (int tc = t_begin; tc < t_end; tc += ST * kChunk) {
        if constexpr (ST == 4) {
          iter(k_st0, v_st0, k_st3, v_st3, tc);
          if (tc + kChunk < t_end) iter(k_st1, v_st1, k_st0, v_st0, tc + kChunk);
          if (tc + 2 * kChunk < t_end) iter(k_st2, v_st2, k_st1, v_st1, tc + 2 * kChunk);
          if (tc + 3 * kChunk < t_end) iter(k_st3, v_st3, k_st2, v_st2, tc + 3 * kChunk);
        } else {
          iter(k_st0, v_st0, k_st1, v_st1, tc);
          if (tc + kChunk < t_end) iter(k_st1, v_st1, k_st0, v_st0, tc + kChunk);
        }
      }
    }

    // Values that are not finite were taken out of masked chunks: their keys' terms are added row
    // by row, for the rows that see them.  (Rare, and slow: one dot product per row and key.)
    if (wave_active && __any(odd)) {
      for (int tc = t_begin; tc < t_end; tc += kChunk) {
        if (!masked(tc)) continue;
        auto row_at = [&](const int j) {
          const int pg = clamp_id(bt[min(j / kBlock, last_page)], p.last_block);
          return (size_t)pg * page_bytes + (size_t)(j % kBlock) * row_bytes + (size_t)kvh * (kHeadDim * kElt);
        };
        auto elem = [&](const uint8_t *row, const int d) {
          if constexpr (FP8) {
            uint32_t o[4];
            fp8x8_to_bf16x8(row[d], 0, o);
            return bf16_bits_to_f32(o[0] & 0xFFFFu);
          } else {
            return bf16_bits_to_f32(*(const uint16_t *)(row + 2 * d));
          }
        };
        auto finite = [](const float x) { return (__float_as_uint(x) & 0x7F800000u) != 0x7F800000u; };
        bool has = false;  // of key tc + lane
        if (tc + lane < v.len) {
          const uint8_t *row = p.v_cache + row_at(tc + lane);
          for (int d = 0; d < kHeadDim; ++d) has |= !finite(elem(row, d));
        }
        uint64_t bad = __ballot(has);
        while (bad) {
          const int b = __builtin_ctzll(bad);
          bad &= bad - 1;
          const uint8_t *krow = p.k_cache + row_at(tc + b), *vrow = p.v_cache + row_at(tc + b);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            const int tl = wtok + 2 * t + (i16 >> 3);
            if (tl < ntok && (chunk_bits(lds_mask[tl], lds_lo[tl], prefix, tc) >> b & 1)) {
              const uint16_t *qr = p.q + ((size_t)(v.row0 + tok0 + tl) * p.num_q_heads + kvh * kGroup + (i16 & 7)) * kHeadDim;
              float dot = 0.f;
              for (int d = 0; d < kHeadDim; ++d) dot += bf16_bits_to_f32(qr[d]) * elem(krow, d);
              const float w = fast_exp2(__builtin_fmaf(dot, c2, -m[t]));
#pragma unroll
              for (int mt = 0; mt < 4; ++mt)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                  const float x = elem(vrow, 16 * mt + 4 * g + r);
                  if (!finite(x)) acc[t][mt][r] += w * x;
                }
            }
          }
        }
      }
    }

    // ---- this piece's rows: the answer, or a partial
    const bool whole = n == v.chunks;
    const int part = c0 == 0 ? 1 : 0;  // a range holds at most one piece of each kind that is not whole
    _Float16 *ws_o = p.ws_o + ((size_t)(range * Hkv + kvh) * 2 + part) * (kRows * kHeadDim);
    TreeStats *ws_ml = p.ws_ml + ((size_t)(range * Hkv + kvh) * 2 + part) * kRows;
    if (c0 == 0 && kvh == 0 && tid == 0 && !p.whole) {  // the tile begins here: where its pieces are
      const int last = u + v.chunks - 1;    // its last unit
      p.ws_rec[s * p.max_tiles + tile] = {range, last / place.per - range + 1};
    }
    if (wave_active) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int tl = wtok + 2 * t + (i16 >> 3);
        const float lt = LSE ? rowgroup_sum(l[t]) : l[t];
        if (tl >= ntok) continue;
        if (whole) {
          const int head = kvh * kGroup + (i16 & 7);
          const float sink = p.sinks ? p.sinks[head] * kLog2e : -INFINITY;
          // (a row that sees nothing, m = kNegBig, has only its sink)
          const float M = max2(m[t], sink), a = fast_exp2(m[t] - M);
          const float den = lt * a + fast_exp2(sink - M);
          const bool any = den > 0.f || den != den;
          const float f = any ? vs * a / den : 0.f;
          const size_t orow = (size_t)(v.row0 + tok0 + tl) * p.num_q_heads + head;
#pragma unroll
          for (int mt = 0; mt < 4; ++mt) {
            u32x2 w;
            w[0] = pack_bf16(acc[t][mt][0] * f, acc[t][mt][1] * f);
            w[1] = pack_bf16(acc[t][mt][2] * f, acc[t][mt][3] * f);
            *(u32x2 *)(p.out + orow * kHeadDim + 16 * mt + 4 * g) = w;
          }
          if (p.lse && g == 0) p.lse[orow] = any ? (M + __log2f(den)) * kLn2 : -INFINITY;
        } else {
          // The outputs go out as fp16 beside a power of two of the row's own, which brings its largest
          // (finite) one to [2^14, 2^15): roundings of 2^-11 of an output down to 2^-28 of the largest, and of
          // 2^-39 of the largest below, against the 2^-8 of the bf16 that the answer is rounded to; and
          // half the bytes of fp32.  The power stands apart from m and l, which do not depend on V: moved
          // into them it would overflow l where all outputs of a piece are tiny.
          const int row = tl * kGroup + (i16 & 7);
          float top = 0.f;
#pragma unroll
          for (int mt = 0; mt < 4; ++mt)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float x = fabsf(acc[t][mt][r]);
              top = fmaxf(top, x < INFINITY ? x : 0.f);
            }
          const int e = top_exponent(rowgroup_max(top)) - 15;
#pragma unroll
          for (int h = 0; h < 2; ++h) {  // (a lane's 16 dims next to each other: 16 mt + 4 g + r at 16 g + 4 mt + r)
            f16x8 x;
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = (_Float16)ldexpf(acc[t][2 * h + i / 4][i & 3], -e);
            *(f16x8 *)(ws_o + (size_t)row * kHeadDim + 16 * g + 8 * h) = x;
          }
          if (g == 0) ws_ml[row] = TreeStats{m[t], lt, e, 0};
        }
      }
    }
    u += n;
  }
}

// Joins the pieces of a tile that range ends cut: out = sum 2^(m + e - M) o / (sum 2^(m - M) l + 2^(sink - M)).
// Eight lanes take a row, PG lane groups every PG-th of its pieces, four at a time; a workgroup holds
// 32 / PG rows of one tile.  Bound by launch and memory latency: 4-7 us (16 trees of 16 tokens: 5 us).
template <int PG>
__global__ __launch_bounds__(256) void tree_merge_kernel(const TreeParams p, const int tile_tok) {
  constexpr int kTokens = 4 / PG;  // of a workgroup (PG 1: four, PG 4: one)
  const int Hkv = p.num_kv_heads, kvh = blockIdx.x % Hkv;
  const int b = blockIdx.x / Hkv, tiles = p.num_seqs * p.max_tiles, at = b % tiles, tok = b / tiles * kTokens;
  const int s = at / p.max_tiles, tok0 = at % p.max_tiles * tile_tok;
  const const_i32_ptr cu = as_constant(p.cu_seqlens_q), sl = as_constant(p.seq_lens);
  const TreeSeq v = tree_seq(p, cu[s], cu[s + 1], sl[s], tile_tok);
  const int ntok = min(v.qlen - tok0, tile_tok);
  if (tok >= ntok) return;
  const TreeRecord rec = p.ws_rec[at];
  if (rec.pieces < 2) return;  // a range held it whole
  // lane = 8 pg + eighth, so that a row's piece groups are lanes of one wave
  const int eighth = threadIdx.x & 7, pg = (threadIdx.x >> 3) % PG, row = threadIdx.x / (8 * PG);
  const int tl = tok + (row >> 3), h = row & 7;
  const int rows = tile_tok * kGroup;
  const size_t cell0 = (size_t)(rec.range * Hkv + kvh) * 2 * rows + tl * kGroup + h;
  const int head = kvh * kGroup + h;
  float o[8], M = kNegBig, den = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) o[k] = 0.f;
  if (tl < ntok) {
    for (int i = pg; i < rec.pieces; i += 4 * PG) {
      TreeStats ml[4];
      f16x8 x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = min(i + e * PG, rec.pieces - 1);  // (past the end the last one again, without weight)
        const size_t c = cell0 + (size_t)j * Hkv * 2 * rows + (j == 0 ? rows : 0);
        ml[e] = p.ws_ml[c];
        x[e] = *(const f16x8 *)(p.ws_o + c * kHeadDim + 8 * eighth);
      }
      float M1 = M;
#pragma unroll
      for (int e = 0; e < 4; ++e) M1 = i + e * PG < rec.pieces ? max2(M1, ml[e].m) : M1;
      const float a = fast_exp2(M - M1);
      den *= a;
#pragma unroll
      for (int k = 0; k < 8; ++k) o[k] *= a;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e * PG < rec.pieces) {
          const float w = fast_exp2(ml[e].m - M1), wo = ldexpf(w, ml[e].e);
          den += ml[e].l * w;
#pragma unroll
          for (int k = 0; k < 8; ++k) o[k] += (float)x[e][k] * wo;
        }
      M = M1;
    }
  }
  const float sink = p.sinks ? p.sinks[head] * kLog2e : -INFINITY;
  float all = M;
#pragma unroll
  for (int d = 8; d < 8 * PG; d <<= 1) all = max2(all, __shfl_xor(all, d));
  all = max2(all, sink);
  const float a = fast_exp2(M - all);
  den *= a;
#pragma unroll
  for (int k = 0; k < 8; ++k) o[k] *= a;
#pragma unroll
  for (int d = 8; d < 8 * PG; d <<= 1) {
    den += __shfl_xor(den, d);
#pragma unroll
    for (int k = 0; k < 8; ++k) o[k] += __shfl_xor(o[k], d);
  }
  den += fast_exp2(sink - all);
  if (tl >= ntok || pg > 0) return;
  const float vs = p.v_scale ? p.v_scale[kvh] : 1.0f;
  const bool any = den > 0.f || den != den;
  const float f = any ? vs / den : 0.f;
  const size_t orow = (size_t)(v.row0 + tok0 + tl) * p.num_q_heads + head;
  // value 16 g + 4 mt + r of a piece is dim 16 mt + 4 g + r
  uint16_t *dst = p.out + orow * kHeadDim + 4 * (eighth >> 1) + 32 * (eighth & 1);
#pragma unroll
  for (int k = 0; k < 2; ++k)
    *(u32x2 *)(dst + 16 * k) = u32x2{pack_bf16(o[4 * k] * f, o[4 * k + 1] * f), pack_bf16(o[4 * k + 2] * f, o[4 * k + 3] * f)};
  if (p.lse && eighth == 0) p.lse[orow] = any ? (all + __log2f(den)) * kLn2 : -INFINITY;
}

}  // namespace

// 16-row tiles per wave: a tree is cut into the fewest tiles of at most 32 tokens, of about equal size,
// in steps of 8 tokens.  16 trees of 40 tokens behind 8k keys: two tiles of 24 145 us, of 32 164 us;
// 8 tokens: a tile of 8 59 us, of 32 79 us.
int tree_tiles(const int max_q_len) {
  const int tiles = (max_q_len + 31) / 32;
  return ((max_q_len + tiles - 1) / tiles + 7) / 8;
}
int tree_tile_tokens(const int max_q_len) { return 2 * tree_tiles(max_q_len) * kTreeWaves; }

template <bool FP8, bool LSE>
static void launch_tree_tiles(const TreeParams &p, const int nt, hipStream_t st) {
  const dim3 grid((unsigned)(p.ranges * p.num_kv_heads)), block(kTreeWaves * 64);
  if (nt == 1) tree_kernel<1, FP8, LSE><<<grid, block, 0, st>>>(p);
  else if (nt == 2) tree_kernel<2, FP8, LSE><<<grid, block, 0, st>>>(p);
  else if (nt == 3) tree_kernel<3, FP8, LSE><<<grid, block, 0, st>>>(p);
  else tree_kernel<4, FP8, LSE><<<grid, block, 0, st>>>(p);
}

hipError_t launch_tree(const TreeParams &p, const bool fp8, hipStream_t st) {
  const int nt = tree_tiles(p.max_q_len);
  if (fp8) p.lse ? launch_tree_tiles<true, true>(p, nt, st) : launch_tree_tiles<true, false>(p, nt, st);
  else p.lse ? launch_tree_tiles<false, true>(p, nt, st) : launch_tree_tiles<false, false>(p, nt, st);
  return hipGetLastError();
}

hipError_t launch_tree_merge(const TreeParams &p, hipStream_t st) {
  // Many pieces of few tiles: their pieces side by side (1 x 16 behind 16k keys: 22 us against 28); else
  // a workgroup takes more rows (32 x 16 behind 4k, two pieces a tile: 73 us against 78).
  const int tile = tree_tile_tokens(p.max_q_len);
  const unsigned tiles = (unsigned)(p.num_seqs * p.max_tiles), cells = tiles * (unsigned)p.num_kv_heads;
  if ((unsigned)p.ranges > 4 * tiles) tree_merge_kernel<4><<<cells * tile, 256, 0, st>>>(p, tile);
  else tree_merge_kernel<1><<<cells * (tile / 4), 256, 0, st>>>(p, tile);
  return hipGetLastError();
}

}  // namespace eid
