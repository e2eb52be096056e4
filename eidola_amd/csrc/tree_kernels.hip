// gfx950 kernels of the attention for trees of drafted tokens over the paged cache.
#include "eid_cache_params.h"
#include "eid_device.h"

namespace eid {

namespace {

typedef const __attribute__((address_space(4))) int32_t *const_i32_ptr;
__device__ __forceinline__ const_i32_ptr as_constant(const int32_t *p) { return (const_i32_ptr)(uintptr_t)p; }
__device__ __forceinline__ int clamp_id(const int id, const int last) { return min(max(id, 0), last); }

// LDS row strides of the K and V tiles (see the prefill kernel: K is read 16 bytes per lane by 16
// lanes of one row each, V^T through the transposing read)
constexpr int kKRow = 144, kVRow = 160;
constexpr float kLazyLog2 = 8.0f;  // a row's reference moves when a score outgrows it by this

// What one sequence gives the kernels: `chunks` 64-key chunks from key `begin` on for each of
// `tiles` tiles of drafted tokens.
struct TreeSeq {
  int row0, qlen, len, begin, chunks, tiles;
};

// The rows at and behind prefix = len - qlen stand for the drafted tokens.  A token's position is
// prefix + (ancestors it sees) >= prefix - 1, so no row sees keys below prefix - window.
__device__ __forceinline__ TreeSeq tree_seq(const TreeParams &p, const int s, const int tile_tok) {
  TreeSeq v;
  const const_i32_ptr cu = as_constant(p.cu_seqlens_q), sl = as_constant(p.seq_lens);
  v.row0 = cu[s];
  v.qlen = cu[s + 1] - v.row0;
  v.len = min(sl[s], p.max_blocks_per_seq * kBlock);
  // (junk lengths: nothing of the sequence is computed, nothing is read)
  if (v.qlen < 0 || v.qlen > kTreeMax || v.qlen > p.mask_words * 64 || v.len < v.qlen || v.row0 < 0 ||
      v.row0 + v.qlen > p.num_q_tokens)
    v.qlen = 0;
  v.begin = p.window > 0 ? max(0, v.len - v.qlen - p.window) & ~(kBlock - 1) : 0;
  v.tiles = (v.qlen + tile_tok - 1) / tile_tok;
  v.chunks = v.qlen > 0 ? (v.len - v.begin + kChunk - 1) / kChunk : 0;
  return v;
}
__device__ __forceinline__ long long units_of(const TreeSeq &v) { return (long long)v.tiles * v.chunks; }

__device__ __forceinline__ long long uniform64(const long long x) {
  return (long long)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)x) |
                     (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32);
}

// Units of all sequences, and those of the sequences before `upto`: by every wave for itself.
__device__ __forceinline__ void count_units(const TreeParams &p, const int tile_tok, const int upto,
                                            long long &total, long long &before) {
  const int lane = threadIdx.x & 63;
  long long a = 0, b = 0;
  for (int s = lane; s < p.num_seqs; s += 64) {
    const long long u = units_of(tree_seq(p, s, tile_tok));
    a += u;
    if (s < upto) b += u;
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) {
    a += __shfl_xor(a, d);
    b += __shfl_xor(b, d);
  }
  total = uniform64(a);
  before = uniform64(b);
}

// Sequence that holds unit u and the units before it.
__device__ __forceinline__ int find_seq(const TreeParams &p, const int tile_tok, const long long u,
                                        long long &before) {
  const int lane = threadIdx.x & 63;
  long long base = 0;
  for (int s0 = 0; s0 < p.num_seqs; s0 += 64) {
    const int s = s0 + lane;
    const long long n = s < p.num_seqs ? units_of(tree_seq(p, s, tile_tok)) : 0;
    long long incl = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const long long o = __shfl_up(incl, d);
      if (lane >= d) incl += o;
    }
    const unsigned long long hit = __ballot(base + incl > u);
    if (hit) {
      const int i = __builtin_ctzll(hit);
      before = uniform64(base + __shfl(incl, i) - __shfl(n, i));
      return s0 + i;
    }
    base += uniform64(__shfl(incl, 63));
  }
  before = base;
  return p.num_seqs;
}

// Chunks per workgroup: equal contiguous ranges of the launch's units.
__device__ __forceinline__ long long range_units(const TreeParams &p, const long long total) {
  const long long q = (total + p.ranges - 1) / p.ranges;
  return q > p.min_chunks ? q : p.min_chunks;
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
  const int cut = min(min(lo, prefix) - tc, 64);  // context keys below the window
  if (cut >= 64) w = 0;
  else if (cut > 0) w &= ~((1ull << cut) - 1);
  return w;
}

// ---------------------------------------------------------------------------------------
// out[i] = sum_j vis(i, j) e^(c q_i.k_j) v_j / (sum_j vis(i, j) e^(c q_i.k_j) + e^sink), with
// vis(i, j) = j < prefix, or bit j - prefix of row i's mask; one pass with a running reference.
//
// A workgroup of four waves owns tile_tok = 8 NT drafted tokens x the 8 query heads of one KV
// head: 16 NT rows per wave.  The launch's (sequence, tile) pairs, 64 keys at a time, are laid
// out in a line and cut into `ranges` equal pieces, one per workgroup, so that a batch of unequal
// contexts loads every CU alike; a range that ends inside a sequence leaves (o, m, l) for
// tree_merge_kernel.  K and V chunks go through LDS, double buffered, and are read by all waves.
// ---------------------------------------------------------------------------------------
template <int NT, bool FP8>
__global__ __launch_bounds__(kTreeWaves * 64, 2) void tree_kernel(const TreeParams p) {
  constexpr int kTok = 2 * NT * kTreeWaves;  // tokens of a tile
  constexpr int kRows = kTok * kGroup;
  constexpr int kElt = FP8 ? 1 : 2;
  __shared__ __align__(16) uint8_t lds_k[2][kChunk * kKRow];
  __shared__ __align__(16) uint8_t lds_v[2][kChunk * kVRow];
  __shared__ uint64_t lds_mask[kTok][kTreeWordsMax];
  __shared__ int lds_lo[kTok];
  __shared__ uint32_t lds_bad[3][2];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i16 = lane & 15, g = lane >> 4;
  const int Hkv = p.num_kv_heads;
  const int kvh = blockIdx.x % Hkv, range = blockIdx.x / Hkv;
  const float c2 = p.softmax_scale * kLog2e * (FP8 ? p.k_scale[kvh] : 1.0f);
  const float vs = FP8 ? p.v_scale[kvh] : 1.0f;

  long long total, ignored;
  count_units(p, kTok, 0, total, ignored);
  const long long per = range_units(p, total);
  long long u = per * range;
  const long long u_end = min(total, u + per);
  if (u >= u_end) return;
  long long before;
  int s = find_seq(p, kTok, u, before);

  const uint32_t row_bytes = (uint32_t)Hkv * kHeadDim * kElt;
  const size_t page_bytes = (size_t)kBlock * row_bytes;
  const int ld_row = tid >> 2, ld_seg = tid & 3;  // loader: row of the chunk, 16-element segment
  const uint32_t gl_off = (uint32_t)(ld_row & 15) * row_bytes + (uint32_t)kvh * (kHeadDim * kElt) +
                          (uint32_t)ld_seg * (16 * kElt);

  while (u < u_end) {
    TreeSeq v = tree_seq(p, s, kTok);
    if (u - before >= units_of(v)) {  // next sequence (those without rows have no units)
      before += units_of(v);
      ++s;
      continue;
    }
    const int tile = (int)((u - before) / v.chunks);
    const int c0 = (int)((u - before) - (long long)tile * v.chunks);
    const int n = (int)min((long long)(v.chunks - c0), u_end - u);
    const int prefix = v.len - v.qlen;
    const int tok0 = tile * kTok;  // first token of the tile, in the sequence
    const int t_begin = v.begin + c0 * kChunk;
    const int t_end = min(v.len, t_begin + n * kChunk);
    const const_i32_ptr bt = as_constant(p.block_table + (size_t)s * p.max_blocks_per_seq);
    const int last_page = (v.len + kBlock - 1) / kBlock - 1;

    // ---- the tile's masks: bits of tokens of this sequence, those outside the window taken out
    __syncthreads();  // (the last piece's readers are done)
    if (tid < kTok) {
      const int tok = tok0 + tid;
      int depth = -1;
#pragma unroll
      for (int w = 0; w < kTreeWordsMax; ++w) {
        uint64_t m = 0;
        if (tok < v.qlen && w < p.mask_words) m = p.mask[(size_t)(v.row0 + tok) * p.mask_words + w];
        const int left = v.qlen - 64 * w;
        if (left <= 0) m = 0;
        else if (left < 64) m &= (1ull << left) - 1;
        lds_mask[tid][w] = m;
        depth += __popcll(m);
      }
      lds_lo[tid] = p.window > 0 ? prefix + depth - p.window + 1 : 0;
    }
    if (tid < 6) (&lds_bad[0][0])[tid] = 0;
    __syncthreads();
    if (p.window > 0 && p.window < v.qlen) {  // an ancestor may lie outside the window
      uint64_t keep = 0;
      const int tl = tid / kTreeWordsMax, w = tid % kTreeWordsMax;
      if (tl < kTok) {
        uint64_t m = lds_mask[tl][w];
        keep = m;
        while (m) {
          const int b = __builtin_ctzll(m);
          m &= m - 1;
          const int j = 64 * w + b;  // an ancestor: its depth comes from its own mask
          int dj = -1;
          for (int x = 0; x < p.mask_words; ++x) {
            uint64_t a = p.mask[(size_t)(v.row0 + j) * p.mask_words + x];
            const int left = v.qlen - 64 * x;
            if (left <= 0) a = 0;
            else if (left < 64) a &= (1ull << left) - 1;
            dj += __popcll(a);
          }
          if (prefix + dj < lds_lo[tl]) keep &= ~(1ull << b);
        }
      }
      __syncthreads();
      if (tl < kTok) lds_mask[tl][w] = keep;
      __syncthreads();
    }

    // ---- Q operands: row i16 of 16-row tile t is token 2 t + i16 / 8, head i16 % 8
    const int wtok = wave * 2 * NT;  // the wave's first token in the tile
    const bool wave_active = tok0 + wtok < v.qlen;
    Frag8 qf[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int tok = tok0 + wtok + 2 * t + (i16 >> 3);
      qf[t][0].u = qf[t][1].u = u32x4{0, 0, 0, 0};
      if (tok < v.qlen) {
        const uint16_t *src = p.q + ((size_t)(v.row0 + tok) * p.num_q_heads + kvh * kGroup + (i16 & 7)) * kHeadDim + 16 * g;
        qf[t][0].u = *(const u32x4 *)src;
        qf[t][1].u = *(const u32x4 *)(src + 8);
      }
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

    // ---- loader
    u32x4 kr[kElt], vr[kElt];
    auto fetch = [&](const int tc) {
      const int page = clamp_id(bt[min(tc / kBlock + wave, last_page)], p.last_block);
      const uint8_t *kp = p.k_cache + (size_t)page * page_bytes + gl_off;
      const uint8_t *vp = p.v_cache + (size_t)page * page_bytes + gl_off;
#pragma unroll
      for (int e = 0; e < kElt; ++e) {
        kr[e] = *(const u32x4 *)(kp + 16 * e);
        vr[e] = *(const u32x4 *)(vp + 16 * e);
      }
    };
    // A chunk that not every row sees whole: keys past the end read as zero; a value that is not
    // finite must not reach rows that do not see it (0 x inf is NaN in the matrix product), so it
    // is taken out of the tile and its key remembered (see below).
    auto masked = [&](const int tc) {
      return tc + kChunk > prefix || (p.window > 0 && tc < prefix + v.qlen - p.window);
    };
    auto stash = [&](const int tc, const int buf, const int slot) {
      u32x4 k0, k1, v0, v1;
      if constexpr (FP8) {
        uint32_t a[4], b[4];
        fp8x8_to_bf16x8(kr[0][0], kr[0][1], a);
        fp8x8_to_bf16x8(kr[0][2], kr[0][3], b);
        k0 = u32x4{a[0], a[1], a[2], a[3]};
        k1 = u32x4{b[0], b[1], b[2], b[3]};
        fp8x8_to_bf16x8(vr[0][0], vr[0][1], a);
        fp8x8_to_bf16x8(vr[0][2], vr[0][3], b);
        v0 = u32x4{a[0], a[1], a[2], a[3]};
        v1 = u32x4{b[0], b[1], b[2], b[3]};
      } else {
        k0 = kr[0];
        k1 = kr[kElt - 1];
        v0 = vr[0];
        v1 = vr[kElt - 1];
      }
      if (masked(tc)) {
        const bool past = tc + ld_row >= v.len;
        bool bad = false;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          auto clean = [&](uint32_t x) {
            if (past) return 0u;
            const bool hi = (x & 0x7F800000u) == 0x7F800000u, lo = (x & 0x7F80u) == 0x7F80u;
            bad |= hi | lo;
            return x & (hi ? 0xFFFFu : ~0u) & (lo ? 0xFFFF0000u : ~0u);
          };
          v0[i] = clean(v0[i]);
          v1[i] = clean(v1[i]);
        }
        if (bad) atomicOr(&lds_bad[slot][ld_row >> 5], 1u << (ld_row & 31));
      }
      *(u32x4 *)(&lds_k[buf][ld_row * kKRow + ld_seg * 32]) = k0;
      *(u32x4 *)(&lds_k[buf][ld_row * kKRow + ld_seg * 32 + 16]) = k1;
      *(u32x4 *)(&lds_v[buf][ld_row * kVRow + ld_seg * 32]) = v0;
      *(u32x4 *)(&lds_v[buf][ld_row * kVRow + ld_seg * 32 + 16]) = v1;
    };

    auto step = [&](const int tc, const int buf, const bool need_mask) {
      const uint8_t *k_rd = &lds_k[buf][0] + i16 * kKRow + g * 32;
      const uint8_t *v_rd = &lds_v[buf][0] + (4 * g + (i16 >> 2)) * kVRow + 8 * (i16 & 3);
      Frag8 kf[4][2], vf[4][2];
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        kf[b][0].u = *(const u32x4 *)(k_rd + b * (kBlock * kKRow));
        kf[b][1].u = *(const u32x4 *)(k_rd + b * (kBlock * kKRow) + 16);
      }
#pragma unroll
      for (int mt = 0; mt < 4; ++mt)
#pragma unroll
        for (int pr = 0; pr < 2; ++pr) {
          const u32x2 a = lds_read_tr16(v_rd + 32 * mt + (2 * pr) * (kBlock * kVRow));
          const u32x2 b = lds_read_tr16(v_rd + 32 * mt + (2 * pr + 1) * (kBlock * kVRow));
          vf[mt][pr].w[0] = a[0];
          vf[mt][pr].w[1] = a[1];
          vf[mt][pr].w[2] = b[0];
          vf[mt][pr].w[3] = b[1];
        }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        f32x4 S[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          S[b] = mfma16x32(kf[b][0], qf[t][0], f32x4{0.f, 0.f, 0.f, 0.f});
          S[b] = mfma16x32(kf[b][1], qf[t][1], S[b]);
        }
        if (need_mask) {
          const int tl = wtok + 2 * t + (i16 >> 3);
          const uint64_t w = chunk_bits(lds_mask[tl], lds_lo[tl], prefix, tc) >> (4 * g);
#pragma unroll
          for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (!((w >> (16 * b + r)) & 1)) S[b][r] = -INFINITY;
        }
        float mx = max3(S[0][0], S[0][1], S[0][2]);
#pragma unroll
        for (int o = 1; o < 7; ++o) mx = max3(mx, S[(2 * o + 1) >> 2][(2 * o + 1) & 3], S[(2 * o + 2) >> 2][(2 * o + 2) & 3]);
        mx = max2(mx, S[3][3]) * c2;
        if (__any(mx > m[t] + kLazyLog2)) {
          const float mrow = rowgroup_max(mx);
          const float m_new = mrow > m[t] + kLazyLog2 ? mrow : m[t];
          const float alpha = fast_exp2(m[t] - m_new);
          l[t] *= alpha;
#pragma unroll
          for (int mt = 0; mt < 4; ++mt)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[t][mt][r] *= alpha;
          m[t] = m_new;
        }
        Frag8 P[2];
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float p0 = fast_exp2(__builtin_fmaf(S[(2 * k) >> 2][(2 * k) & 3], c2, -m[t]));
          const float p1 = fast_exp2(__builtin_fmaf(S[(2 * k + 1) >> 2][(2 * k + 1) & 3], c2, -m[t]));
          sum += p0 + p1;
          P[k >> 2].w[k & 3] = pack_bf16(p0, p1);
        }
        l[t] += sum;
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
          acc[t][mt] = mfma16x32(vf[mt][0], P[0], acc[t][mt]);
          acc[t][mt] = mfma16x32(vf[mt][1], P[1], acc[t][mt]);
        }
      }
    };

    // Values that are not finite, taken out of a masked chunk's tile: their keys' terms are added
    // row by row, for the rows that see them.  (Rare, and slow: one dot product per row and key.)
    auto add_bad = [&](const int tc, uint64_t bad) {
      while (bad) {
        const int b = __builtin_ctzll(bad);
        bad &= bad - 1;
        const int j = tc + b;
        const int page = clamp_id(bt[min(j / kBlock, last_page)], p.last_block);
        const size_t off = (size_t)page * page_bytes + (size_t)(j % kBlock) * row_bytes + (size_t)kvh * (kHeadDim * kElt);
        auto elem = [&](const uint8_t *base, const int d) {
          if constexpr (FP8) {
            uint32_t o[4];
            fp8x8_to_bf16x8(base[off + d], 0, o);
            return bf16_bits_to_f32(o[0] & 0xFFFFu);
          } else {
            return bf16_bits_to_f32(*(const uint16_t *)(base + off + 2 * d));
          }
        };
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const int tl = wtok + 2 * t + (i16 >> 3), tok = tok0 + tl;
          if (tok < v.qlen && (chunk_bits(lds_mask[tl], lds_lo[tl], prefix, tc) >> b & 1)) {
            const uint16_t *qr = p.q + ((size_t)(v.row0 + tok) * p.num_q_heads + kvh * kGroup + (i16 & 7)) * kHeadDim;
            float dot = 0.f;
            for (int d = 0; d < kHeadDim; ++d) dot += bf16_bits_to_f32(qr[d]) * elem(p.k_cache, d);
            const float w = fast_exp2(__builtin_fmaf(dot, c2, -m[t]));
#pragma unroll
            for (int mt = 0; mt < 4; ++mt)
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const float x = elem(p.v_cache, 16 * mt + 4 * g + r);
                if ((__float_as_uint(x) & 0x7F800000u) == 0x7F800000u) acc[t][mt][r] += w * x;
              }
          }
        }
      }
    };

    fetch(t_begin);
    stash(t_begin, 0, 0);
    __syncthreads();
    int cur = 0, slot = 0;
    for (int tc = t_begin; tc < t_end; tc += kChunk, cur ^= 1) {
      const bool has_next = tc + kChunk < t_end;
      const int slot1 = slot == 2 ? 0 : slot + 1, slot2 = slot1 == 2 ? 0 : slot1 + 1;
      if (has_next) fetch(tc + kChunk);
      const bool mk = masked(tc);
      if (tid < 2) lds_bad[slot2][tid] = 0;  // (read last before the barrier that opened this chunk)
      if (wave_active) {
        step(tc, cur, mk);
        if (mk) {
          const uint64_t bad = (uint64_t)__builtin_amdgcn_readfirstlane(lds_bad[slot][0]) |
                               (uint64_t)__builtin_amdgcn_readfirstlane(lds_bad[slot][1]) << 32;
          if (bad) add_bad(tc, bad);
        }
      }
      if (has_next) stash(tc + kChunk, cur ^ 1, slot1);
      __syncthreads();
      slot = slot1;
    }

    // ---- this piece's rows: the answer, or a partial
    const bool whole = n == v.chunks;
    const int part = c0 == 0 ? 1 : 0;  // a range holds at most one piece of each kind that is not whole
    float *ws_o = p.ws_o + ((size_t)(range * Hkv + kvh) * 2 + part) * (kRows * kHeadDim);
    float *ws_ml = p.ws_ml + ((size_t)(range * Hkv + kvh) * 2 + part) * (kRows * 2);
    if (wave_active) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int tl = wtok + 2 * t + (i16 >> 3), tok = tok0 + tl;
        const float lt = rowgroup_sum(l[t]);
        if (tok >= v.qlen) continue;
        if (whole) {
          const int head = kvh * kGroup + (i16 & 7);
          const float sink = p.sinks ? p.sinks[head] * kLog2e : -INFINITY;
          // (a row that sees nothing, m = kNegBig, has only its sink)
          const float M = max2(m[t], sink), a = fast_exp2(m[t] - M);
          const float den = lt * a + fast_exp2(sink - M);
          const float f = den > 0.f || den != den ? vs * a / den : 0.f;
          const size_t orow = (size_t)(v.row0 + tok) * p.num_q_heads + head;
#pragma unroll
          for (int mt = 0; mt < 4; ++mt) {
            u32x2 w;
            w[0] = pack_bf16(acc[t][mt][0] * f, acc[t][mt][1] * f);
            w[1] = pack_bf16(acc[t][mt][2] * f, acc[t][mt][3] * f);
            *(u32x2 *)(p.out + orow * kHeadDim + 16 * mt + 4 * g) = w;
          }
          if (p.lse && g == 0) p.lse[orow] = den > 0.f || den != den ? (M + __log2f(den)) * kLn2 : -INFINITY;
        } else {
          const int row = tl * kGroup + (i16 & 7);
#pragma unroll
          for (int mt = 0; mt < 4; ++mt) *(f32x4 *)(ws_o + (size_t)row * kHeadDim + 16 * mt + 4 * g) = acc[t][mt];
          if (g == 0) {
            ws_ml[2 * row] = m[t];
            ws_ml[2 * row + 1] = lt;
          }
        }
      }
    }
    u += n;
  }
}

// Joins the pieces of the rows that a range's end cut: out = sum 2^(m - M) o / (sum 2^(m - M) l + 2^(sink - M)).
// One workgroup per (row, KV head); a thread per (head, pair of dims).
__global__ __launch_bounds__(256) void tree_merge_kernel(const TreeParams p, const int tile_tok) {
  const int Hkv = p.num_kv_heads, kvh = blockIdx.x % Hkv, row = blockIdx.x / Hkv;
  int lo = 0, hi = p.num_seqs - 1;
  while (lo < hi) {  // the last sequence that starts at or before the row
    const int mid = (lo + hi + 1) >> 1;
    if (p.cu_seqlens_q[mid] <= row) lo = mid; else hi = mid - 1;
  }
  const int s = lo;
  const TreeSeq v = tree_seq(p, s, tile_tok);
  const int tok = row - v.row0;
  if (tok < 0 || tok >= v.qlen) return;
  long long total, before;
  count_units(p, tile_tok, s, total, before);
  const long long per = range_units(p, total);
  const int tile = tok / tile_tok;
  const long long u0 = before + (long long)tile * v.chunks, u1 = u0 + v.chunks;
  const int r0 = (int)(u0 / per), r1 = (int)((u1 - 1) / per);
  if (r0 == r1) return;  // one range held it whole
  const int h = threadIdx.x >> 5, d = (threadIdx.x & 31) * 2;
  const int head = kvh * kGroup + h, prow = (tok - tile * tile_tok) * kGroup + h;
  const float sink = p.sinks ? p.sinks[head] * kLog2e : -INFINITY;
  const int rows = tile_tok * kGroup;
  auto cell = [&](const int r) { return ((size_t)(r * Hkv + kvh) * 2 + (r == r0 ? 1 : 0)) * rows + prow; };
  float M = max2(sink, kNegBig), den = 0.f, o0 = 0.f, o1 = 0.f;
  for (int r = r0; r <= r1; ++r) {
    const size_t c = cell(r);
    const float2 ml = *(const float2 *)(p.ws_ml + 2 * c);
    const float2 o = *(const float2 *)(p.ws_o + c * kHeadDim + d);
    const float M1 = max2(M, ml.x), a = fast_exp2(M - M1), w = fast_exp2(ml.x - M1);
    den = den * a + ml.y * w;
    o0 = o0 * a + o.x * w;
    o1 = o1 * a + o.y * w;
    M = M1;
  }
  den += fast_exp2(sink - M);
  const float vs = p.v_scale ? p.v_scale[kvh] : 1.0f;
  const bool any = den > 0.f || den != den;
  const float f = any ? vs / den : 0.f;
  const size_t orow = (size_t)row * p.num_q_heads + head;
  *(uint32_t *)(p.out + orow * kHeadDim + d) = pack_bf16(o0 * f, o1 * f);
  if (p.lse && d == 0) p.lse[orow] = any ? (M + __log2f(den)) * kLn2 : -INFINITY;
}

}  // namespace

// 16-row tiles per wave: the fewest that hold the longest tree in one workgroup, or the most.
int tree_tiles(const int max_q_len) { return max_q_len <= 8 ? 1 : max_q_len <= 16 ? 2 : 4; }
int tree_tile_tokens(const int max_q_len) { return 2 * tree_tiles(max_q_len) * kTreeWaves; }

hipError_t launch_tree(const TreeParams &p, const bool fp8, hipStream_t st) {
  const int nt = tree_tiles(p.max_q_len);
  const dim3 grid((unsigned)(p.ranges * p.num_kv_heads)), block(kTreeWaves * 64);
  if (nt == 1) {
    if (fp8) tree_kernel<1, true><<<grid, block, 0, st>>>(p);
    else tree_kernel<1, false><<<grid, block, 0, st>>>(p);
  } else if (nt == 2) {
    if (fp8) tree_kernel<2, true><<<grid, block, 0, st>>>(p);
    else tree_kernel<2, false><<<grid, block, 0, st>>>(p);
  } else {
    if (fp8) tree_kernel<4, true><<<grid, block, 0, st>>>(p);
    else tree_kernel<4, false><<<grid, block, 0, st>>>(p);
  }
  return hipGetLastError();
}

hipError_t launch_tree_merge(const TreeParams &p, hipStream_t st) {
  tree_merge_kernel<<<(unsigned)p.num_kv_heads * (unsigned)p.num_q_tokens, 256, 0, st>>>(p, tree_tile_tokens(p.max_q_len));
  return hipGetLastError();
}

}  // namespace eid
