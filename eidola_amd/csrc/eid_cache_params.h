// Launch descriptors of the tree attention and of the operators that thin a paged cache out
// (internal to the library).
#pragma once
#include "eid_params.h"

namespace eid {

constexpr int kTreeWordsMax = 4;              // mask words per drafted token
constexpr int kTreeMax = 64 * kTreeWordsMax;  // drafted tokens per sequence
constexpr int kTreeWaves = 4;
// 64-key chunks per range, at least: 1 x 16 tokens behind 4k keys 13.9 us with 2, 15.7 with 1, 14.8 with 4
constexpr int kTreeMinChunks = 2;

// Where the pieces of a tile of drafted tokens are.
struct TreeRecord {
  int32_t range, pieces;  // first range that holds some of it, and how many do
};

// Statistics of one row of a piece.
struct alignas(16) TreeStats {
  float m, l;    // reference (log2 units) and sum of the row's weights
  int32_t e;     // the row's outputs are kept as 2^-e of themselves
  int32_t unused;
};

struct TreeParams {
  const uint16_t *q;
  uint16_t *out;
  float *lse;  // may be null
  const uint8_t *k_cache, *v_cache;
  const int32_t *block_table, *cu_seqlens_q, *seq_lens;
  const float *sinks;             // may be null
  const float *k_scale, *v_scale; // fp8 only
  const uint64_t *mask;           // [num_q_tokens][mask_words]
  TreeRecord *ws_rec;  // [num_seqs][max_tiles]
  _Float16 *ws_o;  // [ranges][Hkv][2][tile rows][64]  2^-e sum of 2^(s-m) v of a piece, not normalised
  TreeStats *ws_ml;    // [ranges][Hkv][2][tile rows]      m (log2 units), l, e
  int32_t num_seqs, num_q_heads, num_kv_heads, max_blocks_per_seq, last_block;
  int32_t num_q_tokens, mask_words, window, max_q_len, max_kv_len;
  int32_t max_tiles;  // tiles of the longest tree
  int32_t ranges;     // workgroups per KV head
  int32_t whole;      // 1: a range per (sequence, tile), nothing is cut
  int32_t min_chunks; // smallest range
  float softmax_scale;
};

constexpr long long kScoreOwnKeys = 1 << 20;  // keys x KV heads beyond which sequences of few rows get their own launch
constexpr int kScoreFewRows = 2;   // q_len that the few-rows kernel takes
constexpr int kScoreWaves = 4;     // of a workgroup of the rows kernel
constexpr int kScoreKeys = 128;    // keys of a wave of the rows kernel
constexpr int kScorePartsMax = 64;
constexpr int kScoreTile = kScoreWaves * kScoreKeys;

struct ScoreParams {
  const uint16_t *q;
  const float *lse;
  const uint8_t *k_cache;
  const int32_t *block_table, *cu_seqlens_q, *seq_lens;
  const float *k_scale;  // fp8 only
  float *scores;         // [num_blocks][Hkv][16]
  int32_t num_seqs, num_q_heads, num_kv_heads, max_blocks_per_seq, last_block;
  int32_t num_q_tokens, window, max_q_len, max_kv_len;
  int32_t ranges;     // workgroups per eight KV heads of the stream kernel
  int32_t all_rows;   // the rows kernel takes sequences of few rows as well
  int32_t parts;      // the rows kernel's rows are shared out over so many workgroups
  int32_t tile_keys;  // max_kv_len, in whole workgroups' keys
  int32_t ws_tiles;   // tiles of kScoreTile keys that the workspace has for a part and KV head
  float *ws;          // [parts][Hkv][ws_tiles][kScoreTile], the sequences' tiles in a line; parts > 1 only
  float softmax_scale;
};

struct SelectParams {
  const float *scores;
  const int32_t *block_table, *seq_lens;
  int32_t *keep;    // [num_seqs][Hkv][budget]
  int32_t *counts;  // [num_seqs]
  int32_t num_seqs, num_kv_heads, max_blocks_per_seq, last_block;
  int32_t budget, keep_first, keep_last;
  int32_t max_kv_len;  // expected longest sequence: chooses the kernel
};

constexpr int kCompactLayers = 64;  // layers per launch
struct CompactParams {
  uint8_t *k[kCompactLayers], *v[kCompactLayers];
  float *scores[kCompactLayers];  // all null when none were given
  const int32_t *block_table, *seq_lens, *keep, *counts, *starts;  // starts may be null
  int64_t keep_layer, keep_seq, keep_head;  // strides of keep in entries; 0 = shared
  int32_t num_seqs, num_kv_heads, max_blocks_per_seq, last_block;
  int32_t max_rows, elt;  // elt: bytes per cache element
  int32_t has_scores;
};

}  // namespace eid
