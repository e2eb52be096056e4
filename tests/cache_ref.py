"""Plain 64-bit restatements of the tree attention and of the operators that thin a cache out, and
small batches for them (numpy; nothing here calls the library)."""
import numpy as np

import oracle
from eidola_amd import KV_BF16, KV_FP8_E4M3, synth

from helpers import make_batch, logical_tensors, cpu_caches, fp8_scales

BF16_HALF_STEP = 2.0 ** -8    # largest relative error of a rounding to bf16: half of eps = 2^-7


def f64(bits):
    """bf16 bit patterns as doubles."""
    return synth.bf16_bits_to_f32(bits).astype(np.float64)


def fp8_f64(codes):
    """e4m3fn codes as doubles, from the format's definition."""
    c = np.asarray(codes).astype(np.int64)
    sign, e, m = np.where(c & 0x80, -1.0, 1.0), (c >> 3) & 15, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    return np.where((c & 0x7F) == 0x7F, np.nan, sign * v)


def cache_rows(batch, cache, scale, s):
    """[L, Hkv, D] of sequence s, as the values they stand for."""
    rows = cache.reshape(-1, *cache.shape[2:])[batch.all_slots(s)]
    if batch.geom.kv_dtype == KV_FP8_E4M3:
        return fp8_f64(rows) * np.asarray(scale, np.float64)[None, :, None]
    return f64(rows)


def random_parents(n, rng, back=6):
    return [-1] + [int(rng.integers(max(0, i - back), i)) for i in range(1, n)]


def tree_masks(parents_list, words):
    """[T, words] int64 masks of trees given by parents (-1: no parent)."""
    out = []
    for parents in parents_list:
        seen = []
        for i, up in enumerate(parents):
            seen.append((seen[up] if up >= 0 else 0) | 1 << i)
        out += seen
    return masks_from_ints(out, words)


def masks_from_ints(ints, words):
    a = np.array([[(m >> 64 * w) & (1 << 64) - 1 for w in range(words)] for m in ints], dtype=np.uint64)
    return a.view(np.int64).reshape(len(ints), words)


def mask_bits(mask, n):
    """[rows, n] booleans of int64 words."""
    u = mask.view(np.uint64)
    j = np.arange(n)
    return (u[:, j // 64] >> (j % 64).astype(np.uint64) & np.uint64(1)).astype(bool)


def tree_visible(mask, q_len, length, window):
    """[q_len, length]: what the rows of one sequence see."""
    bits = mask_bits(mask, q_len) if q_len else np.zeros((0, 0), bool)
    prefix = length - q_len
    depth = bits.sum(1) - 1
    see = np.concatenate([np.ones((q_len, prefix), bool), bits], 1)
    if window > 0:
        pos = np.concatenate([np.arange(prefix), prefix + depth])
        see &= (prefix + depth)[:, None] - pos[None, :] < window
    return see


def attn_rows(q, k, v, see, scale, sinks):
    """[n, Hq, D] doubles and lse [n, Hq]: rows q over the keys that each sees."""
    n, Hq, _ = q.shape
    group = Hq // k.shape[1]
    out, lse = np.zeros(q.shape), np.full((n, Hq), -np.inf)
    for i in range(n):
        j = np.nonzero(see[i])[0]
        for h in range(Hq):
            s = k[j, h // group] @ q[i, h] * scale
            e = -np.inf if sinks is None else float(sinks[h])
            top = max(s.max() if len(j) else -np.inf, e)
            if top == -np.inf:
                continue
            p = np.exp(s - top)
            den = p.sum() + np.exp(e - top)
            out[i, h] = p @ v[j, h // group] / den
            lse[i, h] = top + np.log(den)
    return out, lse


def attn_tree(batch, q, kc, vc, mask, sinks, k_scale=None, v_scale=None):
    outs, lses = [], []
    for s in range(batch.num_seqs):
        a, b = batch.cu_seqlens_q[s], batch.cu_seqlens_q[s + 1]
        see = tree_visible(mask[a:b], b - a, int(batch.seq_lens[s]), batch.geom.window)
        o, l = attn_rows(f64(q[a:b]), cache_rows(batch, kc, k_scale, s), cache_rows(batch, vc, v_scale, s), see,
                         batch.geom.softmax_scale, sinks)
        outs.append(o)
        lses.append(l)
    return np.concatenate(outs), np.concatenate(lses)


def kv_score(batch, q, lse, kc, scores, k_scale=None):
    """scores [num_blocks, Hkv, 16] doubles after the step (a copy)."""
    new = np.array(scores, np.float64)
    w, Hkv = batch.geom.window, batch.geom.num_kv_heads
    for s in range(batch.num_seqs):
        a, b = batch.cu_seqlens_q[s], batch.cu_seqlens_q[s + 1]
        L, n = int(batch.seq_lens[s]), int(b - a)
        k = cache_rows(batch, kc, k_scale, s)
        slots = batch.all_slots(s)
        page, place = slots // 16, slots % 16
        for h in range(Hkv):
            add = np.zeros(L)
            for i in range(n):
                pos = L - n + i
                j = np.arange(L)
                see = (j <= pos) & ((w <= 0) | (pos - j < w))
                for x in range(8 * h, 8 * h + 8):
                    e = float(lse[a + i, x])
                    if e == -np.inf:
                        continue
                    add += np.where(see, np.exp(k[:, h] @ f64(q[a + i, x]) * batch.geom.softmax_scale - e), 0.0)
            old = np.where(np.arange(L) >= L - n, 0.0, new[page, h, place])
            if n > 0:
                new[page, h, place] = old + add
    return new


def kv_select(batch, scores, budget, first, last):
    S, H = batch.num_seqs, batch.geom.num_kv_heads
    keep = np.full((S, H, budget), -1, np.int32)
    counts = np.minimum(batch.seq_lens, budget).astype(np.int32)
    for s in range(S):
        L = int(batch.seq_lens[s])
        slots = batch.all_slots(s)
        for h in range(H):
            if L <= budget:
                keep[s, h, :L] = np.arange(L)
                continue
            w = scores[slots // 16, h, slots % 16].astype(np.float64)
            mid = list(range(first, L - last))
            mid.sort(key=lambda j: (0, -w[j], j) if w[j] == w[j] else (1, 0.0, j))   # NaN last
            rows = sorted(list(range(first)) + mid[:budget - first - last] + list(range(L - last, L)))
            keep[s, h] = rows
    return keep, counts


def kv_compact(batch, cache, keep, counts, starts, per_head):
    """cache [num_blocks, 16, H, ...] (rows) after the move; keep [S, N] or [S, H, N]."""
    new = cache.copy()
    flat_new, flat_old = new.reshape(-1, *cache.shape[2:]), cache.reshape(-1, *cache.shape[2:])
    for s in range(batch.num_seqs):
        slots = batch.all_slots(s)
        for i in range(int(counts[s])):
            for h in range(cache.shape[2]):
                src = int(keep[s, h, i] if per_head else keep[s, i])
                flat_new[slots[starts[s] + i], h] = flat_old[slots[src], h]
    return new


def filled(seq_lens, q_lens, **kw):
    """(batch, q, k cache, v cache, k scale, v scale, sinks): a batch and its caches on the host."""
    b = make_batch(seq_lens, q_lens, **kw)
    q, k, v, sinks = logical_tensors(b)
    ks, vs = fp8_scales(k, v) if b.geom.kv_dtype == KV_FP8_E4M3 else (None, None)
    kc, vc = cpu_caches(b, k, v, ks, vs)
    return b, q, kc, vc, ks, vs, sinks
